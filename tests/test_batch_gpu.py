"""The operators around a batch's attention on the GPU against the float64 oracle.

Error bounds, from the arithmetic the operators document (u = 2^-8: rounding to bf16 is off by at most
half a step, 2^-8 of the value; f32 2^-24):
  quantize, dequantize, embed   roundings of exact values: equal
  matmul      products of codes and scales are exact; the tensor cores add 64 of them at a time to an f32
              sum and may cut what they add below the sum's last bit (2^-23 of the sum of magnitudes S
              for each of pieces * k / 64 additions, which join up to 8 parts), two factors:
              |error| <= (pieces * k / 64 + 12) 2^-23 S, and u |y| more for bf16
  norm        f32: x r w to 2^-21 of itself (sum of squares, root, two products), the sum to 2^-24, one
              rounding to bf16: |error| <= u |y| + 2^-20 (|residual| + |x r w|)
  beam        scores: f32 exponentials (2^-21 each, ~2^-21 of the sum), 64-bit sums, one rounding
"""

import ctypes
import math

import pytest
import torch

import g4b200 as g4
from oracle import batch as ob

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).bfloat16()


def _sync(ctx):
    torch.cuda.synchronize()
    assert ctx.poll() == 0


def _rows(ctx, n, cols, pieces, seed=0, spread=2.0):
    """Quantised rows from random codes and scales of every size, laid out by the oracle, in a buffer whose
    other bytes are NaN scales and codes of 6; with the values and factors."""
    g = _gen(seed)
    room = n + 3
    r = g4.Nvfp4Rows(ctx, room, cols, pieces)
    for t, v in ((r.codes, 0xFF), (r.scales, 0x7F)):
        t.fill_(v)
    r.factor.fill_(float("nan"))
    codes = torch.randint(0, 16, (pieces, n, cols), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.randn((pieces, n, cols // 16), generator=g, device="cuda") * 8 * spread + 56).clamp(0, 126).byte()
    factor = torch.exp2(torch.randint(-8, 3, (n,), generator=g, device="cuda").float())
    r.codes[:, :n] = ob.pack(codes)
    b = torch.arange(cols // 16, device="cuda")[None, :]
    at = ob.scale_at(torch.arange(n, device="cuda")[:, None], b, cols)
    for p in range(pieces):
        r.scales[p][at] = scales[p]
        if cols % 64:  # columns past the row's end count as zeros
            r.scales[p][ob.scale_at(torch.arange(n, device="cuda")[:, None], b.new_tensor([[cols // 16, cols // 16 + 1]]), cols)] = 0
    r.factor[:n] = factor
    return r, ob.values(codes, scales).sum(0), factor.double()


def _weight(ctx, n, cols, factors=1, seed=1):
    g = _gen(seed)
    codes = torch.randint(0, 16, (n, cols), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.randn((n, cols // 16), generator=g, device="cuda") * 12 + 56).clamp(0, 126).byte()
    factor = torch.rand(factors, generator=g, device="cuda") + 0.01
    return g4.Nvfp4Weight(ctx, ob.pack(codes), scales, factor), ob.values(codes, scales), factor.double()


def _product(ctx, m, n, cols, pieces, f32=False, gap=0, factors=1, seed=0):
    rows, xv, fx = _rows(ctx, m, cols, pieces, seed)
    weight, wv, fw = _weight(ctx, n, cols, factors, seed + 1)
    wide = torch.full((m, (n + 7) // 8 * 8 + gap), 7.0, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    out = wide[:, :n]
    if (n + 7) // 8 * 8 + gap != n and m == 1:
        out = wide.as_strided((1, n), (wide.shape[1], 1))
    g4.nvfp4_matmul(ctx, rows, weight, out)
    _sync(ctx)
    want, size = ob.matmul(xv, wv, fx, fw)
    bound = (pieces * cols / 64 + 12) * 2.0 ** -23 * size + (0 if f32 else U * want.abs())
    assert torch.isfinite(out).all()
    worst = ((out.double() - want).abs() - bound).max().item()
    assert worst <= 0, f"error above its bound by {worst}"
    assert (wide[:, n:] == 7.0).all()
    return out


SHAPES = [
    # m, n, cols, pieces
    (1, 1, 32, 1), (1, 8, 64, 2), (2, 7, 96, 3), (3, 130, 160, 1), (1, 8192, 3840, 2), (5, 515, 3840, 3), (16, 128, 512, 2),
    (17, 256, 512, 1), (31, 129, 480, 2), (32, 3840, 4096, 2), (33, 257, 1056, 3), (64, 640, 1920, 2), (65, 300, 704, 1),
    (127, 384, 256, 2), (128, 128, 128, 1), (129, 1000, 992, 2), (255, 511, 3840, 1), (256, 256, 256, 3), (257, 513, 320, 2),
    (300, 3840, 1024, 2), (509, 1088, 3840, 2), (513, 777, 2080, 3), (1024, 2048, 512, 1), (1111, 512, 3840, 2),
    (700, 3840, 15360, 1), (2, 3840, 15360, 3), (1300, 4096, 96, 2),
    # every tile width and K split with each count of pieces, columns that end inside a stage and inside 64
    (20, 301, 992, 1), (20, 300, 2080, 1), (40, 6001, 2080, 1), (100, 6001, 8192, 1), (100, 4104, 3840, 1), (100, 2049, 8192, 1),
    (3001, 300, 96, 1), (3001, 303, 96, 2), (3001, 300, 96, 3), (2000, 6001, 96, 1), (2000, 6008, 160, 2), (2050, 8192, 96, 3),
    (509, 8704, 3840, 2), (1500, 8192, 352, 3), (2050, 8192, 992, 1),
]


@pytest.mark.parametrize("m, n, cols, pieces", SHAPES)
def test_matmul(gpu_ctx, m, n, cols, pieces):
    _product(gpu_ctx, m, n, cols, pieces)


@pytest.mark.parametrize("m, n, cols, pieces", [(1, 515, 3840, 2), (33, 129, 480, 3), (257, 520, 1056, 1), (640, 300, 3840, 2),
                                                (2000, 6001, 96, 2), (3001, 301, 96, 3), (100, 2049, 8192, 1)])
def test_matmul_f32_strides_and_factors(gpu_ctx, m, n, cols, pieces):
    """f32 sums, rows apart (what lies between them is left alone), a factor for every row of the weight."""
    _product(gpu_ctx, m, n, cols, pieces, f32=True, gap=24, factors=n, seed=5)
    _product(gpu_ctx, m, n, cols, pieces, f32=False, gap=8, factors=n, seed=6)


@pytest.mark.parametrize("m, n, cols, pieces", [(1, 515, 3840, 2), (20, 301, 992, 1), (40, 6001, 2080, 1), (33, 129, 480, 3),
                                                (257, 520, 1056, 1), (509, 8704, 96, 2), (2050, 8192, 96, 3)])
@pytest.mark.parametrize("f32", [False, True])
def test_matmul_factors_far_apart(gpu_ctx, m, n, cols, pieces, f32):
    """Factors of rows and weights whose product, or the sum's with either, leaves f32's range while the result is in it.
    Bounds as above, with half a step of subnormal results more (f32 2^-150, bf16 2^-134); what is twice f32's
    largest number is infinite."""
    rows, xv, fx = _rows(gpu_ctx, m, cols, pieces, 31)
    weight, wv, fw = _weight(gpu_ctx, n, cols, n, 32)
    g = _gen(33)
    pick = lambda exponents, count: torch.exp2(torch.tensor(exponents, device="cuda")[  # noqa: E731
        torch.randint(0, len(exponents), (count,), generator=g, device="cuda")].double()).float()
    rows.factor[:m] = pick([-126.0, -100.0, -60.0, 0.0, 60.0, 100.0, 117.0], m)
    if m == 1:
        rows.factor[0] = 2.0 ** 117
    weight.factor.copy_(pick([-140.0, -126.0, -90.0, -17.0, 0.0, 90.0, 125.0], n) * (1 + torch.rand(n, generator=g, device="cuda")))
    out = torch.empty((m, (n + 7) // 8 * 8), dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")[:, :n]
    g4.nvfp4_matmul(gpu_ctx, rows, weight, out)
    _sync(gpu_ctx)
    want, size = ob.matmul(xv, wv, rows.factor[:m].double(), weight.factor.double())
    bound = (pieces * cols / 64 + 12) * 2.0 ** -23 * size + (2.0 ** -150 if f32 else U * want.abs() + 2.0 ** -134)
    inside, beyond = (want.abs() + bound) < 2.0 ** 127, (want.abs() - bound) > 2.0 ** 129
    assert inside.any() and (m == 1 or beyond.any())
    worst = ((out.double() - want).abs() - bound)[inside].max().item()
    assert worst <= 0, f"error above its bound by {worst}"
    assert torch.isinf(out[beyond]).all()


def test_matmul_repeats_itself(gpu_ctx):
    rows, _, _ = _rows(gpu_ctx, 600, 1920, 2)
    weight, _, _ = _weight(gpu_ctx, 1000, 1920)
    a, b = (torch.empty((600, 1000), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g4.nvfp4_matmul(gpu_ctx, rows, weight, a)
    g4.nvfp4_matmul(gpu_ctx, rows, weight, b)
    _sync(gpu_ctx)
    assert torch.equal(a, b)


@pytest.mark.parametrize("m, n, cols, pieces", [(60, 30720, 256, 2), (200, 30720, 256, 1), (1000, 8192, 96, 2), (2500, 8192, 96, 3)])
def test_matmul_sums_side_by_side(gpu_ctx, m, n, cols, pieces):
    """Several short tiles a pair, whose sums alternate between two places of tensor memory, one read while the next
    tile's are formed in the other: the oracle's, and the same bits again and again."""
    rows, xv, fx = _rows(gpu_ctx, m, cols, pieces, 41)
    weight, wv, fw = _weight(gpu_ctx, n, cols, 1, 42)
    want, size = ob.matmul(xv, wv, fx, fw)
    out, first = torch.empty((m, n), dtype=torch.bfloat16, device="cuda"), None
    for _ in range(30):
        out.fill_(7.0)
        g4.nvfp4_matmul(gpu_ctx, rows, weight, out)
        first = out.clone() if first is None else first
        assert torch.equal(out, first)
    _sync(gpu_ctx)
    assert ((first.double() - want).abs() <= (pieces * cols / 64 + 12) * 2.0 ** -23 * size + U * want.abs()).all()


def test_matmul_of_the_most_rows(gpu_ctx):
    """2^22 rows of 32 values: more tiles than a grid's second dimension has room for."""
    m = 2 ** 22
    rows = g4.Nvfp4Rows(gpu_ctx, m, 32, 1)
    x = _randn(_gen(21), m, 32)
    weight, wv, fw = _weight(gpu_ctx, 8, 32)
    out = torch.empty((m, 8), dtype=torch.float32, device="cuda")
    g4.nvfp4_quantize(gpu_ctx, x, rows)
    g4.nvfp4_matmul(gpu_ctx, rows, weight, out)
    _sync(gpu_ctx)
    for at in (slice(0, 3000), slice(m // 2 - 5, m // 2 + 3000), slice(m - 3000, m)):
        codes, scales, factor = ob.quantize(x[at], 1)
        want, size = ob.matmul(ob.values(codes, scales)[0], wv, factor, fw)
        assert ((out[at].double() - want).abs() <= 13 * 2.0 ** -23 * size).all()


@pytest.mark.parametrize("m, n, cols", [(1, 3840, 15360), (32, 3840, 8192), (17, 300, 2080), (100, 2049, 8192), (1, 8192, 3840)])
@pytest.mark.parametrize("pieces", [2, 3])
def test_matmul_ahead_of_the_quantisation(gpu_ctx, m, n, cols, pieces):
    """A constant weight's first stages are read while the rows are still being quantised, the rest behind that: the
    oracle's values, and the bits of products that read nothing ahead."""
    x = _randn(_gen(m + n), m, cols)
    rows = g4.Nvfp4Rows(gpu_ctx, m, cols, pieces)
    weight, wv, fw = _weight(gpu_ctx, n, cols, 1, 71)
    changing = g4.Nvfp4Weight.__new__(g4.Nvfp4Weight)
    changing._set(weight.codes, weight.scales, weight.factor, n, cols, 0)
    assert weight.desc.constant == 1 and changing.desc.constant == 0
    ahead, after, ordered = (torch.full((m, (n + 7) // 8 * 8), 7.0, dtype=torch.bfloat16, device="cuda")[:, :n] for _ in range(3))
    for _ in range(5):
        g4.nvfp4_quantize(gpu_ctx, x, rows)
        g4.nvfp4_matmul(gpu_ctx, rows, weight, ahead)
        g4.nvfp4_matmul(gpu_ctx, rows, weight, after)  # (a launch lies between)
        g4.nvfp4_quantize(gpu_ctx, x, rows)
        g4.nvfp4_matmul(gpu_ctx, rows, changing, ordered)
        _sync(gpu_ctx)
        assert torch.equal(ahead, after) and torch.equal(ahead, ordered)
    codes, scales, factor = ob.quantize(x, pieces)
    want, size = ob.matmul(ob.values(codes, scales).sum(0), wv, factor, fw)
    assert ((ahead.double() - want).abs() <= (pieces * cols / 64 + 12) * 2.0 ** -23 * size + U * want.abs()).all()


@pytest.mark.parametrize("m, n, cols", [(1, 3840, 4096), (40, 520, 992)])
def test_matmul_ahead_by_quantised_rows(gpu_ctx, m, n, cols):
    """A projection quantised once, just in front of the rows, and used as a constant weight: the same bits as in stream
    order, a new one each time."""
    g = _gen(73)
    rows, made = g4.Nvfp4Rows(gpu_ctx, m, cols), [g4.Nvfp4Rows(gpu_ctx, n, cols, 1) for _ in range(8)]
    x, ws = _randn(g, m, cols), [_randn(g, n, cols, std=0.02) for _ in made]
    ahead, ordered = torch.empty((8, m, n), dtype=torch.bfloat16, device="cuda"), torch.empty((8, m, n), dtype=torch.bfloat16, device="cuda")
    assert g4.Nvfp4Weight.from_rows(made[0], constant=True).desc.constant == 1
    assert g4.Nvfp4Weight.from_rows(made[0]).desc.constant == 0
    for constant, outs in ((True, ahead), (False, ordered)):
        for w, r, out in zip(ws, made, outs):
            r.codes.fill_(0x77), r.scales.fill_(0x38)
            g4.nvfp4_quantize(gpu_ctx, w, r)
            g4.nvfp4_quantize(gpu_ctx, x, rows)
            g4.nvfp4_matmul(gpu_ctx, rows, g4.Nvfp4Weight.from_rows(r, constant=constant), out)
    _sync(gpu_ctx)
    assert torch.equal(ahead, ordered) and torch.isfinite(ahead).all() and ahead.float().std() > 0


def test_matmul_by_what_another_context_makes(gpu_ctx):
    """Two contexts on one stream: one quantises rows, the other then makes the weight (a piece of rows, scale blocks of
    a checkpoint's), and the first multiplies by it."""
    stream = torch.cuda.Stream()
    a, b = g4.Context(0, stream=stream), g4.Context(0, stream=stream)
    g = _gen(72)
    x, w = _randn(g, 3, 4096), _randn(g, 2048, 4096)
    codes = torch.randint(0, 256, (2048, 2048), generator=g, device="cuda", dtype=torch.uint8)
    given = [torch.randint(40, 70, (2048, 256), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    one = torch.ones(1, device="cuda")
    torch.cuda.synchronize()
    rows, made, first = g4.Nvfp4Rows(a, 3, 4096), g4.Nvfp4Rows(b, 2048, 4096, 2), g4.Nvfp4Rows(b, 2048, 4096, 1)
    piece = g4.Nvfp4Weight.from_rows(first)
    piece._set(made.codes, made.scales, made.factor, 2048, 4096, made.device)
    out, want = (torch.empty((3, 2048), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        g4.nvfp4_quantize(b, w, first)
        g4.nvfp4_quantize(a, x, rows)
        torch.cuda.synchronize()
        g4.nvfp4_matmul(a, rows, g4.Nvfp4Weight.from_rows(first), want)
        for _ in range(20):
            made.codes.fill_(0x77), made.scales.fill_(0x38)
            g4.nvfp4_quantize(a, x, rows)
            g4.nvfp4_quantize(b, w, made)
            g4.nvfp4_matmul(a, rows, piece, out)
            assert torch.equal(out, want)
        cx, sx, fx = ob.quantize(x, 2)
        for i in range(20):
            scales = given[i % 2]
            g4.nvfp4_quantize(a, x, rows)
            weight = g4.Nvfp4Weight(b, codes, scales, one)
            g4.nvfp4_matmul(a, rows, weight, out)
            y, size = ob.matmul(ob.values(cx, sx).sum(0), ob.values(ob.unpack(codes), scales), fx, one.double())
            assert ((out.double() - y).abs() <= (2 * 4096 / 64 + 12) * 2.0 ** -23 * size + U * y.abs()).all()
    torch.cuda.synchronize()
    for ctx in (a, b):
        assert ctx.poll() == 0
        ctx.close()


def test_matmul_nan_row_stays_in_its_row(gpu_ctx):
    x = _randn(_gen(3), 140, 512)
    x[7, 100], x[131, 0], x[20] = float("nan"), float("inf"), 0
    rows = g4.Nvfp4Rows(gpu_ctx, 140, 512)
    weight, _, _ = _weight(gpu_ctx, 384, 512)
    out = torch.empty((140, 384), dtype=torch.bfloat16, device="cuda")
    g4.nvfp4_quantize(gpu_ctx, x, rows)
    g4.nvfp4_matmul(gpu_ctx, rows, weight, out)
    _sync(gpu_ctx)
    bad = torch.zeros(140, dtype=torch.bool, device="cuda")
    bad[[7, 131]] = True
    assert out[bad].isnan().all() and torch.isfinite(out[~bad]).all() and (out[20] == 0).all()


def test_matmul_one_row_of_any_width(gpu_ctx):
    """One row's output has no row stride to speak of: wide, odd, by the kernel of many tiles."""
    for m, n in ((1, 160001), (1, 160008), (2, 160008)):
        _product(gpu_ctx, m, n, 32, 2)


def test_quantised_rows_are_a_weight(gpu_ctx):
    g = _gen(9)
    a, b = _randn(g, 70, 768), _randn(g, 200, 768, std=0.02)
    ra, rb = g4.Nvfp4Rows(gpu_ctx, 70, 768, 2), g4.Nvfp4Rows(gpu_ctx, 200, 768, 1)
    out = torch.empty((70, 200), dtype=torch.float32, device="cuda")
    g4.nvfp4_quantize(gpu_ctx, a, ra)
    g4.nvfp4_quantize(gpu_ctx, b, rb)
    g4.nvfp4_matmul(gpu_ctx, ra, g4.Nvfp4Weight.from_rows(rb), out)
    _sync(gpu_ctx)
    ca, sa, fa = ob.quantize(a, 2)
    cb, sb, fb = ob.quantize(b, 1)
    want, size = ob.matmul(ob.values(ca, sa).sum(0), ob.values(cb, sb)[0], fa, fb)
    assert ((out.double() - want).abs() <= (2 * 768 / 64 + 12) * 2.0 ** -23 * size).all()


# ------------------------------------------------------------------------------ quantise
def _check_rows(rows, want, n, cols):
    codes, scales, factor = want
    got = ob.unpack(rows.codes[:, :n])
    assert torch.equal(torch.where(got == 8, 0, got), codes)  # (zero has either sign)
    for p in range(rows.pieces):
        at = ob.scale_at(torch.arange(n, device="cuda")[:, None], torch.arange(cols // 16, device="cuda")[None, :], cols)
        assert torch.equal(rows.scales[p][at], scales[p])
        pad = [b for b in range(cols // 16, -(-cols // 64) * 4)]
        if pad:
            at = ob.scale_at(torch.arange(n, device="cuda")[:, None], torch.tensor([pad], device="cuda"), cols)
            assert (rows.scales[p][at] == 0).all()
    assert torch.equal(rows.factor[:n].double().nan_to_num(-1.0), factor.nan_to_num(-1.0))


@pytest.mark.parametrize("n, cols, pieces", [(1, 32, 1), (1, 3840, 2), (3, 96, 3), (130, 480, 2), (257, 2048, 3), (40, 2080, 1),
                                             (65, 8192, 2), (9, 15360, 3), (300, 16384, 1)])
@pytest.mark.parametrize("gap", [0, 8])
def test_quantize_is_the_oracles(gpu_ctx, n, cols, pieces, gap):
    x = _randn(_gen(n + cols), n, cols + gap)
    x *= torch.exp2(torch.randint(-30, 30, (n, 1), generator=_gen(1), device="cuda")).bfloat16()
    x = x[:, :cols]
    rows = g4.Nvfp4Rows(gpu_ctx, n + 5, cols, pieces)
    for t in (rows.codes, rows.scales):
        t.fill_(0xA5)
    rows.factor.fill_(-3.0)
    g4.nvfp4_quantize(gpu_ctx, x, rows)
    out = torch.full((n, cols + gap), 7.0, dtype=torch.bfloat16, device="cuda")
    g4.nvfp4_dequantize(gpu_ctx, rows, out[:, :cols])
    _sync(gpu_ctx)
    want = ob.quantize(x, pieces)
    _check_rows(rows, want, n, cols)
    assert (rows.codes[:, n:] == 0xA5).all() and (rows.factor[n:] == -3.0).all()
    last = ob.scale_at(torch.arange(n, n + 5, device="cuda")[:, None], torch.arange(cols // 16, device="cuda")[None, :], cols)
    assert all((rows.scales[p][last] == 0xA5).all() for p in range(pieces))
    assert torch.equal(out[:, :cols].double(), (ob.values(want[0], want[1]).sum(0) * want[2][:, None]).bfloat16().double())
    assert (out[:, cols:] == 7.0).all()


@pytest.mark.parametrize("n, cols", [(1, 3840), (50, 3840), (7, 96), (20, 8192), (5, 16384)])
def test_quantize_normed(gpu_ctx, n, cols):
    """The codes are those of the normed rows rounded to bf16: of the f32 products in their order, with a
    root from 64-bit sums."""
    g = _gen(n * cols)
    x, w = _randn(g, n, cols, std=3.0), (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).bfloat16()
    x[0] *= 1e-3
    x[n // 2:] *= 2.0 ** 100  # squares beyond f32
    rows = g4.Nvfp4Rows(gpu_ctx, n, cols, 2)
    g4.nvfp4_quantize(gpu_ctx, x, rows, w)
    _sync(gpu_ctx)
    r = (1 / (x.double().square().mean(1, keepdim=True) + ob.EPS).sqrt()).float()
    y = (x.float() * r * w.float()).bfloat16()
    _check_rows(rows, ob.quantize(y, 2), n, cols)
    exact = ob.rms(x, w)
    assert ((y.double() - exact).abs() <= (U + 2.0 ** -20) * exact.abs() + 2.0 ** -130).all()


@pytest.mark.parametrize("cols", [2048, 2080, 4096, 4128, 8192, 8224, 16384])
@pytest.mark.parametrize("pieces, normed", [(1, False), (2, True), (3, False)])
def test_quantize_many_rows_as_few(gpu_ctx, cols, pieces, normed):
    """A call of more rows than the GPU has SMs and calls of fewer give the same bits, the oracle's."""
    g = _gen(cols + pieces)
    x, w = _randn(g, 301, cols, std=2.0), (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).bfloat16() if normed else None
    x[5] = 0
    many, few = g4.Nvfp4Rows(gpu_ctx, 301, cols, pieces), [g4.Nvfp4Rows(gpu_ctx, 128, cols, pieces) for _ in range(3)]
    for r in (many, *few):
        r.scales.fill_(0)
    g4.nvfp4_quantize(gpu_ctx, x, many, w)
    for i, r in enumerate(few):
        g4.nvfp4_quantize(gpu_ctx, x[128 * i:128 * i + 128], r, w)
    _sync(gpu_ctx)
    assert torch.equal(many.codes, torch.cat([r.codes for r in few], 1)[:, :301])
    assert torch.equal(many.factor, torch.cat([r.factor for r in few])[:301])
    assert torch.equal(many.scales.view(pieces, -1), torch.cat([r.scales.view(pieces, -1) for r in few], 1))
    if not normed:
        _check_rows(many, ob.quantize(x, pieces), 301, cols)


def test_quantize_special_rows(gpu_ctx):
    """Rows of zeros, of the smallest and the largest numbers, ties of both roundings, infinities and NaN."""
    x = torch.zeros((14, 64), dtype=torch.bfloat16, device="cuda")
    x[1, 5] = 2.0 ** -133
    x[2] = _randn(_gen(1), 64) * 2.0 ** -126
    x[3, :] = torch.finfo(torch.bfloat16).max
    x[4, 0], x[4, 17] = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    x[5, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x[5, 8:16] = -x[5, :8]
    x[6, ::16] = torch.tensor([2688.0, 2688 / 2, 204.0, 6 * 17 / 16])  # scale ties
    x[7, 0], x[8, 63], x[9, 2] = float("inf"), -float("inf"), float("nan")
    x[10, 0], x[11, 0] = 42.0, 42.25  # either side of 2688 / 64
    x[12] = -0.0
    x[13, 0], x[13, 16:] = 1.0, 2.0 ** -20
    for pieces in (1, 3):
        rows = g4.Nvfp4Rows(gpu_ctx, 14, 64, pieces)
        g4.nvfp4_quantize(gpu_ctx, x, rows)
        out = torch.empty_like(x)
        g4.nvfp4_dequantize(gpu_ctx, rows, out)
        _sync(gpu_ctx)
        codes, scales, factor = ob.quantize(x, pieces)
        _check_rows(rows, (codes, scales, factor), 14, 64)
        assert out[7:10].isnan().all() and (out[12] == 0).all()
        # one piece of bf16's largest number is past it: max g = 2040, 340 rounds to the scale 352, and 6 of
        # these are 2112 (read back as inf: there is no bf16 for it)
        want = (ob.values(codes, scales).sum(0) * factor[:, None]).bfloat16()
        assert torch.equal(out.nan_to_num(1.0, 2.0, 3.0), want.nan_to_num(1.0, 2.0, 3.0))


def test_scale_blocks(gpu_ctx):
    for n, cols in ((1, 32), (130, 96), (300, 3840)):
        s = torch.randint(0, 127, (n, cols // 16), generator=_gen(n), device="cuda", dtype=torch.uint8)
        w = g4.Nvfp4Weight(gpu_ctx, torch.zeros((n, cols // 2), dtype=torch.uint8, device="cuda"), s.view(torch.float8_e4m3fn),
                           torch.ones(1, device="cuda"))
        _sync(gpu_ctx)
        assert torch.equal(w.scales, ob.scale_blocks(s))


def test_weights_made_in_a_loop_on_another_stream(gpu_ctx):
    """Block scales that are dropped as soon as the constructor is back, on a stream other than the context's, which is
    busy: each weight is laid out from its own, and multiplies as the oracle says."""
    ctx = g4.Context(0, stream=torch.cuda.Stream())
    n, cols = 700, 1024
    g = _gen(81)
    codes = torch.randint(0, 256, (n, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
    kept = [torch.randint(30, 70, (n, cols // 16), generator=g, device="cuda", dtype=torch.uint8) for _ in range(6)]
    rows, xv, fx = _rows(gpu_ctx, 5, cols, 2, 82)
    one, outs = torch.ones(1, device="cuda"), torch.zeros((6, 5, 704), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(ctx.stream):
        torch.cuda._sleep(100_000_000)  # (some 50 ms)
    weights = [g4.Nvfp4Weight(ctx, codes, k.clone().view(torch.float8_e4m3fn), one) for k in kept]
    for w, out in zip(weights, outs):
        g4.nvfp4_matmul(ctx, rows, w, out[:, :n])
    torch.cuda.synchronize()
    assert ctx.poll() == 0
    for w, k, out in zip(weights, kept, outs):
        assert torch.equal(w.scales, ob.scale_blocks(k))
        want, size = ob.matmul(xv, ob.values(ob.unpack(codes), k), fx, one.double())
        assert ((out[:, :n].double() - want).abs() <= (2 * cols / 64 + 12) * 2.0 ** -23 * size + U * want.abs()).all()
    ctx.close()


# ------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("n, vocab, dim, gap", [(1, 262144, 3840, 0), (1, 1, 8, 0), (300, 1000, 3840, 8), (7, 50, 24, 0),
                                                (513, 33, 8192, 16), (4096, 262144, 64, 0)])
def test_embed(gpu_ctx, n, vocab, dim, gap):
    g = _gen(n + dim)
    table = _randn(g, vocab, dim)
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    ids[0], ids[-1] = vocab - 1, 0
    wide = torch.full((n, dim + gap), 7.0, dtype=torch.bfloat16, device="cuda")
    for scale in (62.0, 0.3):
        g4.embed_tokens(gpu_ctx, table, ids, wide[:, :dim], scale)
        _sync(gpu_ctx)
        assert torch.equal(wide[:, :dim], (table[ids.long()].float() * scale).bfloat16())
        assert (wide[:, dim:] == 7.0).all()


def test_embed_ids_outside_the_table(gpu_ctx):
    table = torch.full((10, 16), float("inf"), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([3, -1, 10, 2 ** 31 - 1, -2 ** 31, 9], dtype=torch.int32, device="cuda")
    out = torch.full((6, 16), 7.0, dtype=torch.bfloat16, device="cuda")
    g4.embed_tokens(gpu_ctx, table, ids, out)
    with pytest.raises(g4.G4Error):
        gpu_ctx.poll()
    assert gpu_ctx.poll() == 0
    assert (out[1:5] == 0).all() and out[[0, 5]].isinf().all()


def test_embed_past_32_bits(gpu_ctx):
    """Rows beyond 2^31 elements of the table."""
    vocab, dim = 2 ** 18, 8448  # 2^31.04 elements
    table = torch.zeros((vocab, dim), dtype=torch.bfloat16, device="cuda")
    table[-1], table[0] = 3.0, 1.0
    out = torch.empty((2, dim), dtype=torch.bfloat16, device="cuda")
    g4.embed_tokens(gpu_ctx, table, torch.tensor([vocab - 1, 0], dtype=torch.int32, device="cuda"), out, 2.0)
    _sync(gpu_ctx)
    assert (out[0] == 6.0).all() and (out[1] == 2.0).all()


@pytest.mark.parametrize("n, dim, gap", [(1, 3840, 0), (1, 8, 0), (33, 3840, 8), (300, 24, 0), (5, 1032, 16), (64, 8192, 0), (9, 16384, 8)])
def test_residual_norm(gpu_ctx, n, dim, gap):
    g = _gen(n * dim)
    x, res = _randn(g, n, dim + gap, std=4.0)[:, :dim], _randn(g, n, dim + gap)[:, :dim]
    w = (1 + 0.3 * torch.randn(dim, generator=g, device="cuda")).bfloat16()
    x[0] *= 2.0 ** -20
    x[n // 2 + 1:] *= 2.0 ** 90  # squares beyond f32
    out = torch.full((n, dim + gap), 7.0, dtype=torch.bfloat16, device="cuda")
    g4.residual_norm(gpu_ctx, x, w, res, out[:, :dim])
    _sync(gpu_ctx)
    y = ob.rms(x, w)
    want = res.double() + y
    assert ((out[:, :dim].double() - want).abs() <= U * want.abs() + 2.0 ** -20 * (res.double().abs() + y.abs())).all()
    assert (out[:, dim:] == 7.0).all()
    for given, into in ((res.clone(), "residual"), (x.clone(), "x")):  # in place of either operand
        a, b = (x, given) if into == "residual" else (given, res)
        g4.residual_norm(gpu_ctx, a, w, b, given)
        _sync(gpu_ctx)
        assert torch.equal(given, out[:, :dim])


def test_residual_norm_zero_and_nan_rows(gpu_ctx):
    x = torch.zeros((3, 128), dtype=torch.bfloat16, device="cuda")
    x[1, 5] = float("nan")
    res = _randn(_gen(2), 3, 128)
    out = torch.empty_like(res)
    g4.residual_norm(gpu_ctx, x, torch.ones(128, dtype=torch.bfloat16, device="cuda"), res, out)
    _sync(gpu_ctx)
    assert torch.equal(out[[0, 2]], res[[0, 2]]) and out[1].isnan().all()


# ------------------------------------------------------------------------------ beams
def _select(ctx, logits, scores, k):
    groups = logits.shape[0]
    out = (torch.full((groups, k), 7.0, device="cuda"), *(torch.full((groups, k), -7, dtype=torch.int32, device="cuda") for _ in range(2)))
    g4.beam_select(ctx, logits, scores, *out)
    _sync(ctx)
    return out


def _check_beams(ctx, logits, scores, k):
    got, beams, tokens = _select(ctx, logits, scores, k)
    want, wb, wt = ob.beam_select(logits, scores, k)
    finite = torch.isfinite(want)
    assert torch.equal(beams.long(), wb) and torch.equal(tokens.long(), wt)
    assert torch.equal(finite, torch.isfinite(got)) and (got[~finite] == -math.inf).all()
    err = (got.double() - want)[finite].abs()
    assert (err <= 2.0 ** -20 + 2.0 ** -24 * want[finite].abs()).all()


@pytest.mark.parametrize("groups, beams, vocab, k", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 21), (1, 4, 262144, 8), (32, 4, 262144, 8), (3, 1, 262144, 64), (1, 64, 32003, 64),
    (5, 8, 4097, 16), (2, 64, 1000, 64), (1, 3, 2 ** 20, 7), (1, 64, 2 ** 20, 64), (700, 2, 333, 4), (9, 5, 65537, 3), (1, 2, 40, 64)])
def test_beam_select(gpu_ctx, groups, beams, vocab, k):
    g = _gen(groups + vocab)
    logits = _randn(g, groups, beams, vocab, std=3.0)
    scores = -10 * torch.rand((groups, beams), generator=g, device="cuda")
    _check_beams(gpu_ctx, logits, scores, k)


def test_beam_select_strides(gpu_ctx):
    g = _gen(4)
    wide = _randn(g, 3, 5, 1100, std=3.0)
    scores = torch.rand((3, 4), generator=g, device="cuda")
    for logits in (wide[:, 1:, 3:1004], wide[:, :4, 1:].transpose(0, 1)[:3, :3].contiguous().transpose(0, 1), wide[:, ::2, 5:900]):
        _check_beams(gpu_ctx, logits, scores[:, :logits.shape[1]].contiguous(), 6)


def test_beam_select_a_new_request(gpu_ctx):
    """All beams hold the prompt, only the first counts; one beam in all, none at all."""
    logits = _randn(_gen(5), 1, 1, 3000).expand(3, 4, 3000)
    scores = torch.full((3, 4), -math.inf, device="cuda")
    scores[0, 0], scores[1, 2] = 0.0, -3.5
    _check_beams(gpu_ctx, logits, scores, 8)
    got, beams, tokens = _select(gpu_ctx, logits, scores, 8)
    assert (beams[0] == 0).all() and (beams[1] == 2).all() and (beams[2] == 0).all()
    assert (got[2] == -math.inf).all() and tokens[2].tolist() == list(range(8))


def test_beam_select_equal_scores(gpu_ctx):
    """Constant logits, identical beams, few different values: the lowest (beam, token) first."""
    flat = torch.full((1, 4, 262144), 1.5, dtype=torch.bfloat16, device="cuda")
    _check_beams(gpu_ctx, flat, torch.zeros((1, 4), device="cuda"), 64)
    _check_beams(gpu_ctx, flat[..., :77], torch.tensor([[-1.0, 0.0, 0.0, -1.0]], device="cuda"), 64)
    few = torch.randint(0, 3, (2, 3, 50000), generator=_gen(6), device="cuda").bfloat16()
    few[:, 1] = few[:, 0]
    _check_beams(gpu_ctx, few, torch.zeros((2, 3), device="cuda"), 60)
    # the best ones side by side: all in a few threads' parts
    peak = _randn(_gen(7), 1, 2, 60000)
    peak[0, 0, 1024:65536:256] = 20.0
    peak[0, 1, 512:576] = 25.0
    _check_beams(gpu_ctx, peak, torch.zeros((1, 2), device="cuda"), 64)


def test_beam_select_values_that_are_not_finite(gpu_ctx):
    """Banned tokens (-inf); beams without any continuation: of +inf, NaN, -inf throughout, scores that are not
    finite.  They come after every other, in the order of (beam, token)."""
    logits = _randn(_gen(8), 4, 7, 500)
    logits[:, 0, ::3] = -math.inf
    logits[:, 1, 77] = math.nan
    logits[:, 2, 5] = math.inf
    logits[:, 3] = -math.inf
    logits[:, 6, 10:] = -math.inf
    scores = torch.zeros((4, 7), device="cuda")
    scores[:, 4], scores[:, 5] = math.nan, math.inf
    _check_beams(gpu_ctx, logits, scores, 64)
    wide = torch.full((1, 3, 40000), -math.inf, dtype=torch.bfloat16, device="cuda")
    wide[0, :, 7], wide[0, 0, 39000], wide[0, 1, 8:4000:9] = 1.0, math.nan, math.nan  # NaN with nothing but -inf about it
    _check_beams(gpu_ctx, wide, torch.zeros((1, 3), device="cuda"), 9)
    scores[1, 0], scores[2, 6], scores[3, [0, 6]] = -math.inf, math.nan, -math.inf
    _check_beams(gpu_ctx, logits, scores, 64)


def test_beam_select_lowest_and_largest_numbers(gpu_ctx):
    """Masks of the type's lowest value, rows of nothing else, logits as large as the type's."""
    low, high = torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max
    logits = _randn(_gen(13), 5, 3, 9000)
    logits[0, 0, 5:] = low
    logits[1] = low
    logits[2, 1, ::2], logits[2, 2, 77] = low, high
    logits[3, :, 100:200] = high
    logits[4, 0] = low
    logits[4, 0, 8000] = 2.0 ** 101
    _check_beams(gpu_ctx, logits, torch.tensor([[0.0, -1.0, -2.0]] * 5, device="cuda"), 16)


@pytest.mark.parametrize("k", [1, 8, 16, 17, 64])
def test_beam_select_orders(gpu_ctx, k):
    """Rows in order of value and against it, masked but for a few tokens, masked up to a place or from it, of two
    values: where the best lie together, or a great many are as good as the last one that is in."""
    g = _gen(40 + k)
    logits = _randn(g, 9, 2, 140003, std=3.0)
    logits[0], logits[1] = logits[0].sort(-1).values, logits[1].sort(-1, descending=True).values
    keep = torch.randint(0, 140003, (2, 40), generator=g, device="cuda")
    few = torch.full((2, 140003), -math.inf, dtype=torch.bfloat16, device="cuda")
    logits[2] = few.scatter(1, keep, logits[2].gather(1, keep))
    logits[3] = few.scatter(1, keep[:, :5], 1.0)
    logits[4, :, :70000], logits[5, :, 9000:] = -math.inf, torch.finfo(torch.bfloat16).min
    logits[6] = (torch.arange(140003, device="cuda") % 8192 > 8000).bfloat16()
    logits[7] = (torch.rand((2, 140003), generator=g, device="cuda") < 1e-3).bfloat16()
    logits[8, :, 1:140000] = 0.0  # both ends alone in what no 16-byte piece holds
    _check_beams(gpu_ctx, logits, -torch.rand((9, 2), generator=g, device="cuda"), k)
    _check_beams(gpu_ctx, logits[..., 3:131076], -torch.rand((9, 2), generator=g, device="cuda"), k)


def test_beam_select_one_beam_leads(gpu_ctx):
    """All of the best are one beam's, and a second's between them."""
    logits = _randn(_gen(41), 2, 32, 70001, std=3.0)
    scores = torch.full((2, 32), -300.0, device="cuda")
    scores[0, 7], scores[1, 0], scores[1, 31] = 0.0, 0.0, -0.125
    for k in (64, 33, 17):
        _check_beams(gpu_ctx, logits, scores, k)


def test_beam_select_scores_far_apart(gpu_ctx):
    g = _gen(11)
    logits = _randn(g, 2, 3, 2000, std=20.0)
    _check_beams(gpu_ctx, logits, torch.tensor([[-1e4, 0.0, -2e3], [-900.0, -900.25, -899.5]], device="cuda"), 12)


def test_matmul_by_a_piece_of_the_rows_before(gpu_ctx):
    """The C descriptors let a weight be one piece of rows of several, quantised by the call before."""
    g = _gen(60)
    x, w = _randn(g, 3, 4096), _randn(g, 2048, 4096)
    rows, made, first = g4.Nvfp4Rows(gpu_ctx, 3, 4096), g4.Nvfp4Rows(gpu_ctx, 2048, 4096, 2), g4.Nvfp4Rows(gpu_ctx, 2048, 4096, 1)
    out, want = (torch.empty((3, 2048), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g4.nvfp4_quantize(gpu_ctx, x, rows)
    g4.nvfp4_quantize(gpu_ctx, w, first)
    g4.nvfp4_matmul(gpu_ctx, rows, g4.Nvfp4Weight.from_rows(first), want)
    piece = g4.Nvfp4Weight.from_rows(first)
    piece._set(made.codes, made.scales, made.factor, 2048, 4096, made.device)
    for _ in range(20):
        made.codes.fill_(0x77), made.scales.fill_(0x38)
        g4.nvfp4_quantize(gpu_ctx, w, made)
        g4.nvfp4_matmul(gpu_ctx, rows, piece, out)
        assert torch.equal(out, want)


@pytest.mark.parametrize("vocab, offset", [(46, 7), (15, 1), (30, 5), (3000, 3)])
def test_beam_select_large_logits(gpu_ctx, vocab, offset):
    """Logits some hundreds in size, where a difference of exponents rounded to 32 bits shows in a score, of rows that
    are hardly more than what lies outside 16-byte pieces."""
    g = _gen(vocab)
    logits = _randn(g, 5, 17, vocab + offset, std=60.0)[..., offset:]
    _check_beams(gpu_ctx, logits, -torch.rand((5, 17), generator=g, device="cuda"), min(60, 17 * vocab))


# ------------------------------------------------------------------------------ calls
def test_calls_captured_and_replayed(gpu_ctx):
    """Embed, quantise, multiply, norm and select in one graph, on a stream of the context's own; replays follow
    their inputs."""
    stream = torch.cuda.Stream()
    ctx = g4.Context(0, stream=stream)
    g = _gen(12)
    table, w = _randn(g, 900, 512), torch.ones(512, dtype=torch.bfloat16, device="cuda")
    x, y, z = (torch.zeros((40, 512), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    logits = torch.zeros((40, 1000), dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(40, dtype=torch.int32, device="cuda")
    scores = torch.zeros((10, 4), device="cuda")
    outs = torch.zeros((10, 6), device="cuda"), *(torch.zeros((10, 6), dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    rows = g4.Nvfp4Rows(ctx, 40, 512)
    square, head = _weight(ctx, 512, 512)[0], _weight(ctx, 1000, 512, seed=3)[0]

    def step():
        g4.embed_tokens(ctx, table, ids, x)
        g4.nvfp4_quantize(ctx, x, rows, w)
        g4.nvfp4_matmul(ctx, rows, square, y)
        g4.residual_norm(ctx, y, w, x, z)
        g4.nvfp4_quantize(ctx, z, rows)
        g4.nvfp4_matmul(ctx, rows, head, logits)
        g4.beam_select(ctx, logits.view(10, 4, 1000), scores, *outs)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for i in range(3):
        ids.copy_(torch.randint(0, 900, (40,), generator=g, device="cuda"))
        scores.copy_(torch.rand((10, 4), generator=g, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (logits, *outs)]
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (logits, *outs)))
        assert got[0].float().std() > 0
    assert ctx.poll() == 0
    del graph
    ctx.close()


WORK_ON = """
extern "C" __global__ void work_on(int microseconds, unsigned* out) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  unsigned long long now, end;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
  end = now + 1000ull * microseconds;
  unsigned turns = 0;
  while (now < end && ++turns < 100000000u) asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
  out[0] = turns;
}
"""


@pytest.mark.parametrize("m, n, cols, pieces", [(1, 3840, 4096, 2), (33, 129, 480, 3), (100, 2049, 8192, 1), (600, 2048, 992, 1)])
def test_matmul_behind_a_kernel_that_works_on(gpu_ctx, m, n, cols, pieces):
    """The kernel before lets its dependents start and then takes ten times the context's wait budget: that is no time
    of the product's own waits, which hold and give the oracle's values."""
    ctx = g4.Context(0, stream=torch.cuda.Stream())
    ctx.set_wait_budget(2000)
    work_on = torch.cuda._compile_kernel(WORK_ON, "work_on")
    turns = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows, xv, fx = _rows(gpu_ctx, m, cols, pieces, 51)
    weight, wv, fw = _weight(gpu_ctx, n, cols, 1, 52)
    out = torch.full((m, (n + 7) // 8 * 8), 7.0, dtype=torch.bfloat16, device="cuda")[:, :n]
    torch.cuda.synchronize()
    with torch.cuda.stream(ctx.stream):
        work_on(grid=(1, 1, 1), block=(32, 1, 1), args=[20000, turns])
        g4.nvfp4_matmul(ctx, rows, weight, out)
    torch.cuda.synchronize()
    assert turns.item() > 0 and ctx.poll() == 0
    want, size = ob.matmul(xv, wv, fx, fw)
    assert ((out.double() - want).abs() <= (pieces * cols / 64 + 12) * 2.0 ** -23 * size + U * want.abs()).all()
    ctx.close()


@pytest.mark.parametrize("m, n, cols, pieces", [(1, 3840, 4096, 2), (20, 8192, 3840, 2), (33, 129, 480, 3), (100, 2049, 8192, 1),
                                                (600, 2048, 992, 1)])
def test_matmul_with_a_budget_of_microseconds(gpu_ctx, m, n, cols, pieces):
    """A product whose budget is hardly more than its copies take is right, or the status says that a wait ran out
    (64 tries come before the budget, and may each wait in the hardware, so that few or none do); those behind it are
    right, with nothing of it under way."""
    ctx = g4.Context(0, stream=torch.cuda.Stream())
    rows, xv, fx = _rows(gpu_ctx, m, cols, pieces, 61)
    weight, wv, fw = _weight(gpu_ctx, n, cols, 1, 62)
    out = torch.full((m, (n + 7) // 8 * 8), 7.0, dtype=torch.bfloat16, device="cuda")[:, :n]
    want, size = ob.matmul(xv, wv, fx, fw)
    bound = (pieces * cols / 64 + 12) * 2.0 ** -23 * size + U * want.abs()
    right = lambda: bool(((out.double() - want).abs() <= bound).all())  # noqa: E731

    def told():
        try:
            return ctx.poll() != 0
        except g4.G4Error as e:
            assert e.code == 4  # G4_ERR_TIMEOUT
            return True

    torch.cuda.synchronize()
    for budget in range(1, 31):
        out.fill_(7.0)
        torch.cuda.synchronize()
        ctx.set_wait_budget(budget)
        g4.nvfp4_matmul(ctx, rows, weight, out)
        torch.cuda.synchronize()
        assert told() or right(), budget
        g4.nvfp4_matmul(ctx, rows, weight, out)
        ctx.set_wait_budget(2000000)
        g4.nvfp4_matmul(ctx, rows, weight, out)
        torch.cuda.synchronize()
        assert right()
        told()
        out.fill_(7.0)
        torch.cuda.synchronize()
        g4.nvfp4_matmul(ctx, rows, weight, out)
        torch.cuda.synchronize()
        assert right() and not told()
    ctx.close()


def test_two_contexts_at_once(gpu_ctx):
    """Products (clusters, pairs, single CTAs) and selections of two contexts on two streams, side by side: the same
    bits as one after another."""
    g = _gen(30)
    logits, scores = _randn(g, 3, 4, 20000, std=3.0), torch.rand((3, 4), generator=g, device="cuda")
    shapes = [(1, 3840, 4096, 2), (40, 1024, 3840, 2), (600, 2048, 992, 1), (7, 30720, 512, 2), (300, 3840, 1024, 3)]
    ctxs = [g4.Context(0, stream=torch.cuda.Stream()) for _ in range(2)]
    sets = []
    for ctx in ctxs:
        ops = []
        for m, n, k, p in shapes:
            rows, weight = _rows(ctx, m, k, p)[0], _weight(ctx, n, k)[0]
            ops.append((rows, weight, torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")))
        outs = torch.zeros((3, 9), device="cuda"), *(torch.zeros((3, 9), dtype=torch.int32, device="cuda") for _ in range(2))
        sets.append((ops, outs))

    def run(ctx, ops, outs):
        for rows, weight, out in ops:
            g4.nvfp4_matmul(ctx, rows, weight, out)
        g4.beam_select(ctx, logits, scores, *outs)

    torch.cuda.synchronize()
    want = []
    for ctx, s in zip(ctxs, sets):
        run(ctx, *s)
        torch.cuda.synchronize()
        want.append([t.clone() for t in [o[2] for o in s[0]] + list(s[1])])
        for t in [o[2] for o in s[0]] + list(s[1]):
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for ctx, s in zip(ctxs, sets):
            run(ctx, *s)
    torch.cuda.synchronize()
    for ctx, s, w in zip(ctxs, sets, want):
        assert all(torch.equal(a, b) for a, b in zip([o[2] for o in s[0]] + list(s[1]), w))
        assert ctx.poll() == 0
        ctx.close()


def test_library_refuses(gpu_ctx):
    """The C entry points' own checks: sizes, alignment, strides, null pointers."""
    L, h = g4.LIB, gpu_ctx.handle
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = t.data_ptr()
    rows = lambda codes=p, scales=p, factor=p, m=4, cols=64, pieces=2: g4.batch._RowsDesc(codes, scales, factor, m, cols, pieces)  # noqa: E731
    weight = lambda codes=p, scales=p, factor=p, n=8, cols=64, f=1: g4.batch._WeightDesc(codes, scales, factor, n, cols, f)  # noqa: E731
    bad = [
        L.g4_embed_tokens(h, p, 0, 8, p, 1, 1.0, p, 8), L.g4_embed_tokens(h, p, 4, 12, p, 1, 1.0, p, 16),
        L.g4_embed_tokens(h, p, 4, 8, p + 2, 1, 1.0, p, 8), L.g4_embed_tokens(h, p + 2, 4, 8, p, 1, 1.0, p, 8),
        L.g4_embed_tokens(h, p, 4, 8, p, 2, 1.0, p, 4), L.g4_embed_tokens(h, p, 4, 8, p, 2, 1.0, p, 12),
        L.g4_embed_tokens(h, p, 4, 8, p, -1, 1.0, p, 8), L.g4_embed_tokens(h, p, 4, 8, None, 1, 1.0, p, 8),
        L.g4_residual_norm(h, p, 8, p, p, 8, 2, 12, p, 16), L.g4_residual_norm(h, p, 4, p, p, 8, 2, 8, p, 8),
        L.g4_residual_norm(h, p, 8, None, p, 8, 2, 8, p, 8), L.g4_residual_norm(h, p, 8, p, p, 8, -1, 8, p, 8),
        L.g4_residual_norm(h, p, 32768, p, p, 32768, 1, 32768, p, 32768),
        L.g4_nvfp4_scale_blocks(h, p, 4, 48, p), L.g4_nvfp4_scale_blocks(h, None, 4, 64, p), L.g4_nvfp4_scale_blocks(h, p, 4, 64, p + 4),
        L.g4_nvfp4_quantize(h, p, 64, 5, None, rows()), L.g4_nvfp4_quantize(h, p, 64, 4, None, None),
        L.g4_nvfp4_quantize(h, p, 64, 4, p + 2, rows()), L.g4_nvfp4_quantize(h, p + 2, 64, 4, None, rows()),
        L.g4_nvfp4_quantize(h, p, 32, 4, None, rows()), L.g4_nvfp4_quantize(h, p, 64, 4, None, rows(pieces=4)),
        L.g4_nvfp4_quantize(h, p, 64, 4, None, rows(cols=80)), L.g4_nvfp4_quantize(h, p, 64, 4, None, rows(scales=p + 4)),
        L.g4_nvfp4_quantize(h, p, 64, 4, None, rows(codes=None)), L.g4_nvfp4_quantize(h, p, 64, 0, None, rows(m=0)),
        L.g4_nvfp4_dequantize(h, rows(), 4, p, 32), L.g4_nvfp4_dequantize(h, rows(), 4, None, 64), L.g4_nvfp4_dequantize(h, rows(), -1, p, 64),
        L.g4_nvfp4_matmul(h, rows(), 4, weight(cols=96), p, 8, 0), L.g4_nvfp4_matmul(h, rows(), 4, weight(f=2), p, 8, 0),
        L.g4_nvfp4_matmul(h, rows(), 4, weight(n=0), p, 8, 0), L.g4_nvfp4_matmul(h, rows(), 4, None, p, 8, 0),
        L.g4_nvfp4_matmul(h, rows(), 4, weight(), p, 4, 0), L.g4_nvfp4_matmul(h, rows(), 4, weight(), p, 12, 0),
        L.g4_nvfp4_matmul(h, rows(), 4, weight(codes=p + 8), p, 8, 0), L.g4_nvfp4_matmul(h, rows(), 4, weight(factor=None), p, 8, 0),
        L.g4_nvfp4_matmul(h, rows(), 4, weight(), None, 8, 0), L.g4_nvfp4_matmul(h, rows(), 5, weight(), p, 8, 0),
        L.g4_beam_select(h, p, 9, 9, p, 1, 0, 9, 1, p, p, p), L.g4_beam_select(h, p, 9, 9, p, 1, 1, 9, 10, p, p, p),
        L.g4_beam_select(h, p, 9, 9, p, 1, 65, 9, 1, p, p, p), L.g4_beam_select(h, p, 9, 9, p, 1, 2, 0, 1, p, p, p),
        L.g4_beam_select(h, p, 9, 9, p, 1, 2, 2 ** 20 + 1, 1, p, p, p), L.g4_beam_select(h, p, 9, 9, p, -1, 2, 9, 1, p, p, p),
        L.g4_beam_select(h, p + 1, 9, 9, p, 1, 2, 9, 1, p, p, p), L.g4_beam_select(h, p, 9, -9, p, 1, 2, 9, 1, p, p, p),
        L.g4_beam_select(h, p, 9, 9, p + 2, 1, 2, 9, 1, p, p, p), L.g4_beam_select(h, p, 9, 9, p, 1, 2, 9, 1, p, p, None),
    ]
    assert bad == [1] * len(bad)
    assert L.g4_ctx_last_error(h)
    ok = [L.g4_embed_tokens(h, p, 4, 8, p, 0, 1.0, None, 0), L.g4_nvfp4_quantize(h, None, 0, 0, None, rows()),
          L.g4_nvfp4_matmul(h, rows(), 0, weight(), None, 0, 0), L.g4_beam_select(h, None, 0, 0, None, 0, 2, 9, 1, None, None, None),
          L.g4_residual_norm(h, None, 0, None, None, 0, 0, 8, None, 0), L.g4_nvfp4_scale_blocks(h, None, 0, 64, None)]
    assert ok == [0] * len(ok)
    _sync(gpu_ctx)
    assert not t.any()
    assert ctypes.sizeof(g4.batch._RowsDesc) == 40 and ctypes.sizeof(g4.batch._WeightDesc) == 40


def test_library_refuses_other_constants(gpu_ctx):
    t = torch.zeros(1 << 14, dtype=torch.uint8, device="cuda")
    p = t.data_ptr()
    rows, weight = g4.batch._RowsDesc(p, p, p, 4, 64, 2), g4.batch._WeightDesc(p, p, p, 8, 64, 1, 2)
    assert g4.LIB.g4_nvfp4_matmul(gpu_ctx.handle, rows, 4, weight, p, 8, 0) == 1
    weight.constant = -1
    assert g4.LIB.g4_nvfp4_matmul(gpu_ctx.handle, rows, 4, weight, p, 8, 0) == 1
    _sync(gpu_ctx)


def test_beam_select_zero_of_either_sign(gpu_ctx):
    """-0 and 0 are equal scores: the lower token first, whichever sign it has."""
    logits = torch.full((1, 2, 3000), -5.0, dtype=torch.bfloat16, device="cuda")
    logits[0, 0, 100:140:2], logits[0, 0, 101:140:2] = -0.0, 0.0
    logits[0, 1, 2900:] = -0.0
    _check_beams(gpu_ctx, logits, torch.tensor([[0.0, -0.5]], device="cuda"), 64)


@pytest.mark.parametrize("offset", range(8))
def test_beam_select_alignments(gpu_ctx, offset):
    """Rows that start and end anywhere between 16-byte borders."""
    g = _gen(offset)
    for vocab in (1, 6, 9, 15, 16, 17, 23, 300, 4100):
        wide = _randn(g, 2, 3, vocab + 16 + offset, std=3.0)
        _check_beams(gpu_ctx, wide[:, :, offset:offset + vocab], torch.rand((2, 3), generator=g, device="cuda"), min(5, 3 * vocab))


@pytest.mark.parametrize("offset", range(8))
def test_beam_select_short_rows_of_few_tokens(gpu_ctx, offset):
    """Rows that are hardly more than what lies outside 16-byte pieces, -inf but for none to three tokens, beside a beam
    that counts and one that does not: as many as were asked for come out, whatever their score."""
    g = _gen(70 + offset)
    groups = 24
    for vocab in range(1, 41):
        keep = torch.rand((groups, 2, vocab), generator=g, device="cuda").argsort(-1) < torch.arange(groups, device="cuda")[:, None, None] % 4
        wide = torch.zeros((groups, 2, vocab + 8), dtype=torch.bfloat16, device="cuda")
        logits = wide[..., offset:offset + vocab]
        logits.copy_(torch.where(keep, _randn(g, groups, 2, vocab, std=2.0), -math.inf))
        scores = torch.zeros((groups, 2), device="cuda")
        scores[::2, 1], scores[1::4, 0] = -math.inf, -0.5
        for beams in (1, 2):
            for k in (1, 2, 3, 7, 16, 17, 64):
                if k <= beams * vocab:
                    _check_beams(gpu_ctx, logits[:, :beams], scores[:, :beams].contiguous(), k)


def test_beam_example():
    """Three requests' beams through six layers, their caches reordered at every step: the score that the search kept
    is the one that the best beam's text has when it is run alone.  (24 logits and their sums, each off by what
    bf16 leaves of it and of the residual stream below: a few hundredths of about 4.5 each, at random.)"""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import beam_serving

    r = beam_serving.main()
    assert all(-200 < s < -20 for s in r["scores"])
    assert r["relative difference of the scores"] <= 3e-2
