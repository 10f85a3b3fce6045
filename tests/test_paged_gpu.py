"""Paged caches on the GPU against the float64 oracle: attention of chunks and single tokens
over pages, norm/rotary/store, page copies and compaction, their layouts, edges and refusals.

Error bounds, from the arithmetic the operators document (u = 2^-8: bf16 has 8
significant bits, rounding to nearest is off by at most half a unit in the last):
  attention  the weights of V are rounded to bf16 (u of sum p |v|), the result once more (u of
             |o| <= sum p |v|); scores, softmax and sums are f32 (below 2^-12 of the same sum
             at these score sizes): |error| <= (2u + 2^-11) sum p |v|
  store      f32 throughout (2^-20 of the two products' magnitudes), rounded once:
             |error| <= u |y| + 2^-18 (|a| + |b|)
"""

import math
import random

import pytest
import torch

import g4b200 as g4
from oracle import paged as op

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
SLIDING, FULL = (16, 8, 256), (16, 1, 512)


def _cache_pair(layout, n_pages, page_rows, hkv, d, fill):
    """K and V of shape [n_pages, page_rows, hkv, d] in one of several memory layouts."""
    if layout == "nhd":
        k, v = (torch.full((n_pages, page_rows, hkv, d), fill, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    elif layout == "hnd":
        k, v = (torch.full((n_pages, hkv, page_rows, d), fill, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
                for _ in range(2))
    elif layout == "kv_in_page":
        kv = torch.full((n_pages, 2, page_rows, hkv, d), fill, dtype=torch.bfloat16, device="cuda")
        k, v = kv[:, 0], kv[:, 1]
    else:  # padded rows
        k, v = (torch.full((n_pages, page_rows + 8, hkv + 1, d + 8), fill, dtype=torch.bfloat16,
                           device="cuda")[:, :page_rows, :hkv, :d] for _ in range(2))
    return k, v


def _setup(lens, heads=SLIDING, page_rows=16, window=0, layout="nhd", seed=0, poison=float("nan"), std=2.5,
           bad_entry=-1):
    """Caches that hold `poison` in every row no token may read, tables in random order with
    `bad_entry` where nothing may be looked up."""
    hq, hkv, d = heads
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    need = []
    for s, (n, kv) in enumerate(lens):
        lo = max(0, kv - n - window + 1) if window else 0
        if n:
            need += [(s, p) for p in range(lo // page_rows, -(-kv // page_rows))]
    n_pages = len(need) + 3
    ids = rng.sample(range(n_pages), len(need))
    width = max([1] + [-(-kv // page_rows) for _, kv in lens]) + 1
    tables = [[bad_entry] * width for _ in lens]
    k, v = _cache_pair(layout, n_pages, page_rows, hkv, d, poison)
    for (s, p), i in zip(need, ids):
        tables[s][p] = i
        n, kv = lens[s]
        lo = max(0, kv - n - window + 1) if window else 0
        a, b = max(lo, p * page_rows) - p * page_rows, min(kv, (p + 1) * page_rows) - p * page_rows
        k[i, a:b] = torch.randn((b - a, hkv, d), generator=g, device="cuda").bfloat16()
        v[i, a:b] = torch.randn((b - a, hkv, d), generator=g, device="cuda").bfloat16()
    tokens = sum(n for n, _ in lens)
    q = (torch.randn((tokens, hq, d), generator=g, device="cuda") * (std / math.sqrt(d))).bfloat16()
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = g4.PagedBatch(i32(tables), i32(starts), i32([kv for _, kv in lens]))
    return q, g4.PagedCache(k, v), batch, tables


def _check_attention(out, q, cache, tables, lens, scale=1.0, window=0):
    want, weight = op.attention(q, cache.k, cache.v, tables, lens, scale, window)
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    worst = (err - (2 * U + 2.0 ** -11) * weight).max().item()
    assert worst <= 0, f"error above its bound by {worst} (largest error {err.max().item()})"


def _attend(ctx, q, cache, batch, scale=1.0, window=0):
    out = torch.full_like(q, float("nan"))
    g4.paged_attention(ctx, q, cache, batch, out, scale=scale, window=window)
    torch.cuda.synchronize()
    assert ctx.poll() == 0
    return out


ATTEND = [
    # lens [(new tokens, cache rows)], heads, page_rows, window
    ([(1, 1)], SLIDING, 16, 0),
    ([(1, 1)], FULL, 512, 0),
    ([(1, 1000)], SLIDING, 64, 1024),
    ([(1, 8192)], FULL, 512, 0),
    ([(1, n) for n in (1, 2, 63, 64, 65, 127, 128, 129, 130, 255, 256, 257, 383, 385, 1023)], SLIDING, 8, 0),
    ([(1, n) for n in (1, 2, 63, 64, 65, 127, 128, 129, 130, 255, 256, 257, 383, 385, 1023)], FULL, 24, 0),
    ([(3, 3), (2, 700), (129, 129), (0, 40), (128, 500), (1, 64), (127, 127), (257, 300)], SLIDING, 16, 0),
    ([(3, 3), (2, 700), (9, 129), (0, 40), (16, 500), (1, 64), (17, 127), (33, 300)], FULL, 16, 0),
    ([(1, 5000), (300, 2000), (1, 1), (77, 1100)], SLIDING, 64, 1024),
    ([(40, 1500), (1, 1025), (1, 1024), (1, 1023)], SLIDING, 24, 1024),
    ([(200, 200)], SLIDING, 8, 1),
    ([(200, 333), (1, 9)], SLIDING, 16, 7),
    ([(64, 400), (5, 131)], FULL, 8, 130),
    ([(1, 300)] * 70, SLIDING, 32, 0),
    ([(1, 40 * i + 1) for i in range(40)], FULL, 40, 0),
    ([(5, 9000), (1, 20000)], FULL, 512, 0),
    ([(600, 9001)], SLIDING, 128, 0),
    # more new tokens than rows: the first ones see nothing
    ([(5, 2), (1, 0), (40, 0), (300, 17), (1, 6)], SLIDING, 8, 0),
    ([(20, 3), (1, 0), (2, 130)], FULL, 8, 16),
    # head layouts: a rank's shares, groups that divide nothing
    ([(1, 77), (50, 200)], (4, 2, 256), 16, 0),
    ([(1, 77), (50, 200)], (2, 1, 512), 16, 0),
    ([(100, 200), (1, 333)], (15, 5, 256), 16, 100),
    ([(31, 200), (1, 333)], (7, 1, 512), 16, 0),
    ([(90, 200), (1, 333)], (3, 3, 256), 16, 0),
    ([(9, 150), (1, 333)], (80, 2, 256), 16, 0),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(gpu_ctx, case):
    lens, heads, page_rows, window = ATTEND[case]
    q, cache, batch, tables = _setup(lens, heads, page_rows, window, seed=case)
    out = _attend(gpu_ctx, q, cache, batch, window=window)
    _check_attention(out, q, cache, tables, lens, window=window)
    again = _attend(gpu_ctx, q, cache, batch, window=window)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("layout", ["hnd", "kv_in_page", "padded"])
@pytest.mark.parametrize("heads", [SLIDING, FULL])
def test_attention_layouts_and_strides(gpu_ctx, layout, heads):
    lens, hq, d = [(70, 300), (1, 129), (1, 512)], heads[0], heads[2]
    q, cache, batch, tables = _setup(lens, heads, 16, 0, layout, seed=3, bad_entry=2 ** 30)
    wide = torch.randn(q.shape[0], hq + 3, d + 8, device="cuda").bfloat16()
    wide[:, 2:hq + 2, :d] = q
    out_wide = torch.full((hq, q.shape[0] + 2, d), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    out = out_wide[1:-1]
    g4.paged_attention(gpu_ctx, wide[:, 2:hq + 2, :d], cache, batch, out)
    torch.cuda.synchronize()
    assert gpu_ctx.poll() == 0
    _check_attention(out, q, cache, tables, lens)
    assert (out_wide[0] == 7).all() and (out_wide[-1] == 7).all()


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -3.3895e38, 3.3895e38])
@pytest.mark.parametrize("heads", [SLIDING, FULL])
def test_attention_never_uses_rows_it_may_not_see(gpu_ctx, poison, heads):
    lens = [(130, 200), (1, 61), (3, 390), (1, 128)]
    q, cache, batch, tables = _setup(lens, heads, 64, 50, seed=4, poison=poison)
    _check_attention(_attend(gpu_ctx, q, cache, batch, window=50), q, cache, tables, lens, window=50)


@pytest.mark.parametrize("scale,std", [(0.0, 1.0), (0.0625, 20.0), (-1.0, 2.0), (1.0, 40.0), (1e-3, 1.0)])
@pytest.mark.parametrize("heads", [SLIDING, FULL])
def test_attention_scales(gpu_ctx, scale, std, heads):
    """Flat and very peaked softmaxes (at std 40 scores reach +-150: exp without its maximum
    would overflow).  f32 scores of size 150 carry 2^-24 * 150 * sqrt(d)-ish absolute error, far below
    the bound's 2^-11."""
    lens = [(70, 500), (1, 700)]
    q, cache, batch, tables = _setup(lens, heads, 32, 0, seed=5, std=std)
    _check_attention(_attend(gpu_ctx, q, cache, batch, scale=scale), q, cache, tables, lens, scale=scale)


def test_attention_rising_scores(gpu_ctx):
    """Keys whose scores rise by 30 every 100 rows: the running maximum moves all the way."""
    lens = [(130, 1000), (1, 999)]
    q, cache, batch, tables = _setup(lens, SLIDING, 8, 0, seed=6)
    q.zero_()
    q[:, :, 0] = 1.0
    for s, (n, kv) in enumerate(lens):
        for p in range(-(-kv // 8)):
            rows = torch.arange(8 * p, 8 * p + 8, device="cuda")
            cache.k[tables[s][p], :, :, 0] = torch.where(rows < kv, 0.3 * rows, float("nan"))[:, None].bfloat16()
    _check_attention(_attend(gpu_ctx, q, cache, batch), q, cache, tables, lens)


def test_attention_tokens_of_no_sequence_are_left_alone(gpu_ctx):
    lens = [(3, 30), (1, 20)]
    q, cache, batch, tables = _setup(lens, SLIDING)
    more = torch.cat([q, torch.full_like(q[:2], float("nan"))])
    out = torch.full_like(more, 5.0)
    g4.paged_attention(gpu_ctx, more, cache, batch, out)
    torch.cuda.synchronize()
    assert gpu_ctx.poll() == 0 and (out[4:] == 5).all()
    _check_attention(out[:4], q, cache, tables, lens)


def test_attention_empty_calls(gpu_ctx):
    q, cache, batch, _ = _setup([(2, 20)], SLIDING)
    g4.paged_attention(gpu_ctx, q[:0], cache, batch, q[:0].clone())
    none = g4.PagedBatch(batch.tables[:0], batch.q_start[:1], batch.kv_len[:0])
    out = torch.full_like(q, 5.0)
    g4.paged_attention(gpu_ctx, q, cache, none, out)
    # a sequence without rows in a batch without table columns
    empty = g4.PagedBatch(batch.tables[:, :0], batch.q_start, torch.zeros_like(batch.kv_len))
    zero = torch.full_like(q, 5.0)
    g4.paged_attention(gpu_ctx, q, cache, empty, zero)
    torch.cuda.synchronize()
    assert gpu_ctx.poll() == 0 and (out == 5).all() and (zero == 0).all()


def test_attention_past_32_bit_offsets(gpu_ctx):
    """Pages that lie more than 2^32 bytes (and 2^31 elements) into the cache."""
    hq, hkv, d = SLIDING
    lens = [(3, 40), (1, 17)]
    q, small, batch, tables = _setup(lens, SLIDING, 16)
    stride = 2 ** 31 // 8 + 4096
    n = small.n_pages
    assert n * stride > 2 ** 31
    k, v = (torch.empty(n * stride, dtype=torch.bfloat16, device="cuda").as_strided(
        (n, 16, hkv, d), (stride, hkv * d, d, 1)) for _ in range(2))
    # the pages furthest into the buffer are the ones in use
    order = sorted({p for t in tables for p in t if p >= 0})
    move = dict(zip(order, range(n - len(order), n)))
    for a, b in move.items():
        k[b], v[b] = small.k[a], small.v[a]
    tables = [[move.get(p, -1) for p in t] for t in tables]
    big = g4.PagedBatch(torch.tensor(tables, dtype=torch.int32, device="cuda"), batch.q_start, batch.kv_len)
    cache = g4.PagedCache(k, v)
    _check_attention(_attend(gpu_ctx, q, cache, big), q, cache, tables, lens)


def test_attention_follows_a_captured_batch():
    """One captured call, replayed after the batch's contents changed on the device."""
    stream = torch.cuda.Stream()
    lens = [(3, 200), (1, 500), (2, 90)]
    with torch.cuda.stream(stream):
        ctx = g4.Context(0, stream)
        q, cache, batch, tables = _setup([(n, kv + 60) for n, kv in lens], FULL, 16, seed=8)
        out = torch.empty_like(q)
        g4.paged_attention(ctx, q, cache, batch, out)  # allocates the scratch
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            g4.paged_attention(ctx, q, cache, batch, out)
        for grow in (0, 13, 60):
            now = [(n, kv + grow) for n, kv in lens]
            batch.kv_len.copy_(torch.tensor([kv for _, kv in now], dtype=torch.int32))
            out.fill_(float("nan"))
            graph.replay()
            stream.synchronize()
            _check_attention(out, q, cache, tables, now)
        assert ctx.poll() == 0
        del graph
        ctx.close()


@pytest.mark.parametrize("what", ["page_high", "page_low", "kv_long", "kv_negative", "start_high", "start_falls"])
@pytest.mark.parametrize("heads", [SLIDING, FULL])
def test_attention_flags_a_bad_batch(gpu_ctx, what, heads):
    """Nothing out of range is followed; the status word says so; other sequences are right."""
    lens = [(2, 100), (3, 150)]
    q, cache, batch, tables = _setup(lens, heads, 16, poison=0.0)
    if what == "page_high":
        batch.tables[1, 3] = cache.n_pages
    elif what == "page_low":
        batch.tables[1, 3] = -5
    elif what == "kv_long":
        batch.kv_len[1] = 2 ** 31 - 1
    elif what == "kv_negative":
        batch.kv_len[1] = -7
    elif what == "start_high":
        batch.q_start[2] = 2 ** 30
    else:
        batch.q_start[2] = 1
    out = torch.full_like(q, 5.0)
    g4.paged_attention(gpu_ctx, q, cache, batch, out)
    with pytest.raises(g4.G4Error):
        gpu_ctx.poll()
    assert gpu_ctx.poll() == 0
    _check_attention(out[:2], q[:2], cache, tables[:1], lens[:1])


def test_refusals(gpu_ctx):
    q, cache, batch, _ = _setup([(2, 20)], SLIDING)
    out = torch.empty_like(q)
    bf = torch.bfloat16
    for call, err in [
        (lambda: g4.paged_attention(gpu_ctx, q.float(), cache, batch, out), TypeError),
        (lambda: g4.paged_attention(gpu_ctx, q.cpu(), cache, batch, out), ValueError),
        (lambda: g4.paged_attention(gpu_ctx, q[:, :, :128], cache, batch, out), ValueError),
        (lambda: g4.paged_attention(gpu_ctx, q[:, :15], cache, batch, out[:, :15]), ValueError),
        (lambda: g4.paged_attention(gpu_ctx, q, cache, batch, out[:1]), ValueError),
        (lambda: g4.paged_attention(gpu_ctx, q, cache, batch, out[:1].expand(2, -1, -1)), g4.G4Error),
        (lambda: g4.paged_attention(gpu_ctx, q[0], cache, batch, out), ValueError),
        (lambda: g4.paged_attention(gpu_ctx, q, cache, batch, out, scale=float("nan")), g4.G4Error),
        (lambda: g4.paged_attention(gpu_ctx, q, cache, batch, out, window=-1), g4.G4Error),
        (lambda: g4.PagedCache(cache.k, cache.v[:1]), ValueError),
        (lambda: g4.PagedCache(cache.k.float(), cache.v.float()), TypeError),
        (lambda: g4.PagedCache(cache.k.transpose(2, 3), cache.v.transpose(2, 3)), ValueError),
        (lambda: g4.PagedBatch(batch.tables, batch.q_start[:1], batch.kv_len), ValueError),
        (lambda: g4.PagedBatch(batch.tables.long(), batch.q_start, batch.kv_len), TypeError),
        (lambda: g4.PagedBatch(batch.tables[:, ::2], batch.q_start, batch.kv_len), ValueError),
        (lambda: g4.paged_copy(gpu_ctx, g4.PagedCaches([cache]), batch.kv_len, batch.kv_len, batch.q_start),
         ValueError),
        (lambda: g4.paged_compact(gpu_ctx, g4.PagedCaches([cache]), batch.kv_len, batch.kv_len, batch.tables,
                                  batch.kv_len), ValueError),
    ]:
        with pytest.raises(err):
            call()

    def with_cache(k, v=None):
        g4.paged_attention(gpu_ctx, torch.empty(2, 16, k.shape[3], dtype=bf, device="cuda"),
                           g4.PagedCache(k, k if v is None else v), batch,
                           torch.empty(2, 16, k.shape[3], dtype=bf, device="cuda"))

    buf = torch.zeros(2 ** 16, dtype=bf, device="cuda")
    for k, code in [(buf[:8192].view(4, 8, 2, 128), 5),             # head_dim
                    (buf[:12288].view(1, 12, 4, 256), 1),           # page_rows
                    (buf[4:4 + 16384].view(4, 8, 2, 256), 1),       # alignment
                    (buf.as_strided((4, 8, 2, 256), (4100, 512, 256, 1)), 1),
                    (buf.as_strided((4, 8, 2, 256), (0, 512, 256, 1)), 1),
                    (buf.as_strided((4, 8, 2, 256), (4096, 512, 128, 1)), 1)]:
        with pytest.raises(g4.G4Error) as e:
            with_cache(k)
        assert e.value.code == code, (k.shape, k.stride())
    small = g4.PagedCache(cache.k[:1], cache.v[:1])
    pool = g4.PagePool(cache.n_pages + 1, cache.page_rows)  # not this cache's pool: nothing changes
    s = pool.add()
    pool.extend(s, 30)
    for call in (lambda: pool.compact(gpu_ctx, g4.PagedCaches([cache]), batch.tables),
                 lambda: pool.run_copies(gpu_ctx, g4.PagedCaches([cache]))):
        with pytest.raises(ValueError, match="pool"):
            call()
    assert pool.table(s)[1] == 30
    with pytest.raises(g4.G4Error):
        g4.paged_copy(gpu_ctx, g4.PagedCaches([cache, small]), batch.kv_len, batch.kv_len, batch.kv_len)
    assert gpu_ctx.poll() == 0


# ------------------------------------------------------------------------------ store
STORE = [([(1, 1)], SLIDING, 8), ([(1, 1000)], SLIDING, 64), ([(1, 513)], FULL, 512),
         ([(37, 90), (1, 200), (0, 3), (130, 130), (9, 1000)], SLIDING, 24),
         ([(37, 90), (1, 200), (0, 3), (130, 130), (9, 1000)], FULL, 16),
         ([(1, 17 * i + 1) for i in range(70)], (4, 2, 256), 16), ([(5, 2), (3, 0), (2, 2)], (3, 1, 512), 8)]


def _store_inputs(lens, heads, seed, n_positions=2048):
    hq, hkv, d = heads
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    tokens = sum(n for n, _ in lens)
    size = torch.exp2(torch.randint(-12, 12, (tokens, 1, 1), generator=g, device="cuda").float())
    qkv = (rnd(tokens, hq + 2 * hkv, d) * size).bfloat16()
    ang = rnd(n_positions, d // 2) * 10
    cos = torch.cat([ang.cos(), ang.cos()], 1).bfloat16()
    sin = torch.cat([-ang.sin(), ang.sin()], 1).bfloat16()
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], rnd(d).bfloat16(), rnd(d).bfloat16(), cos, sin


@pytest.mark.parametrize("layout", ["nhd", "hnd", "kv_in_page"])
@pytest.mark.parametrize("case", range(len(STORE)))
def test_store(gpu_ctx, case, layout):
    lens, heads, page_rows = STORE[case]
    _, cache, batch, tables = _setup(lens, heads, page_rows, layout=layout, seed=case, poison=3.0)
    q, k, v, qw, kw, cos, sin = _store_inputs(lens, heads, case)
    before = cache.k.clone(), cache.v.clone()
    out = torch.full(q.shape, 9.0, dtype=torch.bfloat16, device="cuda")
    g4.paged_store_qkv(gpu_ctx, q, k, v, qw, kw, cos, sin, cache, batch, out)
    torch.cuda.synchronize()
    assert gpu_ctx.poll() == 0
    pos = torch.tensor([kv - n + i for n, kv in lens for i in range(n)], device="cuda")
    seq = [s for s, (n, _) in enumerate(lens) for _ in range(n)]
    live = pos >= 0
    c, s_ = cos[pos.clamp(min=0)], sin[pos.clamp(min=0)]

    def close(got, want, size):
        err = (got.double() - want).abs() - (U * want.abs() + 2.0 ** -18 * size)
        assert err.max().item() <= 0

    want, size = op.rotate(op.norm(q, qw), c, s_)
    close(out[live], want[live], size[live])
    assert (out[~live] == 0).all()
    kwant, ksize = op.rotate(op.norm(k, kw), c, s_)
    vwant = op.norm(v)
    touched = torch.zeros(cache.n_pages, page_rows, dtype=torch.bool, device="cuda")
    for i in range(len(seq)):
        p = int(pos[i])
        if p < 0:
            continue
        page, row = tables[seq[i]][p // page_rows], p % page_rows
        touched[page, row] = True
        close(cache.k[page, row], kwant[i], ksize[i])
        close(cache.v[page, row], vwant[i], vwant[i].abs())
    assert torch.equal(cache.k[~touched], before[0][~touched]) and torch.equal(cache.v[~touched], before[1][~touched])


def test_store_in_place_and_zero_rows(gpu_ctx):
    lens = [(6, 40)]
    _, cache, batch, _ = _setup(lens, SLIDING)
    q, k, v, qw, kw, cos, sin = _store_inputs(lens, SLIDING, 1)
    q[2], k[3], v[4] = 0, 0, 0
    apart = torch.empty(q.shape, dtype=torch.bfloat16, device="cuda")
    g4.paged_store_qkv(gpu_ctx, q, k, v, qw, kw, cos, sin, cache, batch, apart)
    first = cache.k.clone(), cache.v.clone()
    g4.paged_store_qkv(gpu_ctx, q, k, v, qw, kw, cos, sin, cache, batch, q)
    torch.cuda.synchronize()
    assert gpu_ctx.poll() == 0
    assert torch.equal(q, apart) and (apart[2] == 0).all() and torch.isfinite(apart).all()
    same = lambda a, b: torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))  # noqa: E731
    assert same(cache.k, first[0]) and same(cache.v, first[1])


@pytest.mark.parametrize("what", ["page", "position"])
def test_store_skips_and_flags_what_is_out_of_range(gpu_ctx, what):
    lens = [(3, 40), (2, 100)]
    _, cache, batch, tables = _setup(lens, SLIDING, poison=3.0)
    q, k, v, qw, kw, cos, sin = _store_inputs(lens, SLIDING, 1, 2048 if what == "page" else 60)
    if what == "page":
        batch.tables[1, 6] = cache.n_pages
    before = cache.k.clone()
    out = torch.full(q.shape, 9.0, dtype=torch.bfloat16, device="cuda")
    g4.paged_store_qkv(gpu_ctx, q, k, v, qw, kw, cos, sin, cache, batch, out)
    with pytest.raises(g4.G4Error):
        gpu_ctx.poll()
    assert (out[3:] == 0).all() and (out[:3] != 9).any()
    page = tables[0][37 // 16]
    changed = (cache.k != before).flatten(1).any(1)
    assert changed[page] and int(changed.sum()) == 1


# ------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("layout", ["nhd", "hnd", "kv_in_page", "padded"])
@pytest.mark.parametrize("page_rows", [8, 24, 64])
def test_copy(gpu_ctx, layout, page_rows):
    rng = random.Random(page_rows)
    layers = [_cache_pair(layout, 50, page_rows, hkv, d, 0.0) for hkv, d in ((8, 256), (1, 512), (3, 256))]
    for k, v in layers:
        k.copy_(torch.randn(k.shape, device="cuda"))
        v.copy_(torch.randn(v.shape, device="cuda"))
    ids = rng.sample(range(50), 40)
    src, dst = ids[:20], ids[20:]
    src[1] = src[0]
    rows = [0, page_rows, 1] + [rng.randint(0, page_rows) for _ in range(17)]
    want = [(k.clone(), v.clone()) for k, v in layers]
    for pair in want:
        for t in pair:
            for s, d, r in zip(src, dst, rows):
                t[d, :r] = t[s, :r]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    caches = g4.PagedCaches([g4.PagedCache(k, v) for k, v in layers])
    g4.paged_copy(gpu_ctx, caches, i32(src), i32(dst), i32(rows))
    torch.cuda.synchronize()
    assert gpu_ctx.poll() == 0
    for pair, expect in zip(layers, want):
        for t, e in zip(pair, expect):
            assert torch.equal(t, e)


def test_copy_skips_and_flags_bad_pages(gpu_ctx):
    k, v = (torch.randn(6, 8, 2, 256, device="cuda").bfloat16() for _ in range(2))
    want = k.clone()
    want[4, :3] = want[0, :3]
    want[5] = want[1]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    g4.paged_copy(gpu_ctx, g4.PagedCaches([g4.PagedCache(k, v)]), i32([0, -1, 6, 2, 1]), i32([4, 3, 3, 6, 5]),
                  i32([3, 8, 8, 8, 100]))
    with pytest.raises(g4.G4Error):
        gpu_ctx.poll()
    assert torch.equal(k, want)
    g4.paged_copy(gpu_ctx, g4.PagedCaches([g4.PagedCache(k, v)]), i32([]), i32([]), i32([]))
    assert gpu_ctx.poll() == 0 and torch.equal(k, want)


def test_many_layers_take_several_launches(gpu_ctx):
    layers = [tuple(torch.randn(4, 8, 1, 512, device="cuda").bfloat16() for _ in range(2)) for _ in range(60)]
    want = [[t.clone() for t in kv] for kv in layers]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    tables = i32([[3, 0, -1], [1, 3, 9]])
    caches = g4.PagedCaches([g4.PagedCache(k, v) for k, v in layers])
    g4.paged_compact(gpu_ctx, caches, i32([3]), i32([2]), tables, i32([0, 1, 2, 2]))
    with pytest.raises(g4.G4Error):  # entry 9
        gpu_ctx.poll()
    assert tables.tolist() == [[2, 0, -1], [1, 2, 9]]
    for kv, e in zip(layers, want):
        for t, x in zip(kv, e):
            x[2] = x[3]
            assert torch.equal(t, x)


def test_pool_on_the_gpu(gpu_ctx):
    """Prefill, fork, append, trim, compact: every sequence attends its own rows throughout."""
    hq, hkv, d = SLIDING
    page_rows, rng = 16, random.Random(0)
    pool = g4.PagePool(64, page_rows)
    k, v = _cache_pair("nhd", 64, page_rows, hkv, d, float("nan"))
    cache = g4.PagedCache(k, v)
    caches = g4.PagedCaches([cache])
    own = {}  # sequence -> its K and V rows, kept apart
    g = torch.Generator(device="cuda").manual_seed(0)

    def append(seqs, counts):
        for s, n in zip(seqs, counts):
            pool.extend(s, n)
        pool.run_copies(gpu_ctx, caches)
        for s, n in zip(seqs, counts):
            new = torch.randn((2, n, hkv, d), generator=g, device="cuda").bfloat16()
            table, rows = pool.table(s)
            for i in range(n):
                r = rows - n + i
                k[table[r // page_rows], r % page_rows] = new[0, i]
                v[table[r // page_rows], r % page_rows] = new[1, i]
            own[s] = torch.cat([own[s], new], 1) if s in own else new
        check(seqs, counts)

    def check(seqs, counts, tables=None):
        batch = pool.batch(gpu_ctx, seqs, counts) if tables is None else tables
        q = (torch.randn((sum(counts), hq, d), generator=g, device="cuda") * 0.15).bfloat16()
        out = _attend(gpu_ctx, q, cache, batch, window=40)
        t0 = 0
        for s, n in zip(seqs, counts):
            kk, vv = (own[s][i][None] for i in range(2))
            want, weight = op.attention(q[t0:t0 + n], kk, vv, [[0]], [(n, own[s].shape[1])], 1.0, 40)
            err = (out[t0:t0 + n].double() - want).abs()
            assert (err <= (2 * U + 2.0 ** -11) * weight).all()
            t0 += n

    a, b = pool.add(), pool.add()
    append([a, b], [75, 20])
    c, e = pool.fork(a), pool.fork(a)
    own[c], own[e] = own[a].clone(), own[a].clone()
    for step in range(6):
        append([a, c, e, b], [1, 3, rng.randint(1, 20), 1])
    pool.free(a)
    del own[a]
    pool.trim(e, own[e].shape[1] - 60)
    batch = pool.batch(gpu_ctx, [e, b, c], [2, 1, 1])
    moved = pool.compact(gpu_ctx, caches, batch.tables)
    assert moved > 0
    assert batch.tables.tolist() == pool.batch(gpu_ctx, [e, b, c], [2, 1, 1]).tables.tolist()
    k[64 - pool.free_pages:] = float("nan")
    v[64 - pool.free_pages:] = float("nan")
    check([e, b, c], [2, 1, 1], batch)
    append([c, b, e], [2, 2, 2])


def test_serving_example():
    """The example's users, served from shared, copied and compacted pages, get what they get
    alone: both sides round each weight and each output to bf16 once, in different tilings
    (2^-8 apiece in relative norm at most)."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import paged_serving

    r = paged_serving.main()
    assert r["pages moved"] > 0 and r["relative difference"] <= 4 * U


# batches near the line between the two kernels (as many tokens as sequences), skewed ones too
SPLIT = [
    ([(33, 33), (0, 5), (0, 0)] + [(0, 7)] * 30, SLIDING, 16, 0),  # as many tokens as sequences
    ([(20, 900), (0, 5), (1, 300), (0, 0)] + [(0, 7)] * 17, FULL, 24, 0),
    ([(1, 700)] * 9 + [(200, 1500)] + [(8, 400), (9, 400), (7, 7)], SLIDING, 8, 100),
    ([(1, 700)] * 9 + [(200, 1500)] + [(2, 400), (3, 400), (0, 9)], FULL, 64, 0),
    ([(1, 300), (1, 1), (5, 260), (6, 131)], (15, 5, 256), 16, 40),
    ([(1, 300), (1, 1), (2, 260), (3, 131)], (7, 1, 512), 16, 0),
    ([(1, 300), (2, 1), (3, 0), (90, 40)], (17, 1, 256), 16, 0),  # no group of 17 is few
    ([(1, 300), (40, 200)], (200, 1, 256), 16, 0),
    ([(1, 12), (4, 4)], (4, 4, 512), 512, 0),
    ([(1, 1 + i % 90) for i in range(1500)], SLIDING, 8, 0),
    ([(i % 3, 1 + i % 90) for i in range(400)], FULL, 16, 33),
    ([(1, 30000), (1, 12345)], SLIDING, 512, 0),
]


@pytest.mark.parametrize("case", range(len(SPLIT)))
def test_attention_split_between_kernels(gpu_ctx, case):
    lens, heads, page_rows, window = SPLIT[case]
    q, cache, batch, tables = _setup(lens, heads, page_rows, window, seed=100 + case)
    out = _attend(gpu_ctx, q, cache, batch, window=window)
    _check_attention(out, q, cache, tables, lens, window=window)
    assert torch.equal(out, _attend(gpu_ctx, q, cache, batch, window=window))


def test_attention_of_one_token_repeated_by_a_zero_stride(gpu_ctx):
    lens = [(40, 100)]
    q, cache, batch, tables = _setup(lens, SLIDING)
    same = q[:1, :1].expand(40, 16, 256)
    out = torch.empty_like(q)
    g4.paged_attention(gpu_ctx, same, cache, batch, out)
    torch.cuda.synchronize()
    assert gpu_ctx.poll() == 0
    _check_attention(out, same.contiguous(), cache, tables, lens)


def test_attention_on_another_stream():
    """The call runs on its context's stream, whatever torch's current stream is."""
    stream = torch.cuda.Stream()
    ctx = g4.Context(0, stream)
    lens = [(50, 300), (1, 77)]
    q, cache, batch, tables = _setup(lens, FULL)
    out = torch.full_like(q, float("nan"))
    stream.wait_stream(torch.cuda.current_stream())
    g4.paged_attention(ctx, q, cache, batch, out)
    torch.cuda.current_stream().wait_stream(stream)
    _check_attention(out, q, cache, tables, lens)
    assert ctx.poll() == 0
    ctx.close()


def test_attention_refuses_more_tiles_than_it_counts(gpu_ctx):
    rows = 65536
    k = torch.zeros(1, rows, 1, 256, dtype=torch.bfloat16, device="cuda")
    tables = torch.zeros(1, 2 ** 21, dtype=torch.int32, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = g4.PagedBatch(tables, i32([0, 2000]), i32([2000]))
    q = torch.zeros(2000, 16, 256, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(g4.G4Error) as e:
        g4.paged_attention(gpu_ctx, q, g4.PagedCache(k, k), batch, q.clone())
    assert e.value.code == 6
