"""The operators around a batch's attention without a GPU: refusals of the bindings, the oracle's roundings,
reordered sequences of a page pool."""

import ctypes
import random

import pytest
import torch

import g4b200 as g4
from oracle import batch as ob
from oracle import ops


class _Ctx:
    """A context of no GPU: what the bindings check passes to the library, which refuses it."""

    device, handle, stream = -1, None, None

    def _check(self, fn, code):
        raise g4.G4Error(fn, code, "")


CTX = _Ctx()
bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
f32 = lambda *s: torch.zeros(s)  # noqa: E731
u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731


def _rows(n=4, cols=64, pieces=2):
    r = object.__new__(g4.Nvfp4Rows)
    r.max_rows, r.cols, r.pieces, r.device, r.desc = n, cols, pieces, -1, g4.batch._RowsDesc()
    r.codes, r.scales, r.factor = u8(pieces, n, cols // 2), u8(pieces, 512), f32(n)
    return r


def _weight(n=8, cols=64):
    w = object.__new__(g4.Nvfp4Weight)
    w.rows, w.cols, w.device, w.desc = n, cols, -1, g4.batch._WeightDesc()
    return w


REFUSED = {
    "tokens of 64 bits": lambda: g4.embed_tokens(CTX, bf(4, 8), i32(2).long(), bf(2, 8)),
    "table of f32": lambda: g4.embed_tokens(CTX, f32(4, 8), i32(2), bf(2, 8)),
    "table not contiguous": lambda: g4.embed_tokens(CTX, bf(4, 16)[:, :8], i32(2), bf(2, 8)),
    "out of another width": lambda: g4.embed_tokens(CTX, bf(4, 8), i32(2), bf(2, 16)),
    "out of other tokens": lambda: g4.embed_tokens(CTX, bf(4, 8), i32(2), bf(3, 8)),
    "no tensor": lambda: g4.embed_tokens(CTX, [[0.0]], i32(2), bf(2, 8)),
    "residual of other rows": lambda: g4.residual_norm(CTX, bf(2, 8), bf(8), bf(3, 8), bf(2, 8)),
    "norm weight of other columns": lambda: g4.residual_norm(CTX, bf(2, 8), bf(16), bf(2, 8), bf(2, 8)),
    "columns apart": lambda: g4.residual_norm(CTX, bf(2, 16)[:, ::2], bf(8), bf(2, 8), bf(2, 8)),
    "x of other columns": lambda: g4.nvfp4_quantize(CTX, bf(2, 32), _rows()),
    "more rows than room": lambda: g4.nvfp4_quantize(CTX, bf(5, 64), _rows()),
    "x of f16": lambda: g4.nvfp4_quantize(CTX, bf(2, 64).half(), _rows()),
    "rms weight of f32": lambda: g4.nvfp4_quantize(CTX, bf(2, 64), _rows(), f32(64)),
    "more rows read back than there are": lambda: g4.nvfp4_dequantize(CTX, _rows(), bf(5, 64)),
    "out of other columns than the weight": lambda: g4.nvfp4_matmul(CTX, _rows(), _weight(), bf(2, 16)),
    "weight of other columns": lambda: g4.nvfp4_matmul(CTX, _rows(), _weight(8, 96), bf(2, 8)),
    "out of f16": lambda: g4.nvfp4_matmul(CTX, _rows(), _weight(), bf(2, 8).half()),
    "columns that are no multiple of 32": lambda: g4.Nvfp4Rows(CTX, 4, 48),
    "four pieces": lambda: g4.Nvfp4Rows(CTX, 4, 64, 4),
    "no rows": lambda: g4.Nvfp4Rows(CTX, 0, 64),
    "too many columns": lambda: g4.Nvfp4Rows(CTX, 4, 32768),
    "codes of half a block": lambda: g4.Nvfp4Weight(CTX, u8(4, 24), u8(4, 3), f32(1)),
    "block scales of another shape": lambda: g4.Nvfp4Weight(CTX, u8(4, 32), u8(4, 3), f32(1)),
    "two global scales for four rows": lambda: g4.Nvfp4Weight(CTX, u8(4, 32), u8(4, 4), f32(2)),
    "a weight of two pieces": lambda: g4.Nvfp4Weight.from_rows(_rows(pieces=2)),
    "logits of f32": lambda: g4.beam_select(CTX, f32(1, 2, 9), f32(1, 2), f32(1, 3), i32(1, 3), i32(1, 3)),
    "logits apart": lambda: g4.beam_select(CTX, bf(1, 2, 18)[..., ::2], f32(1, 2), f32(1, 3), i32(1, 3), i32(1, 3)),
    "scores of other beams": lambda: g4.beam_select(CTX, bf(1, 2, 9), f32(1, 3), f32(1, 3), i32(1, 3), i32(1, 3)),
    "outputs of different counts": lambda: g4.beam_select(CTX, bf(1, 2, 9), f32(1, 2), f32(1, 3), i32(1, 4), i32(1, 3)),
    "more than there are": lambda: g4.beam_select(CTX, bf(1, 1, 9), f32(1, 1), f32(1, 10), i32(1, 10), i32(1, 10)),
    "65 beams": lambda: g4.beam_select(CTX, bf(1, 65, 9), f32(1, 65), f32(1, 3), i32(1, 3), i32(1, 3)),
    "65 selected": lambda: g4.beam_select(CTX, bf(1, 9, 9), f32(1, 9), f32(1, 65), i32(1, 65), i32(1, 65)),
    "none selected": lambda: g4.beam_select(CTX, bf(1, 9, 9), f32(1, 9), f32(1, 0), i32(1, 0), i32(1, 0)),
    "rows past 32 bits": lambda: g4.residual_norm(CTX, bf(1, 8).expand(2 ** 32 + 1, 8), bf(8), bf(1, 8).expand(2 ** 32 + 1, 8),
                                                  bf(1, 8).expand(2 ** 32 + 1, 8)),
}


@pytest.mark.parametrize("case", REFUSED)
def test_bindings_refuse(case):
    with pytest.raises((ValueError, TypeError)):
        REFUSED[case]()


def test_bindings_refuse_tensors_of_another_device():
    ctx = _Ctx()
    ctx.device = 0
    with pytest.raises(ValueError, match="context is on cuda:0"):
        g4.embed_tokens(ctx, bf(4, 8), i32(2), bf(2, 8))
    with pytest.raises(ValueError, match="context is on cuda:0"):
        g4.nvfp4_matmul(ctx, _rows(), _weight(), bf(2, 8))


def test_calls_of_no_rows_reach_no_library():
    g4.embed_tokens(CTX, bf(4, 8), i32(0), bf(0, 8))
    g4.residual_norm(CTX, bf(0, 8), bf(8), bf(0, 8), bf(0, 8))
    g4.nvfp4_quantize(CTX, bf(0, 64), _rows())
    g4.nvfp4_dequantize(CTX, _rows(), bf(0, 64))
    g4.nvfp4_matmul(CTX, _rows(), _weight(), bf(0, 8))
    g4.beam_select(CTX, bf(0, 2, 9), f32(0, 2), f32(0, 3), i32(0, 3), i32(0, 3))


def test_c_entry_points_refuse_a_null_context():
    L, r, w = g4.LIB, g4.batch._RowsDesc(), g4.batch._WeightDesc()
    assert L.g4_embed_tokens(None, None, 1, 8, None, 1, 1.0, None, 8) == 1
    assert L.g4_residual_norm(None, None, 8, None, None, 8, 1, 8, None, 8) == 1
    assert L.g4_nvfp4_scale_blocks(None, None, 1, 32, None) == 1
    assert L.g4_nvfp4_quantize(None, None, 32, 1, None, r) == 1
    assert L.g4_nvfp4_dequantize(None, r, 1, None, 32) == 1
    assert L.g4_nvfp4_matmul(None, r, 1, w, None, 8, 0) == 1
    assert L.g4_beam_select(None, None, 0, 0, None, 1, 1, 9, 1, None, None, None) == 1


def test_weight_descriptors_in_place():
    """The field behind n_factors fills what was padding: descriptors keep their size."""
    assert ctypes.sizeof(g4.batch._WeightDesc) == 40 and g4.batch._WeightDesc.constant.offset == 36
    assert g4.batch._WeightDesc(1, 2, 3, 4, 5, 6).constant == 0


def test_scale_bytes():
    assert g4.LIB.g4_nvfp4_scale_bytes(1, 32) == 512
    assert g4.LIB.g4_nvfp4_scale_bytes(129, 3840) == 2 * 60 * 512
    assert g4.LIB.g4_nvfp4_scale_bytes(2 ** 22, 16384) == 2 ** 32
    assert g4.LIB.g4_nvfp4_scale_bytes(-1, 64) == 0


def test_scale_blocks_place_every_scale_once():
    for rows, nb in ((1, 2), (200, 6), (128, 4), (129, 10)):
        at = {ob.scale_at(r, b, 16 * nb) for r in range(rows) for b in range(nb)}
        assert len(at) == rows * nb and max(at) < g4.LIB.g4_nvfp4_scale_bytes(rows, 16 * nb)


def test_oracle_rounds_as_the_formats_do():
    """Against the weight quantiser's oracle, which the reference's fixtures pin."""
    v = torch.cat([torch.linspace(0, 7, 7001), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])])
    got = torch.tensor(ob.E2M1)[ob._nearest(v.double(), ob.E2M1)]
    assert torch.equal(got, torch.from_numpy(ops.e2m1_round(v.numpy())))
    v = torch.cat([torch.logspace(-12, 9, 5001, base=2.0), torch.tensor(ob.E4M3)[:-1] + torch.diff(torch.tensor(ob.E4M3)) / 2])
    got = torch.tensor(ob.E4M3)[ob._nearest(v.double(), ob.E4M3)]
    assert torch.equal(got, torch.from_numpy(ops.e4m3_round(v.float().numpy())))
    assert torch.equal(got.float(), v.clamp(max=448).float().to(torch.float8_e4m3fn).float())


def test_oracle_pieces_close_in_on_the_row():
    x = torch.randn(20, 256, generator=torch.Generator().manual_seed(1)).bfloat16()
    left = []
    for p in (1, 2, 3):
        c, s, f = ob.quantize(x, p)
        total = ob.values(c, s).sum(0) * f[:, None]
        left.append(((total - x.double()).norm() / x.double().norm()).item())
    assert 0.05 < left[0] < 0.15 and left[1] < 0.15 * left[0] and left[2] < 0.15 * left[1]


# ------------------------------------------------------------------------------ reordered sequences
def test_reorder_swaps_and_copies():
    pool = g4.PagePool(10, 8)
    a, b, c = (pool.add() for _ in range(3))
    for s, n in ((a, 20), (b, 9), (c, 1)):
        pool.extend(s, n)
    ta, tb = pool.table(a), pool.table(b)
    pool.reorder([a, b, c], [b, a, a])
    assert (pool.table(a), pool.table(b), pool.table(c), pool.free_pages) == (tb, ta, ta, 5)
    pool.extend(c, 1)  # its last page is shared with b: a copy of its own
    assert pool.take_copies() == [([ta[0][2]], [pool.table(c)[0][2]], [4])]
    pool.reorder([], [])
    pool.reorder([a, b, c], [a, a, a])
    assert pool.free_pages == 8 and all(pool.table(s) == tb for s in (a, b, c))
    for s in (a, b, c):
        pool.free(s)
    assert pool.free_pages == 10


def test_reorder_refuses():
    pool = g4.PagePool(10, 8)
    a, b = pool.add(), pool.add()
    pool.extend(a, 8)
    before = pool.table(a), pool.table(b), pool.free_pages
    for seqs, parents in (([a, a], [a, b]), ([a, 7], [a, b]), ([a, b], [a, 7]), ([a, -1], [a, b])):
        with pytest.raises(g4.G4Error):
            pool.reorder(seqs, parents)
    with pytest.raises(ValueError, match="length"):
        pool.reorder([a], [a, b])
    with pytest.raises(ValueError, match="32 bits"):
        pool.reorder([a], [2 ** 32 + a])
    assert g4.LIB.g4_page_pool_reorder(pool.handle, None, None, 1) == 1
    assert g4.LIB.g4_page_pool_reorder(pool.handle, None, None, -1) == 1
    assert g4.LIB.g4_page_pool_reorder(None, None, None, 0) == 1
    assert (pool.table(a), pool.table(b), pool.free_pages) == before


@pytest.mark.parametrize("seed", range(4))
def test_beams_keep_their_rows(seed):
    """Beams that continue one another at random, their rows written through their tables."""
    rng = random.Random(seed)
    pool = g4.PagePool(60, 8)
    first = pool.add()
    beams = [first] + [pool.fork(first) for _ in range(4)]
    store, want = {}, {s: [] for s in beams}
    for step in range(60):
        parents = [rng.choice(beams) for _ in beams]
        pool.reorder(beams, parents)
        want = {s: list(want[p]) for s, p in zip(beams, parents)}
        if step % 7 == 6:
            low = max(0, len(want[first]) - 20)
            for s in beams:
                pool.trim(s, low)
        for s in beams:
            pool.extend(s, 1)
        for src, dst, rows in pool.take_copies():
            new = {(d, r): store.get((s, r)) for s, d, n in zip(src, dst, rows) for r in range(n)}
            store.update(new)
        for s in beams:
            table, rows = pool.table(s)
            store[table[(rows - 1) // 8], (rows - 1) % 8] = (step, s)
            want[s].append((step, s))
        for s in beams:
            table, rows = pool.table(s)
            held = [(r, table[r // 8]) for r in range(rows) if table[r // 8] >= 0]
            assert rows == len(want[s]) and all(store[p, r % 8] == want[s][r] for r, p in held) and len(held) >= min(rows, 20)
    for s in beams:
        pool.free(s)
    assert pool.free_pages == 60


def test_reorder_passes_null_safely():
    n = ctypes.c_int32()
    assert g4.LIB.g4_page_pool_reorder(None, ctypes.byref(n), ctypes.byref(n), 1) == 1
