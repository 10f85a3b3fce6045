"""Paged caches on the GPU: the corners of the paged operators that tests/test_paged_gpu.py does not
reach, against the same float64 oracle (u = 2^-8, half a unit in the last place of bf16)."""

import math

import pytest
import torch

import g4b200 as g4
from oracle import paged as op
from test_paged_gpu import FULL, SLIDING, U, _attend, _check_attention, _setup, _store_inputs

pytestmark = pytest.mark.gpu

# calls of few rows (as many tokens as sequences, or 16 rows at most)
FEW = [
    ([(1, 1000)], SLIDING, 64, 1024),
    ([(1, 8192)], FULL, 512, 0),
    ([(1, n) for n in (1, 2, 127, 130, 700, 1023)], SLIDING, 16, 0),
    ([(1, n) for n in (1, 2, 127, 130, 700, 1023)], FULL, 24, 0),
    ([(1, 40 * i + 300) for i in range(40)], FULL, 40, 0),
    ([(3, 900), (0, 5), (0, 7)], SLIDING, 16, 100),
    ([(8, 500)], SLIDING, 8, 0),
    ([(1, 400)], (5, 1, 256), 16, 0),
    ([(1, 400), (1, 3000)], (9, 1, 512), 16, 0),
]


@pytest.mark.parametrize("case", range(len(FEW)))
def test_few_rows_keep_the_weights_of_v(gpu_ctx, case):
    """The kernel for few rows carries a weight as two bf16: off by u^2 = 2^-16 of itself at most.
    Scores, softmax and sums in f32 are off by less than 2^-15 of sum p |v| (scores of std 2.5: their
    sums of |q k| are below 40, in f32 by a tensor core 2^-22 of that), so 2^-13 covers both with
    room; the output is rounded once."""
    lens, heads, page_rows, window = FEW[case]
    q, cache, batch, tables = _setup(lens, heads, page_rows, window, seed=40 + case)
    out = _attend(gpu_ctx, q, cache, batch, window=window)
    want, weight = op.attention(q, cache.k, cache.v, tables, lens, 1.0, window)
    err = (out.double() - want).abs() - (U * want.abs() + 2.0 ** -13 * weight)
    assert err.max().item() <= 0


WIDE = [
    [(5, 2)],
    [(10, 5), (1, 300), (64, 64)],
    [(10, 5), (1, 300)] + [(0, 3)] * 9,  # as many tokens as sequences: few rows
    [(3, 0), (1, 200), (2, 700)] + [(0, 0)] * 3,
]


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, 1])
@pytest.mark.parametrize("heads", [SLIDING, FULL])
@pytest.mark.parametrize("case", range(len(WIDE)))
def test_attention_windows_beyond_every_position(gpu_ctx, case, heads, window):
    """The largest windows an int holds mask nothing, also beside tokens at negative positions (a
    sequence of more new tokens than rows), which see nothing."""
    lens = WIDE[case]
    q, cache, batch, tables = _setup(lens, heads, 16, window, seed=60 + case)
    _check_attention(_attend(gpu_ctx, q, cache, batch, window=window), q, cache, tables, lens, window=window)


@pytest.mark.parametrize("tokens", [4096, 4097])  # as many tokens as sequences, and not
def test_attention_of_a_batch_that_counts_its_tokens_over_and_over(gpu_ctx, tokens):
    """q_start goes up and down, so that half of the sequences have the same 4096 tokens: 8.6e9 tiles
    of 256 rows (or 1.4e11 of 16), past what an int counts.  The host lets 2^30 through and takes it
    that a token is of one sequence.  Nothing is done, and the status word says so."""
    pages, seqs = 256, 4096  # every table entry is the one page: 2^24 rows a sequence
    k = torch.zeros(1, 65536, 1, 256, dtype=torch.bfloat16, device="cuda")
    cache = g4.PagedCache(k, k)
    i32 = dict(dtype=torch.int32, device="cuda")
    starts = torch.zeros(seqs + 1, **i32)
    starts[1::2] = 4096
    batch = g4.PagedBatch(torch.zeros(seqs, pages, **i32), starts, torch.full((seqs,), pages * 65536, **i32))
    q = torch.zeros(tokens, 2, 256, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 5.0)
    g4.paged_attention(gpu_ctx, q, cache, batch, out)
    with pytest.raises(g4.G4Error):
        gpu_ctx.poll()
    assert gpu_ctx.poll() == 0 and (out == 5).all()


# batches of single tokens over so many tiles that a CTA has several of one item; <= 4 and > 4 rows
TOKENS = [([(1, 9000), (1, 8300), (1, 8999)], SLIDING), ([(1, 16000)] * 4, FULL), ([(1, 16000)] * 4, (5, 1, 256)),
          ([(1, 12000)] * 3, (6, 2, 512))]


@pytest.mark.parametrize("case", range(len(TOKENS)))
def test_few_rows_rising_scores(gpu_ctx, case):
    """Scores that rise by 30 every 100 rows, in a CTA's many tiles of an item: O is scaled again at
    each of them."""
    lens, heads = TOKENS[case]
    q, cache, batch, tables = _setup(lens, heads, 64, 0, seed=80 + case)
    q.zero_()
    q[:, :, 0] = 1.0
    for s, (n, kv) in enumerate(lens):
        for p in range(-(-kv // 64)):
            rows = torch.arange(64 * p, 64 * p + 64, device="cuda")
            cache.k[tables[s][p], :, :, 0] = torch.where(rows < kv, 0.3 * rows, float("nan"))[:, None].bfloat16()
    out = _attend(gpu_ctx, q, cache, batch)
    _check_attention(out, q, cache, tables, lens)
    assert torch.equal(out, _attend(gpu_ctx, q, cache, batch))


@pytest.mark.parametrize("scale,std", [(0.0, 1.0), (0.0625, 20.0), (-1.0, 2.0), (1.0, 40.0), (1e-3, 1.0)])
@pytest.mark.parametrize("case", range(len(TOKENS)))
def test_few_rows_scales(gpu_ctx, case, scale, std):
    """The scales and score sizes of test_attention_scales, where they meet the kernel for few rows."""
    lens, heads = TOKENS[case]
    q, cache, batch, tables = _setup(lens, heads, 32, 0, seed=90 + case, std=std)
    _check_attention(_attend(gpu_ctx, q, cache, batch, scale=scale), q, cache, tables, lens, scale=scale)


@pytest.mark.parametrize("heads,page_rows,window", [((60, 20, 256), 128, 64), ((60, 20, 256), 8, 64),
                                                    ((12, 4, 512), 64, 40), (SLIDING, 64, 200), ((32, 16, 256), 24, 8)])
def test_attention_of_many_short_items(gpu_ctx, heads, page_rows, window):
    """Small windows over a long chunk: every CTA pair has many items of few tiles, hardly any of them
    at a sequence's ends; query groups that TMA can copy and ones that it cannot."""
    lens = [(1800, 2500), (700, 700), (1, 40)]
    q, cache, batch, tables = _setup(lens, heads, page_rows, window, seed=7)
    out = _attend(gpu_ctx, q, cache, batch, window=window)
    _check_attention(out, q, cache, tables, lens, window=window)
    assert torch.equal(out, _attend(gpu_ctx, q, cache, batch, window=window))


NOT_FINITE = [
    [(1, 100)],  # within one CTA, no join
    [(1, 8192)],  # in many CTAs' hands
    [(1, 40), (1, 700), (1, 1000), (1, 2)],
    [(130, 300), (1, 40)],  # not the kernel for few rows
    [(3, 2), (1, 300), (0, 4), (0, 4)],  # some rows see nothing
]


@pytest.mark.parametrize("value", [math.nan, math.inf, 3e38])
@pytest.mark.parametrize("heads", [SLIDING, FULL])
@pytest.mark.parametrize("case", range(len(NOT_FINITE)))
def test_attention_rows_that_are_not_finite(gpu_ctx, case, heads, value):
    """A query head with a NaN, an infinity, or scores past f32's range has no softmax: its output is
    NaN (if it sees anything), in one CTA's hands as in many, and the rows beside it are right.  (Two
    dimensions of q and k are +-value and positive, so that a score is +inf and not only -inf.)"""
    lens = NOT_FINITE[case]
    q, cache, batch, tables = _setup(lens, heads, 16, 0, seed=20 + case)
    tokens, hq, _ = q.shape
    cache.k[..., 1] = torch.where(torch.isnan(cache.k[..., 1]), cache.k[..., 1], 10.0)
    hit = torch.zeros(tokens, hq, dtype=torch.bool, device="cuda")
    hit[::3, ::5] = True
    clean = q.clone()
    q[..., 1][hit] = value
    out = _prefilled(gpu_ctx, q, cache, batch)
    sees = torch.tensor([kv - n + i >= 0 for n, kv in lens for i in range(n)], device="cuda")[:, None].expand(tokens, hq)
    assert torch.isnan(out[hit & sees]).all()
    assert (out[~sees] == 0).all()
    want, weight = op.attention(clean, cache.k, cache.v, tables, lens)
    err = (out.double() - want).abs() - (2 * U + 2.0 ** -11) * weight
    assert err[~hit].max().item() <= 0


def _prefilled(ctx, q, cache, batch):
    out = torch.full_like(q, 7.0)
    g4.paged_attention(ctx, q, cache, batch, out)
    torch.cuda.synchronize()
    assert ctx.poll() == 0
    return out


@pytest.mark.parametrize("what", ["kv_long", "kv_negative", "start_high", "start_falls"])
@pytest.mark.parametrize("heads", [SLIDING, FULL])
def test_store_leaves_the_rows_of_a_sequence_with_bad_numbers(gpu_ctx, what, heads):
    """Where a sequence's new tokens belong is not known when its numbers are out of range: none of
    them is stored over rows that it, or a fork that shares its pages, has already."""
    lens = [(2, 100), (3, 150)]
    _, cache, batch, tables = _setup(lens, heads, 16, poison=3.0)
    q, k, v, qw, kw, cos, sin = _store_inputs(lens, heads, 1)
    if what == "kv_long":
        batch.kv_len[1] = batch.tables.shape[1] * 16 + 5
        batch.tables[1] = batch.tables[1].clamp(min=0)  # every entry a page of the cache
    elif what == "kv_negative":
        batch.kv_len[1] = -7
    elif what == "start_high":
        batch.q_start[2] = 2 ** 30
    else:
        batch.q_start[2] = 1
    before = cache.k.clone(), cache.v.clone()
    out = torch.full(q.shape, 9.0, dtype=torch.bfloat16, device="cuda")
    g4.paged_store_qkv(gpu_ctx, q, k, v, qw, kw, cos, sin, cache, batch, out)
    with pytest.raises(g4.G4Error):
        gpu_ctx.poll()
    assert gpu_ctx.poll() == 0
    page, row = tables[0][98 // 16], 98 % 16  # the other sequence's two tokens
    for now, was in zip((cache.k, cache.v), before):
        changed = (now != was).flatten(2).any(2)
        assert changed[page, row:row + 2].all() and int(changed.sum()) == 2
    assert (out[2:] == (9 if what == "start_falls" else 0)).all() and (out[:2] != 9).any()


def test_attention_numbers_past_32_bits(gpu_ctx):
    """A window past 32 bits masks nothing (its low bits are not taken), one below them is refused."""
    lens = [(40, 300), (1, 77)]
    q, cache, batch, tables = _setup(lens, SLIDING, 16)
    for window in (2 ** 31, 2 ** 32 + 5, 2 ** 63):
        _check_attention(_attend(gpu_ctx, q, cache, batch, window=window), q, cache, tables, lens)
    out = torch.empty_like(q)
    with pytest.raises(g4.G4Error) as e:
        g4.paged_attention(gpu_ctx, q, cache, batch, out, window=-2 ** 32)
    assert e.value.code == 1
    assert gpu_ctx.poll() == 0


@pytest.mark.parametrize("scale", [3e38, -3e38, math.inf, -math.inf])
def test_attention_refuses_scales_past_f32(gpu_ctx, scale):
    """The kernels multiply by scale * log2(e), which has to be finite too."""
    q, cache, batch, _ = _setup([(2, 20)], SLIDING)
    with pytest.raises(g4.G4Error) as e:
        g4.paged_attention(gpu_ctx, q, cache, batch, torch.empty_like(q), scale=scale)
    assert e.value.code == 1 and gpu_ctx.poll() == 0


@pytest.mark.parametrize("heads,lens,layout", [(SLIDING, [(1100, 1500), (1, 77), (0, 9), (199, 199)], "nhd"),
                                               (SLIDING, [(1300, 1300)], "hnd"),
                                               (FULL, [(600, 1900), (1, 2000), (600, 601)], "kv_in_page"),
                                               ((15, 5, 256), [(1, 3), (1700, 1800), (33, 20)], "nhd"),
                                               ((5, 3, 512), [(1200, 1200), (1300, 1999)], "padded")])
def test_store_of_many_tokens(gpu_ctx, heads, lens, layout):
    """Calls so large that a warp takes four heads (or pairs of heads) of a token, also where that leaves
    a rest; the bounds of test_store."""
    hq, hkv, d = heads
    _, cache, batch, tables = _setup(lens, heads, 24, layout=layout, seed=3, poison=3.0)
    q, k, v, qw, kw, cos, sin = _store_inputs(lens, heads, 5)
    before = cache.k.clone(), cache.v.clone()
    out = torch.full(q.shape, 9.0, dtype=torch.bfloat16, device="cuda")
    g4.paged_store_qkv(gpu_ctx, q, k, v, qw, kw, cos, sin, cache, batch, out)
    torch.cuda.synchronize()
    assert gpu_ctx.poll() == 0
    pos = torch.tensor([kv - n + i for n, kv in lens for i in range(n)], device="cuda")
    seq = torch.tensor([s for s, (n, _) in enumerate(lens) for _ in range(n)], device="cuda")
    live = pos >= 0
    at = pos.clamp(min=0)
    page = torch.tensor(tables, device="cuda")[seq, at // 24][live]
    row = (at % 24)[live]

    def close(got, want, size):
        assert ((got.double() - want).abs() - (U * want.abs() + 2.0 ** -18 * size)).max().item() <= 0

    want, size = op.rotate(op.norm(q, qw), cos[at], sin[at])
    close(out[live], want[live], size[live])
    assert (out[~live] == 0).all()
    want, size = op.rotate(op.norm(k, kw), cos[at], sin[at])
    close(cache.k[page, row], want[live], size[live])
    want = op.norm(v)
    close(cache.v[page, row], want[live], want[live].abs())
    touched = torch.zeros(cache.n_pages, 24, dtype=torch.bool, device="cuda")
    touched[page, row] = True
    assert torch.equal(cache.k[~touched], before[0][~touched]) and torch.equal(cache.v[~touched], before[1][~touched])
