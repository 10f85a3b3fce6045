"""Paged attention over the decode runtime's own caches: the full layers' 512-row pages laid back to
back, and the sliding layers' ring as two pages that a table names in turn.  Against the float64
oracle, and beside the single-token entry points on the same rows."""

import ctypes

import pytest
import torch

import g4b200 as g4
from g4b200 import runtime
from g4formats import model as fm
from oracle import paged as op
from test_paged_gpu import U

pytestmark = pytest.mark.gpu

ROWS = 1100  # the ring of 1024 has come round


@pytest.fixture(scope="module")
def decoded():
    """A six-layer model's workspace after ROWS positions."""
    ctx = g4.Context(0, stream=torch.cuda.Stream())
    model = runtime.model_from_synthetic(fm.synthetic_model(6, seed=11, device="cuda", post_norm=0.05,
                                                            layer_scalar=(1.0, 1.0)))
    ws = runtime.Workspace(ctx, model, 2048)
    ws.begin([int(x) for x in ((fm.uniform("p", 11, ROWS, "cpu") + 1) * 0.5 * (fm.W - 1))], 0, 0)
    ws.steps(ROWS)
    torch.cuda.synchronize()
    yield ctx, ws
    assert ctx.poll() == 0
    ws.close()
    model.close()
    ctx.close()


def _paged(ctx, ws, layer, heads, n_pages, table, tokens, window):
    """(q, out) of `tokens` random queries, the last at position ROWS - 1, over the workspace's cache."""
    hq, hkv, d = heads
    k, v, nbytes = ws.kv_cache_ptrs(layer)
    assert nbytes == n_pages * 512 * hkv * d * 2
    strides = (512 * hkv * d, hkv * d, d)
    cache = g4.paged._CacheDesc(k, v, *strides, *strides, n_pages, 512, hkv, d)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = g4.PagedBatch(i32([table]), i32([0, tokens]), i32([ROWS]))
    g = torch.Generator(device="cuda").manual_seed(layer + tokens)
    q = (torch.randn((tokens, hq, d), generator=g, device="cuda") * 2.5 / d ** 0.5).bfloat16()
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    ctx._check("g4_paged_attention", g4.LIB.g4_paged_attention(
        ctx.handle, q.data_ptr(), hq * d, d, hq, ctypes.byref(cache), batch.desc(tokens), 1.0, window, out.data_ptr(),
        hq * d, d))
    torch.cuda.synchronize()
    return q, out


def _near(got, want, weight):
    assert ((got.double() - want).abs() <= (2 * U + 2.0 ** -11) * weight).all()


@pytest.mark.parametrize("tokens", [1, 40])
def test_full_layer_pages(decoded, tokens):
    ctx, ws = decoded
    q, out = _paged(ctx, ws, 5, (16, 1, 512), 4, [0, 1, 2, -1], tokens, 0)
    k, v = (t.view(4, 512, 1, 512) for t in ws.kv_cache(5))
    want, weight = op.attention(q, k, v, [[0, 1, 2, 3]], [(tokens, ROWS)])
    _near(out, want, weight)
    if tokens == 1:
        kp, vp = (torch.tensor([t[i].data_ptr() for i in range(3)], dtype=torch.int64, device="cuda") for t in (k, v))
        single, total = torch.empty_like(q[0]), torch.zeros(16, dtype=torch.float32, device="cuda")
        torch.cuda.synchronize()
        g4.full_attention_paged(ctx, q[0].reshape(-1), kp, vp, 3, ROWS - 1 - 1024, total, single.view(-1))
        torch.cuda.synchronize()
        _near(single, want[0], weight[0])


@pytest.mark.parametrize("tokens", [1, 40])
def test_sliding_layer_ring(decoded, tokens):
    """Positions 512 j .. of the ring are its half j % 2; rows below the window have been written over.
    (Of several tokens all windows have to lie in the ring, so they are shorter by the tokens between.)"""
    ctx, ws = decoded
    window = 1024 - (tokens - 1)
    q, out = _paged(ctx, ws, 0, (16, 8, 256), 2, [0, 1, 0], tokens, window)
    k, v = (t.view(2, 512, 8, 256) for t in ws.kv_cache(0))
    want, weight = op.attention(q, k, v, [[0, 1, 0]], [(tokens, ROWS)], 1.0, window)
    _near(out, want, weight)
    if tokens == 1:
        single = torch.empty_like(q[0])
        mask = torch.ones(1024, dtype=torch.float32, device="cuda")
        torch.cuda.synchronize()
        g4.sliding_attention(ctx, q[0].reshape(-1), k.reshape(-1), v.reshape(-1), mask, single.view(-1))
        torch.cuda.synchronize()
        _near(single, want[0], weight[0])
