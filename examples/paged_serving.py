#!/usr/bin/env python3
"""Several users of one prompt served from a paged KV cache.

    python examples/paged_serving.py

One sliding and one full attention layer (the decoder's two kinds) over one page pool.  The
projections are random bf16 matrices on plain torch products; everything between them is the
library's: pages handed out and shared (PagePool), q/k/v normed, rotated and stored
(paged_store_qkv), attention over the pages (paged_attention), forked pages copied on append
(paged_copy) and the cache compacted after a user left (paged_compact).  At the end every
user's last outputs are compared with a cache of its own that was filled in one piece.
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "furiosa-opt-gemma4-12b_b200"))

import g4b200 as g4  # noqa: E402

HIDDEN, POSITIONS, PAGE_ROWS, PAGES = 3840, 4096, 64, 96
KINDS = {"sliding": (16, 8, 256, 1024, 1e4, 1.0), "full": (16, 1, 512, 0, 1e6, 0.25)}


class Layer:
    """One attention layer: its projection, norm weights, rotary tables and cache."""

    def __init__(self, kind: str, seed: int, pages: int = PAGES):
        self.hq, self.hkv, self.d, self.window, theta, turning = KINDS[kind]
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        kv = 1 if kind == "full" else 2  # full layers use the raw K projection as V too
        self.shared_kv = kv == 1
        self.w = (rnd(HIDDEN, (self.hq + kv * self.hkv) * self.d) / HIDDEN ** 0.5).bfloat16()
        self.q_w, self.k_w = (0.15 + 0.02 * rnd(self.d)).bfloat16(), (1 + 0.1 * rnd(self.d)).bfloat16()
        half = self.d // 2
        inv = torch.zeros(half, device="cuda", dtype=torch.float64)
        n = int(half * turning)
        inv[:n] = theta ** (-2.0 * torch.arange(n, device="cuda", dtype=torch.float64) / self.d)
        ang = torch.arange(POSITIONS, device="cuda", dtype=torch.float64)[:, None] * inv
        self.cos = torch.cat([ang.cos(), ang.cos()], 1).bfloat16()
        self.sin = torch.cat([-ang.sin(), ang.sin()], 1).bfloat16()
        self.cache = self.new_cache(pages)

    def new_cache(self, pages: int) -> g4.PagedCache:
        # what a page holds before it is written must not matter
        return g4.PagedCache(*(torch.full((pages, PAGE_ROWS, self.hkv, self.d), float("nan"), dtype=torch.bfloat16,
                                          device="cuda") for _ in range(2)))

    def attend(self, ctx, x, batch, cache=None):
        """x [tokens, HIDDEN] -> attention output [tokens, heads, head size]."""
        cache = cache or self.cache
        qkv = (x @ self.w).view(x.shape[0], -1, self.d)
        q, k = qkv[:, :self.hq], qkv[:, self.hq:self.hq + self.hkv]
        v = k if self.shared_kv else qkv[:, self.hq + self.hkv:]
        rotated, out = (torch.empty((x.shape[0], self.hq, self.d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        g4.paged_store_qkv(ctx, q, k, v, self.q_w, self.k_w, self.cos, self.sin, cache, batch, rotated)
        g4.paged_attention(ctx, rotated, cache, batch, out, window=self.window)
        return out


def main() -> dict:
    g = torch.Generator(device="cuda").manual_seed(7)
    ctx = g4.Context(0)
    layers = [Layer("sliding", 1), Layer("full", 2)]
    caches = g4.PagedCaches([layer.cache for layer in layers])
    pool = g4.PagePool(PAGES, PAGE_ROWS)
    inputs, outputs = {}, {}  # sequence -> its tokens' inputs, its last outputs per layer

    def step(seqs, counts):
        """Appends counts[i] new tokens to seqs[i], all in one batch."""
        for s, n in zip(seqs, counts):
            pool.extend(s, n)
        pool.run_copies(ctx, caches)
        batch = pool.batch(ctx, seqs, counts)
        x = torch.randn((sum(counts), HIDDEN), generator=g, device="cuda").bfloat16()
        outs = [layer.attend(ctx, x, batch) for layer in layers]
        t = 0
        for s, n in zip(seqs, counts):
            inputs[s] = torch.cat([inputs[s], x[t:t + n]]) if s in inputs else x[t:t + n]
            outputs[s] = [o[t:t + n] for o in outs]
            t += n

    def leave(s):
        pool.free(s)
        del inputs[s], outputs[s]  # (a later sequence may get the same number)

    prompt = pool.add()
    for chunk in (512, 512, 277):  # the prompt in chunks
        step([prompt], [chunk])
    users = [prompt] + [pool.fork(prompt) for _ in range(3)]
    for s in users[1:]:
        inputs[s] = inputs[prompt]
    shared = pool.free_pages
    step(users, [19, 40, 7, 131])  # each user's own question: the shared last page is copied
    for _ in range(20):
        step(users, [1, 1, 1, 1])
    leave(users.pop(1))
    late = pool.add()  # a new user's prompt beside the others' single tokens
    step([late] + users, [300, 1, 1, 1])
    users.append(late)
    leave(users.pop(0))
    moved = pool.compact(ctx, caches, pool.batch(ctx, users, [1] * len(users)).tables)
    step(users, [1] * len(users))

    worst = 0.0
    for s in users:  # the same tokens in one piece, alone in a cache
        alone = g4.PagePool(PAGES, PAGE_ROWS)
        seq = alone.add()
        alone.extend(seq, inputs[s].shape[0])
        batch = alone.batch(ctx, [seq], [inputs[s].shape[0]])
        for layer, got in zip(layers, outputs[s]):
            want = layer.attend(ctx, inputs[s], batch, layer.new_cache(PAGES))[-got.shape[0]:].float()
            worst = max(worst, ((got.float() - want).norm() / want.norm()).item())
    torch.cuda.synchronize()
    assert ctx.poll() == 0
    ctx.close()
    return {"pages free after the prompt": shared, "pages moved": moved, "relative difference": worst}


if __name__ == "__main__":
    print(main())
