#!/usr/bin/env python3
"""Beam search of several requests at once through a small decoder, over a paged KV cache.

    python examples/beam_serving.py

A decoder of six layers (five sliding, one full: the pattern of the model) with random NVFP4
weights and a vocabulary of 2048.  Prompts go in as one batch of chunks, then every step takes
one token of each beam: embedding rows (embed_tokens), and per layer the norm and quantisation
of the rows (nvfp4_quantize), the q/k/v product (nvfp4_matmul), norm + rotary + store
(paged_store_qkv), attention over the pages (paged_attention), the output product, its norm into
the residual stream (residual_norm) and the MLP of all rows (decoder_feedforward_prefill); then the
logits, the best continuations of each request's beams (beam_select), and the caches that
follow them (PagePool.reorder: pages shared, nothing copied but the last page's tail).

At the end each request's best beam is run again, alone and in one piece, and its tokens' log
probabilities are added up: they have to give the score that the search kept.
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "furiosa-opt-gemma4-12b_b200"))

import g4b200 as g4  # noqa: E402

HIDDEN, MLP, VOCAB, LAYERS, POSITIONS = 3840, 15360, 2048, 6, 1024
PAGE_ROWS, PAGES, MAX_ROWS = 16, 256, 512
KINDS = {"sliding": (16, 8, 256, 64, 1e4, 1.0), "full": (16, 1, 512, 0, 1e6, 0.25)}


def weight(ctx, g, n, k):
    """A random projection, quantised on the GPU."""
    rows = g4.Nvfp4Rows(ctx, n, k, 1)
    g4.nvfp4_quantize(ctx, (torch.randn((n, k), generator=g, device="cuda") * k ** -0.5).bfloat16(), rows)
    return g4.Nvfp4Weight.from_rows(rows, constant=True)


def stored(g, n, k):
    """A random projection as a checkpoint stores it: codes, block scales, reciprocal global scale."""
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.full((n, k // 16), 0x38, device="cuda", dtype=torch.uint8)  # 1.0
    return codes, scales, torch.full((1,), 0.3 * k ** -0.5, device="cuda")


def norm_weight(g, n, around=1.0):
    return (around + 0.1 * torch.randn(n, generator=g, device="cuda")).bfloat16()


class Layer:
    def __init__(self, ctx, kind, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.hq, self.hkv, self.d, self.window, theta, turning = KINDS[kind]
        self.shared_kv = kind == "full"  # full layers use the raw K projection as V too
        kv = 1 if self.shared_kv else 2
        self.qkv = weight(ctx, g, (self.hq + kv * self.hkv) * self.d, HIDDEN)
        self.out = weight(ctx, g, HIDDEN, self.hq * self.d)
        self.norms = [norm_weight(g, HIDDEN) for _ in range(2)]
        self.q_norm, self.k_norm = norm_weight(g, self.d, 0.15), norm_weight(g, self.d)
        (up, us, ug), (gate, gs, gg), (down, ds, dg) = stored(g, MLP, HIDDEN), stored(g, MLP, HIDDEN), stored(g, HIDDEN, MLP)
        self.mlp = [norm_weight(g, HIDDEN), up, gate, down, us, gs, ds, ug, gg, dg, norm_weight(g, HIDDEN),
                    torch.ones(8, dtype=torch.bfloat16, device="cuda")]
        half = self.d // 2
        inv = torch.zeros(half, device="cuda", dtype=torch.float64)
        n = int(half * turning)
        inv[:n] = theta ** (-2.0 * torch.arange(n, device="cuda", dtype=torch.float64) / self.d)
        ang = torch.arange(POSITIONS, device="cuda", dtype=torch.float64)[:, None] * inv
        self.cos = torch.cat([ang.cos(), ang.cos()], 1).bfloat16()
        self.sin = torch.cat([-ang.sin(), ang.sin()], 1).bfloat16()
        self.cache = g4.PagedCache(*(torch.full((PAGES, PAGE_ROWS, self.hkv, self.d), float("nan"), dtype=torch.bfloat16,
                                                device="cuda") for _ in range(2)))

    def run(self, ctx, x, batch, rows):
        """x [tokens, HIDDEN], in place."""
        n, hq, d = x.shape[0], self.hq, self.d
        bf = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        qkv, rotated, attended, y = bf(n, self.qkv.rows), bf(n, hq, d), bf(n, hq, d), bf(n, HIDDEN)
        g4.nvfp4_quantize(ctx, x, rows[HIDDEN], self.norms[0])
        g4.nvfp4_matmul(ctx, rows[HIDDEN], self.qkv, qkv)
        heads = qkv.view(n, -1, d)
        q, k = heads[:, :hq], heads[:, hq:hq + self.hkv]
        v = k if self.shared_kv else heads[:, hq + self.hkv:]
        g4.paged_store_qkv(ctx, q, k, v, self.q_norm, self.k_norm, self.cos, self.sin, self.cache, batch, rotated)
        g4.paged_attention(ctx, rotated, self.cache, batch, attended, window=self.window)
        g4.nvfp4_quantize(ctx, attended.view(n, hq * d), rows[hq * d])
        g4.nvfp4_matmul(ctx, rows[hq * d], self.out, y)
        g4.residual_norm(ctx, y, self.norms[1], x, x)
        g4.decoder_feedforward_prefill(ctx, x, *self.mlp)


class Decoder:
    def __init__(self, ctx):
        g = torch.Generator(device="cuda").manual_seed(3)
        self.ctx = ctx
        self.table = (0.02 * torch.randn((VOCAB, HIDDEN), generator=g, device="cuda")).bfloat16()
        self.layers = [Layer(ctx, "full" if i % 6 == 5 else "sliding", i) for i in range(LAYERS)]
        self.final_norm, self.head = norm_weight(g, HIDDEN), weight(ctx, g, VOCAB, HIDDEN)
        self.rows = {k: g4.Nvfp4Rows(ctx, MAX_ROWS, k, 3) for k in (HIDDEN, 16 * 256, 16 * 512)}
        self.pool = g4.PagePool(PAGES, PAGE_ROWS)
        self.caches = g4.PagedCaches([layer.cache for layer in self.layers])

    def append(self, seqs, tokens):
        """The logits [total tokens, VOCAB] of tokens[i] (lists or a tensor of one each) appended to seqs[i]."""
        flat = torch.tensor([t for ts in tokens for t in ts], dtype=torch.int32, device="cuda") if isinstance(tokens, list) else tokens
        counts = [len(ts) for ts in tokens] if isinstance(tokens, list) else [1] * len(seqs)
        for s, n in zip(seqs, counts):
            self.pool.extend(s, n)
        self.pool.run_copies(self.ctx, self.caches)
        batch = self.pool.batch(self.ctx, seqs, counts)
        x = torch.empty((flat.numel(), HIDDEN), dtype=torch.bfloat16, device="cuda")
        g4.embed_tokens(self.ctx, self.table, flat, x)
        for layer in self.layers:
            layer.run(self.ctx, x, batch, self.rows)
        logits = torch.empty((flat.numel(), VOCAB), dtype=torch.bfloat16, device="cuda")
        g4.nvfp4_quantize(self.ctx, x, self.rows[HIDDEN], self.final_norm)
        g4.nvfp4_matmul(self.ctx, self.rows[HIDDEN], self.head, logits)
        return logits


def search(model, prompts, beams=4, steps=24):
    """The best beam of each prompt: (tokens, score)."""
    ctx, pool, groups = model.ctx, model.pool, len(prompts)
    firsts = [pool.add() for _ in prompts]
    logits = model.append(firsts, prompts)
    ends = torch.tensor([len(p) for p in prompts]).cumsum(0) - 1
    seqs = [[f] + [pool.fork(f) for _ in range(beams - 1)] for f in firsts]
    # every beam holds the prompt: only the first one counts at the start
    scores = torch.full((groups, beams), -torch.inf, device="cuda")
    scores[:, 0] = 0.0
    logits = logits[ends.cuda()][:, None].expand(groups, beams, VOCAB)
    texts = [[[] for _ in range(beams)] for _ in range(groups)]
    best = torch.empty((groups, beams), device="cuda")
    parents, tokens = (torch.empty((groups, beams), dtype=torch.int32, device="cuda") for _ in range(2))
    for step in range(steps):
        g4.beam_select(ctx, logits, scores, best, parents, tokens)
        scores.copy_(best)
        chosen = parents.tolist()
        for group, came_from, new in zip(range(groups), chosen, tokens.tolist()):
            texts[group] = [texts[group][b] + [t] for b, t in zip(came_from, new)]
            pool.reorder(seqs[group], [seqs[group][b] for b in came_from])
        if step + 1 < steps:
            logits = model.append([s for group in seqs for s in group], tokens.flatten()).view(groups, beams, VOCAB)
    for group in seqs:
        for s in group:
            pool.free(s)
    return [(t[0], s) for t, s in zip(texts, scores[:, 0].tolist())]


def main() -> dict:
    ctx = g4.Context(0)
    model = Decoder(ctx)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (90, 7, 33)]
    found = search(model, prompts)
    worst = 0.0
    for prompt, (text, score) in zip(prompts, found):
        seq = model.pool.add()
        logits = model.append([seq], [prompt + text[:-1]])[len(prompt) - 1:].float()
        again = torch.log_softmax(logits, 1).gather(1, torch.tensor(text, device="cuda")[:, None]).sum().item()
        model.pool.free(seq)
        worst = max(worst, abs(again - score) / abs(score))
    torch.cuda.synchronize()
    assert ctx.poll() == 0 and model.pool.free_pages == PAGES
    ctx.close()
    return {"scores": [round(s, 3) for _, s in found], "relative difference of the scores": worst}


if __name__ == "__main__":
    print(main())
