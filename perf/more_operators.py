"""Operators around the attention of a batch of sequences, as cases that can be timed and compared.

What a program that serves prompts in chunks, or many sequences at once, calls besides the paged
caches:

* ``embed``    -- the embedding rows of a batch's tokens, scaled;
* ``quantize`` -- activation rows to NVFP4 (E2M1 codes, an E4M3 scale per 16 values, a factor per
  row), as one to three pieces that add up, after an RMSNorm or as they are, and read back;
* ``linear``   -- bf16 rows through a projection stored in NVFP4: quantised as above, then the
  product on the codes;
* ``norm``     -- the projection's rows normed and added to the residual stream;
* ``beam``     -- the best continuations of each group of beams over the vocabulary.

Sizes are the decoder's: hidden 3840, intermediate 15360, vocabulary 262144, attention of 16 heads of
256 (8 KV heads) or of 512 (one), or a tensor-parallel rank's share of them.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

H, L, V = 3840, 15360, 262144
EMBED_SCALE = 62.0  # bf16(sqrt(H))
EPS = 1e-6
#: weight rows and columns: the two attention kinds' fused q/k/v and output projections, the MLP's
PROJECTIONS = {
    "sliding_qkv": ((16 + 8 + 8) * 256, H), "sliding_out": (H, 16 * 256),
    "full_qkv": ((16 + 1) * 512, H), "full_out": (H, 16 * 512),
    "gate_up": (2 * L, H), "down": (H, L),
}
LIMIT = 2.6e11  # products of the largest case: drawn ones stay below


# ------------------------------------------------------------------------------ cases
def _embed(name, tokens, vocab=V, width=H):
    return {"name": name, "op": "embed", "tokens": tokens, "vocab": vocab, "width": width}


def _quantize(name, rows, cols, pieces, norm, gap=0):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "pieces": pieces, "norm": norm, "gap": gap}


def _linear(name, kind, rows, pieces, ranks=1, gap=0):
    return {"name": name, "op": "linear", "kind": kind, "rows": rows, "pieces": pieces, "ranks": ranks, "gap": gap}


def _norm(name, rows, cols):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols}


def _beam(name, groups, beams, select, vocab=V, start=False):
    return {"name": name, "op": "beam", "groups": groups, "beams": beams, "select": select, "vocab": vocab, "start": start}


def listed():
    return [
        # one user's next token, and a prompt of the prefill benchmark's size
        _embed("embed_one_token", 1),
        _embed("embed_4096_tokens", 4096),
        # one token ahead of its projection; a prompt's wide rows (the MLP's h) at the default pieces
        _quantize("quantize_norm_one_token", 1, H, 2, True),
        _quantize("quantize_4096_wide", 4096, L, 2, False),
        # decode: one user's q/k/v, 32 users' output projection; prefill: an odd-sized chunk's q/k/v
        # at the default precision, a whole prompt's at the fastest
        _linear("linear_sliding_qkv_one_token", "sliding_qkv", 1, 2),
        _linear("linear_full_out_32_tokens", "full_out", 32, 2),
        _linear("linear_full_qkv_chunk_509", "full_qkv", 509, 2),
        _linear("linear_sliding_qkv_4096", "sliding_qkv", 4096, 1),
        # the attention's projection into the residual stream: 32 users' tokens, a prompt
        _norm("norm_32_tokens", 32, H),
        _norm("norm_4096_tokens", 4096, H),
        # one request's four beams; a batch of 32 requests, twice as many candidates as beams
        # (some of them will have ended)
        _beam("beam_4_of_one_request", 1, 4, 8),
        _beam("beam_4_of_32_requests", 32, 4, 8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "quantize", "quantize", "linear", "linear", "linear", "linear", "norm", "beam", "beam"])
    if op == "embed":
        c = _embed("", _log(rng, 1, 4096), rng.choice([V, V, 32003]), rng.choice([H, H, 8 * rng.randint(1, 1024)]))
    elif op == "quantize":
        ranks = rng.choice([1, 1, 2, 4, 8])
        cols = rng.choice([H, L // ranks, 16 * 256 // ranks, 16 * 512 // ranks, 32 * rng.randint(1, 320)])
        c = _quantize("", _log(rng, 1, 4096), cols, rng.choice([1, 2, 2, 3]), rng.random() < 0.5, rng.choice([0, 0, 8, 64]))
    elif op == "linear":
        while True:
            kind, ranks = rng.choice(sorted(PROJECTIONS)), rng.choice([1, 1, 2, 4, 8])
            c = _linear("", kind, _log(rng, 1, 4096), rng.choice([1, 2, 2, 3]), ranks, rng.choice([0, 0, 8, 64]))
            if work(c)["flops"] * c["pieces"] <= LIMIT:
                break
    elif op == "norm":
        c = _norm("", _log(rng, 1, 4096), rng.choice([H, H, 8 * rng.randint(1, 1024)]))
    else:
        vocab = rng.choice([V, V, rng.randint(1000, V)])
        beams = rng.randint(1, 8)
        groups = _log(rng, 1, 128 // beams)
        c = _beam("", groups, beams, rng.randint(1, 2 * beams), vocab, rng.random() < 0.2)
    del c["name"]
    return c


def _shape(case):
    """Rows and columns of the rank's projection: outputs are cut where the next operator wants its
    own heads, inputs where the last one left them."""
    n, k = PROJECTIONS[case["kind"]]
    return (n, k // case["ranks"]) if case["kind"].endswith(("out", "down")) else (n // case["ranks"], k)


def work(case):
    op = case["op"]
    if op == "embed":
        return {"bytes": case["tokens"] * (4 + 4 * case["width"]), "flops": case["tokens"] * case["width"]}
    if op == "quantize":
        e = case["rows"] * case["cols"]
        return {"bytes": 4 * e + (2 * case["cols"] if case["norm"] else 0), "flops": e * (4 * case["pieces"] + (4 if case["norm"] else 0))}
    if op == "linear":
        n, k = _shape(case)
        return {"bytes": 2 * case["rows"] * (n + k) + n * k * 9 // 16, "flops": 2 * case["rows"] * n * k}
    if op == "norm":
        e = case["rows"] * case["cols"]
        return {"bytes": 6 * e + 2 * case["cols"], "flops": 6 * e}
    rows = case["groups"] * case["beams"]
    return {"bytes": rows * (2 * case["vocab"] + 4) + 12 * case["groups"] * case["select"], "flops": 3 * rows * case["vocab"]}


# ------------------------------------------------------------------------------ inputs
def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + salt)
    return g


def _randn(g, shape, std=1.0):
    t = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    return t.mul_(std) if std != 1.0 else t


def _activations(g, rows, cols, gap=0):
    """Rows as a residual stream has them: a few channels much larger than the others, rows of
    different sizes; `gap` elements between them (a slice of something wider)."""
    x = torch.empty((rows, cols + gap), device="cuda").normal_(generator=g)
    x *= torch.where(torch.rand(cols + gap, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    x *= torch.exp(0.5 * torch.empty((rows, 1), device="cuda").normal_(generator=g))
    return x.bfloat16()[:, :cols]


def _pack(code):
    """E2M1 codes (0..15) two a byte, the even one low."""
    return (code[..., 0::2] | code[..., 1::2] << 4).contiguous()


def _weight(g, n, k):
    """A projection as a checkpoint stores it: codes [n, k / 2], block scales [n, k / 16], 1 / g."""
    w = torch.empty((n, k), device="cuda").normal_(generator=g).mul_(0.02).view(n, k // 16, 16)
    factor = 2688.0 / w.abs().amax()
    scale = (w.abs().amax(2) / 6 * factor).to(torch.float8_e4m3fn)
    code = _e2m1_code(w * factor / scale.float().clamp(min=2.0 ** -9)[..., None])
    return _pack(code.view(n, k)), scale.view(torch.uint8), (1 / factor).reshape(1)


def _library():
    pkg = str(Path(__file__).resolve().parent.parent / "furiosa-opt-gemma4-12b_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import g4b200

    return g4b200


_ctx = None


def prepare(case, seed):
    global _ctx
    st = _inputs(case, seed)
    if own:  # what a server keeps: its context, its layers' weights, its activation buffers
        g4 = _library()
        if _ctx is None:
            _ctx = g4.Context(torch.cuda.current_device())
        st["g4"], st["ctx"] = g4, _ctx
        if case["op"] == "quantize":
            st["rows"] = g4.Nvfp4Rows(_ctx, case["rows"], case["cols"], case["pieces"])
        if case["op"] == "linear":
            n, k = _shape(case)
            st["rows"] = g4.Nvfp4Rows(_ctx, case["rows"], k, case["pieces"])
            st["weight"] = g4.Nvfp4Weight(_ctx, st["codes"], st["scales"], st["global_scale"])
    return st


def _inputs(case, seed):
    op, g = case["op"], _gen(seed, 1)
    st = {"case": case}
    if op == "embed":
        vocab, width = case["vocab"], case["width"]
        st["table"] = _randn(g, (vocab, width), 0.03)
        # ids as text has them: a few very frequent ones, the rest anywhere
        u = torch.rand(case["tokens"], generator=g, device="cuda", dtype=torch.float64)
        st["tokens"] = (torch.exp(u * math.log(vocab)) - 1).to(torch.int32).clamp_(0, vocab - 1)
        st["out"] = torch.empty((case["tokens"], width), dtype=torch.bfloat16, device="cuda")
    elif op == "quantize":
        st["x"] = _activations(g, case["rows"], case["cols"], case["gap"])
        st["w"] = (1.0 + 0.3 * _randn(g, (case["cols"],)).float()).bfloat16() if case["norm"] else None
        st["out"] = torch.empty((case["rows"], case["cols"]), dtype=torch.bfloat16, device="cuda")
    elif op == "linear":
        n, k = _shape(case)
        st["x"] = _activations(g, case["rows"], k, case["gap"])
        st["codes"], st["scales"], st["global_scale"] = _weight(g, n, k)
        st["out"] = torch.empty((case["rows"], n + case["gap"]), dtype=torch.bfloat16, device="cuda")[:, :n]
    elif op == "norm":
        st["x"] = _activations(g, case["rows"], case["cols"])
        st["w"] = (1.0 + 0.3 * _randn(g, (case["cols"],)).float()).bfloat16()
        st["residual"] = _activations(g, case["rows"], case["cols"])
        st["out"] = torch.empty_like(st["residual"])
    else:
        groups, beams, vocab, select = case["groups"], case["beams"], case["vocab"], case["select"]
        # capped logits as a decoder's: a few likely tokens far above the others, many equal in bf16
        x = torch.empty((groups, beams, vocab), device="cuda").normal_(generator=g).mul_(2.5)
        st["logits"] = (30.0 * torch.tanh((x + 0.004 * x ** 3) / 30.0)).bfloat16()
        scores = -20.0 * torch.rand((groups, beams), generator=g, device="cuda")
        if case["start"]:  # all beams of a new request hold the prompt: only the first counts
            scores[:, 0], scores[:, 1:] = 0.0, -math.inf
        st["scores"] = scores
        st["out_scores"] = torch.empty((groups, select), device="cuda")
        st["out_beams"], st["out_tokens"] = (torch.empty((groups, select), dtype=torch.int32, device="cuda") for _ in range(2))
    return st


# ------------------------------------------------------------------------------ one pass
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    g4, ctx, op = st["g4"], st["ctx"], st["case"]["op"]
    if op == "embed":
        g4.embed_tokens(ctx, st["table"], st["tokens"], st["out"])
    elif op == "quantize":
        g4.nvfp4_quantize(ctx, st["x"], st["rows"], st["w"])
        g4.nvfp4_dequantize(ctx, st["rows"], st["out"])
    elif op == "linear":
        g4.nvfp4_quantize(ctx, st["x"], st["rows"])
        g4.nvfp4_matmul(ctx, st["rows"], st["weight"], st["out"])
    elif op == "norm":
        g4.residual_norm(ctx, st["x"], st["w"], st["residual"], st["out"])
    else:
        g4.beam_select(ctx, st["logits"], st["scores"], st["out_scores"], st["out_beams"], st["out_tokens"])
        return st["out_scores"], st["out_beams"], st["out_tokens"]
    return st["out"]


def _run_plain(st):
    op = st["case"]["op"]
    if op == "embed":
        return (st["table"][st["tokens"].long()].float() * EMBED_SCALE).bfloat16()
    if op == "quantize":
        total, factor = _pieces(_rms(st["x"], st["w"]), st["case"]["pieces"])
        return (total * factor).bfloat16()
    if op == "linear":
        total, factor = _pieces(st["x"].float(), st["case"]["pieces"])
        return (total @ _dequantized(st["codes"], st["scales"]).T * factor * st["global_scale"]).bfloat16()
    if op == "norm":
        x = st["x"].float()
        r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
        return (st["residual"].float() + x * r * st["w"].float()).bfloat16()
    # 64 bits: a sum of 262144 terms, and scores of different beams next to one another
    logits = st["logits"].double()
    top = logits.amax(-1, keepdim=True)
    logsum = top + torch.log(torch.exp(logits - top).sum(-1, keepdim=True))
    scores = (st["scores"].double()[..., None] + logits - logsum).nan_to_num_(-math.inf, math.inf, -math.inf).flatten(1)
    best, at = torch.sort(scores, dim=1, descending=True, stable=True)  # ties: the lowest index first
    best, at = best[:, :st["out_scores"].shape[1]], at[:, :st["out_scores"].shape[1]]
    vocab = logits.shape[-1]
    return best.float(), (at // vocab).int(), (at % vocab).int()


def _rms(x, w):
    """bf16(x r w) with r = 1 / sqrt(mean x^2 + eps), or x itself; r from 64-bit sums: what is next to
    a rounding border would fall on either side by the order of a 32-bit one."""
    if w is None:
        return x.float()
    r = (1 / torch.sqrt(x.double().square().mean(1, keepdim=True) + EPS)).float()
    return (x.float() * r * w.float()).bfloat16().float()


def _e2m1(v):
    """The nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, ties to the even code."""
    a = v.abs()
    up = ((a > 0.25).float() + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) * 0.5 + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5)
    return torch.where(v < 0, -up, up)


def _e2m1_code(v):
    a = v.abs()
    code = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    return code | (v < 0).byte() << 3


def _pieces(x, pieces):
    """(sum of the pieces, 1 / g): g the largest power of two up to 2^126 with max|row| g <= 2688, y_0 = x g,
    s_p = e4m3(max_block |y_p| / 6), c_p = e2m1(y_p / s_p), y_{p+1} = y_p - c_p s_p; a row of zeros is
    pieces of zeros and factor 0."""
    rows, cols = x.shape
    top = x.abs().amax(1)
    mantissa, _ = torch.frexp(room := (2688.0 / top).clamp(max=2.0 ** 126))
    g = room / mantissa / 2
    factor = torch.where(top > 0, 1 / g, torch.zeros_like(g))
    y = (x * g[:, None]).view(rows, cols // 16, 16)
    total = torch.zeros_like(y)
    for _ in range(pieces):
        s = (y.abs().amax(2, keepdim=True) / 6).clamp(max=448.0).to(torch.float8_e4m3fn).float()
        piece = torch.where(s > 0, _e2m1(y / s) * s, torch.zeros_like(y))
        y = y - piece
        total = total + piece
    return total.view(rows, cols), factor[:, None]


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _dequantized(codes, scales):
    n, half = codes.shape
    values = torch.tensor(_E2M1, device=codes.device)
    pair = torch.stack([codes & 15, codes >> 4], 2).view(n, 2 * half)
    return (values[pair.int()].view(n, half // 8, 16) * scales.view(torch.float8_e4m3fn).float()[..., None]).view(n, 2 * half)


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The operators' definitions in 64 bits: roundings to E4M3 and E2M1 as roundings to a multiple of
    the format's step at the value's magnitude."""
    st, op = _inputs(case, seed), case["op"]
    if op == "embed":
        return st["table"][st["tokens"].long()].double() * EMBED_SCALE
    if op == "quantize":
        x = st["x"].double()
        if case["norm"]:
            x = (x * (x.pow(2).mean(1, keepdim=True) + EPS).rsqrt() * st["w"].double()).bfloat16().double()
        return _exact_rows(x, case["pieces"])
    if op == "linear":
        scale = st["scales"].view(torch.float8_e4m3fn).double().repeat_interleave(16, 1)
        nibble = torch.empty(scale.shape, dtype=torch.uint8, device="cuda")
        nibble[:, 0::2], nibble[:, 1::2] = st["codes"] % 16, st["codes"] // 16
        weight = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")[nibble.long()] * scale
        return _exact_rows(st["x"].double(), case["pieces"]) @ weight.T * st["global_scale"].double()
    if op == "norm":
        x = st["x"].double()
        return st["residual"].double() + x * (x.pow(2).mean(1, keepdim=True) + EPS).rsqrt() * st["w"].double()
    # the scores; which beams and tokens they belong to has no value in 64 bits
    scores = (st["scores"].double()[..., None] + torch.log_softmax(st["logits"].double(), -1)).flatten(1)
    return torch.topk(scores, case["select"], 1).values, None, None


def _to_step(v, smallest, mantissa, most):
    """v >= 0 to the nearest multiple of 2^(exponent - mantissa), ties to even, at most `most`."""
    step = torch.exp2(torch.floor(torch.log2(v.clamp(min=2.0 ** smallest))) - mantissa)
    return (torch.round(v / step) * step).clamp(max=most)


def _exact_rows(x, pieces):
    top = x.abs().amax(1, keepdim=True)
    g = torch.exp2(torch.floor(torch.log2((2688.0 / top).clamp(max=2.0 ** 126))))
    left = (x * g).unflatten(1, (-1, 16))
    total = 0
    for _ in range(pieces):
        s = _to_step(left.abs().amax(-1, keepdim=True) / 6, -6, 3, 448.0)
        piece = torch.where(s > 0, torch.sign(left) * _to_step((left / s).abs(), 0, 1, 6.0) * s, 0.0)
        left, total = left - piece, total + piece
    return torch.where(top > 0, total.flatten(1) / g, 0.0)
