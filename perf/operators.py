"""Serving operators over a paged KV cache, as cases that can be timed and compared.

Four operators that a program serving many sequences calls one after another:

* ``store``   -- norm, rotate and store a chunk of new tokens: q gets its per-head RMSNorm
  and rotary positions, k the same and goes to its cache page, v its unweighted RMSNorm and
  goes to its cache page;
* ``attend``  -- attention of the new tokens (a long chunk, one token, or some of each) over
  the pages of their sequences, causal, optionally within a sliding window;
* ``copy``    -- the pages that forked sequences stop sharing, copied in every layer;
* ``compact`` -- pages moved to the front of every layer's cache, block tables rewritten.

Head layouts are the decoder's two attention kinds: sliding (16 query heads over 8 KV heads
of 256, window 1024) and full (16 query heads over one KV head of 512), or a rank's share.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

POSITIONS = 32768  # rows of the rotary tables
EPS = 1e-6
WINDOW = 1024
KINDS = {"sliding": (16, 8, 256, WINDOW), "full": (16, 1, 512, 0)}


# ------------------------------------------------------------------------------ cases
def _attend(name, kind, page_rows, chunks, chunk, singles, context, ranks=1, ragged=True):
    return {"name": name, "op": "attend", "kind": kind, "page_rows": page_rows, "chunks": chunks, "chunk": chunk,
            "singles": singles, "context": context, "ranks": ranks, "ragged": ragged}


def _store(name, kind, page_rows, seqs, chunk, context, ranks=1):
    return {"name": name, "op": "store", "kind": kind, "page_rows": page_rows, "seqs": seqs, "chunk": chunk,
            "context": context, "ranks": ranks}


def _move(name, op, page_rows, pages, moves, sliding_layers, full_layers, ranks=1):
    return {"name": name, "op": op, "page_rows": page_rows, "pages": pages, "moves": moves,
            "sliding_layers": sliding_layers, "full_layers": full_layers, "ranks": ranks}


def listed():
    return [
        # one user's next token early in a chat: nothing but latency
        _attend("attend_sliding_one_token", "sliding", 64, 0, 1, 1, 1000, ragged=False),
        # one user's next token at the context the decode benchmark uses, doubled
        _attend("attend_full_one_token_8192", "full", 512, 0, 1, 1, 8192, ragged=False),
        # a batch of 32 users' next tokens, contexts anywhere up to 8192
        _attend("attend_full_32_tokens", "full", 512, 0, 1, 32, 8192),
        # 31 users' next tokens beside one new user's odd-sized chunk, small pages
        _attend("attend_sliding_mixed", "sliding", 16, 1, 509, 31, 4096),
        # the second chunk of a long document: few rows against a long cache
        _attend("attend_full_chunk_256_of_16384", "full", 512, 1, 256, 0, 16384, ragged=False),
        # whole prompts of the prefill benchmark's size
        _attend("attend_sliding_prompt_4096", "sliding", 64, 1, 4096, 0, 4096, ragged=False),
        _attend("attend_full_prompt_4096", "full", 512, 1, 4096, 0, 4096, ragged=False),
        # the same user's single token, and a whole prompt, on their way into the cache
        _store("store_sliding_one_token", "sliding", 64, 1, 1, 1000),
        _store("store_sliding_4096_tokens", "sliding", 64, 3, 1365, 4096),
        # three sequences that fork off one prompt stop sharing their last page: one layer group
        _move("copy_3_tails", "copy", 64, 96, 3, 5, 1),
        # a beam of 48 continuations goes separate ways, small pages
        _move("copy_48_tails", "copy", 16, 1024, 48, 20, 4),
        # after many sequences ended: the pages still in use move to the front
        _move("compact_200_pages", "compact", 64, 640, 200, 10, 2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend"] * 4 + ["store", "copy", "compact"])
    ranks = rng.choice([1, 1, 2, 4])
    if op == "attend":
        limit = 2.7e11
        while True:
            kind = rng.choice(["sliding", "full"])
            page = rng.choice([8, 16, 24, 64, 128, 512])
            shape = rng.choice(["tokens", "chunk", "mixed"])
            chunks = 0 if shape == "tokens" else rng.randint(1, 3)
            chunk = _log(rng, 2, 4096) if chunks else 1
            singles = 0 if shape == "chunk" else _log(rng, 1, 32)
            context = max(chunk, _log(rng, 1, 16384))
            c = _attend("", kind, page, chunks, chunk, singles, context, ranks, rng.random() < 0.7)
            del c["name"]
            if work(c)["flops"] <= limit:
                return c
    if op == "store":
        kind = rng.choice(["sliding", "full"])
        seqs = _log(rng, 1, 32)
        chunk = _log(rng, 1, max(1, 4096 // seqs))
        c = _store("", kind, rng.choice([8, 16, 24, 64, 512]), seqs, chunk, max(chunk, _log(rng, 1, 8192)), ranks)
    else:
        page = rng.choice([16, 24, 64])
        moves = _log(rng, 1, 200 if op == "compact" else 64)
        c = _move("", op, page, 2 * moves + rng.randint(0, 200), moves, rng.randint(0, 10), rng.randint(1, 2), ranks)
    del c["name"]
    return c


def _lens(case):
    """(new tokens, cache length with them) of each sequence: a function of the case alone."""
    rng = random.Random(case["context"] * 1009 + case["chunk"] * 31 + case.get("singles", 0))
    out = []
    for _ in range(case.get("chunks", case.get("seqs", 0))):
        n = case["chunk"]
        kv = rng.randint(n, case["context"]) if case.get("ragged", True) else case["context"]
        out.append((n, kv))
    for _ in range(case.get("singles", 0)):
        kv = rng.randint(1, case["context"]) if case.get("ragged", True) else case["context"]
        out.append((1, kv))
    if out and case.get("ragged", True):  # one sequence always has the whole context
        i = rng.randrange(len(out))
        out[i] = (out[i][0], case["context"])
    rng.shuffle(out)
    return out


def _heads(case):
    """(query heads, KV heads, head size, window) of one rank."""
    hq, hkv, d, window = KINDS[case["kind"]]
    return hq // case["ranks"], max(1, hkv // case["ranks"]), d, window


def _layer_rows(case):
    """(KV heads, head size) of each layer that a page move goes through."""
    out = []
    for kind in ("sliding", "full"):
        _, hkv, d, _ = KINDS[kind]
        out += [(max(1, hkv // case["ranks"]), d)] * case[kind + "_layers"]
    return out


def _tail_rows(case):
    rng = random.Random(case["moves"] * 7919 + case["page_rows"])
    return [rng.randint(1, case["page_rows"]) for _ in range(case["moves"])]


def work(case):
    if case["op"] == "attend":
        hq, hkv, d, window = _heads(case)
        seen = rows = tokens = pages = 0
        for n, kv in _lens(case):
            first = kv - n
            lo = max(0, first - window + 1) if window else 0
            rows += kv - lo
            tokens += n
            pages += (kv - 1) // case["page_rows"] - lo // case["page_rows"] + 1
            if not window:
                seen += n * first + n * (n + 1) // 2
            else:  # row p sees min(p + 1, window) keys
                ramp = max(0, min(kv, window) - first)
                seen += ramp * first + ramp * (ramp + 1) // 2 + (n - ramp) * window
        return {"bytes": 2 * (2 * tokens * hq * d + 2 * rows * hkv * d) + 4 * pages, "flops": 4 * d * hq * seen}
    if case["op"] == "store":
        hq, hkv, d, _ = _heads(case)
        lens = _lens(case)
        tokens = sum(n for n, _ in lens)
        positions = {p for n, kv in lens for p in range(kv - n, kv)}
        pages = sum((kv - 1) // case["page_rows"] - (kv - n) // case["page_rows"] + 1 for n, kv in lens)
        return {"bytes": 2 * (2 * tokens * (hq + 2 * hkv) * d + 2 * len(positions) * d + 2 * d) + 4 * pages,
                "flops": tokens * (hq * 7 + hkv * 7 + hkv * 3) * d}
    rows = sum(_tail_rows(case)) if case["op"] == "copy" else case["moves"] * case["page_rows"]
    row_bytes = sum(2 * 2 * hkv * d for hkv, d in _layer_rows(case))
    return {"bytes": 2 * rows * row_bytes + 8 * case["moves"] + (8 * case["pages"] if case["op"] == "compact" else 0),
            "flops": 0}


# ------------------------------------------------------------------------------ inputs
def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + salt)
    return g


def _randn(g, shape, std=1.0):
    t = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    return t.mul_(std) if std != 1.0 else t


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(lens, page_rows, window, rng):
    """Block tables of pages handed out in random order, -1 where a sequence holds none (past
    its end; below its window, where a server has given the page back), and the page count."""
    need = []
    for s, (n, kv) in enumerate(lens):
        lo = max(0, kv - n - window + 1) if window else 0
        need += [(s, p) for p in range(lo // page_rows, (kv + page_rows - 1) // page_rows)]
    n_pages = len(need) + max(2, len(need) // 8)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    width = max((kv + page_rows - 1) // page_rows for _, kv in lens)
    table = [[-1] * width for _ in lens]
    for (s, p), i in zip(need, ids):
        table[s][p] = i
    return table, n_pages


def _rotary(d, kind):
    """cos/sin [POSITIONS, d] in bf16, the sine of the low half negated: theta 1e4 over every
    pair (sliding), theta 1e6 over the first quarter of the pairs (full)."""
    half = d // 2
    turning = half if kind == "sliding" else half // 4
    theta = 1e4 if kind == "sliding" else 1e6
    inv = torch.zeros(half, dtype=torch.float64, device="cuda")
    inv[:turning] = theta ** (-2.0 * torch.arange(turning, dtype=torch.float64, device="cuda") / d)
    ang = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inv
    cos, sin = ang.cos(), ang.sin()
    return torch.cat([cos, cos], 1).bfloat16(), torch.cat([-sin, sin], 1).bfloat16()


_ctx = None


def _library():
    pkg = str(Path(__file__).resolve().parent.parent / "furiosa-opt-gemma4-12b_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import g4b200

    return g4b200


def prepare(case, seed):
    global _ctx
    st = _inputs(case, seed)
    if own:  # what a server keeps: its context, its layers' caches and its batch
        g4 = _library()
        if _ctx is None:
            _ctx = g4.Context(torch.cuda.current_device())
        st["ctx"] = _ctx
        if case["op"] in ("attend", "store"):
            st["cache"] = g4.PagedCache(st["k_cache"], st["v_cache"])
            st["batch"] = g4.PagedBatch(st["tables"], st["q_start"], st["kv_len"])
        else:
            st["caches"] = g4.PagedCaches([g4.PagedCache(k, v) for k, v in st["layers"]])
    return st


def _inputs(case, seed):
    rng = random.Random(seed * 7 + 11)
    st = {"case": case}
    if case["op"] in ("attend", "store"):
        hq, hkv, d, window = _heads(case)
        lens = _lens(case)
        table, n_pages = _tables(lens, case["page_rows"], window if case["op"] == "attend" else 0, rng)
        tokens = sum(n for n, _ in lens)
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        g = _gen(seed, 1)
        st.update(lens=lens, starts=starts, window=window, tables=_i32(table), q_start=_i32(starts),
                  kv_len=_i32([kv for _, kv in lens]))
        st["k_cache"] = _randn(g, (n_pages, case["page_rows"], hkv, d))
        st["v_cache"] = _randn(g, (n_pages, case["page_rows"], hkv, d))
        st["out"] = torch.empty((tokens, hq, d), dtype=torch.bfloat16, device="cuda")
        if case["op"] == "attend":
            # q . k of normed heads spreads over a few units
            st["q"] = _randn(g, (tokens, hq, d), 2.5 / math.sqrt(d))
        else:
            # one fused projection's rows: q, k and v side by side
            qkv = _randn(g, (tokens, (hq + 2 * hkv), d), 1.7)
            st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
            st["q_w"], st["k_w"] = (1.0 + 0.3 * _randn(g, (d,)).float()).bfloat16(), _randn(g, (d,), 0.5)
            st["cos"], st["sin"] = _rotary(d, case["kind"])
        return st
    # page moves: sources are pages in use, destinations free ones
    n, moves = case["pages"], case["moves"]
    g = _gen(seed, 2)
    st["layers"] = [tuple(_randn(g, (n, case["page_rows"], hkv, d)) for _ in range(2)) for hkv, d in _layer_rows(case)]
    if case["op"] == "copy":
        ids = rng.sample(range(n), 2 * moves)
        src, dst = ids[:moves], ids[moves:]
        if moves >= 3:  # forks of one prompt leave the same page
            src[1] = src[2] = src[0]
        st["rows_list"] = _tail_rows(case)
        st["rows"] = _i32(st["rows_list"])
        st["row_index"] = (torch.arange(case["page_rows"], device="cuda") < st["rows"][:, None]).nonzero(as_tuple=True)
    else:
        # `used` pages stay, `moves` of them beyond the front; the front has as many free ones
        used = moves + (n - 2 * moves) // 3
        src = sorted(rng.sample(range(used, n), moves))
        dst = sorted(rng.sample(range(used), moves))
        page_map = list(range(n))
        for s, t in zip(src, dst):
            page_map[s] = t
        free = set(dst)
        held = [p for p in range(used) if p not in free] + src
        rng.shuffle(held)
        seqs = 16
        width = (len(held) + seqs - 1) // seqs + 3
        table = [held[i::seqs] + [-1] * (width - len(held[i::seqs])) for i in range(seqs)]
        st["tables"], st["page_map"] = _i32(table), _i32(page_map)
    st["src_list"], st["dst_list"] = src, dst
    st["src"], st["dst"] = _i32(src), _i32(dst)
    st["src_index"], st["dst_index"] = st["src"].long(), st["dst"].long()
    return st


# ------------------------------------------------------------------------------ one pass
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    g4, ctx, op = _library(), st["ctx"], st["case"]["op"]
    if op == "attend":
        g4.paged_attention(ctx, st["q"], st["cache"], st["batch"], st["out"], window=st["window"])
        return st["out"]
    if op == "store":
        g4.paged_store_qkv(ctx, st["q"], st["k"], st["v"], st["q_w"], st["k_w"], st["cos"], st["sin"], st["cache"],
                           st["batch"], st["out"])
        return st["out"], st["k_cache"], st["v_cache"]
    if op == "copy":
        g4.paged_copy(ctx, st["caches"], st["src"], st["dst"], st["rows"])
        return [t for kv in st["layers"] for t in kv]
    g4.paged_compact(ctx, st["caches"], st["src"], st["dst"], st["tables"], st["page_map"])
    return [t for kv in st["layers"] for t in kv] + [st["tables"]]


def _rows(cache, table_row, lo, hi):
    """Rows [lo, hi) of one sequence: [hi - lo, KV heads, head size]."""
    page_rows = cache.shape[1]
    pos = torch.arange(lo, hi, device=cache.device)
    return cache[table_row[pos // page_rows].long(), pos % page_rows]


def _softmax_rows(scores, visible):
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _run_plain(st):
    case, op = st["case"], st["case"]["op"]
    if op == "attend":
        hq, hkv, d, window = _heads(case)
        group = hq // hkv
        out = torch.empty_like(st["out"])
        for s, (n, kv) in enumerate(st["lens"]):
            first = kv - n
            lo = max(0, first - window + 1) if window else 0
            k = _rows(st["k_cache"], st["tables"][s], lo, kv).float().permute(1, 2, 0)  # [hkv, d, keys]
            v = _rows(st["v_cache"], st["tables"][s], lo, kv).float().permute(1, 0, 2)
            q = st["q"][st["starts"][s]:st["starts"][s + 1]].float()
            q = q.view(n, hkv, group, d).permute(1, 0, 2, 3).reshape(hkv, n * group, d)
            row = torch.arange(first, kv, device=q.device).repeat_interleave(group)[:, None]
            key = torch.arange(lo, kv, device=q.device)[None, :]
            visible = key <= row
            if window:
                visible &= key > row - window
            o = torch.matmul(_softmax_rows(torch.matmul(q, k), visible), v)
            o = o.view(hkv, n, group, d).permute(1, 0, 2, 3).reshape(n, hq, d)
            out[st["starts"][s]:st["starts"][s + 1]] = o.to(out.dtype)
        return out
    if op == "store":
        page_rows = case["page_rows"]
        pos = torch.cat([torch.arange(kv - n, kv, device="cuda") for n, kv in st["lens"]])
        page = torch.cat([st["tables"][s][torch.arange(kv - n, kv, device="cuda") // page_rows]
                          for s, (n, kv) in enumerate(st["lens"])]).long()
        cos, sin = st["cos"][pos].float()[:, None], st["sin"][pos].float()[:, None]

        def norm(x, w=None):
            x = x.float()
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            return x if w is None else x * w.float()

        def rotate(x):
            half = x.shape[-1] // 2
            return x * cos + torch.cat([x[..., half:], x[..., :half]], -1) * sin

        out = rotate(norm(st["q"], st["q_w"])).bfloat16()
        st["k_cache"][page, pos % page_rows] = rotate(norm(st["k"], st["k_w"])).bfloat16()
        st["v_cache"][page, pos % page_rows] = norm(st["v"]).bfloat16()
        return out, st["k_cache"], st["v_cache"]
    if op == "copy":
        i, row = st["row_index"]
        for kv in st["layers"]:
            for t in kv:
                t[st["dst_index"][i], row] = t[st["src_index"][i], row]
        return [t for kv in st["layers"] for t in kv]
    for kv in st["layers"]:
        for t in kv:
            t[st["dst_index"]] = t[st["src_index"]]
    held = st["tables"] >= 0
    moved = st["page_map"][st["tables"].clamp(min=0).long()]
    st["tables"].copy_(torch.where(held, moved, st["tables"]))
    return [t for kv in st["layers"] for t in kv] + [st["tables"]]


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """What ``run`` returns, from the definitions, in float64; None for the page moves, which
    compute no numbers."""
    if case["op"] not in ("attend", "store"):
        return None
    st = _inputs(case, seed)
    hq, hkv, d, window = _heads(case)
    page_rows = case["page_rows"]
    tables = st["tables"].tolist()
    if case["op"] == "attend":
        out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
        for s, (n, kv) in enumerate(st["lens"]):
            low = max(0, kv - n - window + 1) if window else 0
            index = torch.tensor([tables[s][p // page_rows] * page_rows + p % page_rows for p in range(low, kv)],
                                 device="cuda")
            for h in range(hkv):
                keys = st["k_cache"].flatten(0, 1)[index, h].double()
                values = st["v_cache"].flatten(0, 1)[index, h].double()
                for g in range(hq // hkv):
                    head = h * (hq // hkv) + g
                    for b in range(0, n, 1024):
                        e = min(n, b + 1024)
                        at = torch.arange(kv - n + b, kv - n + e, device="cuda", dtype=torch.float64)
                        j = torch.arange(low, kv, device="cuda", dtype=torch.float64)
                        distance = at[:, None] - j[None, :]
                        bad = distance < 0
                        if window:
                            bad |= distance >= window
                        q = st["q"][st["starts"][s] + b:st["starts"][s] + e, head].double()
                        w = (q @ keys.T).masked_fill_(bad, -math.inf)
                        w = (w - w.logsumexp(1, keepdim=True)).exp_()
                        out[st["starts"][s] + b:st["starts"][s] + e, head] = w @ values
        return out
    q_out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
    where, at = [], []
    for s, (n, kv) in enumerate(st["lens"]):
        for p in range(kv - n, kv):
            where.append(tables[s][p // page_rows] * page_rows + p % page_rows)
            at.append(p)
    where, at = torch.tensor(where, device="cuda"), torch.tensor(at, device="cuda")
    c, s_ = st["cos"][at].double(), st["sin"][at].double()
    half = d // 2

    def head(x, w):
        x = x.double()
        y = x / ((x * x).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        lo, hi = y[..., :half], y[..., half:]
        return torch.cat([lo * c[:, :half] + hi * s_[:, :half], hi * c[:, half:] + lo * s_[:, half:]], -1)

    for h in range(hq):
        q_out[:, h] = head(st["q"][:, h], st["q_w"])
    for h in range(hkv):
        k_cache.flatten(0, 1)[where, h] = head(st["k"][:, h], st["k_w"])
        x = st["v"][:, h].double()
        v_cache.flatten(0, 1)[where, h] = x / ((x * x).sum(-1, keepdim=True) / d + EPS).sqrt()
    return q_out, k_cache, v_cache
