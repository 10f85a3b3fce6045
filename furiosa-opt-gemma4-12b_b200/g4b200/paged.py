"""Host binding of the paged KV caches (include/g4.h, g4_paged_* and g4_page_pool_*): the
attention side of serving many sequences or a prompt in chunks, which the reference's host
runs one position per dispatch (src/host/generate.rs:194-211).

A layer's cache is a `PagedCache`, the sequences of a call a `PagedBatch`; both only describe
tensors the caller owns (they keep them alive), are checked once and can be used for any
number of calls while the tensors' contents change.  `PagePool` hands out the pages.

    pool = PagePool(n_pages, page_rows)
    seq = pool.add(); pool.extend(seq, len(prompt))          # pages for the new rows
    child = pool.fork(seq)                                    # shares them; copies on append
    pool.run_copies(ctx, caches)                              # before the rows are written
    batch = pool.batch(ctx, [seq], [len(prompt)])
    paged_store_qkv(ctx, q, k, v, ..., cache, batch, q_out)   # per layer
    paged_attention(ctx, q_out, cache, batch, out, window=1024)
"""

from __future__ import annotations

import ctypes
import operator

import torch

from . import LIB, Context, G4Error, _i32, _i64, _vp

_f32 = ctypes.c_float


class _CacheDesc(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp)] + [(f"{t}_{s}_stride", _i64) for t in "kv" for s in ("page", "row", "head")] + [
        (n, _i32) for n in ("n_pages", "page_rows", "n_kv_heads", "head_dim")]


class _BatchDesc(ctypes.Structure):
    _fields_ = [("tables", _vp), ("table_stride", _i64), ("q_start", _vp), ("kv_len", _vp),
                ("max_pages", _i32), ("n_seqs", _i32), ("n_tokens", _i32)]


_p_i32 = ctypes.POINTER(_i32)
LIB.g4_paged_attention.argtypes = [_vp, _vp, _i64, _i64, _i32, ctypes.POINTER(_CacheDesc), ctypes.POINTER(_BatchDesc),
                                   _f32, _i32, _vp, _i64, _i64]
LIB.g4_paged_store_qkv.argtypes = [_vp, _vp, _i64, _i64, _i32, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _vp, _vp,
                                   _i32, ctypes.POINTER(_CacheDesc), ctypes.POINTER(_BatchDesc), _vp, _i64, _i64]
LIB.g4_paged_copy.argtypes = [_vp, ctypes.POINTER(_CacheDesc), _i32, _vp, _vp, _vp, _i32]
LIB.g4_paged_compact.argtypes = [_vp, ctypes.POINTER(_CacheDesc), _i32, _vp, _vp, _i32, _vp, _i64, _i32, _i32, _vp]
LIB.g4_page_pool_create.argtypes = [_i32, _i32, ctypes.POINTER(_vp)]
LIB.g4_page_pool_destroy.argtypes = [_vp]
LIB.g4_page_pool_last_error.argtypes = [_vp]
LIB.g4_page_pool_last_error.restype = ctypes.c_char_p
LIB.g4_page_pool_add.argtypes = [_vp, _p_i32]
LIB.g4_page_pool_extend.argtypes = [_vp, _i32, _i32]
LIB.g4_page_pool_fork.argtypes = [_vp, _i32, _p_i32]
LIB.g4_page_pool_reorder.argtypes = [_vp, _p_i32, _p_i32, _i32]
LIB.g4_page_pool_trim.argtypes = [_vp, _i32, _i32]
LIB.g4_page_pool_free.argtypes = [_vp, _i32]
LIB.g4_page_pool_compact.argtypes = [_vp, _p_i32, _p_i32, _p_i32, _p_i32]
LIB.g4_page_pool_take_copies.argtypes = [_vp, _p_i32, _p_i32, _p_i32, _i32, _p_i32]
LIB.g4_page_pool_table.argtypes = [_vp, _i32, _p_i32, _i32, _p_i32]
LIB.g4_page_pool_free_pages.argtypes = [_vp, _p_i32]


def _int32(name: str, value) -> int:
    """An integer as the library's 32-bit int (ctypes would keep the low bits of a larger one)."""
    v = operator.index(value)
    if not -2 ** 31 <= v < 2 ** 31:
        raise ValueError(f"{name}: {v} does not fit 32 bits")
    return v


def _cuda(name: str, t, dtype, dims: int):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name}: {t.dim()} dimensions, expected {dims}")
    return t


def _same_device(ctx: Context, **named) -> None:
    for name, t in named.items():
        if t.get_device() != ctx.device:
            raise ValueError(f"{name}: on {t.device}, the context is on cuda:{ctx.device}")


def _rows(ctx: Context, name: str, t, tokens: int, heads: int, dim: int) -> tuple:
    """A [tokens, heads, dim] bf16 operand on the context's device; returns its pointer and its
    token and head strides in elements (0 along a dimension of size one)."""
    _cuda(name, t, torch.bfloat16, 3)
    if t.shape != (tokens, heads, dim):
        raise ValueError(f"{name}: shape {list(t.shape)}, expected [{tokens}, {heads}, {dim}]")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name}: on {t.device}, the context is on cuda:{ctx.device}")
    token_stride, head_stride, last = t.stride()
    if last != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return t.data_ptr(), token_stride if tokens > 1 else 0, head_stride if heads > 1 else 0


def _row_strides(name: str, t, dims) -> tuple:
    """The strides of `dims`; the last dimension must be contiguous (a stride of a dimension of
    size one means nothing and is passed on as 0)."""
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return tuple(t.stride(i) if t.shape[i] > 1 else 0 for i in dims)


def _tokens_heads(name: str, t) -> tuple:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor")
    if t.dim() != 3:
        raise ValueError(f"{name}: {t.dim()} dimensions, expected 3")
    return t.shape[0], t.shape[1]


class PagedCache:
    """One layer's K and V pages (g4_paged_cache): bf16 CUDA tensors of shape
    [n_pages, page_rows, n_kv_heads, head_dim] with any strides of multiples of 8 over a
    contiguous last dimension, so a [n_pages, n_kv_heads, page_rows, head_dim] tensor is
    passed as its transpose(1, 2)."""

    def __init__(self, k, v):
        for name, t in (("k", k), ("v", v)):
            _cuda(name, t, torch.bfloat16, 4)
        if k.shape != v.shape:
            raise ValueError(f"k and v differ in shape: {list(k.shape)}, {list(v.shape)}")
        if k.device != v.device:
            raise ValueError("k and v are on different devices")
        self.k, self.v = k, v
        self.n_pages, self.page_rows, self.n_kv_heads, self.head_dim = k.shape
        self.device = k.get_device()
        self.desc = _CacheDesc(k.data_ptr(), v.data_ptr(), *_row_strides("k", k, (0, 1, 2)),
                               *_row_strides("v", v, (0, 1, 2)), *k.shape)


class PagedCaches:
    """The layers that page copies and compaction go through at once (PagedCache objects of
    equal page_rows and n_pages)."""

    def __init__(self, layers):
        self.layers = list(layers)
        if not self.layers:
            raise ValueError("no layers")
        if len({c.k.device for c in self.layers}) > 1:
            raise ValueError("layers on different devices")
        self.desc = (_CacheDesc * len(self.layers))(*[c.desc for c in self.layers])


class PagedBatch:
    """The sequences of a call (g4_paged_batch): int32 CUDA tensors tables [n_seqs, max_pages],
    q_start [n_seqs + 1], kv_len [n_seqs].  Their contents are read on the stream by every
    call, so they may be updated in place between calls."""

    def __init__(self, tables, q_start, kv_len):
        _cuda("tables", tables, torch.int32, 2)
        for name, t in (("q_start", q_start), ("kv_len", kv_len)):
            _cuda(name, t, torch.int32, 1)
            if not t.is_contiguous():
                raise ValueError(f"{name}: must be contiguous")
        n = kv_len.numel()
        if tables.shape[0] != n or q_start.numel() != n + 1:
            raise ValueError(f"tables, q_start and kv_len have {tables.shape[0]}, {q_start.numel()} and {n} entries: "
                             "expected n, n + 1 and n")
        if tables.shape[1] > 1 and tables.stride(1) != 1:
            raise ValueError("tables: rows must be contiguous")
        if not tables.device == q_start.device == kv_len.device:
            raise ValueError("tables, q_start and kv_len are on different devices")
        self.tables, self.q_start, self.kv_len, self.n_seqs = tables, q_start, kv_len, n
        width = tables.shape[1]
        self.stride = max(tables.stride(0), width) if n > 1 else width
        if n > 1 and tables.stride(0) < width:
            raise ValueError("tables: rows overlap")
        self.device = kv_len.get_device()
        self._fields = tables.data_ptr(), self.stride, q_start.data_ptr(), kv_len.data_ptr(), width, n

    def desc(self, n_tokens: int) -> _BatchDesc:
        """A descriptor of the call's own: calls of other threads may be under way on this batch."""
        return _BatchDesc(*self._fields, n_tokens)


def paged_attention(ctx: Context, q, cache: PagedCache, batch: PagedBatch, out, *, scale: float = 1.0,
                    window: int = 0) -> None:
    """Attention of every new token of the batch over its sequence's pages, causal, within the
    last `window` positions if window > 0 (g4_paged_attention).  q, out: bf16
    [n_tokens, n_heads, head_dim]; the model's scale is 1."""
    n, heads = _tokens_heads("q", q)
    qa = _rows(ctx, "q", q, n, heads, cache.head_dim)
    oa = _rows(ctx, "out", out, n, heads, cache.head_dim)
    if cache.device != ctx.device or batch.device != ctx.device:
        raise ValueError(f"cache or batch: not on the context's device cuda:{ctx.device}")
    if heads % cache.n_kv_heads:
        raise ValueError(f"q: {heads} heads is not a multiple of the cache's {cache.n_kv_heads}")
    if n == 0:
        return
    window = max(-1, min(int(window), 2 ** 31 - 1))  # (no position is past that: larger ones mask nothing)
    ctx._check("g4_paged_attention", LIB.g4_paged_attention(
        ctx.handle, *qa, heads, cache.desc, batch.desc(n), float(scale), window, *oa))


def paged_store_qkv(ctx: Context, q, k, v, q_rms_weight, k_rms_weight, cos, sin, cache: PagedCache,
                    batch: PagedBatch, q_out) -> None:
    """q_out = rope(rmsnorm(q) * q_rms_weight); k the same and v = rmsnorm(v) into the cache rows
    of the new tokens (g4_paged_store_qkv).  q, q_out: bf16 [n_tokens, n_heads, head_dim]; k, v:
    [n_tokens, n_kv_heads, head_dim] (slices of a fused projection are fine; full layers
    pass k as v); cos, sin: [n_positions, head_dim] with sin's low half negated."""
    n, heads = _tokens_heads("q", q)
    d, hkv = cache.head_dim, cache.n_kv_heads
    qa, oa = _rows(ctx, "q", q, n, heads, d), _rows(ctx, "q_out", q_out, n, heads, d)
    ka, va = _rows(ctx, "k", k, n, hkv, d), _rows(ctx, "v", v, n, hkv, d)
    if cache.device != ctx.device or batch.device != ctx.device:
        raise ValueError(f"cache or batch: not on the context's device cuda:{ctx.device}")
    for name, t, dims in (("q_rms_weight", q_rms_weight, 1), ("k_rms_weight", k_rms_weight, 1), ("cos", cos, 2),
                          ("sin", sin, 2)):
        _cuda(name, t, torch.bfloat16, dims)
        if t.shape[-1] != d or not t.is_contiguous() or t.get_device() != ctx.device:
            raise ValueError(f"{name}: must be contiguous with {d} columns, on cuda:{ctx.device}")
    if cos.shape != sin.shape:
        raise ValueError("cos and sin differ in shape")
    if n == 0:
        return
    ctx._check("g4_paged_store_qkv", LIB.g4_paged_store_qkv(
        ctx.handle, *qa, heads, *ka, *va, q_rms_weight.data_ptr(), k_rms_weight.data_ptr(), cos.data_ptr(),
        sin.data_ptr(), cos.shape[0], cache.desc, batch.desc(n), *oa))


def _words(name: str, t, n: int | None = None):
    _cuda(name, t, torch.int32, 1)
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name}: {t.numel()} entries, expected {n}")
    return t.data_ptr()


def _check_tables(tables) -> None:
    _cuda("tables", tables, torch.int32, 2)
    if tables.shape[1] > 1 and tables.stride(1) != 1:
        raise ValueError("tables: rows must be contiguous")
    if tables.shape[0] > 1 and tables.stride(0) < tables.shape[1]:
        raise ValueError("tables: rows overlap")


def paged_copy(ctx: Context, caches: PagedCaches, src, dst, rows) -> None:
    """Rows [0, rows[i]) of page src[i] into page dst[i] in K and V of every layer
    (g4_paged_copy; int32 CUDA tensors).  No dst may be another dst or any src."""
    n = src.numel()
    a = _words("src", src), _words("dst", dst, n), _words("rows", rows, n)
    _same_device(ctx, src=src, dst=dst, rows=rows, caches=caches.layers[0].k)
    if n:
        ctx._check("g4_paged_copy", LIB.g4_paged_copy(ctx.handle, caches.desc, len(caches.layers), *a, n))


def paged_compact(ctx: Context, caches: PagedCaches, src, dst, tables, page_map) -> None:
    """Whole pages src[i] into dst[i] in every layer, and tables = page_map[tables] where an
    entry is not negative (g4_paged_compact), in one launch per 56 layers."""
    n = src.numel()
    a = _words("src", src), _words("dst", dst, n)
    _check_tables(tables)
    seqs, width = tables.shape
    m = _words("page_map", page_map, caches.layers[0].n_pages)
    _same_device(ctx, src=src, dst=dst, tables=tables, page_map=page_map, caches=caches.layers[0].k)
    ctx._check("g4_paged_compact", LIB.g4_paged_compact(
        ctx.handle, caches.desc, len(caches.layers), *a, n, tables.data_ptr(), tables.stride(0) if seqs > 1 else width,
        seqs, width, m))


class PagePool:
    """Which pages the sequences of a cache hold (g4_page_pool, host bookkeeping): pages are
    counted by their users, forks share pages and copy the last one when they append.

    `run_copies` (the copies that `extend` asked for) must run before anything writes the
    cache rows those extends made room for."""

    def __init__(self, n_pages: int, page_rows: int):
        h = _vp()
        n_pages, page_rows = _int32("n_pages", n_pages), _int32("page_rows", page_rows)
        code = LIB.g4_page_pool_create(n_pages, page_rows, ctypes.byref(h))
        if code != 0:
            raise G4Error("g4_page_pool_create", code, f"n_pages={n_pages}, page_rows={page_rows}")
        self.handle, self.n_pages, self.page_rows = h, n_pages, page_rows
        self._copies = []  # groups taken from the library's pool, not launched yet
        self._moves = None  # (src, dst, page_map) of a compaction that is not launched yet

    def _check(self, fn: str, code: int) -> None:
        if code != 0:
            raise G4Error(fn, code, LIB.g4_page_pool_last_error(self.handle).decode())

    def add(self) -> int:
        s = _i32()
        self._check("g4_page_pool_add", LIB.g4_page_pool_add(self.handle, ctypes.byref(s)))
        return s.value

    def extend(self, seq: int, n_rows: int) -> None:
        self._check("g4_page_pool_extend", LIB.g4_page_pool_extend(
            self.handle, _int32("seq", seq), _int32("n_rows", n_rows)))

    def fork(self, seq: int) -> int:
        s = _i32()
        self._check("g4_page_pool_fork", LIB.g4_page_pool_fork(
            self.handle, _int32("seq", seq), ctypes.byref(s)))
        return s.value

    def reorder(self, seqs, parents) -> None:
        """Every seqs[i] becomes a copy of what parents[i] was, all at once and without moving a row:
        the pages are shared as by a fork (g4_page_pool_reorder).  For beams: parents[i] is the
        sequence of the beam that beam i continues."""
        a, b = ([_int32(name, s) for s in x] for name, x in (("seqs", seqs), ("parents", parents)))
        if len(a) != len(b):
            raise ValueError("seqs and parents differ in length")
        self._check("g4_page_pool_reorder", LIB.g4_page_pool_reorder(
            self.handle, (_i32 * len(a))(*a), (_i32 * len(b))(*b), len(a)))

    def trim(self, seq: int, first_row: int) -> None:
        """Gives back the pages wholly below row first_row (below a sliding window)."""
        self._check("g4_page_pool_trim", LIB.g4_page_pool_trim(
            self.handle, _int32("seq", seq), _int32("first_row", first_row)))

    def free(self, seq: int) -> None:
        self._check("g4_page_pool_free", LIB.g4_page_pool_free(self.handle, _int32("seq", seq)))

    @property
    def free_pages(self) -> int:
        n = _i32()
        self._check("g4_page_pool_free_pages", LIB.g4_page_pool_free_pages(self.handle, ctypes.byref(n)))
        return n.value

    def table(self, seq: int) -> tuple[list[int], int]:
        """(the sequence's pages in order, -1 where given back; its rows)."""
        self._check_moved()
        seq = _int32("seq", seq)
        rows = _i32()
        code = LIB.g4_page_pool_table(self.handle, seq, None, 0, ctypes.byref(rows))
        if code != 6:  # (no room for its pages: has rows, their number is set)
            self._check("g4_page_pool_table", code)
        out = (_i32 * ((rows.value + self.page_rows - 1) // self.page_rows))()
        self._check("g4_page_pool_table", LIB.g4_page_pool_table(self.handle, seq, out, len(out), ctypes.byref(rows)))
        return out[:], rows.value

    def _check_caches(self, ctx: Context, caches: PagedCaches) -> None:
        for c in caches.layers:
            if (c.n_pages, c.page_rows) != (self.n_pages, self.page_rows) or c.device != ctx.device:
                raise ValueError(f"caches: a layer of {c.n_pages} pages of {c.page_rows} rows on cuda:{c.device}, the pool "
                                 f"has {self.n_pages} of {self.page_rows}, the context is on cuda:{ctx.device}")

    def _collect_copies(self) -> None:
        self._check_moved()
        while True:
            src, dst, rows = ((_i32 * 4096)() for _ in range(3))
            n = _i32()
            self._check("g4_page_pool_take_copies",
                        LIB.g4_page_pool_take_copies(self.handle, src, dst, rows, 4096, ctypes.byref(n)))
            if n.value == 0:
                return
            self._copies.append((list(src[:n.value]), list(dst[:n.value]), list(rows[:n.value])))

    def take_copies(self) -> list[tuple[list[int], list[int], list[int]]]:
        """The waiting page copies as (src, dst, rows) groups, to be run one after another."""
        self._collect_copies()
        groups, self._copies = self._copies, []
        return groups

    def run_copies(self, ctx: Context, caches: PagedCaches) -> None:
        """Runs the waiting copies on the context's stream.  After an error, those that were not
        launched still wait."""
        self._check_caches(ctx, caches)
        self._collect_copies()
        while self._copies:
            paged_copy(ctx, caches, *[_upload(ctx, x) for x in self._copies[0]])
            del self._copies[0]

    def compact(self, ctx: Context, caches: PagedCaches, tables) -> int:
        """Moves the pages in use to the front of every layer's cache and rewrites `tables`
        (int32 CUDA [n_seqs, max_pages], as `batch` makes them); returns the pages moved.  After
        an error on the way to the GPU the pool's pages are known by their new numbers, but not
        moved: until another call with the same tables has moved them, the pool hands out no
        tables, batches or copies."""
        self._check_caches(ctx, caches)  # before the pool forgets where the pages were
        _check_tables(tables)
        _same_device(ctx, tables=tables)
        if self._moves is None:
            if self._copies:
                raise G4Error("g4_page_pool_compact", 1, "page copies wait to be run")
            src, dst, page_map = ((_i32 * self.n_pages)() for _ in range(3))
            n = _i32()
            self._check("g4_page_pool_compact",
                        LIB.g4_page_pool_compact(self.handle, src, dst, page_map, ctypes.byref(n)))
            self._moves = src[:n.value], dst[:n.value], page_map[:]
        src, dst, page_map = self._moves
        paged_compact(ctx, caches, _upload(ctx, src), _upload(ctx, dst), tables, _upload(ctx, page_map))
        self._moves = None
        return len(src)

    def _check_moved(self) -> None:
        if self._moves is not None:
            raise G4Error("g4_page_pool_compact", 1, "a compaction did not move its pages: call compact again")

    def batch(self, ctx: Context, seqs, new_tokens) -> PagedBatch:
        """The batch of `seqs` with their last `new_tokens[i]` rows as new tokens, in that
        order in the token dimension."""
        rows = [self.table(s) for s in seqs]
        width = max([len(t) for t, _ in rows], default=0)
        starts = [0]
        for n in new_tokens:
            starts.append(starts[-1] + int(n))
        if len(starts) != len(rows) + 1:
            raise ValueError("seqs and new_tokens differ in length")
        tables = _upload(ctx, [t + [-1] * (width - len(t)) for t, _ in rows]).view(len(rows), width)
        return PagedBatch(tables, _upload(ctx, starts), _upload(ctx, [r for _, r in rows]))

    def close(self) -> None:
        if getattr(self, "handle", None) is not None:
            LIB.g4_page_pool_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _upload(ctx: Context, values):
    """An int32 CUDA tensor written on the context's stream (so the calls that read it, and
    the reuse of its memory, are in stream order)."""
    with torch.cuda.stream(ctx.stream):
        return torch.tensor(values, dtype=torch.int32, device=f"cuda:{ctx.device}")


__all__ = ["PagedCache", "PagedCaches", "PagedBatch", "PagePool", "paged_attention", "paged_store_qkv", "paged_copy",
           "paged_compact"]
