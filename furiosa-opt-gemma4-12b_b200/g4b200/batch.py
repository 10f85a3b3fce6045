"""Host binding of the operators around the attention of a batch (include/g4.h: g4_embed_tokens,
g4_nvfp4_*, g4_residual_norm, g4_beam_select), for programs that run many sequences or prompt
chunks where the reference's host runs one position per dispatch (src/host/generate.rs:194-211).

    rows = Nvfp4Rows(ctx, max_tokens, 3840)                  # kept: codes, scales, factors
    qkv_w = Nvfp4Weight(ctx, codes, block_scales, gscale)    # once per projection
    embed_tokens(ctx, table, tokens, x)
    nvfp4_quantize(ctx, x, rows, input_rms_weight)           # per layer
    nvfp4_matmul(ctx, rows, qkv_w, qkv)
    ...                                                      # paged_store_qkv, paged_attention
    nvfp4_quantize(ctx, attended, o_rows)
    nvfp4_matmul(ctx, o_rows, o_w, y)
    residual_norm(ctx, y, post_rms_weight, x, x)
    ...
    beam_select(ctx, logits, scores, best_scores, beams, next_tokens)
    pool.reorder(seqs, [seqs[b] for b in beams])             # each group's caches follow
"""

from __future__ import annotations

import ctypes

import torch

from . import LIB, Context, _i32, _i64, _vp

_f32 = ctypes.c_float
EMBED_SCALE = 62.0  # G4_EMBED_SCALE
BEAM_MAX = 64  # G4_BEAM_MAX


class _RowsDesc(ctypes.Structure):
    _fields_ = [("codes", _vp), ("scales", _vp), ("factor", _vp), ("max_rows", _i32), ("cols", _i32), ("pieces", _i32)]


class _WeightDesc(ctypes.Structure):
    _fields_ = [("codes", _vp), ("scales", _vp), ("factor", _vp), ("rows", _i32), ("cols", _i32), ("n_factors", _i32),
                ("constant", _i32)]


_rows_p, _weight_p = ctypes.POINTER(_RowsDesc), ctypes.POINTER(_WeightDesc)
LIB.g4_embed_tokens.argtypes = [_vp, _vp, _i32, _i32, _vp, _i32, _f32, _vp, _i64]
LIB.g4_residual_norm.argtypes = [_vp, _vp, _i64, _vp, _vp, _i64, _i32, _i32, _vp, _i64]
LIB.g4_nvfp4_scale_bytes.argtypes = [_i32, _i32]
LIB.g4_nvfp4_scale_bytes.restype = ctypes.c_uint64
LIB.g4_nvfp4_scale_blocks.argtypes = [_vp, _vp, _i32, _i32, _vp]
LIB.g4_nvfp4_quantize.argtypes = [_vp, _vp, _i64, _i32, _vp, _rows_p]
LIB.g4_nvfp4_dequantize.argtypes = [_vp, _rows_p, _i32, _vp, _i64]
LIB.g4_nvfp4_matmul.argtypes = [_vp, _rows_p, _i32, _weight_p, _vp, _i64, _i32]
LIB.g4_beam_select.argtypes = [_vp, _vp, _i64, _i64, _vp, _i32, _i32, _i32, _i32, _vp, _vp, _vp]

_g4_embed_tokens, _g4_residual_norm, _g4_beam_select = LIB.g4_embed_tokens, LIB.g4_residual_norm, LIB.g4_beam_select
_g4_nvfp4_quantize, _g4_nvfp4_dequantize, _g4_nvfp4_matmul = LIB.g4_nvfp4_quantize, LIB.g4_nvfp4_dequantize, LIB.g4_nvfp4_matmul

_BF16, _F32, _I32, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


def _tensor(ctx: Context, name: str, t, dtypes: tuple, dims: int):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name}: on {t.device}, the context is on cuda:{ctx.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype}, expected {dtypes[0]}")
    if t.dim() != dims:
        raise ValueError(f"{name}: {t.dim()} dimensions, expected {dims}")
    if t.numel() >= 2 ** 31 and max(t.shape) >= 2 ** 31:  # (ctypes would keep the low 32 bits)
        raise ValueError(f"{name}: shape {list(t.shape)} does not fit 32 bits")
    return t


def _matrix(ctx: Context, name: str, t, rows, cols, dtypes=(_BF16,)) -> tuple:
    """A [rows, cols] operand (None: any) with contiguous rows: (pointer, row stride)."""
    shape = _tensor(ctx, name, t, dtypes, 2).shape
    if (rows is not None and shape[0] != rows) or (cols is not None and shape[1] != cols):
        raise ValueError(f"{name}: shape {list(shape)}, expected [{'n' if rows is None else rows}, {'any' if cols is None else cols}]")
    row, col = t.stride()
    if col != 1 and shape[1] > 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return t.data_ptr(), row if shape[0] > 1 else max(row, shape[1])


def _operand(ctx: Context, name: str, t, rows, cols, dtype=_BF16) -> tuple:
    """_matrix, and its rows and columns: (rows, columns, pointer, row stride), in few steps where all is well
    (a call of few rows takes the GPU less than its checks take the host)."""
    try:
        if t.get_device() == ctx.device and t.dtype is dtype:
            (r, c), (stride, one) = t.shape, t.stride()
            if one == 1 and (rows is None or r == rows) and (cols is None or c == cols) and r < 2 ** 31 > c:
                return r, c, t.data_ptr(), stride if r > 1 else c
    except (AttributeError, ValueError):
        pass
    at = _matrix(ctx, name, t, rows, cols, (dtype,))
    return *t.shape, *at


def _vector(ctx: Context, name: str, t, n, dtype) -> int:
    """A contiguous [n] operand's pointer."""
    try:
        if t.dtype is dtype and t.dim() == 1 and t.numel() == n and t.get_device() == ctx.device and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    return _whole(ctx, name, t, (n,), (dtype,))


def _exact(ctx: Context, name: str, t, shape: tuple, dtype) -> int:
    """A contiguous operand's pointer."""
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == ctx.device and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    return _whole(ctx, name, t, shape, (dtype,))


def _whole(ctx: Context, name: str, t, shape: tuple, dtypes) -> int:
    _tensor(ctx, name, t, dtypes, len(shape))
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: shape {list(t.shape)}, expected {list(shape)}, contiguous")
    return t.data_ptr()


def embed_tokens(ctx: Context, table, tokens, out, scale: float = EMBED_SCALE) -> None:
    """out[t] = bf16(table[tokens[t]] * scale) (g4_embed_tokens): table bf16 [vocab, dim] contiguous,
    tokens int32 [n], out bf16 [n, dim].  An id outside the table gives zeros and a device status bit."""
    vocab, dim, rows, stride = _operand(ctx, "table", table, None, None)
    n, _, to, out_stride = _operand(ctx, "out", out, None, dim)
    ids = _vector(ctx, "tokens", tokens, n, _I32)
    if stride != dim:
        raise ValueError("table: must be contiguous")
    if n and (code := _g4_embed_tokens(ctx.handle, rows, vocab, dim, ids, n, scale, to, out_stride)):
        ctx._check("g4_embed_tokens", code)


def residual_norm(ctx: Context, x, rms_weight, residual, out) -> None:
    """out = bf16(residual + rmsnorm(x) * rms_weight) by rows (g4_residual_norm); out may be residual."""
    n, dim, xp, xs = _operand(ctx, "x", x, None, None)
    _, _, rp, rs = _operand(ctx, "residual", residual, n, dim)
    _, _, op, os = (n, dim, rp, rs) if out is residual else _operand(ctx, "out", out, n, dim)
    w = _vector(ctx, "rms_weight", rms_weight, dim, _BF16)
    if n and (code := _g4_residual_norm(ctx.handle, xp, xs, w, rp, rs, n, dim, op, os)):
        ctx._check("g4_residual_norm", code)


class Nvfp4Rows:
    """Room for `max_rows` rows of `cols` values as 1 to 3 NVFP4 pieces (g4_nvfp4_rows), on the
    context's device.  Filled by nvfp4_quantize; calls take the first rows of it."""

    def __init__(self, ctx: Context, max_rows: int, cols: int, pieces: int = 2):
        if not 1 <= max_rows <= 2 ** 22 or cols % 32 or not 32 <= cols <= 16384 or not 1 <= pieces <= 3:
            raise ValueError(f"{max_rows} rows of {cols} values in {pieces} pieces: expected 1..2^22 rows of a multiple of "
                             "32 up to 16384 in 1..3 pieces")
        self.max_rows, self.cols, self.pieces, self.device = max_rows, cols, pieces, ctx.device
        blocks = LIB.g4_nvfp4_scale_bytes(max_rows, cols)
        with torch.cuda.stream(ctx.stream):  # (the memory is used on, and given back to, this stream)
            dev = f"cuda:{ctx.device}"
            self.codes = torch.empty((pieces, max_rows, cols // 2), dtype=_U8, device=dev)
            self.scales = torch.empty((pieces, blocks), dtype=_U8, device=dev)
            self.factor = torch.empty(max_rows, dtype=_F32, device=dev)
        self.desc = _RowsDesc(self.codes.data_ptr(), self.scales.data_ptr(), self.factor.data_ptr(), max_rows, cols, pieces)


class Nvfp4Weight:
    """A projection [rows, cols] for nvfp4_matmul (g4_nvfp4_weight): the checkpoint's codes uint8
    [rows, cols / 2] (kept, not copied), its block scales [rows, cols / 16], which are laid out anew, and
    the reciprocal global scale f32 [1], or a factor for every row, f32 [rows] (projections stacked
    along their rows).  Codes and scales are constant (g4.h): nothing may write them between the nvfp4_quantize
    and the nvfp4_matmul of a product, which reads them ahead; a weight that changes is one of from_rows."""

    def __init__(self, ctx: Context, codes, block_scales, global_scale):
        n, half = _tensor(ctx, "codes", codes, (_U8,), 2).shape
        cols = 2 * half
        if n < 1 or cols % 32 or not 32 <= cols <= 16384:
            raise ValueError(f"codes: [{n}, {half}] bytes, expected rows of a multiple of 16 up to 8192")
        _whole(ctx, "codes", codes, (n, half), (_U8,))
        given = _whole(ctx, "block_scales", block_scales, (n, cols // 16), (_U8, torch.float8_e4m3fn))
        _tensor(ctx, "global_scale", global_scale, (_F32,), 1)
        if global_scale.numel() not in (1, n) or not global_scale.is_contiguous():
            raise ValueError(f"global_scale: {global_scale.numel()} values, expected 1 or {n}, contiguous")
        with torch.cuda.stream(ctx.stream):
            scales = torch.empty(LIB.g4_nvfp4_scale_bytes(n, cols), dtype=_U8, device=f"cuda:{ctx.device}")
        ctx._check("g4_nvfp4_scale_blocks", LIB.g4_nvfp4_scale_blocks(ctx.handle, given, n, cols, scales.data_ptr()))
        block_scales.record_stream(ctx.stream)  # (not kept: their memory is nobody else's until that has read them)
        self._set(codes, scales, global_scale, n, cols, ctx.device, 1)

    @classmethod
    def from_rows(cls, rows: Nvfp4Rows, constant: bool = False) -> "Nvfp4Weight":
        """The matrix that nvfp4_quantize wrote into `rows` (one piece, all of its rows), as a weight; constant: the
        rows stay what they are (a projection quantised once), and products may read them ahead."""
        if rows.pieces != 1:
            raise ValueError(f"rows: {rows.pieces} pieces, a weight has one")
        w = cls.__new__(cls)
        w._set(rows.codes, rows.scales, rows.factor, rows.max_rows, rows.cols, rows.device, int(constant))
        return w

    def _set(self, codes, scales, factor, n, cols, device, constant=0):
        self.codes, self.scales, self.factor, self.rows, self.cols, self.device = codes, scales, factor, n, cols, device
        self.desc = _WeightDesc(codes.data_ptr(), scales.data_ptr(), factor.data_ptr(), n, cols, factor.numel(), constant)


def _rows_of(ctx: Context, rows: Nvfp4Rows, n: int) -> None:
    if rows.device != ctx.device:
        raise ValueError(f"rows: on cuda:{rows.device}, the context is on cuda:{ctx.device}")
    if n > rows.max_rows:
        raise ValueError(f"rows: room for {rows.max_rows}, the call has {n}")


def nvfp4_quantize(ctx: Context, x, rows: Nvfp4Rows, rms_weight=None) -> None:
    """x (bf16 [n, cols]), or rmsnorm(x) * rms_weight rounded to bf16, into the first n rows of `rows`
    (g4_nvfp4_quantize)."""
    n, _, xp, xs = _operand(ctx, "x", x, None, rows.cols)
    _rows_of(ctx, rows, n)
    w = None if rms_weight is None else _vector(ctx, "rms_weight", rms_weight, rows.cols, _BF16)
    if n and (code := _g4_nvfp4_quantize(ctx.handle, xp, xs, n, w, rows.desc)):
        ctx._check("g4_nvfp4_quantize", code)


def nvfp4_dequantize(ctx: Context, rows: Nvfp4Rows, out) -> None:
    """The values of the first n rows, rounded to bf16, into out [n, cols] (g4_nvfp4_dequantize)."""
    n, _, op, os = _operand(ctx, "out", out, None, rows.cols)
    _rows_of(ctx, rows, n)
    if n and (code := _g4_nvfp4_dequantize(ctx.handle, rows.desc, n, op, os)):
        ctx._check("g4_nvfp4_dequantize", code)


def nvfp4_matmul(ctx: Context, rows: Nvfp4Rows, weight: Nvfp4Weight, out) -> None:
    """out [n, weight.rows] = the first n rows times the weight's rows (g4_nvfp4_matmul); out bf16, or
    f32 (a tensor-parallel rank's partial sums)."""
    f32 = isinstance(out, torch.Tensor) and out.dtype is _F32
    n, _, op, os = _operand(ctx, "out", out, None, weight.rows, _F32 if f32 else _BF16)
    _rows_of(ctx, rows, n)
    if weight.device != ctx.device:
        raise ValueError(f"weight: on cuda:{weight.device}, the context is on cuda:{ctx.device}")
    if weight.cols != rows.cols:
        raise ValueError(f"rows of {rows.cols} values, a weight of {weight.cols}")
    if n and (code := _g4_nvfp4_matmul(ctx.handle, rows.desc, n, weight.desc, op, os, f32)):
        ctx._check("g4_nvfp4_matmul", code)


def beam_select(ctx: Context, logits, scores, out_scores, out_beams, out_tokens) -> None:
    """Each group's best continuations (g4_beam_select): logits bf16 [groups, beams, vocab] over any
    strides with a contiguous last dimension, scores f32 [groups, beams] (-inf: the beam does not
    count); out_scores f32, out_beams and out_tokens int32 [groups, select], best first, equal scores
    in the order of (beam, token)."""
    try:
        fits = logits.dtype is _BF16 and logits.get_device() == ctx.device
        (groups, beams, vocab), (group_stride, beam_stride, one) = logits.shape, logits.stride()
        fits = fits and groups < 2 ** 31
    except (AttributeError, ValueError):
        fits = False
    if not fits:
        groups, beams, vocab = _tensor(ctx, "logits", logits, (_BF16,), 3).shape
        group_stride, beam_stride, one = logits.stride()
    if vocab > 1 and one != 1:
        raise ValueError("logits: the last dimension must be contiguous")
    given = _exact(ctx, "scores", scores, (groups, beams), _F32)
    two = isinstance(out_scores, torch.Tensor) and out_scores.dim() == 2
    select = (out_scores if two else _tensor(ctx, "out_scores", out_scores, (_F32,), 2)).shape[1]
    best = _exact(ctx, "out_scores", out_scores, (groups, select), _F32)
    of = _exact(ctx, "out_beams", out_beams, (groups, select), _I32)
    to = _exact(ctx, "out_tokens", out_tokens, (groups, select), _I32)
    if not 1 <= beams <= BEAM_MAX or not 1 <= select <= BEAM_MAX or not 1 <= vocab <= 2 ** 20 or select > beams * vocab:
        raise ValueError(f"{select} of {beams} beams of {vocab} tokens: expected up to {BEAM_MAX} of up to {BEAM_MAX} beams of up "
                         "to 2^20 tokens, no more than there are")
    if groups and (code := _g4_beam_select(ctx.handle, logits.data_ptr(), group_stride, beam_stride, given, groups, beams,
                                           vocab, select, best, of, to)):
        ctx._check("g4_beam_select", code)


__all__ = ["Nvfp4Rows", "Nvfp4Weight", "embed_tokens", "residual_norm", "nvfp4_quantize", "nvfp4_dequantize",
           "nvfp4_matmul", "beam_select"]
