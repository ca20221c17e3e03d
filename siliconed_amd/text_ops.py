"""A text decoder's operators: the norm that writes a product's 8-bit operand, products of block-scaled e4m3 codes,
and a paged key-value cache with its append and its attention (the sq8_* entries of include/siliconed_q8.h).

`TensorGEMM` has them as methods; everything is queued on its stream. With them, a decoder layer's step is

    codes, sx, x = ctx.add_norm_quantized(y, w_norm, eps, residual=x)
    qkv = ctx.product_f8(codes, sx, w_qkv, s_qkv)
    q = ctx.append_kv(q, k, v, cache, positions, slots, table)
    o = ctx.paged_attention(q, cache, pages, lengths)
    y = ctx.product_f8_quantized(o.flatten(1), w_out, s_out)
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _abi as abi

GROUP = 128  # values of K that share a scale

_ACTIVATIONS = {torch.bfloat16: abi.BF16, torch.float32: abi.F32}
_F8 = torch.float8_e4m3fn
_CACHES = {torch.bfloat16: abi.BF16, _F8: abi.FP8_E4M3}
_EPILOGUES = {None: abi.EPI_NONE, "none": abi.EPI_NONE, "silu_glu": abi.EPI_SILU_GLU, "swiglu": abi.EPI_SILU_GLU}


def _groups(k: int) -> int:
    return -(-k // GROUP)


def _rows(t: torch.Tensor, what: str, shape=None) -> int:
    """The leading dimension of a matrix on the GPU whose rows are contiguous, its shape checked."""
    if not t.is_cuda:
        raise ValueError(f"{what} must be on the GPU")
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError(f"{what} must be {'2-D' if shape is None else shape}, not {tuple(t.shape)}")
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1 and rows > 0:
        raise ValueError(f"{what} must have contiguous rows")
    return ld if rows > 1 else max(cols, 1)


def _activation(t: torch.Tensor, what: str) -> int:
    dtype = _ACTIVATIONS.get(t.dtype)
    if dtype is None:
        raise ValueError(f"{what} must be bfloat16 or float32, not {t.dtype}")
    return dtype


def _vector(t: Optional[torch.Tensor], count: int, what: str, dtype=torch.float32):
    """A contiguous vector's address (None: null)."""
    if t is None:
        return None
    if t.dtype != dtype or t.numel() != count or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"{what} must be {count} contiguous {dtype} values on the GPU")
    return t.data_ptr()


def _heads(t: torch.Tensor, what: str, rows: int, heads: Optional[int], dim: int):
    """(address, row stride, head stride) of bf16 [rows, heads, dim]."""
    shape = t.shape
    if (t.dtype != torch.bfloat16 or len(shape) != 3 or shape[0] != rows or shape[2] != dim or not t.is_cuda
            or (heads is not None and shape[1] != heads)):
        raise ValueError(f"{what} must be bfloat16 [{rows}, {'heads' if heads is None else heads}, {dim}] on the GPU")
    a, b, c = t.stride()
    if c != 1 and dim > 1:
        raise ValueError(f"{what} must have contiguous heads")
    return t.data_ptr(), a, b


class PagedCache:
    """Two pools of pages, [pages, page, kv_heads, head_dim] of bfloat16, or of float8_e4m3fn standing for code ·
    scale (`k_scale`, `v_scale`: float32 [kv_heads], None: 1). Any strides with the values of a head contiguous. Made
    once for the pools; what it says is what append_kv writes and paged_attention reads."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        dtype = _CACHES.get(k.dtype)
        if dtype is None or v.dtype != k.dtype:
            raise ValueError("a cache's pools are both bfloat16 or both float8_e4m3fn")
        if k.dim() != 4 or v.shape != k.shape or not k.is_cuda or v.device != k.device:
            raise ValueError("a cache's pools are [pages, page, kv_heads, head_dim] on one GPU")
        pages, page, heads, dim = k.shape
        if page == 0 or heads == 0 or dim == 0:
            raise ValueError("a cache has tokens in a page, heads and values in a head")
        if dim > 1 and (k.stride(3) != 1 or v.stride(3) != 1):
            raise ValueError("a cache's heads must be contiguous")
        if dtype == abi.BF16 and (k_scale is not None or v_scale is not None):
            raise ValueError("scales belong to float8_e4m3fn pools")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.page, self.kv_heads, self.dim = pages, page, heads, dim
        self._args = abi.PagedCacheArgs(k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3],
                                        _vector(k_scale, heads, "k_scale"), _vector(v_scale, heads, "v_scale"), dtype,
                                        pages, page, heads, dim)
        self._ref = ctypes.byref(self._args)


class TextOps:
    """The operators as methods of a context (`TensorGEMM`)."""

    def add_norm_quantized(self, x: torch.Tensor, w: torch.Tensor, eps: float = 1e-6, *,
                           residual: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None,
                           dtype: torch.dtype = _F8, codes: Optional[torch.Tensor] = None,
                           scales: Optional[torch.Tensor] = None):
        """RMS norm of residual + x [rows, cols] (or of x), times w, in 8 bits: (codes, scales, the new residual).
        `dtype` float8_e4m3fn: a scale per 128 columns [rows, ⌈cols/128⌉] (product_f8's operand); int8: one per row
        [rows] (product_w8a8's). The sum goes to `residual_out`, by default into `residual` itself; its rounding to
        the stream's type comes after the norm has taken it."""
        ldx = _rows(x, "x")
        rows, cols = x.shape
        int8 = dtype == torch.int8
        if not int8 and dtype != _F8:
            raise ValueError(f"codes are float8_e4m3fn or int8, not {dtype}")
        if codes is None:
            codes = torch.empty((rows, cols), dtype=dtype, device=x.device)
        elif codes.dtype != dtype:
            raise ValueError(f"codes must be {dtype}")
        lds = 0
        if int8:
            if scales is None:
                scales = torch.empty(rows, dtype=torch.float32, device=x.device)
            at = _vector(scales, rows, "scales")
        else:
            if scales is None:
                scales = torch.empty((rows, _groups(cols)), dtype=torch.float32, device=x.device)
            elif scales.dtype != torch.float32:
                raise ValueError("scales must be float32")
            lds, at = _rows(scales, "scales", (rows, _groups(cols))), scales.data_ptr()
        rp, rt, ldr, op, ldo = None, 0, 0, None, 0
        if residual is not None:
            if residual_out is None:
                residual_out = residual
            elif residual_out.dtype != residual.dtype:
                raise ValueError("residual_out must be of the residual's type")
            rp, rt, ldr = residual.data_ptr(), _activation(residual, "residual"), _rows(residual, "residual", (rows, cols))
            op, ldo = residual_out.data_ptr(), _rows(residual_out, "residual_out", (rows, cols))
        elif residual_out is not None:
            raise ValueError("residual_out needs a residual")
        st = abi.load().sq8_add_norm_quantized(self._h, x.data_ptr(), _activation(x, "x"), ldx, rp, rt, ldr, op, ldo,
                                               _vector(w, cols, "w"), eps, codes.data_ptr(),
                                               abi.INT8 if int8 else abi.FP8_E4M3, _rows(codes, "codes", (rows, cols)),
                                               at, lds, rows, cols)
        abi.check(st, "sq8_add_norm_quantized")
        return codes, scales, residual_out

    def quantize_groups(self, x: torch.Tensor, *, codes: Optional[torch.Tensor] = None,
                        scales: Optional[torch.Tensor] = None):
        """x [rows, cols] (bfloat16 or float32) as float8_e4m3fn codes and a scale per 128 columns of a row."""
        ldx = _rows(x, "x")
        rows, cols = x.shape
        if codes is None:
            codes = torch.empty((rows, cols), dtype=_F8, device=x.device)
        if scales is None:
            scales = torch.empty((rows, _groups(cols)), dtype=torch.float32, device=x.device)
        if codes.dtype != _F8 or scales.dtype != torch.float32:
            raise ValueError("codes must be float8_e4m3fn, scales float32")
        st = abi.load().sq8_quantize_groups(self._h, x.data_ptr(), _activation(x, "x"), ldx, rows, cols, codes.data_ptr(),
                                            _rows(codes, "codes", (rows, cols)), scales.data_ptr(),
                                            _rows(scales, "scales", (rows, _groups(cols))))
        abi.check(st, "sq8_quantize_groups")
        return codes, scales

    def _f8(self, name, lead, m, k, w, scale, bias, epilogue, out, out_dtype, timed, device):
        if epilogue not in _EPILOGUES:
            raise ValueError(f"a block-scaled product's epilogue is None or 'silu_glu', not {epilogue!r}")
        epi = _EPILOGUES[epilogue]
        if w.dtype != _F8:
            raise ValueError(f"w must be float8_e4m3fn codes [n, k], not {w.dtype}")
        n = w.shape[0]
        ldw = _rows(w, "w", (n, k))
        h = n
        blocks = _groups(n)
        if epi == abi.EPI_SILU_GLU:
            if n % 2:
                raise ValueError("a GLU weight has an even number of rows")
            h = n // 2
            blocks = 2 * _groups(h)
        if scale.dtype != torch.float32:
            raise ValueError("scale must be float32")
        lds = _rows(scale, "scale", (blocks, _groups(k)))
        if out is None:
            out = torch.empty((m, h), dtype=out_dtype, device=device)
        ldc = _rows(out, "out", (m, h))
        secs = ctypes.c_double(0.0) if timed else None
        st = getattr(abi.load(), name)(self._h, *lead, w.data_ptr(), ldw, scale.data_ptr(), lds, _vector(bias, n, "bias"),
                                       epi, out.data_ptr(), _activation(out, "out"), ldc, m, k, n,
                                       None if secs is None else ctypes.byref(secs))
        abi.check(st, name)
        return (out, secs.value) if timed else out

    def product_f8(self, codes: torch.Tensor, sx: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, *,
                   bias: Optional[torch.Tensor] = None, epilogue=None, out: Optional[torch.Tensor] = None,
                   out_dtype: torch.dtype = torch.bfloat16, timed: bool = False):
        """act(Σ over blocks of 128 of K of sx · scale · (codes · wᵀ) + bias): codes float8_e4m3fn [m, k] with sx
        [m, ⌈k/128⌉] (add_norm_quantized's, quantize_groups'), w float8_e4m3fn [n, k] with scale [⌈n/128⌉, ⌈k/128⌉] as
        published. `epilogue="silu_glu"`: n = 2h rows, gate then up, each half blocked by itself (scale
        [2·⌈h/128⌉, ⌈k/128⌉]), output [m, h]."""
        if codes.dtype != _F8 or sx.dtype != torch.float32:
            raise ValueError("codes float8_e4m3fn [m, k], sx float32 [m, ⌈k/128⌉]")
        lda = _rows(codes, "codes")
        m, k = codes.shape
        lead = (codes.data_ptr(), lda, sx.data_ptr(), _rows(sx, "sx", (m, _groups(k))))
        return self._f8("sq8_linear_f8", lead, m, k, w, scale, bias, epilogue, out, out_dtype, timed, codes.device)

    def product_f8_quantized(self, x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, *,
                             bias: Optional[torch.Tensor] = None, epilogue=None, out: Optional[torch.Tensor] = None,
                             out_dtype: torch.dtype = torch.bfloat16, timed: bool = False):
        """product_f8 on x [m, k] (bfloat16 or float32), quantized by groups first."""
        ldx = _rows(x, "x")
        m, k = x.shape
        return self._f8("sq8_linear_f8_quantized", (x.data_ptr(), _activation(x, "x"), ldx), m, k, w, scale, bias, epilogue,
                        out, out_dtype, timed, x.device)

    def append_kv(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedCache, positions: torch.Tensor,
                  slots: torch.Tensor, table: torch.Tensor, *, q_out: Optional[torch.Tensor] = None,
                  interleaved: bool = False) -> torch.Tensor:
        """Turns q [tokens, q_heads, dim] and k by their positions' angles, writes k and v [tokens, kv_heads, dim] (bf16,
        any row and head strides) to the cache's slots (slot = page · tokens a page + place, −1: none), and returns
        the turned q (`q_out`; q itself turns it in place). `table` float32 [positions, rot]: rot/2 cosines, then the
        sines, of a head's first rot values, paired (i, i + rot/2), or (2i, 2i + 1) when `interleaved`. positions,
        slots int32 [tokens]."""
        tokens = q.shape[0]
        qa = _heads(q, "q", tokens, None, cache.dim)
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty((tokens, heads, cache.dim), dtype=torch.bfloat16, device=q.device)
        if table.dtype != torch.float32:
            raise ValueError("table must be float32 [positions, rot]")
        rows = _rows(table, "table")
        st = abi.load().sq8_append_kv(self._h, *qa, *_heads(k, "k", tokens, cache.kv_heads, cache.dim),
                                      *_heads(v, "v", tokens, cache.kv_heads, cache.dim),
                                      *_heads(q_out, "q_out", tokens, heads, cache.dim), cache._ref,
                                      _vector(positions, tokens, "positions", torch.int32),
                                      _vector(slots, tokens, "slots", torch.int32), table.data_ptr(), rows,
                                      table.shape[0], table.shape[1], interleaved, tokens, heads)
        abi.check(st, "sq8_append_kv")
        return q_out

    def paged_attention(self, q: torch.Tensor, cache: PagedCache, pages: torch.Tensor, lengths: torch.Tensor, *,
                        scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of each sequence's new token q [batch, q_heads, dim] (bf16) over its cached tokens: `pages` int32
        [batch, most pages] page indices in order, `lengths` int32 [batch] (0: zeros). `scale` defaults to
        1/sqrt(dim); `softcap` c > 0: scores c · tanh(s/c); `window` w > 0: the last w tokens only."""
        batch = q.shape[0]
        qa = _heads(q, "q", batch, None, cache.dim)
        heads = q.shape[1]
        if out is None:
            out = torch.empty((batch, heads, cache.dim), dtype=torch.bfloat16, device=q.device)
        if pages.dtype != torch.int32 or pages.dim() != 2 or pages.shape[0] != batch:
            raise ValueError(f"pages must be int32 [{batch}, most pages]")
        row = _rows(pages, "pages")
        oa = _heads(out, "out", batch, heads, cache.dim)
        st = abi.load().sq8_paged_attention(self._h, *qa, cache._ref, pages.data_ptr(), row, pages.shape[1],
                                            _vector(lengths, batch, "lengths", torch.int32),
                                            1.0 / math.sqrt(cache.dim) if scale is None else scale, softcap, window,
                                            *oa, batch, heads)
        abi.check(st, "sq8_paged_attention")
        return out
