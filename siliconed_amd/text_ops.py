"""A text decoder's operators: the norm that writes a product's 8-bit operand, products of block-scaled e4m3 codes,
and a paged key-value cache with its append and its attention; heads normed in the pass that turns and appends them, attention of
packed prompts and of chunks over the cache, and the draw of the next tokens (the sq8_* entries of include/siliconed_q8.h).

`TensorGEMM` has them as methods; everything is queued on its stream. Outputs that a call allocates are torch's, of its
current stream: make calls with the context's stream current (`torch.cuda.stream`), or hand in outputs and order the two
streams. With them, a decoder layer's step is

    codes, sx, x = ctx.add_norm_quantized(y, w_norm, eps, residual=x)
    qkv = ctx.product_f8(codes, sx, w_qkv, s_qkv)
    q = ctx.append_kv(q, k, v, cache, positions, slots, table)
    o = ctx.paged_attention(q, cache, pages, lengths)
    y = ctx.product_f8_quantized(o.flatten(1), w_out, s_out)

with normed heads norm_append_kv, with several new tokens of a sequence chunk_attention, and after the last layer

    tokens, logprobs = ctx.sample_tokens(logits, uniform, temperature=t, top_p=p)
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _abi as abi

_F8 = torch.float8_e4m3fn
_CACHES = {torch.bfloat16: abi.BF16, _F8: abi.FP8_E4M3}
_EPILOGUES = {None: False, "none": False, "silu_glu": True, "swiglu": True}  # True: a GLU


def _vector(t: Optional[torch.Tensor], count: int, what: str, device: torch.device):
    """A contiguous fp32 vector's address (None: null)."""
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != count or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what} must be {count} contiguous float32 values on {device}")
    return t.data_ptr()


def _strides(pool: torch.Tensor):
    """A pool's strides but the last; of a dimension of one, which torch leaves anything, 0."""
    return [stride if size > 1 else 0 for size, stride in zip(pool.shape[:3], pool.stride())]


def _glu(epilogue) -> bool:
    if epilogue not in _EPILOGUES:
        raise ValueError(f"a block-scaled product's epilogue is None or 'silu_glu', not {epilogue!r}")
    return _EPILOGUES[epilogue]


def _is_f32(dtype: torch.dtype) -> bool:
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"outputs are bfloat16 or float32, not {dtype}")
    return dtype == torch.float32


def _done(result, what: str):
    """A native call's outputs; a status is the library's refusal."""
    if type(result) is int:
        abi.check(result, what)
    return result


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
        self.pages, self.page, self.kv_heads, self.dim, self.device = pages, page, heads, dim, k.device.index
        self._args = abi.PagedCacheArgs(k.data_ptr(), v.data_ptr(), *_strides(k), *_strides(v),
                                        _vector(k_scale, heads, "k_scale", k.device), _vector(v_scale, heads, "v_scale", k.device),
                                        dtype, pages, page, heads, dim)


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
        int8 = dtype == torch.int8
        if not int8 and dtype != _F8:
            raise ValueError(f"codes are float8_e4m3fn or int8, not {dtype}")
        return _done(abi.text.add_norm_quantized(self._h, x, w, eps, residual, residual_out, int8, codes, scales),
                     "sq8_add_norm_quantized")

    def quantize_groups(self, x: torch.Tensor, *, codes: Optional[torch.Tensor] = None,
                        scales: Optional[torch.Tensor] = None):
        """x [rows, cols] (bfloat16 or float32) as float8_e4m3fn codes and a scale per 128 columns of a row."""
        return _done(abi.text.quantize_groups(self._h, x, codes, scales), "sq8_quantize_groups")

    def product_f8(self, codes: torch.Tensor, sx: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, *,
                   bias: Optional[torch.Tensor] = None, epilogue=None, out: Optional[torch.Tensor] = None,
                   out_dtype: torch.dtype = torch.bfloat16, timed: bool = False):
        """act(Σ over blocks of 128 of K of sx · scale · (codes · wᵀ) + bias), sums in fp32 with `out_dtype` float32 (a
        bfloat16 output's leave out what is under 2^-13 of the largest of 8 products): codes float8_e4m3fn [m, k] with sx
        [m, ⌈k/128⌉] (add_norm_quantized's, quantize_groups'), w float8_e4m3fn [n, k] with scale [⌈n/128⌉, ⌈k/128⌉] as
        published. `epilogue="silu_glu"`: n = 2h rows, gate then up, each half blocked by itself (scale
        [2·⌈h/128⌉, ⌈k/128⌉]), output [m, h]."""
        if sx is None:
            raise ValueError("sx float32 [m, ⌈k/128⌉] belongs to codes (product_f8_quantized takes values)")
        return _done(abi.text.product_f8(self._h, codes, sx, w, scale, bias, _glu(epilogue), out, _is_f32(out_dtype),
                                         timed), "sq8_linear_f8")

    def product_f8_quantized(self, x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, *,
                             bias: Optional[torch.Tensor] = None, epilogue=None, out: Optional[torch.Tensor] = None,
                             out_dtype: torch.dtype = torch.bfloat16, timed: bool = False):
        """product_f8 on x [m, k] (bfloat16 or float32), quantized by groups first."""
        return _done(abi.text.product_f8(self._h, x, None, w, scale, bias, _glu(epilogue), out, _is_f32(out_dtype),
                                         timed), "sq8_linear_f8_quantized")

    def _args_of(self, cache: PagedCache):
        """What the native calls take of a cache, which lies on this context's GPU."""
        if cache.device != self.device:
            raise ValueError(f"the cache must be on the context's GPU, cuda:{self.device}, not cuda:{cache.device}")
        return cache._args

    def append_kv(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedCache, positions: torch.Tensor,
                  slots: torch.Tensor, table: torch.Tensor, *, q_out: Optional[torch.Tensor] = None,
                  interleaved: bool = False) -> torch.Tensor:
        """Turns q [tokens, q_heads, dim] and k by their positions' angles, writes k and v [tokens, kv_heads, dim] (bf16,
        any row and head strides) to the cache's slots (slot = page · tokens a page + place, −1: none), and returns
        the turned q (`q_out`; q itself turns it in place). `table` float32 [positions, rot]: rot/2 cosines, then the
        sines, of a head's first rot values, paired (i, i + rot/2), or (2i, 2i + 1) when `interleaved`. positions,
        slots int32 [tokens]."""
        return _done(abi.text.append_kv(self._h, q, k, v, self._args_of(cache), positions, slots, table, q_out, interleaved),
                     "sq8_append_kv")

    def paged_attention(self, q: torch.Tensor, cache: PagedCache, pages: torch.Tensor, lengths: torch.Tensor, *,
                        scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of each sequence's new token q [batch, q_heads, dim] (bf16) over its cached tokens: `pages` int32
        [batch, most pages] page indices in order, `lengths` int32 [batch] (0: zeros). `scale` defaults to
        1/sqrt(dim); `softcap` c > 0 (inf: none): scores c · tanh(s/c); `window` w > 0: the last w tokens only."""
        return _done(abi.text.paged_attention(self._h, q, self._args_of(cache), pages, lengths, scale, softcap, window, out),
                     "sq8_paged_attention")

    def norm_append_kv(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedCache, positions: torch.Tensor,
                       slots: torch.Tensor, table: torch.Tensor, *, q_norm: Optional[torch.Tensor] = None,
                       k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
                       interleaved: bool = False) -> torch.Tensor:
        """append_kv with every query and key head's RMS norm (times `q_norm`, `k_norm` float32 [dim]; None: not normed) before
        its turn, in the same pass: nothing is rounded in between. Heads of up to 512."""
        return _done(abi.text.norm_append_kv(self._h, q, k, v, self._args_of(cache), positions, slots, table, q_norm, k_norm, eps,
                                             q_out, interleaved), "sq8_norm_append_kv")

    def norm_rotate(self, q: torch.Tensor, k: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                    table: Optional[torch.Tensor] = None, *, q_norm: Optional[torch.Tensor] = None,
                    k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
                    k_out: Optional[torch.Tensor] = None, interleaved: bool = False):
        """The same without a cache: q [tokens, q_heads, dim] and k [tokens, kv_heads, dim] (None: q alone) normed and turned:
        (q_out, k_out), which may be q and k themselves. No positions and table: normed only."""
        return _done(abi.text.norm_rotate(self._h, q, k, positions, table, q_norm, k_norm, eps, q_out, k_out, interleaved),
                     "sq8_norm_rotate")

    def prompt_attention(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: Optional[torch.Tensor] = None, *,
                         causal: bool = True, scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of whole sequences over their own keys and values: q [tokens, q_heads, dim], k and v [tokens, kv_heads,
        dim] (bf16, any row and head strides of whole 16 bytes), sequence b in rows starts[b] to starts[b + 1] − 1 (`starts`
        int32 [sequences + 1] on the GPU; None: one sequence). `causal`: a token sees those up to itself, with `window` w > 0
        the last w of them; else all of its sequence. Rows of no sequence are left as they were: of an `out` that the call
        allocates, anything. `scale` and `softcap` as paged_attention."""
        return _done(abi.text.prompt_attention(self._h, q, k, v, starts, scale, softcap, window, causal, out), "sq8_prompt_attention")

    def chunk_attention(self, q: torch.Tensor, cache: PagedCache, pages: torch.Tensor, lengths: torch.Tensor,
                        starts: Optional[torch.Tensor] = None, *, scale: Optional[float] = None, softcap: float = 0.0,
                        window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of each sequence's newest tokens over its cached ones, these included: q [tokens, q_heads, dim] (bf16) in
        rows as prompt_attention's (`starts`), `pages` int32 [sequences, most pages] and `lengths` int32 [sequences] as
        paged_attention's. A draft to verify, a piece of a long prompt, or both in one batch."""
        return _done(abi.text.chunk_attention(self._h, q, self._args_of(cache), pages, lengths, starts, scale, softcap, window, out),
                     "sq8_chunk_attention")

    def sample_tokens(self, logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Optional[torch.Tensor] = None,
                      top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                      min_p: Optional[torch.Tensor] = None, tokens: Optional[torch.Tensor] = None,
                      logprobs: Optional[torch.Tensor] = None):
        """The next token of each row of logits [rows, vocab] (bfloat16 or float32), drawn with `uniform` float32 [rows] in [0, 1):
        (tokens int32 [rows], the logs of the probabilities they were drawn with, float32 [rows]). Each row its own, float32
        [rows]: `temperature` (None: 1; 0: the largest logit, the first of equal ones), `top_p` (None: 1), `min_p` (None: 0), and
        `top_k` int32 [rows] (None or 0: all): of the tokens by falling logit the first top_k, of these the fewest that hold top_p
        of their probability, of these the ones of at least min_p of the likeliest's. A row of nothing but -inf and NaN gives
        −1. The same inputs give the same tokens always."""
        return _done(abi.text.sample_tokens(self._h, logits, uniform, temperature, top_k, top_p, min_p, tokens, logprobs),
                     "sq8_sample_tokens")
