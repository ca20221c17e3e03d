"""A text decoder's layer on block-scaled e4m3 weights and a paged key-value cache, from this library's operators:

    x += y;  q, k, v = Wqkv · RMS(x)·w_in       sq8_add_norm_quantized, sq8_linear_f8
    q, k turned by their positions, k, v kept   sq8_append_kv
    o = softmax(q · Kᵀ / sqrt(dim)) · V         sq8_paged_attention (a prompt: torch's fused SDPA)
    y = Wout · o                                sq8_linear_f8_quantized
    x += y;  g, u = Wgu · RMS(x)·w_post         sq8_add_norm_quantized, sq8_linear_f8 with the SiLU-GLU epilogue
    y = Wdown · (SiLU(g) · u)                   sq8_linear_f8_quantized

A layer takes and returns (y, x): the branch not yet added, and the fp32 residual stream, which it updates in place.
Weights are e4m3 codes with an fp32 scale per 128 × 128 block, as published (random here); heads of a group share their
keys and values. `step` runs one new token of each sequence and launches eight kernels (ten past a few sequences, whose
operands two passes quantize), all of which a HIP graph can hold; `prompt` runs one sequence's first tokens. Both queue
everything on torch's current stream (a capture's: one that a step has run on before). With the
sizes below a step's layer takes 76 us for one sequence of 2000 tokens, 103 for 16 and 125 for 64 of 1000; the weights
alone, 192 MB, are 38.

    python -m siliconed_amd.text_block --layers 4 --batch 16 --context 2000

times a decode step of such layers, as calls and as a graph.
"""
from __future__ import annotations

import torch

from .tensor_gemm import TensorGEMM, context
from .text_ops import PagedCache

EPS = 1e-6
BLOCK = 128
F8 = torch.float8_e4m3fn


def quantize_f8_blocks(w: torch.Tensor):
    """[n, k] as e4m3 codes with a scale per 128 × 128 block: s = amax/448, code = e4m3(w / s)."""
    n, k = w.shape
    rows, cols = -(-n // BLOCK), -(-k // BLOCK)
    padded = torch.zeros(rows * BLOCK, cols * BLOCK, device=w.device)
    padded[:n, :k] = w
    blocks = padded.view(rows, BLOCK, cols, BLOCK)
    s = (blocks.abs().amax(dim=(1, 3)) / 448.0).clamp_min(1e-30)
    codes = (blocks / s[:, None, :, None]).view(rows * BLOCK, cols * BLOCK)[:n, :k]
    return codes.to(F8).contiguous(), s


def widen_f8_blocks(codes: torch.Tensor, s: torch.Tensor, glu: bool = False) -> torch.Tensor:
    """What the codes and block scales stand for, float64 (`glu`: both halves blocked by themselves)."""
    if glu:
        h, rows = codes.shape[0] // 2, s.shape[0] // 2
        return torch.cat([widen_f8_blocks(codes[:h], s[:rows]), widen_f8_blocks(codes[h:], s[rows:])])
    n, k = codes.shape
    return codes.double() * s.double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def rotation_table(positions: int, dim: int, theta: float = 1e6, device="cuda") -> torch.Tensor:
    """append_kv's table: row p holds cos, then sin, of p · theta^(−2i/dim)."""
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


class TextBlock:
    """One layer's weights on one device."""

    def __init__(self, d: int = 4096, heads: int = 32, kv_heads: int = 8, dim: int = 128, hidden: int = 12288,
                 seed: int = 0, device: int = 0, ctx: TensorGEMM | None = None):
        if heads % kv_heads:
            raise ValueError("query heads share key heads in equal groups")
        self.ctx = ctx or context(device)
        self.d, self.heads, self.kv_heads, self.dim, self.hidden = d, heads, kv_heads, dim, hidden
        g = torch.Generator(device=f"cuda:{device}").manual_seed(seed)

        def normal(n, k):
            return torch.randn(n, k, generator=g, device=g.device) * k ** -0.5

        self.qkv = quantize_f8_blocks(normal((heads + 2 * kv_heads) * dim, d))
        self.out = quantize_f8_blocks(normal(d, heads * dim))
        gate, up = quantize_f8_blocks(normal(hidden, d)), quantize_f8_blocks(normal(hidden, d))
        self.gate_up = torch.cat([gate[0].view(torch.int8), up[0].view(torch.int8)]).view(F8), torch.cat([gate[1], up[1]])
        self.down = quantize_f8_blocks(normal(d, hidden))
        self.w_in = 1 + 0.1 * torch.randn(d, generator=g, device=g.device)
        self.w_post = 1 + 0.1 * torch.randn(d, generator=g, device=g.device)

    def cache(self, pages: int, page: int = 64, dtype: torch.dtype = F8, scale: float = 1 / 32) -> PagedCache:
        """Pools for this layer's keys and values; an e4m3 one stands for code · `scale`."""
        dev = self.w_in.device
        k, v = (torch.zeros(pages, page, self.kv_heads, self.dim, dtype=torch.bfloat16, device=dev).to(dtype) for _ in "kv")
        s = torch.full((self.kv_heads,), scale, device=dev) if dtype == F8 else None
        return PagedCache(k, v, s, s)

    def _here(self) -> TensorGEMM:
        """The context, on torch's current stream: what torch does before, between and after the library's kernels is
        queued there (the context may be shared, and moved by whoever used it last)."""
        self.ctx.set_stream(torch.cuda.current_stream(self.ctx.device))
        return self.ctx

    def _append(self, y, x, cache, positions, slots, table):
        """The layer up to its attention: the turned q [tokens, heads, dim] and the stream."""
        ctx = self._here()
        codes, sx, x = ctx.add_norm_quantized(y, self.w_in, EPS, residual=x)
        qkv = ctx.product_f8(codes, sx, *self.qkv).view(-1, self.heads + 2 * self.kv_heads, self.dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
        return ctx.append_kv(q, k, v, cache, positions, slots, table, q_out=q), x

    def _finish(self, o, x):
        """The layer after its attention."""
        y = self.ctx.product_f8_quantized(o.flatten(1), *self.out)
        codes, sx, x = self.ctx.add_norm_quantized(y, self.w_post, EPS, residual=x)
        hidden = self.ctx.product_f8(codes, sx, *self.gate_up, epilogue="silu_glu")
        return self.ctx.product_f8_quantized(hidden, *self.down), x

    def step(self, y, x, cache, positions, slots, pages, lengths, table):
        """One new token of each sequence: y bf16 and x fp32 [batch, d]; its position and cache slot, the sequence's
        pages [batch, most] and its length with this token (int32)."""
        q, x = self._append(y, x, cache, positions, slots, table)
        return self._finish(self.ctx.paged_attention(q, cache, pages, lengths), x)

    def prompt(self, y, x, cache, positions, slots, pages, table):
        """One sequence's first tokens, [tokens, d], its pages int32 in order."""
        q, x = self._append(y, x, cache, positions, slots, table)
        tokens = q.shape[0]

        def held(pool, scale):
            t = pool[pages.long()].flatten(0, 1)[:tokens].to(torch.bfloat16)
            if scale is not None:
                t = (t.float() * scale[:, None]).to(torch.bfloat16)
            return t.repeat_interleave(self.heads // self.kv_heads, 1).transpose(0, 1)[None]

        from torch.nn.attention import SDPBackend, sdpa_kernel
        with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
            o = torch.nn.functional.scaled_dot_product_attention(
                q.transpose(0, 1)[None].contiguous(), held(cache.k, cache.k_scale).contiguous(),
                held(cache.v, cache.v_scale).contiguous(), is_causal=True)[0]
        return self._finish(o.transpose(0, 1).contiguous(), x)


def main() -> None:
    import argparse
    import time

    a = argparse.ArgumentParser(description="times a decode step")
    a.add_argument("--layers", type=int, default=4)
    a.add_argument("--batch", type=int, default=16)
    a.add_argument("--context", type=int, default=2000)
    a.add_argument("--steps", type=int, default=50)
    a.add_argument("--page", type=int, default=64)
    a = a.parse_args()
    most = -(-a.context // a.page)
    layers = [TextBlock(seed=i) for i in range(a.layers)]
    caches = [block.cache(a.batch * most, a.page) for block in layers]
    d, dev = layers[0].d, layers[0].w_in.device
    i32 = dict(dtype=torch.int32, device=dev)
    pages = torch.randperm(a.batch * most, device=dev).to(torch.int32).view(a.batch, most)
    lengths = torch.full((a.batch,), a.context, **i32)
    positions = lengths - 1
    slots = (pages[:, -1] * a.page + (a.context - 1) % a.page).contiguous()
    table = rotation_table(a.context, layers[0].dim)
    token = torch.randn(a.batch, d, device=dev).to(torch.bfloat16)
    stream = torch.zeros(a.batch, d, device=dev)

    def run():
        y, x = token, stream.zero_()
        for block, cache in zip(layers, caches):
            y, x = block.step(y, x, cache, positions, slots, pages, lengths, table)
        return y

    def timed(f):
        f()
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(a.steps):
            f()
        torch.cuda.synchronize()
        return (time.perf_counter() - t) / a.steps * 1e6

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls = timed(run)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
        replays = timed(graph.replay)
    print(f"{a.layers} layers, {a.batch} sequences of {a.context} tokens: {calls:.0f} us a step as calls, "
          f"{replays:.0f} us as a graph ({replays / a.layers:.1f} a layer), {a.batch / replays * 1e6:.0f} tokens/s")


if __name__ == "__main__":
    main()
