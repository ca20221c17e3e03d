"""A text decoder's layer on block-scaled e4m3 weights and a paged key-value cache, from this library's operators:

    x += y;  q, k, v = Wqkv · RMS(x)·w_in       sq8_add_norm_quantized, sq8_linear_f8
    q, k turned by their positions, k, v kept   sq8_append_kv (heads normed first: sq8_norm_append_kv)
    o = softmax(q · Kᵀ / sqrt(dim)) · V         sq8_paged_attention, sq8_chunk_attention (`prompt`: torch's fused SDPA)
    y = Wout · o                                sq8_linear_f8_quantized
    x += y;  g, u = Wgu · RMS(x)·w_post         sq8_add_norm_quantized, sq8_linear_f8 with the SiLU-GLU epilogue
    y = Wdown · (SiLU(g) · u)                   sq8_linear_f8_quantized

A layer takes and returns (y, x): the branch not yet added, and the fp32 residual stream, which it updates in place.
Weights are e4m3 codes with an fp32 scale per 128 × 128 block, as published (random here); heads of a group share their
keys and values. `step` runs one new token of each sequence and launches eight kernels (ten past a few sequences, whose
operands two passes quantize), all of which a HIP graph can hold; `prompt` runs one sequence's first tokens; `chunk` any
number of new tokens of each sequence (prompts, pieces of them, drafts to verify, one token beside them); `encode` packed
prompts without a cache, as a text encoder's layer (sq8_norm_rotate, sq8_prompt_attention). All queue
everything on torch's current stream (a capture's: one that a step has run on before). `TextHead` turns the last layer's
output into logits and draws the next tokens (sq8_sample_tokens). With the
sizes below a step's layer takes 76 us for one sequence of 2000 tokens, 103 for 16 and 125 for 64 of 1000; the weights
alone, 192 MB, are 38.

    python -m siliconed_amd.text_block --layers 4 --batch 16 --context 2000

times a decode step of such layers, as calls and as a graph; --new 4 a step of four tokens a sequence, --vocab 128000 with
the draw of the next tokens.
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
                 seed: int = 0, device: int = 0, ctx: TensorGEMM | None = None, norm_heads: bool = False):
        """`norm_heads`: every query and key head is normed before its turn (RMS, with weights of its own)."""
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
        self.w_q, self.w_k = (1 + 0.1 * torch.randn(dim, generator=g, device=g.device) if norm_heads else None for _ in "qk")

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

    def _project(self, y, x):
        """The heads' rows [tokens, heads, dim] of q, k and v, and the stream."""
        codes, sx, x = self._here().add_norm_quantized(y, self.w_in, EPS, residual=x)
        qkv = self.ctx.product_f8(codes, sx, *self.qkv).view(-1, self.heads + 2 * self.kv_heads, self.dim)
        return *qkv.split([self.heads, self.kv_heads, self.kv_heads], 1), x

    def _append(self, y, x, cache, positions, slots, table):
        """The layer up to its attention: the turned q [tokens, heads, dim] and the stream."""
        q, k, v, x = self._project(y, x)
        if self.w_q is None:
            return self.ctx.append_kv(q, k, v, cache, positions, slots, table, q_out=q), x
        return self.ctx.norm_append_kv(q, k, v, cache, positions, slots, table, q_norm=self.w_q, k_norm=self.w_k, eps=EPS, q_out=q), x

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

    def chunk(self, y, x, cache, positions, slots, pages, lengths, starts, table):
        """New tokens of each sequence, sequence b's in rows starts[b] to starts[b + 1] − 1 (int32 [batch + 1]) of y and x
        [tokens, d]; each token's position and cache slot, and the sequences' pages and lengths with these tokens as step's."""
        q, x = self._append(y, x, cache, positions, slots, table)
        return self._finish(self.ctx.chunk_attention(q, cache, pages, lengths, starts), x)

    def encode(self, y, x, positions, starts, table, causal: bool = True):
        """Whole prompts packed in rows as chunk's, over their own keys and values: nothing is kept."""
        q, k, v, x = self._project(y, x)
        self.ctx.norm_rotate(q, k, positions, table, q_norm=self.w_q, k_norm=self.w_k, eps=EPS, q_out=q, k_out=k)
        return self._finish(self.ctx.prompt_attention(q, k, v, starts, causal=causal), x)

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


class TextHead:
    """What follows the last layer: its branch added, the norm, logits over a vocabulary and the draw of the next tokens."""

    def __init__(self, d: int = 4096, vocab: int = 128000, seed: int = 0, device: int = 0, ctx: TensorGEMM | None = None):
        self.ctx = ctx or context(device)
        g = torch.Generator(device=f"cuda:{device}").manual_seed(seed)
        self.weight = quantize_f8_blocks(torch.randn(vocab, d, generator=g, device=g.device) * d ** -0.5)
        self.w_norm = 1 + 0.1 * torch.randn(d, generator=g, device=g.device)

    def logits(self, y, x):
        """[rows, vocab] in bf16, of a last layer's (y, x)."""
        self.ctx.set_stream(torch.cuda.current_stream(self.ctx.device))
        codes, sx, x = self.ctx.add_norm_quantized(y, self.w_norm, EPS, residual=x)
        return self.ctx.product_f8(codes, sx, *self.weight)

    def draw(self, y, x, uniform, **options):
        """The rows' next tokens and their log probabilities: sample_tokens' `uniform` and options."""
        return self.ctx.sample_tokens(self.logits(y, x), uniform, **options)


def main() -> None:
    import argparse
    import time

    a = argparse.ArgumentParser(description="times a decode step")
    a.add_argument("--layers", type=int, default=4)
    a.add_argument("--batch", type=int, default=16)
    a.add_argument("--context", type=int, default=2000)
    a.add_argument("--steps", type=int, default=50)
    a.add_argument("--page", type=int, default=64)
    a.add_argument("--new", type=int, default=1, help="tokens of each sequence a step")
    a.add_argument("--vocab", type=int, default=0, help="logits a sequence, and the draw of its next token from the nucleus of 0.9")
    a = a.parse_args()
    if not 1 <= a.new <= a.context:
        raise SystemExit("--new: at least one token, and no more than --context")
    most = -(-a.context // a.page)
    layers = [TextBlock(seed=i) for i in range(a.layers)]
    caches = [block.cache(a.batch * most, a.page) for block in layers]
    d, dev = layers[0].d, layers[0].w_in.device
    i32 = dict(dtype=torch.int32, device=dev)
    pages = torch.randperm(a.batch * most, device=dev).to(torch.int32).view(a.batch, most)
    lengths = torch.full((a.batch,), a.context, **i32)
    starts = torch.arange(a.batch + 1, **i32) * a.new
    place = torch.arange(a.context - a.new, a.context, **i32)  # of a sequence's new tokens
    positions = place.repeat(a.batch)
    slots = (pages[:, (place // a.page).long()] * a.page + place % a.page).flatten().contiguous()
    table = rotation_table(a.context, layers[0].dim)
    token = torch.randn(a.batch * a.new, d, device=dev).to(torch.bfloat16)
    stream = torch.zeros(a.batch * a.new, d, device=dev)
    head = TextHead(d, a.vocab) if a.vocab else None
    uniform, top_p = torch.rand(a.batch, device=dev), torch.full((a.batch,), 0.9, device=dev)
    newest = (starts[1:] - 1).long()

    def run():
        y, x = token, stream.zero_()
        for block, cache in zip(layers, caches):
            if a.new == 1:
                y, x = block.step(y, x, cache, positions, slots, pages, lengths, table)
            else:
                y, x = block.chunk(y, x, cache, positions, slots, pages, lengths, starts, table)
        if head:
            head.draw(y[newest], x[newest], uniform, top_p=top_p)
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
    what = (f", {a.new} new tokens each" if a.new > 1 else "") + (f", the next of {a.vocab}" if a.vocab else "")
    print(f"{a.layers} layers, {a.batch} sequences of {a.context} tokens{what}: {calls:.0f} us a step as calls, "
          f"{replays:.0f} us as a graph ({replays / a.layers:.1f} a layer), {a.batch * a.new / replays * 1e6:.0f} tokens/s")


if __name__ == "__main__":
    main()
