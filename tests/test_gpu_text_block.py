"""A decoder layer run on the text operators together, against the layer's formula in 64 bits on the same weights.

The formula takes the activations as they are; the layer rounds four products' operands to e4m3, whose relative error
is 2.55 % root mean square (a uniform error within ± 2^-4 of the binade, over a mantissa of 1 to 2). On normal operands
a product's output carries its operand's relative error. The attention's branch carries it three times over (the values',
3.6 % from both sides of the scores, the output's), 5.1 % in all; the MLP's carries its operand's error in gate and up
(√2 · 2.55 % and the slope of SiLU, under 1.1), and the hidden values', 4.7 %, besides what the attention's share of
its input carried (under 5.1 %). An e4m3 cache adds 2.55 % to the keys and to the values each. So what the layer adds
to the stream is within 10 % of the formula's in norm; a wrong wire is off by its whole size.
"""
import pytest
import torch

import siliconed_amd as sq

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOUND = 0.10


def text_block():
    from siliconed_amd import text_block as tb
    return tb


def formula(block, streams, table):
    """The layer in 64 bits on whole sequences (a list of [tokens, d]): what it adds to each stream."""
    tb = text_block()
    qkv, out, down = (tb.widen_f8_blocks(*w) for w in (block.qkv, block.out, block.down))
    gate_up = tb.widen_f8_blocks(*block.gate_up, glu=True)
    half, dim, heads, kv = block.dim // 2, block.dim, block.heads, block.kv_heads

    def norm(x, w):
        return x * (x.square().mean(1, keepdim=True) + tb.EPS).rsqrt() * w.double()

    def turn(t):
        c, s = table[:len(t), None, :half].double(), table[:len(t), None, half:].double()
        return torch.cat([t[..., :half] * c - t[..., half:] * s, t[..., half:] * c + t[..., :half] * s], -1)

    added = []
    for x in streams:
        x = x.double()
        n = len(x)
        q, k, v = (norm(x, block.w_in) @ qkv.T).view(n, heads + 2 * kv, dim).split([heads, kv, kv], 1)
        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(heads // kv, 1) for t in (k, v))
        ahead = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
        o = torch.empty(n, heads, dim, dtype=torch.float64, device=x.device)
        for h in range(heads):
            p = (q[:, h] @ k[:, h].T * dim ** -0.5).masked_fill(ahead, -torch.inf).softmax(1)
            o[:, h] = p @ v[:, h]
        attention = o.flatten(1) @ out.T
        g, u = (norm(x + attention, block.w_post) @ gate_up.T).chunk(2, 1)
        added.append(attention + (torch.nn.functional.silu(g) * u) @ down.T)
    return added


def layout(lengths, page, most):
    """Pages for the sequences, scattered: [sequences, most]."""
    g = torch.Generator().manual_seed(5)
    return torch.randperm(len(lengths) * most, generator=g).to(torch.int32).view(len(lengths), most).to(DEV)


def slots_of(pages, page, start, stop):
    t = torch.arange(start, stop, device=DEV)
    return (pages[t // page] * page + t % page).to(torch.int32)


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.bfloat16])
@pytest.mark.parametrize("sizes", [(512, 8, 2, 64, 640), (384, 3, 3, 128, 200)])
def test_prompts_then_steps_follow_the_formula(dtype, sizes):
    tb = text_block()
    d, heads, kv, dim, hidden = sizes
    block = tb.TextBlock(d, heads, kv, dim, hidden, seed=3)
    lengths, more, page, most = [37, 1, 64], 3, 16, 6
    pages = layout(lengths, page, most)
    cache = block.cache(pages.numel(), page, dtype)
    table = tb.rotation_table(80, dim)
    torch.manual_seed(11)
    streams = [torch.randn(n + more, d, device=DEV).to(torch.bfloat16) for n in lengths]
    want = formula(block, streams, table)

    def started(y):
        return y, torch.zeros(y.shape, device=DEV)

    for i, n in enumerate(lengths):
        at = torch.arange(n, dtype=torch.int32, device=DEV)
        y, x = block.prompt(*started(streams[i][:n]), cache, at, slots_of(pages[i], page, 0, n), pages[i], table)
        assert off(x + y - streams[i][:n], want[i][:n]) < BOUND
    for t in range(more):
        now = torch.tensor([n + t for n in lengths], dtype=torch.int32, device=DEV)
        token = torch.stack([s[n + t] for s, n in zip(streams, lengths)])
        slots = torch.cat([slots_of(pages[i], page, n + t, n + t + 1) for i, n in enumerate(lengths)])
        y, x = block.step(*started(token), cache, now, slots, pages, now + 1, table)
        assert off(x + y - token, torch.stack([w[n + t] for w, n in zip(want, lengths)])) < BOUND


def test_a_graph_s_steps_are_the_calls():
    """Replays over new tokens, with calls in between, give what the calls give, bit for bit."""
    tb = text_block()
    ctx = sq.TensorGEMM.make(0)
    block = tb.TextBlock(512, 8, 2, 64, 640, seed=4, ctx=ctx)
    batch, page, most = 5, 16, 4
    pages = layout([0] * batch, page, most)
    caches = [block.cache(pages.numel(), page) for _ in range(2)]
    table = tb.rotation_table(64, 64)
    token = torch.zeros(batch, 512, dtype=torch.bfloat16, device=DEV)
    stream = torch.zeros(batch, 512, device=DEV)
    now = torch.zeros(batch, dtype=torch.int32, device=DEV)
    slots, lengths = torch.zeros_like(now), torch.zeros_like(now)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.set_stream(side)
        block.step(token, stream, caches[0], now, slots, pages, lengths, table)  # buffers at their sizes
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y, x = block.step(token, stream.zero_(), caches[0], now, slots, pages, lengths, table)
        for t in range(40):
            token.copy_(torch.randn(batch, 512, device=DEV))
            now.fill_(t)
            lengths.fill_(t + 1)
            slots.copy_(pages[:, t // page] * page + t % page)
            graph.replay()
            side.synchronize()
            y2, x2 = block.step(token, torch.zeros_like(stream), caches[1], now, slots, pages, lengths, table)
            side.synchronize()
            assert torch.equal(y, y2) and torch.equal(x, x2), t
        ctx.set_stream(torch.cuda.default_stream())
    torch.cuda.current_stream().wait_stream(side)
