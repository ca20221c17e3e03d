"""A decoder layer stage by stage: each operator's call inside a step and a prompt is noted, and its outputs are compared with the
formula in 64 bits on the inputs that it was given, which have to be the outputs of the stages before. So no rounding
of one stage hides a fault of a later one.

Bounds, relative and in norm: a bf16 output is rounded by 2^-8 of each value at most, besides what fp32 sums and the e4m3
instructions leave out, 2^-13 with room; torch's attention of a prompt also rounds its probabilities to bf16, which is taken
as another 2^-7 of the output. An e4m3 code is within 2^-4 of its value, or 2^-10 of its scale, elementwise.
"""
import pytest
import torch

import siliconed_amd as sq

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
ROUNDED = 2.0 ** -8 + 2.0 ** -13


class Noted:
    """A context whose text operators' calls are noted: (name, arguments, keywords, outputs), tensors as they were."""

    def __init__(self, ctx):
        self.ctx, self.calls, self.device = ctx, [], ctx.device

    def __getattr__(self, name):
        method = getattr(self.ctx, name)
        if name not in ("add_norm_quantized", "product_f8", "product_f8_quantized", "append_kv", "paged_attention"):
            return method

        def copy(v):
            return v.clone() if isinstance(v, torch.Tensor) else v

        def call(*a, **kw):
            before = [copy(v) for v in a], {k: copy(v) for k, v in kw.items()}
            found = method(*a, **kw)
            self.calls.append((name, *before, tuple(map(copy, found)) if isinstance(found, tuple) else copy(found)))
            return found
        return call


def close(got, want, bound=ROUNDED):
    got, want = got.double(), want.double()
    error = ((got - want).norm() / want.norm()).item()
    assert error <= bound, error


def coded(got, want, scale):
    """got, what e4m3 codes stand for, is want rounded to them."""
    step = torch.maximum(want.abs() * 2.0 ** -4, scale.double() * 2.0 ** -10)
    assert ((got.double() - want).abs() <= step * (1 + 2.0 ** -10)).all()


def widened(codes, sx):
    return codes.double() * sx.double().repeat_interleave(128, 1)[:, :codes.shape[1]]


class Layer:
    """The noted calls of a layer, in turn, against the formula of each."""

    def __init__(self, block, calls):
        from siliconed_amd import text_block as tb
        self.tb, self.block, self.calls = tb, block, iter(calls)

    def next(self, name):
        found = next(self.calls)
        assert found[0] == name
        return found[1:]

    def norm(self, y, x, weight):
        """The branch y and the stream x come in; the stream and the codes go out."""
        (got_y, w, eps), kw, (codes, sx, stream) = self.next("add_norm_quantized")
        assert torch.equal(got_y, y) and torch.equal(kw["residual"], x) and torch.equal(w, weight) and eps == self.tb.EPS
        s = x.double() + y.double()
        close(stream, s, 2.0 ** -23)
        want = s / (s.square().mean(1, keepdim=True) + eps).sqrt() * weight.double()
        coded(widened(codes, sx), want, sx.repeat_interleave(128, 1)[:, :want.shape[1]])
        return codes, sx, stream

    def product(self, codes, sx, weight, glu=False):
        (a, s, *w), kw, out = self.next("product_f8")
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip((a, s, *w), (codes, sx, *weight)))
        assert kw == ({"epilogue": "silu_glu"} if glu else {})
        want = widened(codes, sx) @ self.tb.widen_f8_blocks(*weight, glu=glu).T
        if glu:
            g, u = want.chunk(2, 1)
            want = torch.nn.functional.silu(g) * u
        close(out, want)
        return out

    def product_of_values(self, x, weight):
        (got, *w), kw, out = self.next("product_f8_quantized")
        assert torch.equal(got, x) and not kw
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(w, weight))
        codes, sx = self.block.ctx.ctx.quantize_groups(x)
        coded(widened(codes, sx), x.double(), sx.repeat_interleave(128, 1)[:, :x.shape[1]])
        close(out, widened(codes, sx) @ self.tb.widen_f8_blocks(*weight).T)
        return out

    def append(self, qkv, cache, positions, slots, table):
        """The turned q, and the tokens' keys and values as the pools hold them."""
        (q, k, v, got_cache, *where), _, out = self.next("append_kv")
        assert got_cache is cache and all(torch.equal(a, b) for a, b in zip(where, (positions, slots, table)))
        b = self.block
        parts = qkv.view(len(qkv), -1, b.dim).split([b.heads, b.kv_heads, b.kv_heads], 1)
        assert all(torch.equal(a, p) for a, p in zip((q, k, v), parts))
        c, s = (t[:, None].double() for t in table[positions.long()].chunk(2, 1))

        def turned(t):
            x, y = t.double().chunk(2, 2)
            return torch.cat([x * c - y * s, y * c + x * s], 2)

        close(out, turned(q))
        for pool, scale, want in ((cache.k, cache.k_scale, turned(k)), (cache.v, cache.v_scale, v.double())):
            held = pool.view(torch.uint8).flatten(0, 1)[slots.long()].view(pool.dtype).double()
            if scale is None:
                close(held, want)
            else:
                coded(held * scale.double()[:, None], want, scale[:, None])
        return out

    def attention(self, q, cache, pages, length):
        """One query at the end of a sequence."""
        t = torch.arange(length, device=DEV)
        k, v = (pool.view(torch.uint8)[pages[t // cache.page].long(), t % cache.page].view(pool.dtype).double() for pool in (cache.k, cache.v))
        if cache.k_scale is not None:
            k, v = k * cache.k_scale.double()[:, None], v * cache.v_scale.double()[:, None]
        k, v = (x.repeat_interleave(self.block.heads // self.block.kv_heads, 1) for x in (k, v))
        p = torch.softmax((k * q.double()).sum(2) * self.block.dim ** -0.5, 0)
        return (p[..., None] * v).sum(0)

    def rest(self, o, x):
        y = self.product_of_values(o, self.block.out)
        codes, sx, x = self.norm(y, x, self.block.w_post)
        return self.product_of_values(self.product(codes, sx, self.block.gate_up, glu=True), self.block.down), x


@pytest.mark.parametrize("dtype", [F8, torch.bfloat16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("sizes", [(512, 8, 2, 64, 640), (1024, 8, 4, 128, 1536), (384, 3, 3, 128, 200)])
def test_every_stage_of_a_layer(dtype, sizes):
    from siliconed_amd import text_block as tb
    block = tb.TextBlock(*sizes, seed=7, ctx=Noted(sq.context(0)))
    lengths, page, most = [90, 1, 200], 16, 13
    g = torch.Generator().manual_seed(2)
    pages = torch.randperm(len(lengths) * most, generator=g).to(torch.int32).view(len(lengths), most).to(DEV)
    cache = block.cache(pages.numel(), page, dtype)
    table = tb.rotation_table(210, block.dim)
    torch.manual_seed(12)

    def started(rows):
        return torch.randn(rows, block.d, device=DEV).to(torch.bfloat16), torch.randn(rows, block.d, device=DEV)

    def slots(i, start, stop):
        t = torch.arange(start, stop, device=DEV)
        return (pages[i, t // page] * page + t % page).to(torch.int32)

    for i, n in enumerate(lengths):
        y, x = started(n)
        at, to = torch.arange(n, dtype=torch.int32, device=DEV), slots(i, 0, n)
        block.ctx.calls.clear()
        out = block.prompt(y, x.clone(), cache, at, to, pages[i], table)
        layer = Layer(block, block.ctx.calls)
        codes, sx, x = layer.norm(y, x, block.w_in)
        q = layer.append(layer.product(codes, sx, block.qkv), cache, at, to, table)
        o = block.ctx.calls[3][1][0]  # torch's attention: what the next product was given
        close(o, torch.stack([layer.attention(q[t], cache, pages[i], t + 1) for t in range(n)]).flatten(1), ROUNDED + 2.0 ** -7)
        y, x = layer.rest(o, x)
        assert torch.equal(out[0], y) and torch.equal(out[1], x) and next(layer.calls, None) is None
    for t in range(2):
        y, x = started(len(lengths))
        now = torch.tensor([n + t for n in lengths], dtype=torch.int32, device=DEV)
        to = torch.cat([slots(i, n + t, n + t + 1) for i, n in enumerate(lengths)])
        block.ctx.calls.clear()
        out = block.step(y, x.clone(), cache, now, to, pages, now + 1, table)
        layer = Layer(block, block.ctx.calls)
        codes, sx, x = layer.norm(y, x, block.w_in)
        q = layer.append(layer.product(codes, sx, block.qkv), cache, now, to, table)
        (got_q, got_cache, got_pages, got_lengths), kw, o = layer.next("paged_attention")
        assert torch.equal(got_q, q) and got_cache is cache and not kw
        assert torch.equal(got_pages, pages) and torch.equal(got_lengths, now + 1)
        close(o, torch.stack([layer.attention(q[i], cache, pages[i], n + t + 1) for i, n in enumerate(lengths)]))
        y, x = layer.rest(o.flatten(1), x)
        assert torch.equal(out[0], y) and torch.equal(out[1], x) and next(layer.calls, None) is None
