"""The operators of prompts, chunks and drawn tokens together, as a decoder uses them: a layer's `chunk` and `encode`, the head
that draws, on torch's current stream, as calls and in graphs, and beside each other on the layer's own context.

Each operator's outputs inside a layer are compared with the formula in 64 bits on the inputs that it was given, which have to be
the outputs of the stage before, so no rounding of one stage hides a fault of a later one (attend_reference.py says where the
attention's tolerances come from). A head normed and turned and rounded to bf16 once is within 2^-8 of each value, with fp32's
sums of 64 squares and products, 2^-17 of the pair's size; in e4m3 within 2^-4 of it or 2^-10 of its scale."""
import ctypes
import sys

import pytest
import torch

import siliconed_amd as sq
from attend_reference import attended, within
from siliconed_amd import _abi as abi
from siliconed_amd import text_block as tb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F8 = torch.bfloat16, torch.float8_e4m3fn
NOTED = ("append_kv", "norm_append_kv", "norm_rotate", "prompt_attention", "chunk_attention", "product_f8", "product_f8_quantized")


class Noted:
    """A context whose calls of the names above are noted: (name, arguments, keywords, outputs), tensors as they were."""

    def __init__(self, ctx):
        self.ctx, self.calls, self.device = ctx, [], ctx.device

    def __getattr__(self, name):
        method = getattr(self.ctx, name)
        if name not in NOTED:
            return method

        def copy(v):
            return v.clone() if isinstance(v, torch.Tensor) else tuple(map(copy, v)) if isinstance(v, tuple) else v

        def call(*a, **kw):
            before = tuple(map(copy, a)), {k: copy(v) for k, v in kw.items()}
            found = method(*a, **kw)
            self.calls.append((name, *before, copy(found)))
            return found
        return call

    def take(self, name):
        return next(c for c in self.calls if c[0] == name)[1:]


def turned(x, w, positions, table, eps):
    """RMS(x) · w turned by the positions' angles, 64 bits, and the size that errors are relative to."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = x.shape[-1] // 2
    cos, sin = (t[positions.long()].double()[:, None] for t in table.split(half, 1))
    a, b = x[..., :half], x[..., half:]
    size = (a.abs() + b.abs()).repeat(1, 1, 2)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1), size


def near(got, want, size, what):
    within(got, want, want.abs() * 2.0 ** -8 + size * 2.0 ** -17 + 1e-30, what)


class Batch:
    """Sequences of (new, held) tokens in pages of 16 in a random order."""

    def __init__(self, block, chunks, dtype, seed=1):
        g = torch.Generator(device=DEV).manual_seed(seed)
        most = -(-max(m for _, m in chunks) // 16)
        i32 = dict(dtype=torch.int32, device=DEV)
        self.chunks = chunks
        self.pages = torch.randperm(len(chunks) * most, generator=g, device=DEV).to(torch.int32).view(len(chunks), most)
        self.cache = block.cache(len(chunks) * most, 16, dtype)
        self.lengths = torch.tensor([m for _, m in chunks], **i32)
        self.starts = torch.tensor([sum(n for n, _ in chunks[:i]) for i in range(len(chunks) + 1)], **i32)
        self.positions = torch.cat([torch.arange(m - n, m, **i32) for n, m in chunks])
        of = torch.cat([torch.full((n,), b, device=DEV) for b, (n, _) in enumerate(chunks)])
        self.slots = self.pages[of, (self.positions // 16).long()] * 16 + self.positions % 16
        self.table = tb.rotation_table(most * 16, block.dim)
        self.y = torch.randn(len(of), block.d, generator=g, device=DEV).to(BF)
        self.x = torch.randn(len(of), block.d, generator=g, device=DEV)

    def held(self, b, scale_of):
        """What the cache holds for sequence b: k, v [held, kv heads, dim]."""
        m = self.chunks[b][1]
        found = []
        for pool, scale in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            t = pool[self.pages[b].long()].flatten(0, 1)[:m].float()
            found.append(t if scale is None else t * scale[:, None])
        return found

    def fill(self, seed=3):
        """The tokens that were there before."""
        g = torch.Generator(device=DEV).manual_seed(seed)
        for pool, scale in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            t = torch.randn(pool.shape, generator=g, device=DEV)
            pool.copy_((t if scale is None else t / scale[:, None]).to(pool.dtype))

    def run(self, block):
        return block.chunk(self.y, self.x.clone(), self.cache, self.positions, self.slots, self.pages, self.lengths, self.starts, self.table)


@pytest.fixture(scope="module")
def ctx():
    c = sq.TensorGEMM.make(0)
    yield c
    torch.cuda.synchronize()
    c.close()


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("normed", [False, True], ids=["plain", "normed"])
@pytest.mark.parametrize("chunks", [[(1, 1), (3, 40), (70, 70), (20, 150)], [(1, 90), (1, 17)], [(200, 300), (4, 9)]])
def test_a_layer_s_chunk(ctx, chunks, normed, dtype):
    noted = Noted(ctx)
    block = tb.TextBlock(256, 8, 2, 64, 384, seed=6, ctx=noted, norm_heads=normed)
    b = Batch(block, chunks, dtype)
    b.fill()
    before = b.cache.k.float().clone(), b.cache.v.float().clone()
    y, x = b.run(block)
    rows = noted.take("product_f8")[2].view(-1, 12, 64)
    a, kw, q = noted.take("norm_append_kv" if normed else "append_kv")
    assert all(torch.equal(p, r) for p, r in zip(a[:3], rows.split([8, 2, 2], 1)))
    near(q, *turned(rows[:, :8], block.w_q, b.positions, b.table, tb.EPS), "q")
    # The cache: the new tokens' slots, and nothing else.
    want_k, size = turned(rows[:, 8:10], block.w_k, b.positions, b.table, tb.EPS)
    page, place = (b.slots // 16).long(), (b.slots % 16).long()
    for pool, want, size, old, scale in ((b.cache.k, want_k, size, before[0], b.cache.k_scale),
                                         (b.cache.v, rows[:, 10:].double(), rows[:, 10:].double().abs(), before[1], b.cache.v_scale)):
        got = pool[page, place].double()
        if scale is None:
            near(got, want, size, "the cache")
        else:
            got = got * scale.double()[:, None]
            step = torch.maximum(want.abs() * 2.0 ** -4, scale.double()[:, None] * 2.0 ** -10)
            within(got, want.clamp(-448 * float(scale[0]), 448 * float(scale[0])), step * (1 + 2.0 ** -8) + size * 2.0 ** -17, "the cache")
        rest = pool.float().clone()
        rest[page, place] = old[page, place]
        assert torch.equal(rest, old)
    a, kw, o = noted.take("chunk_attention")
    assert torch.equal(a[0], q)
    for i, (n, m) in enumerate(chunks):
        lo = int(b.starts[i])
        want, tol = attended(q[lo:lo + n], *b.held(i, dtype), m - n)
        within(o[lo:lo + n], want, tol, f"sequence {i}")
    assert torch.equal(noted.take("product_f8_quantized")[0][0], o.flatten(1))
    assert torch.isfinite(y.float()).all() and torch.isfinite(x).all()


@pytest.mark.parametrize("normed", [False, True], ids=["plain", "normed"])
@pytest.mark.parametrize("causal", [True, False])
def test_a_layer_s_packed_prompts(ctx, normed, causal):
    noted = Noted(ctx)
    block = tb.TextBlock(256, 4, 4, 64, 384, seed=7, ctx=noted, norm_heads=normed)
    b = Batch(block, [(33, 33), (1, 1), (0, 0), (200, 200)], BF)
    y, x = block.encode(b.y, b.x.clone(), b.positions, b.starts, b.table, causal=causal)
    rows = noted.take("product_f8")[2].view(-1, 12, 64)
    _, _, (q, k) = noted.take("norm_rotate")
    near(q, *turned(rows[:, :4], block.w_q, b.positions, b.table, tb.EPS), "q")
    near(k, *turned(rows[:, 4:8], block.w_k, b.positions, b.table, tb.EPS), "k")
    a, kw, o = noted.take("prompt_attention")
    assert torch.equal(a[0], q) and torch.equal(a[1], k) and torch.equal(a[2], rows[:, 8:])
    for i, (n, _) in enumerate(b.chunks):
        lo = int(b.starts[i])
        want, tol = attended(q[lo:lo + n], k[lo:lo + n], rows[lo:lo + n, 8:], 0, causal=causal)
        within(o[lo:lo + n], want, tol, f"prompt {i}")
    assert torch.isfinite(y.float()).all() and torch.isfinite(x).all()


def test_the_head_draws_from_its_logits(ctx):
    head = tb.TextHead(256, 5000, seed=2, ctx=ctx)
    g = torch.Generator(device=DEV).manual_seed(4)
    y, x = torch.randn(6, 256, generator=g, device=DEV).to(BF), torch.randn(6, 256, generator=g, device=DEV)
    u = torch.rand(6, generator=g, device=DEV)
    logits = head.logits(y, x.clone())
    assert logits.shape == (6, 5000) and logits.dtype == BF
    w = tb.widen_f8_blocks(*head.weight)
    s = x.double() + y.double()
    want = (s / (s.square().mean(1, keepdim=True) + tb.EPS).sqrt() * head.w_norm.double()) @ w.T
    # The operand's codes are within 2^-4 of each value: independent errors, far under 2^-4 of the whole in norm.
    assert ((logits.double() - want).norm() / want.norm()).item() <= 2.0 ** -4
    tokens, logprobs = head.draw(y, x.clone(), u, top_k=torch.full((6,), 40, dtype=torch.int32, device=DEV))
    again = ctx.sample_tokens(logits, u, top_k=torch.full((6,), 40, dtype=torch.int32, device=DEV))
    assert torch.equal(tokens, again[0]) and torch.equal(logprobs, again[1])
    top = logits.double().topk(40, 1).values
    assert (logits.double().gather(1, tokens.long()[:, None]) >= top[:, -1:]).all()
    greedy = head.draw(y, x.clone(), u, temperature=torch.zeros(6, device=DEV))[0]
    assert torch.equal(greedy.long(), logits.float().argmax(1)) and (logprobs < 0).all()


def test_a_decoder_s_graphs(ctx):
    """Two layers and the head in one graph, drafts of other lengths and other numbers at every replay, calls of the same context in
    between, bit for bit what the calls give. A second graph, of packed prompts, shares the context's scratch and counters."""
    layers = [tb.TextBlock(256, 8, 2, 64, 384, seed=i, ctx=ctx, norm_heads=True) for i in range(2)]
    head = tb.TextHead(256, 3000, ctx=ctx)
    b = Batch(layers[0], [(4, 900), (4, 64), (4, 333)], F8)
    caches = [Batch(layers[0], b.chunks, F8, seed=s).cache for s in (5, 6)]
    p = Batch(layers[0], [(70, 70), (200, 200), (5, 5)], BF)
    uniform, last = torch.rand(3, device=DEV), (b.starts[1:] - 1).long()
    tokens, logprobs = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(3, device=DEV)
    lengths, positions, slots = b.lengths.clone(), b.positions.clone(), b.slots.clone()
    x, xp = b.x.clone(), p.x.clone()

    def decode():
        y, s = b.y, x.copy_(b.x)
        for block, cache in zip(layers, caches):
            y, s = block.chunk(y, s, cache, positions, slots, b.pages, lengths, b.starts, b.table)
        head.draw(y[last], s[last], uniform, top_p=None, tokens=tokens, logprobs=logprobs)
        return y

    def encode():
        y, s = p.y, xp.copy_(p.x)
        for block in layers:
            y, s = block.encode(y, s, p.positions, p.starts, p.table)
        return y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode(), encode()
        side.synchronize()
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        outs = []
        for graph, f in zip(graphs, (decode, encode)):
            with torch.cuda.graph(graph, stream=side):
                outs.append(f())
        for i in range(5):
            back = torch.tensor([100 * i, 10 * i, 60 * i], dtype=torch.int32, device=DEV)
            lengths.copy_(b.lengths - back)
            positions.copy_(b.positions - back.repeat_interleave(4))
            of = torch.arange(3, device=DEV).repeat_interleave(4)
            slots.copy_(b.pages[of, (positions // 16).long()] * 16 + positions % 16)
            uniform.copy_(torch.rand(3, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV))
            for graph in graphs:
                graph.replay()
            side.synchronize()
            got = [outs[0].clone(), outs[1].clone(), tokens.clone(), logprobs.clone()]
            want = [decode(), encode(), tokens, logprobs]
            side.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(got, want)), i
    torch.cuda.current_stream().wait_stream(side)
    ctx.set_stream(torch.cuda.default_stream())


def test_layers_follow_torch_s_current_stream(ctx):
    block = tb.TextBlock(256, 8, 2, 64, 384, seed=6, ctx=ctx, norm_heads=True)
    head = tb.TextHead(256, 3000, ctx=ctx)
    u = torch.rand(83, device=DEV)

    def run():
        b = Batch(block, [(3, 40), (60, 70), (20, 150)], F8)
        y, x = b.run(block)
        return [y, x, *block.encode(b.y, b.x.clone(), b.positions, b.starts, b.table), *head.draw(y, x, u)]

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert all(torch.equal(a, c) for a, c in zip(run(), want))
    torch.cuda.synchronize()


def test_two_contexts_at_once(ctx):
    """Two contexts on two streams, each with scratch and counters of its own, their calls interleaved."""
    other = sq.TensorGEMM.make(0)
    g = torch.Generator(device=DEV).manual_seed(8)
    sides = [torch.cuda.Stream() for _ in range(2)]
    blocks = [tb.TextBlock(256, 8, 2, 64, 384, seed=6, ctx=c) for c in (ctx, other)]
    batches = [Batch(b, [(4, 900), (4, 64), (4, 333)], BF, seed=i) for i, b in enumerate(blocks)]
    for b in batches:
        b.fill()
    q = [torch.randn(12, 8, 64, generator=g, device=DEV).to(BF) for _ in range(2)]
    logits, u = torch.randn(12, 4000, generator=g, device=DEV), torch.rand(12, generator=g, device=DEV)

    def calls(i):
        c, b = blocks[i]._here(), batches[i]
        return [c.chunk_attention(q[i], b.cache, b.pages, b.lengths, b.starts), *c.sample_tokens(logits, u)]

    want = [calls(i) for i in range(2)]
    torch.cuda.synchronize()
    found = []
    for _ in range(20):
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                found.append((i, calls(i)))
    torch.cuda.synchronize()
    for i, got in found:
        assert all(torch.equal(a, c) for a, c in zip(got, want[i]))
    ctx.set_stream(torch.cuda.default_stream())
    other.close()


def test_the_command(monkeypatch, capsys):
    for more in ([], ["--new", "3", "--vocab", "1000"]):
        monkeypatch.setattr(sys, "argv", ["text_block", "--layers", "1", "--batch", "2", "--context", "100", "--steps", "2", *more])
        tb.main()
        said = capsys.readouterr().out
        assert "2 sequences of 100 tokens" in said and ("3 new tokens each" in said) == bool(more)
    monkeypatch.setattr(sys, "argv", ["text_block", "--context", "3", "--new", "4"])
    with pytest.raises(SystemExit):
        tb.main()


@pytest.mark.parametrize("S,d,heads,route", [(256, 384, 3, "bf16"), (300, 256, 2, "w8a8")])
def test_an_image_block_on_this_library_s_attention(S, d, heads, route):
    """The bar of the block with torch's attention: the update within 2e-2 of the fp32 block's."""
    from dit_reference import reference
    from siliconed_amd.dit_block import DiTBlock
    blk = DiTBlock(d=d, heads=heads, mlp=4, seed=S, keep_codes=True, route=route, group=64 if route == "w8a8" else 0, attend="own")
    g = torch.Generator(device=DEV).manual_seed(1)
    x, temb = torch.randn((S, d), device=DEV, generator=g), torch.randn(d, device=DEV, generator=g)
    y, ref = blk.forward(x, temb), reference(blk, x, temb)
    rel = float((y - ref).norm() / (ref - x).norm())
    assert torch.isfinite(y).all() and rel <= 2e-2, rel
    with pytest.raises(ValueError):
        DiTBlock(d=d, heads=heads, attend="other")


def test_tensors_on_another_gpu_are_refused(gemm):
    """There is one GPU here: the entries are replaced by stand-ins that say the context is on another and note what is reached."""
    lib, reached, kept = abi.load(), [], []

    def stand_in(name):
        restype, argtypes = abi.SIGNATURES[name]

        def entry(*_):
            if name == "sq8_device":
                return 1
            reached.append(name)
            return abi.EINVAL
        kept.append(ctypes.CFUNCTYPE(restype, *argtypes)(entry))
        return ctypes.cast(kept[-1], ctypes.c_void_p).value

    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    cache = sq.PagedCache(z(2, 16, 2, 64), z(2, 16, 2, 64))
    abi.text.bind(*(stand_in(name) for name in abi.TEXT_ENTRIES))
    try:
        for call in (lambda: gemm.norm_append_kv(z(3, 4, 64), z(3, 2, 64), z(3, 2, 64), cache, i32(3), i32(3), f32(9, 64), q_norm=f32(64)),
                     lambda: gemm.norm_rotate(z(3, 4, 64), z(3, 2, 64), i32(3), f32(9, 64)),
                     lambda: gemm.prompt_attention(z(3, 4, 64), z(3, 2, 64), z(3, 2, 64)),
                     lambda: gemm.chunk_attention(z(3, 4, 64), cache, i32(1, 2), i32(1)),
                     lambda: gemm.sample_tokens(f32(3, 100), f32(3))):
            with pytest.raises(ValueError, match="context's GPU"):
                call()
        assert not reached
    finally:
        abi.text.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in abi.TEXT_ENTRIES))
