"""Heads normed and turned in one pass, into a paged cache or beside them, against the formula in 64 bits.

Tolerances: a bf16 output is rounded by 2^-8 of itself at most. Before it, fp32: the sum of squares of up to 512 values
(under 40 roundings of positive terms), its mean, root and reciprocal and two products move y by less than 50 · 2^-24 of it, a turn
of (a, b) adds three roundings of |a cos| + |b sin|: 60 · 2^-24 of the pair's size in all. An e4m3 code is within max(2^-4 of its
value, 2^-10) of the value over the scale."""
import math

import pytest
import torch

import siliconed_amd as sq
from siliconed_amd import _abi as abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F8 = torch.bfloat16, torch.float8_e4m3fn
FINE = 60 * 2.0 ** -24


def normal(g, *shape):
    return torch.randn(*shape, generator=g).to(DEV)


def formula(x, w, table, positions, eps, interleaved):
    """(turned values, the size of each value's pair) in 64 bits."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(2, keepdim=True) + eps).sqrt() * w.double()
    size = y.abs()
    if table is None or not table.shape[1]:
        return y, size
    rot = table.shape[1]
    c, s = table[positions.long().clamp(max=len(table) - 1)].double()[:, None].chunk(2, 2)
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    pair = a.abs() + b.abs()
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat([u, v], -1))
    return torch.cat([join(a * c - b * s, b * c + a * s), y[..., rot:]], -1), torch.cat([join(pair, pair), size[..., rot:]], -1)


def rounded(got, want, size, what):
    got = got.double()
    bad = ~((got - want).abs() <= want.abs() * 2.0 ** -8 + size * FINE * 1.01)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max())}"


def coded(got, want, size, scale, what):
    code, v = got.double(), (want / scale).clamp(-448.0, 448.0)
    bad = ~((code - v).abs() <= torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + (size / scale) * FINE * 2)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off"


def rotation(positions, rot, g):
    angle = 6.3 * torch.rand(positions, rot // 2, generator=g)
    return torch.cat([angle.cos(), angle.sin()], 1).to(DEV)


DIMS = [(128, 128), (128, 64), (64, 64), (256, 256), (96, 32), (80, 80), (72, 24), (8, 8), (2, 2), (6, 4), (130, 10), (250, 250),
        (512, 512), (510, 2), (40, 0), (16, 16), (504, 8)]


@pytest.mark.parametrize("dim,rot", DIMS)
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_beside(gemm, dim, rot, interleaved):
    g = torch.Generator().manual_seed(dim + rot)
    for tokens, qh, kvh, apart, which in ((1, 3, 1, 0, "qk"), (37, 5, 2, 0, "qk"), (9, 4, 4, 3, "q"), (5, 1, 2, 8, "k"), (3, 2, 1, 0, "")):
        print(f"beside {tokens} x {qh} + {kvh} x {dim} rot {rot} apart {apart} normed {which}", flush=True)
        x = normal(g, tokens, qh + kvh, dim + apart).to(BF)[..., apart // 2:apart // 2 + dim]
        q, k = x.split([qh, kvh], 1)
        w = [1 + 0.2 * normal(g, dim) if n in which else None for n in "qk"]
        table = rotation(50, rot, g)
        at = torch.randint(0, 50, (tokens,), generator=g).to(torch.int32).to(DEV)
        q_out, k_out = gemm.norm_rotate(q, k, at, table, q_norm=w[0], k_norm=w[1], eps=1e-5, interleaved=interleaved)
        assert q_out.shape == q.shape and k_out.shape == k.shape
        for got, t, n in ((q_out, q, w[0]), (k_out, k, w[1])):
            rounded(got, *formula(t, n, table, at, 1e-5, interleaved), f"{tokens} tokens")
        # In place, from a copy: the same bits.
        q2, k2 = q.clone(), k.clone()
        back = gemm.norm_rotate(q2, k2, at, table, q_norm=w[0], k_norm=w[1], eps=1e-5, q_out=q2, k_out=k2, interleaved=interleaved)
        assert back[0] is q2 and back[1] is k2 and torch.equal(q2, q_out) and torch.equal(k2, k_out)


def test_norm_alone_and_q_alone(gemm):
    g = torch.Generator().manual_seed(1)
    q, k, w = normal(g, 20, 3, 64).to(BF), normal(g, 20, 2, 64).to(BF), 1 + 0.1 * normal(g, 64)
    q_out, k_out = gemm.norm_rotate(q, k, q_norm=w, k_norm=w)
    for got, t in ((q_out, q), (k_out, k)):
        rounded(got, *formula(t, w, None, None, 1e-6, False), "normed")
    alone, none = gemm.norm_rotate(q, q_norm=w)
    assert none is None and torch.equal(alone, q_out)
    copied, _ = gemm.norm_rotate(q)
    assert torch.equal(copied, q)
    assert gemm.norm_rotate(q[:0], k[:0])[0].shape == (0, 3, 64)


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (256, 128), (80, 80), (72, 24), (6, 4), (512, 512)])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_appended(gemm, dtype, dim, rot, interleaved):
    g = torch.Generator().manual_seed(dim + rot)
    for tokens, qh, kvh, page, by_head in ((1, 4, 1, 16, False), (41, 6, 2, 16, True), (30, 3, 3, 7, False)):
        print(f"append {tokens} x {qh} + {kvh} x {dim} rot {rot} page {page} {dtype}", flush=True)
        pages = -(-tokens // page) + 2
        scales = [(0.01 + 0.02 * torch.rand(kvh, generator=g)).to(DEV) if dtype == F8 else None for _ in "kv"]
        pools = [torch.zeros(pages, page, kvh, dim, dtype=BF, device=DEV).to(dtype) for _ in "kv"]
        if by_head:
            pools = [p.view(torch.int16 if dtype == BF else torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(dtype) for p in pools]
        for p in pools:
            p.view(torch.uint8).fill_(0x11)
        before = [p.view(torch.uint8).clone() for p in pools]
        cache = sq.PagedCache(*pools, *scales)
        q, k, v = normal(g, tokens, qh + 2 * kvh, dim).to(BF).split([qh, kvh, kvh], 1)
        wq, wk = (1 + 0.2 * normal(g, dim) for _ in "qk")
        table = rotation(30, rot, g)
        at = torch.randint(0, 40, (tokens,), generator=g).to(torch.int32).to(DEV)  # past the table: its last row
        slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
        if tokens > 5:
            slots[3], slots[5] = -1, pages * page  # no slot, and one past the pools
        slots = slots.to(DEV)
        out = gemm.norm_append_kv(q, k, v, cache, at, slots, table, q_norm=wq, k_norm=wk, interleaved=interleaved)
        rounded(out, *formula(q, wq, table, at, 1e-6, interleaved), "q")
        live = (slots >= 0) & (slots < pages * page)
        to = slots[live].long()
        for name, pool, scale, (want, size) in (("k", cache.k, scales[0], formula(k, wk, table, at, 1e-6, interleaved)),
                                                ("v", cache.v, scales[1], (v.double(), v.double().abs()))):
            kept = pool.view(torch.int16 if dtype == BF else torch.uint8).reshape(-1, kvh, dim)[to].view(dtype)
            if scale is None:
                rounded(kept, want[live], size[live], name)
            else:
                coded(kept, want[live], size[live], scale.double()[:, None], name)
        untouched = torch.ones(pages * page, dtype=torch.bool, device=DEV)
        untouched[to] = False
        for pool, was in zip(pools, before):
            wide = pool.view(torch.uint8).reshape(pages * page, kvh, -1), was.reshape(pages * page, kvh, -1)
            assert torch.equal(wide[0][untouched], wide[1][untouched])


def test_without_norms_it_is_append_kv(gemm):
    g = torch.Generator().manual_seed(2)
    q, k, v = normal(g, 20, 8, 64).to(BF).split([4, 2, 2], 1)
    table, at = rotation(20, 64, g), torch.arange(20, dtype=torch.int32, device=DEV)
    caches = [sq.PagedCache(*(torch.zeros(2, 16, 2, 64, dtype=BF, device=DEV) for _ in "kv")) for _ in range(2)]
    a = gemm.append_kv(q, k, v, caches[0], at, at, table)
    b = gemm.norm_append_kv(q, k, v, caches[1], at, at, table)
    assert torch.equal(a, b) and torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)


def test_a_head_of_zeros_infinities_and_nans(gemm):
    """A head's row is its own: zeros stay zeros, an infinity makes its head's other values 0 and itself a NaN."""
    g = torch.Generator().manual_seed(3)
    x = normal(g, 4, 2, 128).to(BF)
    w = torch.ones(128, device=DEV)
    clean, _ = gemm.norm_rotate(x, q_norm=w)
    x[0, 0] = 0
    x[1, 0, 5] = math.inf
    x[2, 0, 5] = math.nan
    got, _ = gemm.norm_rotate(x, q_norm=w)
    assert (got[0, 0] == 0).all() and torch.isnan(got[1, 0, 5]) and (got[1, 0, :5] == 0).all()
    assert torch.isnan(got[2, 0]).all()
    assert torch.equal(got[:, 1], clean[:, 1]) and torch.equal(got[3], clean[3])


def test_many_tokens(gemm):
    g = torch.Generator().manual_seed(4)
    q, k = normal(g, 5000, 6, 128).to(BF).split([4, 2], 1)
    w, table = 1 + 0.1 * normal(g, 128), rotation(5000, 128, g)
    at = torch.arange(5000, dtype=torch.int32, device=DEV)
    for got, t in zip(gemm.norm_rotate(q, k, at, table, q_norm=w, k_norm=w), (q, k)):
        rounded(got, *formula(t, w, table, at, 1e-6, False), "many")


def test_refusals(gemm):
    g = torch.Generator().manual_seed(5)
    q, k, v = normal(g, 8, 8, 64).to(BF).split([4, 2, 2], 1)
    w, table, at = torch.ones(64, device=DEV), rotation(8, 64, g), torch.arange(8, dtype=torch.int32, device=DEV)
    refused = lambda kind, f, *a, **kw: pytest.raises(kind, f, *a, **kw)  # noqa: E731
    for f, args in ((gemm.norm_rotate, (q, k, at, table)),
                    (gemm.norm_append_kv, (q, k, v, sq.PagedCache(*(torch.zeros(2, 16, 2, 64, dtype=BF, device=DEV) for _ in "kv")), at, at, table))):
        refused(ValueError, f, q.float(), *args[1:])
        refused(ValueError, f, q, k[:7], *args[2:])
        refused(ValueError, f, *args, q_norm=w[:32])
        refused(ValueError, f, *args, k_norm=w.to(BF))
        refused(ValueError, f, *args, q_norm=w.cpu())
        refused(ValueError, f, *args[:-1], table.to(BF))
        refused(ValueError, f, *args[:-2], at.long(), table)
        refused(ValueError, f, *args, q_out=q[:, :2])
        refused(abi.SQ8Error, f, *args[:-1], rotation(8, 128, g))  # turned values past the head
        refused(abi.SQ8Error, f, *args[:-1], table[:0])
        refused(abi.Unsupported, f, *args[:-1], table[:, :3])
    refused(ValueError, gemm.norm_rotate, q, k, at)  # positions without a table
    refused(ValueError, gemm.norm_rotate, q, k_norm=w)
    refused(ValueError, gemm.norm_rotate, q, k_out=k)
    long = torch.zeros(2, 1, 514, dtype=BF, device=DEV)
    refused(abi.Unsupported, gemm.norm_rotate, long)
    refused(abi.Unsupported, gemm.norm_rotate, long[..., :63])


def test_a_graph_s_replays(gemm):
    ctx = sq.TensorGEMM.make(0)
    side = torch.cuda.Stream()
    g = torch.Generator().manual_seed(6)
    x, w, table = torch.zeros(30, 6, 64, dtype=BF, device=DEV), 1 + 0.1 * normal(g, 64), rotation(30, 64, g)
    q, k = x.split([4, 2], 1)
    at = torch.arange(30, dtype=torch.int32, device=DEV)
    outs = [torch.zeros(30, n, 64, dtype=BF, device=DEV) for n in (4, 2)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.set_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ctx.norm_rotate(q, k, at, table, q_norm=w, k_norm=w, q_out=outs[0], k_out=outs[1])
        for i in range(4):
            x.copy_(torch.randn(x.shape, device=DEV))
            graph.replay()
            side.synchronize()
            for got, want in zip(outs, ctx.norm_rotate(q, k, at, table, q_norm=w, k_norm=w)):
                assert torch.equal(got, want), i
        ctx.set_stream(torch.cuda.default_stream())
    torch.cuda.current_stream().wait_stream(side)
