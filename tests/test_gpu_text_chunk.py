"""Attention of chunks of new tokens over a paged cache, against the formula in 64 bits (attend_reference.py says where the
tolerances come from)."""
import math

import pytest
import torch

import siliconed_amd as sq
from attend_reference import attended, within
from siliconed_amd import _abi as abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F8 = torch.bfloat16, torch.float8_e4m3fn
BOTH = pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])


def normal(g, *shape):
    return torch.randn(*shape, generator=g).to(DEV)


def ints(*n):
    return torch.tensor(n, dtype=torch.int32, device=DEV)


class Batch:
    """Sequences of (new tokens, cached tokens with them) in pages in random order; what no sequence holds is NaN. `bad`:
    (sequence, page number, index) of page table entries replaced by an index outside the pools."""

    def __init__(self, chunks, qh, kvh, dim, page, dtype, *, by_head=False, bad=(), seed=0, spare=0, extra_pages=2):
        g = torch.Generator().manual_seed(seed + sum(n + m for n, m in chunks) + dim + qh + page)
        self.chunks, self.spare = chunks, spare
        each = max(1, max(-(-m // page) for _, m in chunks)) + 1
        total = sum(-(-m // page) for _, m in chunks) + extra_pages
        order = torch.randperm(total, generator=g)
        table = torch.full((len(chunks), each), -7, dtype=torch.int32)
        pools = [torch.full((total, page, kvh, dim), math.nan, device=DEV) for _ in range(2)]
        scales = [(0.5 + torch.rand(kvh, generator=g)).to(DEV) for _ in range(2)] if dtype == F8 else [None, None]
        self.values, at = [], 0
        for b, (_, m) in enumerate(chunks):
            count = -(-m // page)
            ids = order[at:at + count]
            table[b, :count] = ids.to(torch.int32)
            at += count
            kv = [normal(g, m, kvh, dim).to(dtype).float() for _ in range(2)]
            for pool, t in zip(pools, kv):
                token = torch.arange(m)
                pool[ids[token // page].to(DEV), (token % page).to(DEV)] = t
            self.values.append([t if s is None else t * s[:, None] for t, s in zip(kv, scales)])
        self.dead = [torch.zeros(m, dtype=torch.bool, device=DEV) for _, m in chunks]
        for b, i, index in bad:
            table[b, i] = index
            self.dead[b][i * page:(i + 1) * page] = True
        pools = [p.to(dtype) for p in pools]
        if by_head:
            pools = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in pools]
        self.cache = sq.PagedCache(*pools, *scales)
        self.table = table.to(DEV)
        self.lengths = ints(*(m for _, m in chunks))
        self.starts = ints(*(sum(n for n, _ in chunks[:i]) for i in range(len(chunks) + 1)))
        self.q = normal(g, int(self.starts[-1]) + spare, qh, dim).to(BF)

    def roomy(self):
        """The table with room for two million tokens: many rows a sequence then go by larger tiles."""
        page = self.cache.k.shape[1]
        room = torch.full((len(self.chunks), (1 << 21) // page), -5, dtype=torch.int32, device=DEV)
        room[:, :self.table.shape[1]] = self.table
        return room

    def run(self, gemm, table=None, **options):
        out = torch.full_like(self.q, 7.0)
        got = gemm.chunk_attention(self.q, self.cache, self.table if table is None else table, self.lengths, self.starts, out=out, **options)
        assert got is out
        return out

    def check(self, gemm, **options):
        print(f"chunks {self.chunks[:6]} q {tuple(self.q.shape)} pools {tuple(self.cache.k.shape)} {self.cache.k.dtype} {options}", flush=True)
        out, again = self.run(gemm, **options), self.run(gemm, self.roomy(), **options)
        for b, (n, m) in enumerate(self.chunks):
            lo = int(self.starts[b])
            want, tol = attended(self.q[lo:lo + n], *self.values[b], m - n, dead=self.dead[b], **options)
            within(out[lo:lo + n], want, tol, f"sequence {b}: {n} of {m}")
            within(again[lo:lo + n], want, tol, f"sequence {b}: {n} of {m}, a roomy table")
        assert (out[len(out) - self.spare:] == 7.0).all() and (again[len(out) - self.spare:] == 7.0).all()
        return out


CHUNKS = [(1, 1), (0, 40), (1, 33), (3, 16), (5, 300), (17, 17), (16, 129), (40, 64), (2, 2), (33, 500), (1, 128), (4, 15)]


@BOTH
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64])
def test_lengths_and_pages(gemm, dtype, page):
    Batch(CHUNKS, 8, 2, 128, page, dtype, spare=3).check(gemm)
    Batch(CHUNKS, 2, 2, 64, page, dtype, by_head=True).check(gemm)


@BOTH
@pytest.mark.parametrize("qh,kvh,dim", [(1, 1, 64), (8, 8, 128), (5, 1, 96), (40, 8, 128), (32, 1, 128), (20, 1, 64), (6, 2, 256),
                                        (3, 3, 16), (4, 2, 80), (4, 1, 192), (12, 4, 48)])
def test_heads_and_dims(gemm, dtype, qh, kvh, dim):
    for page in (16, 7):
        Batch([(3, 200), (0, 5), (20, 65), (1, 70)], qh, kvh, dim, page, dtype, by_head=page == 7).check(gemm)


@pytest.mark.parametrize("dim", [8, 24, 40, 72, 120, 136])
def test_narrow_dims_in_bf16(gemm, dim):
    Batch([(9, 90), (4, 4)], 4, 2, dim, 16, BF).check(gemm)


# Each tile of rows: 16, 32, 64, 128 and 256 rows (a sequence's, or as many as a table's room makes worth while).
@BOTH
@pytest.mark.parametrize("new", [1, 7, 13, 30, 70, 200])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (128, 24), (256, 32)])
def test_every_tile(gemm, dtype, new, dim, page):
    Batch([(new, 700), (new, new), (new, 1300)], 8, 2, dim, page, dtype).check(gemm)


@BOTH
@pytest.mark.parametrize("window", [1, 16, 50, 128, 500, 5000, (1 << 31) - 1])
def test_windows(gemm, dtype, window):
    Batch([(3, 3), (1, 49), (20, 51), (60, 700), (0, 9), (5, 1400)], 8, 2, 64, 16, dtype).check(gemm, window=window)
    Batch([(70, 129), (2, 260)], 4, 4, 128, 3, dtype).check(gemm, window=window)


@pytest.mark.parametrize("softcap", [0.5, 30.0, math.inf])
def test_softcap_and_scale(gemm, softcap):
    Batch([(1, 1), (9, 140), (40, 500)], 8, 2, 128, 16, BF).check(gemm, softcap=softcap)
    Batch([(1, 1), (9, 140), (40, 500)], 8, 2, 128, 16, F8).check(gemm, softcap=softcap, scale=0.5)
    Batch([(9, 140)], 8, 2, 64, 16, BF).check(gemm, scale=-0.3)
    Batch([(9, 140)], 8, 2, 64, 16, BF).check(gemm, scale=0.0)


@BOTH
def test_shared_over_workgroups(gemm, dtype):
    Batch([(4, 9001)], 4, 1, 128, 16, dtype).check(gemm)
    Batch([(2, 5000), (0, 0), (3, 3), (1, 8000), (30, 130)], 16, 2, 64, 32, dtype).check(gemm)
    Batch([(100, 3000), (2, 1500)], 2, 2, 256, 9, dtype).check(gemm)
    Batch([(300, 4000), (200, 900)], 8, 2, 128, 64, dtype).check(gemm)
    Batch([(300, 4000), (200, 900)], 8, 2, 128, 64, dtype).check(gemm, window=700)


def test_many_sequences(gemm):
    Batch([((5 * i) % 7, (5 * i) % 7 + (37 * i) % 290) for i in range(150)], 4, 2, 64, 16, BF).check(gemm)
    Batch([(0, 30)] * 130 + [(5, 5)], 4, 2, 64, 16, F8).check(gemm)


def test_one_new_token_is_paged_attention(gemm):
    b = Batch([(1, n) for n in (1, 15, 200, 1000, 64)], 8, 2, 128, 16, BF)
    want = gemm.paged_attention(b.q, b.cache, b.table, b.lengths)
    within(b.check(gemm), want.double(), want.double().abs() * 2.0 ** -7 + 1e-5, "one token")


def test_pages_outside_the_pools_are_masked(gemm):
    for page, dtype in ((16, BF), (5, BF), (16, F8), (24, F8)):
        for new in (3, 60):
            Batch([(new, 200), (new, 64)], 4, 2, 64, page, dtype, bad=[(0, 1, -1), (0, 3, 1 << 30), (1, 0, 99999)]).check(gemm)
    out = Batch([(4, 16), (5, 40)], 4, 2, 128, 16, BF, bad=[(0, 0, -1)]).check(gemm)
    assert (out[:4] == 0).all()


def test_lengths_are_cut_and_chunks_past_them_give_zeros(gemm):
    g = torch.Generator().manual_seed(9)
    k, v = (normal(g, 3, 16, 1, 64).to(BF) for _ in range(2))
    cache = sq.PagedCache(k, v)
    q = normal(g, 12, 2, 64).to(BF)
    table = torch.tensor([[2, 0], [1, 2], [0, 1]], dtype=torch.int32, device=DEV)
    starts = ints(0, 4, 8, 12)
    got = gemm.chunk_attention(q, cache, table, ints(1 << 30, -4, 32), starts)
    want = gemm.chunk_attention(q, cache, table, ints(32, 0, 32), starts)
    assert torch.equal(got, want) and (got[4:8] == 0).all()
    got = gemm.chunk_attention(q, cache, table, ints(2, 4, 32), starts)  # four new tokens, of which two are there
    assert (got[:2] == 0).all()
    flat = lambda pool, b: pool[table[b].long()].flatten(0, 1)  # noqa: E731
    o, tol = attended(q[2:4], flat(k, 0)[:2], flat(v, 0)[:2], 0)
    within(got[2:4], o, tol, "the two that are there")
    for window in (5, (1 << 31) - 1):  # eleven new tokens, of which three are there, the others nowhere
        wide = gemm.chunk_attention(q[:11], cache, table[:1], ints(3), window=window)
        o, tol = attended(q[8:11], flat(k, 0)[:3], flat(v, 0)[:3], 0)
        assert (wide[:8] == 0).all()
        within(wide[8:], o, tol, "the three that are there")
    assert gemm.chunk_attention(q[:0], cache, table, ints(5, 5, 5), ints(0, 0, 0, 0)).shape == (0, 2, 64)
    none = gemm.chunk_attention(q, cache, table[:, :0], ints(5, 5, 5), starts)
    assert (none == 0).all()
    empty = sq.PagedCache(k[:0], v[:0])
    assert (gemm.chunk_attention(q, empty, table, ints(5, 5, 5), starts) == 0).all()


@pytest.mark.parametrize("roomy", [False, True])
@pytest.mark.parametrize("starts", [[4, 2, 9, 3], [0, 12, 1, 11], [50, 60, 70, 80]])
def test_starts_that_do_not_ascend_stay_inside(gemm, starts, roomy):
    """Whatever is written, rows outside stay, and the counters that workgroups share are left as they were found."""
    b = Batch([(4, 2000), (4, 900), (4, 3000)], 24, 1, 64, 16, BF, spare=4)
    b.check(gemm)
    table = b.roomy() if roomy else b.table
    want = b.run(gemm, table)
    out = torch.full((20, 24, 64), 3.0, dtype=BF, device=DEV)
    gemm.chunk_attention(b.q[:12], b.cache, table, b.lengths, ints(*starts), out=out[:12])
    assert (out[12:] == 3.0).all()
    assert torch.equal(b.run(gemm, table), want)


def test_starts_that_count_more_tiles_than_32_bits_hold(gemm):
    """4096 sequences of 32 768 tokens that all claim the same 4096 rows: nothing past the rows is written, and calls go on."""
    good = Batch([(4, 2000), (4, 900)], 32, 8, 64, 16, BF)
    want = good.check(gemm)
    k, v = (torch.zeros(2, 16, 8, 64, dtype=BF, device=DEV) for _ in "kv")
    table = torch.zeros(4096, 2048, dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 4096] * 2048 + [0], dtype=torch.int32, device=DEV)
    out = torch.full((4104, 32, 64), 3.0, dtype=BF, device=DEV)
    q = torch.zeros(4096, 32, 64, dtype=BF, device=DEV)
    gemm.chunk_attention(q, sq.PagedCache(k, v), table, torch.full((4096,), 32768, dtype=torch.int32, device=DEV), starts, out=out[:4096])
    assert (out[4096:] == 3.0).all()
    assert torch.equal(good.run(gemm, good.roomy()), good.run(gemm, good.roomy())) and torch.equal(good.run(gemm), want)


def test_offsets_past_32_bits(gemm):
    """A pool of 5 GB, the sequence's pages at its end."""
    pages, page, dim = 40000, 64, 128
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("a small card")
    k, v = (torch.zeros(pages, page, 8, dim, dtype=BF, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(3)
    ids = torch.tensor([pages - 1, 7, pages - 2], device=DEV)
    for pool in (k, v):
        pool[ids] = normal(g, 3, page, 8, dim).to(BF)
    q = normal(g, 40, 16, dim).to(BF)
    table = ids.to(torch.int32)[None]
    got = gemm.chunk_attention(q, sq.PagedCache(k, v), table, ints(170))
    want, tol = attended(q, k[ids].flatten(0, 1)[:170], v[ids].flatten(0, 1)[:170], 130)
    within(got, want, tol, "the pool's end")


@BOTH
@pytest.mark.parametrize("roomy", [False, True])
def test_infinite_and_nan_values_are_their_tokens(gemm, dtype, roomy):
    b = Batch([(40, 100), (40, 100)], 4, 2, 64, 16, dtype)
    b.check(gemm)
    table = b.roomy() if roomy else None
    clean = b.run(gemm, table)
    page, place = int(b.table[0, 5]), 0  # token 80 of the first sequence: the chunk's twentieth
    pool = b.cache.v.view(torch.uint8)
    pool[page, place, 0, :2 if dtype == BF else 1] = 0xFF  # a NaN
    out = b.run(gemm, table)
    # Rows beside those that see it may be done without the matrix cores, their probabilities not rounded: the formula's tolerance
    # covers either, another sequence keeps its bits.
    want, tol = attended(b.q[:40], *b.values[0], 60)
    within(out[:20], want[:20], tol[:20], "before the token")
    within(out[20:40, 2:], want[20:, 2:], tol[20:, 2:], "another kv head")
    assert torch.equal(out[40:], clean[40:])
    assert torch.isnan(out[20:40, :2, 0]).all()
    within(out[20:40, :2, 1:], want[20:, :2, 1:], tol[20:, :2, 1:], "its other values")


def test_refusals(gemm):
    b = Batch([(4, 20), (3, 9)], 4, 2, 64, 16, BF)
    a = (b.q, b.cache, b.table, b.lengths, b.starts)
    refused = lambda kind, *a, **kw: pytest.raises(kind, gemm.chunk_attention, *a, **kw)  # noqa: E731
    refused(ValueError, b.q.float(), *a[1:])
    refused(ValueError, b.q, b.cache, b.table.long(), b.lengths, b.starts)
    refused(ValueError, b.q, b.cache, b.table, b.lengths[:1], b.starts)
    refused(ValueError, b.q, b.cache, b.table, b.lengths, b.starts[:2])
    refused(ValueError, b.q, b.cache, b.table, b.lengths)  # no starts, two sequences' pages
    refused(ValueError, b.q, b.cache, b.table, b.lengths.cpu(), b.starts)
    refused(ValueError, *a, out=b.q[:3])
    refused(ValueError, b.q[..., :32], *a[1:])
    refused(abi.SQ8Error, b.q[:, :3], *a[1:])
    refused(abi.SQ8Error, *a, window=-1)
    refused(abi.SQ8Error, *a, softcap=-1.0)
    refused(abi.SQ8Error, *a, softcap=math.nan)
    narrow = sq.PagedCache(*(torch.zeros(2, 16, 2, 24, dtype=BF, device=DEV).to(F8) for _ in "kv"))
    refused(abi.Unsupported, torch.zeros(7, 4, 24, dtype=BF, device=DEV), narrow, *a[2:])
    wide = torch.zeros(7, 4, 65, dtype=BF, device=DEV)[..., :64]
    refused(abi.Unsupported, wide, *a[1:])


def test_a_graph_s_replays_beside_other_attention(gemm):
    """A captured chunk attention and a captured one-token attention share the context's scratch and counters: other lengths
    at every replay, calls in between, bit for bit what calls give."""
    ctx = sq.TensorGEMM.make(0)
    side = torch.cuda.Stream()
    b = Batch([(8, 3000), (8, 2000), (8, 600)], 8, 2, 128, 16, BF)
    one = b.q[::8].contiguous()
    out, single = torch.zeros_like(b.q), torch.zeros_like(one)
    lengths = b.lengths.clone()

    def calls(o, s):
        ctx.chunk_attention(b.q, b.cache, b.table, lengths, b.starts, out=o)
        ctx.paged_attention(one, b.cache, b.table, lengths, out=s)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.set_stream(side)
        calls(out, single)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            calls(out, single)
        for i in range(6):
            lengths.copy_(b.lengths - ints(400 * i, 300 * i, 90 * i))
            out.zero_()
            single.zero_()
            graph.replay()
            side.synchronize()
            o, s = torch.zeros_like(out), torch.zeros_like(single)
            calls(o, s)
            side.synchronize()
            assert torch.equal(out, o) and torch.equal(single, s), i
        ctx.set_stream(torch.cuda.default_stream())
    torch.cuda.current_stream().wait_stream(side)


@BOTH
@pytest.mark.parametrize("dim", [80, 96, 48])
def test_a_sequence_s_nan_stays_with_it(gemm, dtype, dim):
    """Heads narrower than their tiles, many sequences to a workgroup: a NaN in every seventh's cache is in no other's output."""
    b = Batch([(20, 70)] * 300, 16, 4, dim, 64, dtype)
    room = torch.full((300, 1 << 15), -5, dtype=torch.int32, device=DEV)
    room[:, :b.table.shape[1]] = b.table
    for table in (None, room):
        clean = b.run(gemm, table).view(300, 20, 16, dim)
        pool, kept = b.cache.v.view(torch.uint8), b.cache.v.view(torch.uint8).clone()
        for i in range(0, 300, 7):
            pool[int(b.table[i, 0]), 0] = 0xFF  # the first token, which every row sees
        out = b.run(gemm, table).view(300, 20, 16, dim)
        pool.copy_(kept)
        others = torch.arange(300, device=DEV) % 7 != 0
        assert torch.equal(out[others], clean[others]) and torch.isnan(out[~others]).all()
