"""Attention of whole packed prompts over their own keys and values, against the formula in 64 bits (attend_reference.py says
where the tolerances come from)."""
import math

import pytest
import torch

import siliconed_amd as sq
from attend_reference import attended, within
from siliconed_amd import _abi as abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def normal(g, *shape):
    return torch.randn(*shape, generator=g).to(DEV)


def run_prompt(gemm, lengths, qh, kvh, dim, *, spare=0, lead=0, seed=0, apart=0, **options):
    """Packed sequences behind `lead` rows and before `spare` ones, which stay as they are. `apart`: values between heads."""
    print(f"prompt {lengths[:6]} heads {qh}/{kvh} dim {dim} spare {spare} lead {lead} {options}", flush=True)
    g = torch.Generator().manual_seed(seed + sum(lengths) + dim + qh)
    rows = lead + sum(lengths) + spare
    qkv = (normal(g, rows, qh + 2 * kvh, dim + apart)).to(BF)
    q, k, v = qkv[..., :dim].split([qh, kvh, kvh], 1)
    starts = torch.tensor([lead + sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=DEV)
    out = torch.full((rows, qh, dim), 7.0, dtype=BF, device=DEV)
    got = gemm.prompt_attention(q, k, v, starts, out=out, **options)
    assert got is out
    for lo, n in zip(starts.tolist(), lengths):
        want, tol = attended(q[lo:lo + n], k[lo:lo + n], v[lo:lo + n], 0, **options)
        within(out[lo:lo + n], want, tol, f"{n} rows from {lo}")
    assert (out[:lead] == 7.0).all() and (out[rows - spare:] == 7.0).all()
    return out


LENGTHS = [1, 2, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257, 300]


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "whole"])
@pytest.mark.parametrize("qh,kvh,dim", [(8, 2, 128), (4, 4, 64), (2, 1, 256), (5, 1, 96)])
def test_lengths(gemm, causal, qh, kvh, dim):
    run_prompt(gemm, LENGTHS, qh, kvh, dim, causal=causal, spare=3, lead=2)


@pytest.mark.parametrize("qh,kvh,dim", [(1, 1, 8), (3, 1, 16), (6, 2, 40), (7, 1, 72), (12, 4, 80), (16, 2, 120), (4, 1, 136),
                                        (2, 2, 192), (33, 1, 64), (40, 1, 128), (8, 8, 248)])
def test_heads_and_dims(gemm, qh, kvh, dim):
    run_prompt(gemm, [70, 1, 130], qh, kvh, dim)
    run_prompt(gemm, [150], qh, kvh, dim, causal=False, apart=8)


# Each tile of rows: 256, 128, 64 and 32 of them, by the units that there are for a card of 256 CUs.
@pytest.mark.parametrize("lengths,qh,kvh", [([5000, 3200], 32, 8), ([2000], 32, 8), ([700, 300], 32, 8), ([200], 8, 8), ([90], 4, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_every_tile(gemm, lengths, qh, kvh, dim):
    run_prompt(gemm, lengths, qh, kvh, dim)
    run_prompt(gemm, lengths[:1], qh, kvh, dim, causal=False)


@pytest.mark.parametrize("length,qh,kvh", [(4100, 16, 8), (600, 4, 2)])
def test_tiles_of_heads_of_256(gemm, length, qh, kvh):
    run_prompt(gemm, [length], qh, kvh, 256)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 200, 5000, (1 << 31) - 1])
def test_windows(gemm, window):
    run_prompt(gemm, [1, 300, 64, 700], 8, 2, 128, window=window)
    run_prompt(gemm, [333], 2, 2, 64, window=window)


def test_softcap_and_scale(gemm):
    for softcap in (0.5, 30.0, math.inf):
        run_prompt(gemm, [140, 40], 8, 2, 128, softcap=softcap)
        run_prompt(gemm, [140], 8, 2, 64, softcap=softcap, scale=1.0, causal=False)
    for scale in (-0.3, 0.0, 2.0, 1e-6):
        run_prompt(gemm, [140], 8, 2, 64, scale=scale)
        run_prompt(gemm, [140], 2, 1, 64, scale=scale, softcap=5.0)


def test_no_starts_is_one_sequence(gemm):
    g = torch.Generator().manual_seed(1)
    q, k, v = (normal(g, 77, h, 64).to(BF) for h in (4, 2, 2))
    want = gemm.prompt_attention(q, k, v, torch.tensor([0, 77], dtype=torch.int32, device=DEV))
    assert torch.equal(gemm.prompt_attention(q, k, v), want)


def test_many_sequences(gemm):
    run_prompt(gemm, [(7 * i) % 40 for i in range(150)], 4, 2, 64)
    run_prompt(gemm, [0] * 100 + [9] + [0] * 30, 4, 1, 128, spare=1)


def test_starts_outside_the_rows_are_cut(gemm):
    g = torch.Generator().manual_seed(2)
    q, k, v = (normal(g, 50, h, 64).to(BF) for h in (2, 1, 1))
    out = torch.full_like(q, 3.0)
    gemm.prompt_attention(q, k, v, torch.tensor([-5, 20, 1 << 30], dtype=torch.int32, device=DEV), out=out)
    for lo, hi in ((0, 20), (20, 50)):
        want, tol = attended(q[lo:hi], k[lo:hi], v[lo:hi], 0)
        within(out[lo:hi], want, tol, f"rows {lo} to {hi}")


@pytest.mark.parametrize("starts", [[40, 20, 30], [0, 50, 10, 45], [60, 70, 80], [0, 0, 0]])
def test_starts_that_do_not_ascend_stay_inside(gemm, starts):
    """Such sequences overlap or are empty: whatever is written, rows outside them all stay."""
    g = torch.Generator().manual_seed(3)
    q, k, v = (normal(g, 50, h, 64).to(BF) for h in (2, 1, 1))
    out = torch.full((60, 2, 64), 3.0, dtype=BF, device=DEV)
    gemm.prompt_attention(q, k, v, torch.tensor(starts, dtype=torch.int32, device=DEV), out=out[:50])
    assert (out[50:] == 3.0).all()
    want, tol = attended(q, k, v, 0)
    within(gemm.prompt_attention(q, k, v), want, tol, "the next call")


@pytest.mark.parametrize("dim,qh,kvh", [(128, 4, 1), (64, 2, 2), (256, 1, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_what_a_row_does_not_see_may_be_anything(gemm, dim, qh, kvh, causal):
    """Infinite and NaN keys and values of later tokens, of the neighbouring sequences and of unused rows."""
    g = torch.Generator().manual_seed(4)
    q, k, v = (normal(g, 200, h, dim).to(BF) for h in (qh, kvh, kvh))
    lo, hi, at = 30, 170, 100
    wild_k, wild_v = k.clone(), v.clone()
    for t in (wild_k, wild_v):
        t[:lo] = math.nan
        t[hi:] = math.inf
    starts = torch.tensor([lo, hi], dtype=torch.int32, device=DEV)
    got = gemm.prompt_attention(q, wild_k, wild_v, starts, causal=causal, out=torch.zeros_like(q))
    want, tol = attended(q[lo:hi], k[lo:hi], v[lo:hi], 0, causal=causal)
    within(got[lo:hi], want, tol, "beside other rows")
    if not causal:
        return
    for bad_k, bad_v in ((0.0, math.nan), (0.0, math.inf), (math.nan, 0.0), (math.inf, -math.inf)):
        wild_k[at, 0], wild_v[at, 0] = k[at, 0] + bad_k, v[at, 0] + bad_v
        for window in (0, 20):
            got = gemm.prompt_attention(q, wild_k, wild_v, starts, window=window, out=torch.zeros_like(q))
            want, tol = attended(q[lo:hi], k[lo:hi], v[lo:hi], 0, window=window)
            clean = torch.ones(hi - lo, dtype=torch.bool, device=DEV)
            clean[at - lo:at - lo + (window or hi)] = False
            within(got[lo:hi][clean], want[clean], tol[clean], f"before a token of {bad_k}, {bad_v}, window {window}")
            if not bad_k:  # seen by all the others with some weight
                heads = range(qh // kvh)  # of its kv head
                rest = got[lo:hi][~clean][:, list(heads)]
                assert (~torch.isfinite(rest)).all()


def test_rows_of_the_lowest_scores(gemm):
    """A row whose every score is -inf gives zeros; finite scores however low are a softmax as any."""
    q = torch.ones(40, 1, 64, dtype=BF, device=DEV)
    k = torch.full((40, 1, 64), -math.inf, dtype=BF, device=DEV)
    g = torch.Generator().manual_seed(5)
    v = normal(g, 40, 1, 64).to(BF)
    assert (gemm.prompt_attention(q, k, v) == 0).all()
    k.fill_(torch.finfo(BF).min / 1024)
    want, tol = attended(q, torch.zeros_like(k), v, 0)
    within(gemm.prompt_attention(q, k, v), want, tol, "low scores")


def test_refusals(gemm):
    g = torch.Generator().manual_seed(6)
    q, k, v = (normal(g, 20, h, 64).to(BF) for h in (4, 2, 2))
    starts = torch.tensor([0, 20], dtype=torch.int32, device=DEV)
    refused = lambda kind, *a, **kw: pytest.raises(kind, gemm.prompt_attention, *a, **kw)  # noqa: E731
    refused(ValueError, q.float(), k, v, starts)
    refused(ValueError, q, k.float(), v, starts)
    refused(ValueError, q, k[:19], v, starts)
    refused(ValueError, q, k, v[:, :1], starts)
    refused(ValueError, q, k, v, starts.long())
    refused(ValueError, q, k, v, starts.cpu())
    refused(ValueError, q, k, v, starts[:0])
    refused(ValueError, q, k, v, starts, out=q[:, :2])
    refused(ValueError, q.cpu(), k, v, starts)
    refused(ValueError, q.transpose(1, 2).contiguous().transpose(1, 2), k, v, starts)
    refused(abi.SQ8Error, q[:, :3], k, v, starts)  # three heads on two
    refused(abi.SQ8Error, q, k, v, starts, window=-1)
    refused(abi.SQ8Error, q, k, v, starts, window=4, causal=False)
    refused(abi.SQ8Error, q, k, v, starts, softcap=-1.0)
    refused(abi.SQ8Error, q, k, v, starts, softcap=math.nan)
    refused(abi.Unsupported, q[..., :60], k[..., :60], v[..., :60], starts)  # dim not a multiple of 8
    wide = torch.zeros(20, 2, 65, dtype=BF, device=DEV)
    refused(abi.Unsupported, q, wide[..., :64], v, starts)  # rows not 16-byte aligned
    far = torch.zeros(20, 1, 264, dtype=BF, device=DEV)
    refused(abi.Unsupported, far, far, far, starts)
    assert gemm.prompt_attention(q[:0], k[:0], v[:0], starts).shape == (0, 4, 64)
    out = torch.full_like(q, 5.0)
    gemm.prompt_attention(q, k, v, starts[:1], out=out)  # no sequence
    assert (out == 5.0).all()


def test_a_graph_s_replays(gemm):
    """Other lengths and values at every replay, calls in between: bit for bit what calls give."""
    ctx = sq.TensorGEMM.make(0)
    side = torch.cuda.Stream()
    q, k, v = (torch.zeros(900, h, 128, dtype=BF, device=DEV) for h in (8, 2, 2))
    starts = torch.zeros(4, dtype=torch.int32, device=DEV)
    out = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.set_stream(side)
        ctx.prompt_attention(q, k, v, starts, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ctx.prompt_attention(q, k, v, starts, out=out)
        for i in range(5):
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, device=DEV))
            starts.copy_(torch.tensor([0, 100 + i, 400 - 37 * i, 900 - i], dtype=torch.int32))
            out.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(out, ctx.prompt_attention(q, k, v, starts, out=torch.zeros_like(q))), i
        ctx.set_stream(torch.cuda.default_stream())
    torch.cuda.current_stream().wait_stream(side)
