"""The next token of rows of logits, against the definition in 64 bits: sorted, cut, summed, on the CPU.

Tokens have to be equal. Both sides' sums are within 2^-40 of the whole, so a random number or a border lies between them with a
chance of some 2^-40 for each token kept, under 2^-20 a row; where the sums are whole numbers of equal weights both are exact.
Log probabilities: a float32's rounding, 2^-24 of them, and of the sum's 2^-40."""
import math

import pytest
import torch

import siliconed_amd as sq
from siliconed_amd import _abi as abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
TYPES = pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])


def kept_of(x, t, k, p, m):
    """The weights in 64 bits of the tokens that are kept, 0 for others; None for a row of nothing."""
    x = torch.where(torch.isnan(x), -math.inf, x.double())
    top = x.max()
    if top == -math.inf:
        return None
    if not t > 0:
        k, t = 1, 1.0
    w = (x == math.inf).double() if top == math.inf else torch.exp((x - top) / t)
    w = torch.where(x == -math.inf, 0.0, w)
    order = torch.sort(x, descending=True, stable=True).indices
    w = w[order]
    keep = torch.ones(len(w), dtype=torch.bool)
    if k > 0:
        keep[k:] = False
    if not p >= 1:
        kept = torch.where(keep, w, 0.0)
        upto = kept.cumsum(0)
        before = torch.cat([upto.new_zeros(1), upto[:-1]])
        keep &= before < p * upto[-1]
    keep &= w >= m
    keep[0] = True
    found = torch.zeros_like(w)
    found[order] = torch.where(keep, w, 0.0)
    return found


def drawn(x, u, t=1.0, k=0, p=1.0, m=0.0):
    w = kept_of(x, t, k, p, m)
    if w is None:
        return -1, -math.inf
    u = min(max(0.0 if math.isnan(u) else u, 0.0), 1 - 2.0 ** -24)
    upto = w.cumsum(0)
    token = int((upto > u * upto[-1]).nonzero()[0])
    return token, math.log(w[token] / upto[-1])


def run(gemm, x, u, temperature=None, top_k=None, top_p=None, min_p=None, what=""):
    """Rows of logits (on the CPU) and their lists of options: tokens and log probabilities as the definition has them."""
    def f(v, dtype=torch.float32):
        return None if v is None else torch.tensor(v, dtype=dtype).to(DEV)
    print(f"sample {tuple(x.shape)} {x.dtype} {what}", flush=True)
    u = torch.tensor(u, dtype=torch.float32)
    tokens, logprobs = gemm.sample_tokens(x.to(DEV), u.to(DEV), temperature=f(temperature), top_k=f(top_k, torch.int32),
                                          top_p=f(top_p), min_p=f(min_p))
    tokens, logprobs = tokens.cpu(), logprobs.cpu()
    at = lambda v, b, none: none if v is None else torch.tensor(v[b], dtype=torch.float32).item()  # noqa: E731
    for b in range(len(x)):
        options = dict(t=at(temperature, b, 1.0), k=0 if top_k is None else top_k[b], p=at(top_p, b, 1.0), m=at(min_p, b, 0.0))
        token, logprob = drawn(x[b].float(), u[b].item(), **options)
        assert int(tokens[b]) == token, f"{what} row {b} {options} u {u[b].item()}: {int(tokens[b])} for {token}"
        got = float(logprobs[b])
        assert got == logprob or abs(got - logprob) <= 2.0 ** -23 * abs(logprob) + 1e-11, f"{what} row {b}: log {got} for {logprob}"
    return tokens


def logits(g, rows, vocab, dtype=torch.float32):
    """The heavy head of a language model's, a few forbidden."""
    x = torch.randn(rows, vocab, generator=g) + 1.5 * torch.empty(rows, vocab).exponential_(generator=g)
    if vocab > 8:
        x[:, torch.randperm(vocab, generator=g)[:vocab // 8]] = -math.inf
    return x.to(dtype)


def uniform(g, rows):
    return torch.rand(rows, generator=g).tolist()


VOCABS = [1, 2, 3, 63, 100, 1000, 1023, 1025, 4095, 4096, 4097, 5000, 32000, 50257, 128001]


@TYPES
@pytest.mark.parametrize("vocab", VOCABS)
def test_vocabularies(gemm, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    rows = 6 if vocab < 20000 else 3
    x = logits(g, rows, vocab, dtype)
    t = [0.5 + 0.3 * i for i in range(rows)]
    run(gemm, x, uniform(g, rows), what="plain")
    run(gemm, x, uniform(g, rows), t, what="temperature")
    run(gemm, x, uniform(g, rows), t, [1, 2, 50, 300, 1000, 0][:rows], what="top_k")
    run(gemm, x, uniform(g, rows), t, None, [0.05, 0.5, 0.9, 0.97, 0.999, 1.0][-rows:], what="top_p")
    run(gemm, x, uniform(g, rows), t, None, None, [0.0, 1e-6, 0.01, 0.1, 0.9, 1.0][:rows], what="min_p")
    run(gemm, x, uniform(g, rows), t, [5, 40, 100, 1, 2000, 0][:rows], [0.9, 0.8, 0.95, 0.5, 0.99, 0.7][:rows],
        [0.0, 0.05, 0.01, 0.0, 0.001, 0.3][:rows], what="all")
    run(gemm, x, uniform(g, rows), [0.0] * rows, what="greedy")


@TYPES
@pytest.mark.parametrize("vocab", [700, 9000, 40000])
def test_flat_rows(gemm, dtype, vocab):
    """Hot or plain normal logits: a nucleus of most of the vocabulary."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(5, vocab, generator=g).to(dtype)
    t = [1.0, 2.0, 5.0, 100.0, math.inf]
    for p in (0.3, 0.9, 0.999):
        run(gemm, x, uniform(g, 5), t, None, [p] * 5, what=f"flat top_p {p}")
        run(gemm, x, uniform(g, 5), t, [vocab // 2] * 5, [p] * 5, what=f"flat half, top_p {p}")
    run(gemm, x, uniform(g, 5), t, [vocab - 3, vocab, vocab + 9, vocab // 3, 5000], what="flat top_k")
    run(gemm, x, uniform(g, 5), t, None, None, [0.5, 0.1, 0.6, 0.97, 1.0], what="flat min_p")


@TYPES
@pytest.mark.parametrize("vocab", [1, 5, 1000, 6000, 20000])
def test_equal_logits(gemm, dtype, vocab):
    """Ties go to the lowest index, exactly: whole numbers of equal weights."""
    x = torch.full((4, vocab), -2.5, dtype=dtype)
    for u in (0.0, 0.25, 0.5, 0.999):
        run(gemm, x, [u] * 4, what="equal")
        tokens = run(gemm, x, [u] * 4, None, [1, 2, 7, vocab], what="equal top_k")
        assert all(int(n) < k for n, k in zip(tokens, (1, 2, 7, vocab)))
        run(gemm, x, [u] * 4, None, None, [0.125, 0.25, 0.5, 0.75], what="equal top_p")
        run(gemm, x, [u] * 4, None, [vocab // 2, 3, 4, 0], [0.5, 0.5, 0.25, 1.0], [1.0, 0.5, 0.0, 0.0], what="equal all")


@TYPES
@pytest.mark.parametrize("vocab", [600, 9000, 30000])
def test_few_levels(gemm, dtype, vocab):
    """Logits of few values: the cut lies among many equal ones."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randint(0, 5, (6, vocab), generator=g).to(dtype)
    x[1, 3::2] = -math.inf
    x[2] = -x[2] * 0.0  # zeros of both signs: equal
    k = [1, vocab // 3, 2, vocab // 4, 10, vocab - 1]
    run(gemm, x, uniform(g, 6), None, k, what="levels top_k")
    run(gemm, x, uniform(g, 6), None, None, [0.1, 0.3, 0.5, 0.7, 0.9, 0.99], what="levels top_p")
    run(gemm, x, uniform(g, 6), None, k, [0.9, 0.3, 0.5, 0.7, 0.9, 0.99], [0.0, 0.02, 0.0, 0.1, 0.5, 1.0], what="levels all")


@TYPES
def test_masked_infinite_and_nan_logits(gemm, dtype):
    g = torch.Generator().manual_seed(1)
    for vocab in (50, 5000):
        x = logits(g, 10, vocab, dtype)
        x[0] = -math.inf
        x[1] = math.nan
        x[2, :] = -math.inf
        x[2, vocab - 1] = -3.0
        x[3, 7] = math.inf
        x[4, 3::3] = math.inf
        x[5, 1::2] = math.nan
        x[6, 5] = torch.finfo(dtype).max
        x[6, 9] = torch.finfo(dtype).min
        x[7] = torch.finfo(dtype).min  # a mask of the type's lowest value, one token left
        x[7, 11] = 0.5
        x[8] = torch.finfo(dtype).min  # none left: all alike
        tiny = torch.finfo(dtype).tiny
        x[9] = torch.arange(vocab) * tiny  # logits that differ by next to nothing
        for k, p, m in ((None, None, None), (4, None, None), (None, 0.7, None), (3, 0.7, 0.1), (vocab - 1, 0.99, None)):
            run(gemm, x, uniform(g, 10), None, None if k is None else [k] * 10, None if p is None else [p] * 10,
                None if m is None else [m] * 10, what=f"masked {vocab} {k} {p} {m}")
        run(gemm, x, uniform(g, 10), [0.0] * 10, what="masked greedy")


def test_numbers_at_their_ends(gemm):
    g = torch.Generator().manual_seed(2)
    x = logits(g, 12, 3000)
    run(gemm, x, [0.0, 1.0, -1.0, 2.0, math.nan, 1 - 2.0 ** -24, 2.0 ** -30, math.inf, -math.inf, 0.5, 0.5, 0.5], what="u")
    u = uniform(g, 12)
    run(gemm, x, u, [0.0, -1.0, math.nan, 1e-30, 1e-3, 0.01, 50.0, 1e30, math.inf, 1e-45, 0.1, 3e38], what="temperatures")
    run(gemm, x, u, None, [-5, 0, 1, 2, 3, 2999, 3000, 3001, 1 << 30, -(1 << 31), (1 << 31) - 1, 64], what="top_k")
    run(gemm, x, u, None, None, [0.0, -1.0, 1e-30, 1e-7, 0.5, 1 - 2.0 ** -24, 1.0, 1.5, math.inf, 0.999999, 0.2, 0.8], what="top_p")
    run(gemm, x, u, None, None, None, [0.0, -1.0, 1e-30, 1e-13, 0.5, 1.0, 1.5, math.inf, 1e-3, 2.0 ** -20, 0.2, 0.8], what="min_p")


def test_one_far_above_the_rest(gemm):
    """Weights that end before the second logit, and a row whose big logits lie all in one thread's places."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 20000, generator=g)
    x[0, 777] = 500.0
    x[1, ::4096] = 30.0 + torch.arange(len(x[1, ::4096]))
    x[2, 100:3000] += 20.0  # more near the top than the threads' own largest tell
    x[3, :4096] = 9.0
    for k, p in ((None, None), (50, None), (None, 0.9), (700, 0.95), (4000, None)):
        run(gemm, x, uniform(g, 4), None, None if k is None else [k] * 4, None if p is None else [p] * 4, what=f"{k} {p}")


def test_the_largest_vocabulary(gemm):
    g = torch.Generator().manual_seed(4)
    x = logits(g, 2, 1 << 20, BF)
    run(gemm, x, uniform(g, 2), None, [100, 0], [1.0, 0.9], what="2^20")
    run(gemm, torch.zeros(2, 1 << 20), [0.75, 0.3], None, None, [1.0, 0.5], what="2^20 alike")


def test_draws_follow_the_probabilities(gemm):
    """All of u's range over a row: each token as often as its weight says, within a step of the grid at either end."""
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, -math.inf, 0.5]).repeat(1 << 14, 1)
    u = (torch.arange(1 << 14) + 0.5) / (1 << 14)
    tokens, _ = gemm.sample_tokens(x.to(DEV), u.to(DEV))
    share = torch.bincount(tokens.cpu().long(), minlength=6) / (1 << 14)
    assert ((share - torch.softmax(x[0].double(), 0)).abs() <= 2.0 ** -13).all()


@TYPES
def test_strided_and_unaligned_rows(gemm, dtype):
    g = torch.Generator().manual_seed(5)
    x = logits(g, 5, 5003, dtype)
    u = torch.rand(5, generator=g).to(DEV)
    k, p = torch.tensor([3, 50, 0, 900, 7], dtype=torch.int32, device=DEV), torch.full((5,), 0.9, device=DEV)
    want = gemm.sample_tokens(x.to(DEV), u, top_k=k, top_p=p)
    wide = torch.full((5, 5010), math.inf, dtype=dtype, device=DEV)
    for offset in (0, 1, 3):
        view = wide[:, offset:offset + 5003]
        view.copy_(x)
        tokens, logprobs = torch.zeros(5, dtype=torch.int32, device=DEV), torch.zeros(5, device=DEV)
        back = gemm.sample_tokens(view, u, top_k=k, top_p=p, tokens=tokens, logprobs=logprobs)
        assert back[0] is tokens and back[1] is logprobs
        assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])
        wide.fill_(math.inf)


def test_the_same_inputs_give_the_same_tokens(gemm):
    g = torch.Generator().manual_seed(6)
    x, u = logits(g, 300, 9000).to(DEV), torch.rand(300, generator=g).to(DEV)
    p = torch.full((300,), 0.98, device=DEV)
    want = gemm.sample_tokens(x, u, top_p=p)
    for _ in range(3):
        got = gemm.sample_tokens(x, u, top_p=p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    each = [gemm.sample_tokens(x[i:i + 1], u[i:i + 1], top_p=p[:1])[0] for i in range(0, 300, 37)]
    assert torch.equal(torch.cat(each), want[0][::37])  # a row does not depend on its neighbours


def test_refusals(gemm):
    x, u = torch.zeros(3, 40, device=DEV), torch.zeros(3, device=DEV)
    refused = lambda kind, *a, **kw: pytest.raises(kind, gemm.sample_tokens, *a, **kw)  # noqa: E731
    refused(ValueError, x.half(), u)
    refused(ValueError, x[0], u)
    refused(ValueError, x.cpu(), u)
    refused(ValueError, x, u[:2])
    refused(ValueError, x, u.double())
    refused(ValueError, x, u.cpu())
    refused(ValueError, x.T.contiguous().T, u)
    for name in ("temperature", "top_p", "min_p"):
        refused(ValueError, x, u, **{name: u[:1]})
        refused(ValueError, x, u, **{name: u.int()})
    refused(ValueError, x, u, top_k=u)
    refused(ValueError, x, u, tokens=u)
    refused(ValueError, x, u, logprobs=u.int())
    refused(abi.SQ8Error, x[:, :0], u)
    refused(abi.Unsupported, torch.zeros(1, (1 << 20) + 1, device=DEV), u[:1])
    tokens, logprobs = gemm.sample_tokens(x[:0], u[:0])
    assert tokens.shape == (0,) and logprobs.shape == (0,)


def test_a_graph_s_replays(gemm):
    ctx = sq.TensorGEMM.make(0)
    side = torch.cuda.Stream()
    x, u = torch.zeros(7, 6000, device=DEV), torch.zeros(7, device=DEV)
    t, p = torch.ones(7, device=DEV), torch.full((7,), 0.9, device=DEV)
    k = torch.zeros(7, dtype=torch.int32, device=DEV)
    tokens, logprobs = torch.zeros(7, dtype=torch.int32, device=DEV), torch.zeros(7, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.set_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ctx.sample_tokens(x, u, temperature=t, top_k=k, top_p=p, tokens=tokens, logprobs=logprobs)
        for i in range(5):
            x.copy_(4 * torch.randn(x.shape, device=DEV))
            u.copy_(torch.rand(7, device=DEV))
            k.fill_(40 * i)
            t.fill_(0.5 * i)
            graph.replay()
            side.synchronize()
            want = ctx.sample_tokens(x, u, temperature=t, top_k=k, top_p=p)
            assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1]), i
        ctx.set_stream(torch.cuda.default_stream())
    torch.cuda.current_stream().wait_stream(side)
