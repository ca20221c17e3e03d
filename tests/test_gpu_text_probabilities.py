"""The paged attention's probabilities are not rounded to bf16: its output is the formula's, in 64 bits, rounded once.

Before its one rounding an output is within e of the formula's, so it lies between the formula's less e and plus e, both
rounded (rounding keeps order). e: a probability is within 2^-17 of its own in the product with v, and within 2^-23 · (8 +
|s| log2 e) of the formula's by its exponent's rounding and the exponential, |s| < 8 here: under 2^-18; its score's own sum
(dim products of 8 by 8 bits, exact, added in fp32) is off by dim · 2^-24 · Σ|q k| · scale, Σ|q k| < 1.5 dim on these inputs,
under 2^-11 at dim 128 were every rounding the largest and alike, and 2^-15 with ten times their root mean square, which
is taken. The sums of up to 4000 terms in fp32 of one sign: 2^-24 · 64 (32 steps of a lane, the joins). So e = 2^-14 Σ p|v|.
"""
import math

import pytest
import torch

import siliconed_amd as sq

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
F8 = torch.float8_e4m3fn


def cache_of(g, n, page, heads, dim, dtype):
    """One sequence's cache of n tokens, in order; keys and values in 64 bits."""
    pages = -(-n // page)
    k, v = (torch.randn(pages, page, heads, dim, generator=g, device=DEV).to(dtype) for _ in "kv")
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    return sq.PagedCache(k, v), table, k.double().flatten(0, 1)[:n], v.double().flatten(0, 1)[:n]


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("n,page,heads,dim", [(2, 16, 2, 128), (3, 5, 1, 64), (40, 16, 2, 64), (777, 16, 8, 128), (600, 24, 2, 256),
                                              (4000, 64, 1, 128)])
def test_outputs_are_the_formula_s_rounded_once(gemm, dtype, n, page, heads, dim):
    g = torch.Generator(device=DEV).manual_seed(n + dim)
    cache, table, k, v = cache_of(g, n, page, heads, dim, dtype)
    q = torch.randn(1, 4 * heads, dim, generator=g, device=DEV).to(BF)
    got = gemm.paged_attention(q, cache, table, torch.tensor([n], dtype=torch.int32, device=DEV))[0].double()
    for h in range(4 * heads):
        p = torch.softmax(k[:, h // 4] @ q[0, h].double() / math.sqrt(dim), 0)
        want, size = p @ v[:, h // 4], p @ v[:, h // 4].abs()
        least, most = ((want + e * 2.0 ** -14 * size).to(BF).double() for e in (-1, 1))
        assert ((least <= got[h]) & (got[h] <= most)).all(), h


@pytest.mark.parametrize("n", [1, 2, 300])
def test_an_infinite_value_is_infinite(gemm, n):
    """An infinity among the values that a sequence holds gives infinities of its sign, whatever bits its probability has."""
    g = torch.Generator(device=DEV).manual_seed(n)
    cache, table, k, v = cache_of(g, n, 16, 1, 64, BF)
    q = torch.randn(1, 8, 64, generator=g, device=DEV).to(BF)
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    clean = gemm.paged_attention(q, cache, table, lengths)
    for i, value in ((3, math.inf), (40, -math.inf)):
        cache.v.flatten(0, 1)[n // 2, 0, i] = value
    got = gemm.paged_attention(q, cache, table, lengths)
    assert (got[..., 3] == math.inf).all() and (got[..., 40] == -math.inf).all()
    rest = [i for i in range(64) if i not in (3, 40)]
    assert torch.equal(got[..., rest], clean[..., rest])
