"""Arguments at the ends of their ranges: what the attention gives for them is what it gives for the plain value they mean."""
import math

import pytest
import torch

import siliconed_amd as sq

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
F8 = torch.float8_e4m3fn


def held(batch, page, most, heads, dim, dtype=BF, seed=0):
    """A cache whose pages `table` [batch, most] scatters, and queries of two heads a key head."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    k, v = (torch.randn(batch * most, page, heads, dim, generator=g, device=DEV).to(dtype) for _ in "kv")
    table = torch.randperm(batch * most, generator=g, device=DEV).to(torch.int32).view(batch, most)
    q = torch.randn(batch, 2 * heads, dim, generator=g, device=DEV).to(BF)
    return sq.PagedCache(k, v), table, q


def lengths(*n):
    return torch.tensor(n, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
def test_a_cap_that_no_score_comes_near_is_none(gemm, dtype):
    cache, table, q = held(3, 16, 20, 2, 64, dtype)
    n = lengths(300, 1, 0)
    want = gemm.paged_attention(q, cache, table, n)
    for cap in (math.inf, 3.4e38, 1e31):
        assert torch.equal(gemm.paged_attention(q, cache, table, n, softcap=cap), want), cap
    # Just inside: the formula's own value, s to a relative 2^-22 for |s| < 30, whose exponential is within 2^-16.
    near = gemm.paged_attention(q, cache, table, n, softcap=1e30)
    assert ((near.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -15 * 5).all()


def test_a_cap_of_nothing_averages(gemm):
    """Scores within 1e-20 of 0: every exponential is 1 in fp32, and the output the values' mean."""
    cache, table, q = held(2, 16, 8, 1, 64)
    want = gemm.paged_attention(q, cache, table, lengths(100, 3), scale=0.0)
    for cap in (1e-20, 1e-39, 1e-45):
        assert torch.equal(gemm.paged_attention(q, cache, table, lengths(100, 3), softcap=cap), want), cap


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
def test_a_window_past_every_length_is_none(gemm, dtype):
    """Up to the largest int, the usual "no window"; the work is split as without one, so the bits are the same."""
    cache, table, q = held(2, 16, 300, 1, 128, dtype)
    n = lengths(4777, 130)
    want = gemm.paged_attention(q, cache, table, n)
    for window in (2 ** 31 - 1, 2 ** 31 - 31, 2 ** 31 - 32, 2 ** 30):
        assert torch.equal(gemm.paged_attention(q, cache, table, n, window=window), want), window


def test_the_stride_of_a_single_row_is_nothing(gemm):
    """One token's query, one key head, one page: torch leaves the stride of a dimension of one anything, odd values too."""
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn(2, 16, 1, 64, generator=g, device=DEV).to(BF) for _ in "kv")
    q = torch.randn(1, 4, 64, generator=g, device=DEV).to(BF)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    want = gemm.paged_attention(q, sq.PagedCache(k, v), table, lengths(29))
    odd = [t.as_strided(t.shape, (1024, 64, 3, 1)) for t in (k, v)]
    out = torch.empty(4 * 64, dtype=BF, device=DEV).as_strided((1, 4, 64), (257, 64, 1))
    gemm.paged_attention(q.as_strided(q.shape, (257, 64, 1)), sq.PagedCache(*odd), table, lengths(29), out=out)
    assert torch.equal(out, want)
    one = gemm.paged_attention(q[:, :1].as_strided((1, 1, 64), (5, 3, 1)), sq.PagedCache(*odd), table, lengths(29))
    assert torch.equal(one, want[:, :1])
    last = [t[1:].as_strided((1, 16, 1, 64), (7, 64, 3, 1), t[1:].storage_offset()) for t in (k, v)]
    first = gemm.paged_attention(q, sq.PagedCache(*last), torch.zeros_like(table), lengths(16))
    assert torch.equal(first, gemm.paged_attention(q, sq.PagedCache(k, v), table, lengths(16)))
