"""Prompt and chunk attention at the ends of what a cap and a scale may be, against the formula in 64 bits without the cap.

attend_reference's tolerance holds a cap's error relative to the cap, which says nothing here: below a cap c of 1e28 or more tanh is its
argument to 2^-60, so the score is the uncapped one, off by the roundings on its way in and out of units of the cap, 4 · 2^-24 of
it beside those that the tolerance counts. With |s| < 20, as here, that is 4 · 1.45 · 20 · 2^-24 < 2^-17 of A = Σ p|v| / Σ p, and the
tolerance holds 2^-8 of A: a factor of 1 + 2^-8 is more than enough."""
import math

import pytest
import torch

from attend_reference import attended, within
from test_gpu_text_chunk import Batch, normal

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F8 = torch.bfloat16, torch.float8_e4m3fn
CAPS = [1e28, 1e29, 1e30, 2.0 ** 100, 1e31, 1e38, math.inf]


def check_prompt(gemm, lengths, qh, kvh, dim, *, by=1.0, scale=None, causal=True, **options):
    """Queries and keys times `by`."""
    print(f"prompt {lengths} {qh} {kvh} {dim} by {by} scale {scale} {causal} {options}", flush=True)
    g = torch.Generator().manual_seed(sum(lengths) + dim + qh)
    q, k, v = (normal(g, sum(lengths), h, dim) for h in (qh, kvh, kvh))
    q, k, v = (q * by).to(BF), (k * by).to(BF), v.to(BF)
    starts = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=DEV)
    out = gemm.prompt_attention(q, k, v, starts, scale=scale, causal=causal, **options)
    for lo, n in zip(starts.tolist(), lengths):
        want, tol = attended(q[lo:lo + n], k[lo:lo + n], v[lo:lo + n], 0, scale=scale, causal=causal)
        within(out[lo:lo + n], want, tol * (1 + 2.0 ** -8), f"{n} rows from {lo}")


def check_chunk(gemm, b, *, scale=None, **options):
    """A tight table and a roomy one: the narrow kernel's tiles and the wide one's."""
    print(f"chunks {b.chunks} {tuple(b.q.shape)} {b.cache.k.dtype} scale {scale} {options}", flush=True)
    for what, table in (("tight", None), ("roomy", b.roomy())):
        out = b.run(gemm, table, scale=scale, **options)
        for i, (n, m) in enumerate(b.chunks):
            lo = int(b.starts[i])
            want, tol = attended(b.q[lo:lo + n], *b.values[i], m - n, scale=scale)
            within(out[lo:lo + n], want, tol * (1 + 2.0 ** -8), f"sequence {i}: {n} of {m}, {what}")


@pytest.mark.parametrize("cap", CAPS)
def test_a_cap_that_no_score_comes_near_is_none(gemm, cap):
    for dim in (64, 128, 200, 256):
        check_prompt(gemm, [140, 40], 8, 2, dim, softcap=cap)
    check_prompt(gemm, [700, 300], 32, 8, 128, softcap=cap)
    check_prompt(gemm, [150], 4, 4, 64, causal=False, softcap=cap)
    check_prompt(gemm, [150], 4, 4, 64, scale=-0.2, softcap=cap)
    for dtype in (BF, F8):
        check_chunk(gemm, Batch([(1, 1), (9, 140), (40, 500)], 8, 2, 128, 16, dtype), softcap=cap)
        check_chunk(gemm, Batch([(3, 90), (30, 200)], 4, 1, 64, 24, dtype), softcap=cap, scale=-0.2)
        check_chunk(gemm, Batch([(20, 90)], 4, 1, 256, 16, dtype), softcap=cap)


def test_a_large_cap_on_the_largest_tiles(gemm):
    check_prompt(gemm, [4100], 16, 8, 128, softcap=1e30)


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
def test_a_large_cap_of_scores_by_a_small_scale(gemm, dtype):
    """The product of both scales over the cap is what matters, not the scores' size."""
    b = Batch([(9, 140), (40, 500)], 8, 2, 128, 16, dtype)
    b.q = (b.q.float() * 2.0 ** 16).to(BF)
    for cap in (1e24, 1e27, 1e30):
        check_chunk(gemm, b, softcap=cap, scale=2.0 ** -16 / math.sqrt(128))


@pytest.mark.parametrize("cap", [0.0, 5.0, 1e10, 1e29, 1e30, math.inf])
def test_a_scale_of_nothing_averages(gemm, cap):
    check_prompt(gemm, [140, 1, 33], 8, 2, 128, scale=0.0, softcap=cap)
    check_prompt(gemm, [140, 1, 33], 8, 2, 128, scale=0.0, softcap=cap, by=1e17)
    check_prompt(gemm, [300], 4, 4, 64, scale=0.0, softcap=cap, causal=False)
    for dtype in (BF, F8):
        check_chunk(gemm, Batch([(1, 1), (9, 140), (40, 500)], 8, 2, 128, 16, dtype), scale=0.0, softcap=cap)


@pytest.mark.parametrize("by,scale", [(1e15, 1e-31), (1e17, 1e-35), (1e17, -1e-35), (4e17, 1e-36), (1e18, 1e-37)])
def test_a_tiny_scale_of_large_heads(gemm, by, scale):
    """Queries and keys whose products near fp32's end, scaled to scores of a few units."""
    for dim in (64, 128):
        check_prompt(gemm, [140, 40], 8, 2, dim, by=by, scale=scale)
    check_prompt(gemm, [150], 4, 4, 128, by=by, scale=scale, causal=False)
    b = Batch([(9, 140), (40, 500)], 8, 2, 128, 16, BF)
    b.q = (b.q.float() * by).to(BF)
    b.cache.k.copy_((b.cache.k.float() * by).to(BF))
    b.values = [[(k * by).to(BF).float(), v] for k, v in b.values]
    check_chunk(gemm, b, scale=scale)


@pytest.mark.parametrize("cap", [1e-20, 1e-39, 1e-45])
def test_a_cap_of_nothing_averages(gemm, cap):
    """Scores within 1e-18 of 0: every exponential is 1 in fp32."""
    q, k, v = (normal(torch.Generator().manual_seed(7 + h), 150, h, 64).to(BF) for h in (8, 2, 2))
    assert torch.equal(gemm.prompt_attention(q, k, v, softcap=cap), gemm.prompt_attention(q, k, v, scale=0.0))
    for dtype in (BF, F8):
        b = Batch([(1, 1), (9, 140), (40, 500)], 8, 2, 128, 16, dtype)
        for table in (None, b.roomy()):
            assert torch.equal(b.run(gemm, table, softcap=cap), b.run(gemm, table, scale=0.0))
