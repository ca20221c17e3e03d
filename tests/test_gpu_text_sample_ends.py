"""The draw at the ends of what a temperature and a min_p may be, against the definition in 64 bits (test_gpu_text_sample.py)."""
import math

import pytest
import torch

from test_gpu_text_sample import logits, run, uniform

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
TYPES = pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])


@TYPES
@pytest.mark.parametrize("vocab", [4097, 9001, 32001, 50257])
def test_a_nucleus_at_an_infinite_temperature(gemm, dtype, vocab):
    """Every logit but -inf and NaN weighs the same, whatever the row's last run is filled up with: whole numbers, exactly."""
    g = torch.Generator().manual_seed(vocab)
    x = logits(g, 6, vocab, dtype)
    x[1] = torch.randn(vocab, generator=g).to(dtype)  # nothing forbidden
    x[2, 5::7] = math.nan
    x[3, vocab // 3:] = -math.inf
    for p in (0.001, 0.02, 0.05, 0.2, 0.9):
        run(gemm, x, uniform(g, 6), [math.inf] * 6, None, [p] * 6, what=f"infinite, top_p {p}")
        run(gemm, x, uniform(g, 6), [math.inf] * 6, None, [p] * 6, [0.0, 0.5, 1.0, 0.1, 0.0, 0.0], what=f"infinite, top_p {p}, min_p")
    run(gemm, x, uniform(g, 6), [math.inf] * 6, [7, 300, 3000, 0, 4096, vocab], [0.3] * 6, what="infinite, top_k")
    run(gemm, x, uniform(g, 6), [math.inf] * 6, what="infinite")


@TYPES
@pytest.mark.parametrize("vocab", [1000, 9001, 30000])
def test_a_nucleus_of_logits_of_every_size(gemm, dtype, vocab):
    """Differences past the type's largest number, at temperatures that bring them back to units."""
    g = torch.Generator().manual_seed(vocab)
    x = (3.3e38 * (2 * torch.rand(5, vocab, generator=g) - 1)).to(dtype)
    x[1, 3::8] = -math.inf
    for t in (1e37, 5e37, 1e38, 3e38):
        for p in (0.05, 0.5, 0.97):
            run(gemm, x, uniform(g, 5), [t] * 5, None, [p] * 5, what=f"wide {t} top_p {p}")
        run(gemm, x, uniform(g, 5), [t] * 5, [vocab // 3, 5, 0, vocab, 2000], [0.9] * 5, what=f"wide {t} top_k")
        run(gemm, x, uniform(g, 5), [t] * 5, None, None, [0.0, 0.01, 0.1, 0.5, 0.9], what=f"wide {t} min_p")


@pytest.mark.parametrize("vocab", [1000, 9001])
def test_a_nucleus_at_temperatures_of_next_to_nothing(gemm, vocab):
    """Logits that differ by as little."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(4, vocab, generator=g).double()
    for t in (1e-20, 1e-30, 1e-36, 1e-38, 1e-41, 1e-44):
        row = (x * t).float()
        for p in (0.05, 0.5, 0.97):
            run(gemm, row, uniform(g, 4), [t] * 4, None, [p] * 4, what=f"tiny {t} top_p {p}")


@TYPES
@pytest.mark.parametrize("vocab", [3, 700, 9000])
def test_a_min_p_above_one_keeps_the_first(gemm, dtype, vocab):
    """No weight is as much, and the first of the order is always kept: of equal largest logits the lowest index alone."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(6, vocab, generator=g).to(dtype)
    x[0, 1:] = 9.0
    x[1, vocab // 2::2] = 7.5
    x[2] = -2.5
    x[3, vocab - 2:] = math.inf
    x[4, ::2] = -math.inf
    m = [1.5, 1.0 + 2.0 ** -23, math.inf, 2.0, 3e38, 1.0001]
    for u in (0.0, 0.5, 0.999):
        run(gemm, x, [u] * 6, None, None, None, m, what=f"min_p {u}")
        run(gemm, x, [u] * 6, [2.0, 0.5, math.inf, 1.0, 1e-3, 1.0], [0, 2, 5, vocab, 3, 0], [0.9, 1.0, 0.5, 0.7, 0.99, 0.0], m, what=f"all {u}")
        run(gemm, x, [u] * 6, None, None, None, [1.0] * 6, what=f"one {u}")  # every one of the largest
