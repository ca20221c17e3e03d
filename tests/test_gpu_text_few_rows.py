"""Block-scaled products of a few rows at a decoder's sizes of K and N, against the formula in 64 bits: from codes, and from
values that are quantized on the way or before."""
import pytest
import torch

from f8_shapes import FEW, VALUES, operands, product

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OUTS = pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])


def check(got, want, bound):
    off = (got.double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


@OUTS
@pytest.mark.parametrize("m,k,n,glu", [s for s, _ in FEW])
def test_codes(gemm, m, k, n, glu, out):
    a, sx, w, sw, bias = operands(m, k, n, glu, m + k + n)
    for b in (None, bias):
        got = gemm.product_f8(a, sx, w, sw, bias=b, epilogue="silu_glu" if glu else None, out_dtype=out)
        check(got, *product(a, sx, w, sw, b, glu, out))


@OUTS
@pytest.mark.parametrize("m,k,n", [s for s, _ in VALUES])
def test_values(gemm, m, k, n, out):
    """The formula is on the codes that quantize_groups gives, which has its own tests."""
    _, _, w, sw, bias = operands(1, k, n, False, m + k + n)
    x = torch.randn(m, k, device=DEV, generator=torch.Generator(device=DEV).manual_seed(k)).to(torch.bfloat16)
    x *= torch.exp(torch.arange(m, device=DEV) - 3.0)[:, None]  # rows that are not of one size
    a, sx = gemm.quantize_groups(x)
    for b in (None, bias):
        got = gemm.product_f8_quantized(x, w, sw, bias=b, out_dtype=out)
        check(got, *product(a, sx, w, sw, b, False, out))


@pytest.mark.parametrize("m", [1, 8, 16])
def test_a_row_of_nan_stays_alone(gemm, m):
    """Values and weights that are NaN make their row and their column NaN, and nothing else."""
    _, _, w, sw, _ = operands(1, 1024, 200, False, 5)
    x = torch.randn(m, 1024, device=DEV).to(torch.bfloat16)
    x[m - 1, 700] = float("nan")
    w.view(torch.uint8)[77, 1000] = 0x7F
    got = torch.isnan(gemm.product_f8_quantized(x, w, sw))
    want = torch.zeros(m, 200, dtype=torch.bool, device=DEV)
    want[m - 1], want[:, 77] = True, True
    assert torch.equal(got, want)
