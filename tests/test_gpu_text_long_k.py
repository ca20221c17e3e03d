"""Block-scaled products of many rows whose K is long: more than 64 blocks in one workgroup, and split over several, against
the formula in 64 bits at rows from all over and the edges."""
import pytest
import torch

from f8_shapes import LONG, operands, product

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("m,k,n,glu", [s for s, *_ in LONG])
def test_long_sums(gemm, m, k, n, glu, out):
    a, sx, w, sw, bias = operands(m, k, n, glu, m + k + n)
    got = gemm.product_f8(a, sx, w, sw, bias=bias, epilogue="silu_glu" if glu else None, out_dtype=out)
    g = torch.Generator().manual_seed(m)
    rows = torch.unique(torch.cat([torch.randint(0, m, (12,), generator=g), torch.tensor([0, 1, m - 2, m - 1])])).to(DEV)
    want, bound = product(a[rows], sx[rows], w, sw, bias, glu, out)
    off = (got[rows].double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
