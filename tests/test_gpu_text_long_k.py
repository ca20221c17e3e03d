"""Block-scaled products of many rows whose K is long: more than 64 blocks in one workgroup, and split over several, against
the formula in 64 bits at rows from all over and the edges; and the bits of rows in chunks."""
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


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("k,n,glu", [(8192, 2048, False), (8208, 1026, True), (1040, 4100, False), (640, 8196, True)])
def test_tall_products_have_the_same_bits_in_chunks(gemm, k, n, glu, out):
    """Chunks of 4096 rows and more of a weight of more than 1024 columns; the tiles differ among these."""
    m = 9000
    a, sx, w, sw, bias = operands(m, k, n, glu, k + n)
    call = lambda *at: gemm.product_f8(a[slice(*at)], sx[slice(*at)], w, sw, bias=bias, epilogue="silu_glu" if glu else None, out_dtype=out)  # noqa: E731
    whole = call(0, m)
    for at in ((0, 4097), (4097, m), (0, 4096), (1, 5001), (3000, 8192)):
        assert torch.equal(call(*at), whole[slice(*at)]), at
