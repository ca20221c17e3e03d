"""Values that are not finite through the text operators: a product of their codes has to be as unfinite as the formula's."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.mark.parametrize("cols", [8, 129, 1000, 4096, 20001])
def test_int8_norm_keeps_what_is_not_finite(gemm, cols):
    """int8 has no code for a NaN: the row's scale carries it, and so does every product of the row. An infinite weight
    makes its row's scale infinite. The other rows are as without them."""
    torch.manual_seed(cols)
    x, r = torch.randn(6, cols, device=DEV).to(BF), torch.randn(6, cols, device=DEV)
    w = 1 + 0.1 * torch.randn(cols, device=DEV)
    clean, clean_scales, _ = gemm.add_norm_quantized(x, w, 1e-6, residual=r.clone(), dtype=torch.int8)
    x[1, cols - 1] = math.nan
    x[2, cols // 2] = math.inf
    r[4, 0] = -math.inf
    codes, scales, _ = gemm.add_norm_quantized(x, w, 1e-6, residual=r.clone(), dtype=torch.int8)
    assert torch.isnan(scales).tolist() == [False, True, True, False, True, False]
    for i in (0, 3, 5):
        assert torch.equal(codes[i], clean[i]) and scales[i] == clean_scales[i]
    if cols % 8 == 0:
        q = torch.randint(-127, 128, (16, cols), dtype=torch.int8, device=DEV)
        y = gemm.product_w8a8(codes, scales, q, torch.ones(16, device=DEV))
        assert torch.isnan(y).all(dim=1).tolist() == [False, True, True, False, True, False]
        assert torch.isfinite(y[[0, 3, 5]]).all()
    w[cols // 3] = math.nan
    _, scales, _ = gemm.add_norm_quantized(x, w, 1e-6, residual=r.clone(), dtype=torch.int8)
    assert torch.isnan(scales).all()
    w[cols // 3] = math.inf
    _, scales, _ = gemm.add_norm_quantized(x[:1], w, 1e-6, residual=r[:1].clone(), dtype=torch.int8)
    assert torch.isinf(scales).all()
