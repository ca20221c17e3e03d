"""Block-scaled products wide enough for each tile of many rows, against the formula in 64 bits.

Bounds: a sum in fp32 of a block's four instructions and of K / 128 scaled blocks rounds at most K / 128 + 8 times, each
by 2^-24 of the terms' sizes summed (doubled: an instruction's own sum may round more than once); the instructions of a
bf16 C also drop what is under 2^-13 of the largest of eight products, at most 7 of them. A gate's error reaches the output
by the slope of SiLU, under 1.1, times up, an up's by SiLU(gate), and their product; SiLU itself and its product are
within 2^-20 of theirs. A bf16 C is then rounded by 2^-8 at most (a half unit would be 2^-9).
"""
import pytest
import torch

import siliconed_amd as sq

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn


def formula(a, sx, w, sw):
    """The sums, and the sizes of their terms and of the largest of each eight summed, in 64 bits."""
    y = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    size, largest = torch.zeros_like(y), torch.zeros_like(y)
    for b in range(-(-a.shape[1] // 128)):
        at = slice(128 * b, min(a.shape[1], 128 * b + 128))
        scale = sx[:, b, None].double() * sw[:, b].double().repeat_interleave(128)[: w.shape[0]]
        x, z = a[:, at].double(), w[:, at].double()
        y += scale * (x @ z.T.contiguous())
        size += scale * (x.abs() @ z.abs().T.contiguous())
        for c in range(0, x.shape[1], 8):
            largest += scale * (x[:, None, c:c + 8].float() * z[None, :, c:c + 8].float()).abs().amax(-1)
    return y, size, largest


# (rows, K, N) that a bf16 C takes in 256 x 256 tiles; 128 x 128 at two a CU and at one; 64 x 128; 64 x 64; all with edges.
SHAPES = [(2100, 528, 4100), (1000, 656, 6100), (1000, 1040, 4000), (250, 400, 8100), (200, 272, 2500)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("glu", [False, True], ids=["plain", "glu"])
def test_tiles_follow_the_formula(m, k, n, out, glu):
    g = torch.Generator(device=DEV).manual_seed(m + n)
    h = n // 2 if glu else n
    rows, blocks = -(-h // 128), -(-k // 128)
    a = (torch.randn(m, k, generator=g, device=DEV) * 60).to(F8)
    w = (torch.randn(n, k, generator=g, device=DEV) * 60).to(F8)
    sx = torch.rand(m, blocks, generator=g, device=DEV) * 2e-2 + 1e-3
    sw = torch.rand(rows * (2 if glu else 1), blocks, generator=g, device=DEV) * 1e-3 + 1e-4
    bias = torch.randn(n, generator=g, device=DEV)
    got = sq.context(0).product_f8(a, sx, w, sw, bias=bias, epilogue="silu_glu" if glu else None, out_dtype=out).double()

    def half(part):
        at = slice(part * h, part * h + h)
        y, size, largest = formula(a, sx, w[at], sw[part * rows:part * rows + rows])
        y += bias[at].double()
        off = 2 * (k / 128 + 8) * 2.0 ** -24 * (size + bias[at].double().abs())
        if out == torch.bfloat16:
            off += 7 * 2.0 ** -13 * largest
        return y, off

    y, bound = half(0)
    if glu:
        u, up = half(1)
        s = torch.nn.functional.silu(y)
        y, bound = s * u, 1.1 * bound * u.abs() + s.abs() * up + 1.1 * bound * up + 2.0 ** -20 * (s * u).abs()
    if out == torch.bfloat16:
        bound += 2.0 ** -8 * (y.abs() + bound)
    assert ((got - y).abs() <= bound).all()
