"""append_kv by runs of four: heads, or turned parts of them, that are a multiple of 8 and not of 16; and rows at odd places."""
import pytest
import torch

import siliconed_amd as sq
import test_gpu_text_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
F8 = torch.float8_e4m3fn
DTYPES = pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])


@DTYPES
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(120, 120), (40, 40), (40, 24), (80, 40), (72, 0), (72, 8), (8, 8), (24, 16)])
def test_runs_of_four(gemm, dtype, interleaved, dim, rot):
    """The formula's check of test_gpu_text_ops, on heads of these sizes."""
    ops.test_append(gemm, dtype, interleaved, 37, 6, 2, dim, rot, 16)


def moved(t, by):
    """A copy of t on the GPU whose first value lies `by` elements past an aligned address."""
    size = t.element_size()
    raw = torch.zeros(t.numel() * size + 64, dtype=torch.uint8, device=DEV)
    found = raw[by * size:(by + t.numel()) * size].view(t.dtype).view(t.shape)
    found.view(torch.uint8).copy_(t.view(torch.uint8))
    return found


@DTYPES
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 32), (120, 120), (40, 24), (18, 10)])
@pytest.mark.parametrize("by", [1, 3])
def test_rows_at_odd_places(gemm, dtype, interleaved, dim, rot, by):
    """The same bits wherever the rows, the table, the pools and the output begin."""
    g = torch.Generator(device=DEV).manual_seed(dim + by)
    tokens, heads, kv, page, pages = 19, 3, 2, 8, 4
    q, k, v = (torch.randn(tokens, h, dim, generator=g, device=DEV).to(BF) for h in (heads, kv, kv))
    angles = 6.3 * torch.rand(30, rot // 2, generator=g, device=DEV)
    table = torch.cat([angles.cos(), angles.sin()], 1)
    positions = torch.randint(0, 30, (tokens,), generator=g, dtype=torch.int32, device=DEV)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens].to(torch.int32)
    scale = torch.full((kv,), 0.05, device=DEV) if dtype == F8 else None
    empty = torch.zeros(pages, page, kv, dim, dtype=BF, device=DEV).to(dtype)

    def run(place):
        pools = [place(empty), place(empty)]
        out = place(torch.zeros_like(q))
        cache = sq.PagedCache(*pools, scale, scale)
        gemm.append_kv(place(q), place(k), place(v), cache, positions, slots, place(table), q_out=out, interleaved=interleaved)
        return [out.view(torch.int16), *(p.view(torch.uint8) for p in pools)]

    for got, want in zip(run(lambda t: moved(t, by)), run(torch.clone)):
        assert torch.equal(got, want)
