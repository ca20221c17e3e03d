"""A value that every row of its tile sees may be an infinity or a NaN: it is in its own column of the outputs, and the other columns
keep their bits, under a cap as without one."""
import math

import pytest
import torch

from test_gpu_text_chunk import Batch, normal

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,rows", [(128, 300), (64, 1200), (256, 300)])
def test_prompts(gemm, softcap, causal, dim, rows):
    g = torch.Generator().manual_seed(rows + dim)
    q, k, v = (normal(g, rows, h, dim).to(BF) for h in (8, 2, 2))
    options = dict(softcap=softcap, causal=causal)
    clean = gemm.prompt_attention(q, k, v, **options)
    for value in (math.nan, math.inf):
        wild = v.clone()
        wild[0, 1, 5] = value  # the first token, which every row sees
        if not causal:
            wild[rows - 1, 1, 5] = wild[rows // 2, 1, 5] = value
        got = gemm.prompt_attention(q, k, wild, **options)
        own = got[:, 4:, 5].clone()
        assert (torch.isnan(own) if math.isnan(value) else own == value).all(), value
        got[:, 4:, 5] = clean[:, 4:, 5]
        assert torch.equal(got, clean), value


@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 24)])
def test_chunks(gemm, softcap, dtype, dim, page):
    b = Batch([(70, 400), (100, 129)], 8, 2, dim, page, dtype)
    for table in (None, b.roomy()):
        clean = b.run(gemm, table, softcap=softcap)
        pool = b.cache.v.view(torch.uint8)
        kept = pool.clone()
        for t in (0, 70, 131):  # of the first sequence's cached tokens
            place = int(b.table[0, t // page]), t % page, 1
            pool[place][:2 if dtype == BF else 1] = 0xFF  # a NaN
        got = b.run(gemm, table, softcap=softcap)
        pool.copy_(kept)
        assert torch.isnan(got[:70, 4:, 0]).all()
        got[:70, 4:, 0] = clean[:70, 4:, 0]
        assert torch.equal(got, clean)
