"""Chunks of few rows keep their probabilities in two bf16 parts: against the formula in 64 bits with the tolerance that this leaves
(narrow_chunks.py), which rounded ones fail (test_narrow_chunks.py)."""
import pytest
import torch

from attend_reference import within
from narrow_chunks import attended_narrow
from test_gpu_text_chunk import Batch

pytestmark = pytest.mark.gpu
BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def check(gemm, b, **options):
    print(f"chunks {b.chunks[:6]} q {tuple(b.q.shape)} pools {tuple(b.cache.k.shape)} {b.cache.k.dtype} {options}", flush=True)
    out = b.run(gemm, **options)
    for i, (n, m) in enumerate(b.chunks):
        lo = int(b.starts[i])
        want, tol = attended_narrow(b.q[lo:lo + n], *b.values[i], m - n, dead=b.dead[i], **options)
        within(out[lo:lo + n], want, tol, f"sequence {i}: {n} of {m}")


# At most 16, 32 and 64 rows of a sequence and kv head, in tables of their lengths: the narrow kernel's, also where parts are joined.
@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (128, 24), (96, 16), (256, 16)])
def test_chunks_of_few_rows(gemm, dtype, dim, page):
    check(gemm, Batch([(4, 200), (0, 5), (1, 70), (3, 3)], 8, 2, dim, page, dtype))
    check(gemm, Batch([(8, 90), (4, 1300)], 8, 2, dim, page, dtype), softcap=20.0)
    check(gemm, Batch([(2, 5000)], 4, 2, dim, page, dtype), window=700)
    if dim <= 128:
        check(gemm, Batch([(16, 700), (16, 40)], 8, 2, dim, page, dtype))
