"""Sizes at the end of what 32 bits count: refused before anything is launched, or done in parts. (Expanded tensors: their rows or heads
all lie in one place, so that such sizes take no memory.)"""
import pytest
import torch

import siliconed_amd as sq
from siliconed_amd import _abi as abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
MOST = (1 << 31) - 1


@pytest.mark.parametrize("dim", [64, 24, 10])
def test_more_heads_of_a_token_than_32_bits_count(gemm, dim):
    many = torch.zeros(1, 1, dim, dtype=BF, device=DEV).expand(1, MOST, dim)
    few = torch.zeros(1, 2, dim, dtype=BF, device=DEV)
    at, table = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dim, device=DEV)
    cache = sq.PagedCache(*(torch.zeros(1, 16, 2, dim, dtype=BF, device=DEV) for _ in "kv"))
    for append in (gemm.append_kv, gemm.norm_append_kv):
        with pytest.raises(abi.Unsupported):
            append(many, few, few, cache, at, at, table, q_out=many)
    with pytest.raises(abi.Unsupported):
        gemm.norm_rotate(many, few, q_out=many, k_out=few)


def test_windows_that_begin_before_what_32_bits_count(gemm):
    """2^31 - 4097 new tokens of a sequence that holds fewer: with a window their places less it would wrap."""
    tokens = MOST - 4096
    q = torch.zeros(1, 1, 8, dtype=BF, device=DEV).expand(tokens, 1, 8)
    cache = sq.PagedCache(*(torch.zeros(1, 64, 1, 8, dtype=BF, device=DEV) for _ in "kv"))
    pages, length = torch.zeros(1, 256, dtype=torch.int32, device=DEV), torch.full((1,), 16000, dtype=torch.int32, device=DEV)
    with pytest.raises(abi.Unsupported):
        gemm.chunk_attention(q, cache, pages, length, window=16000, out=q)


def test_more_rows_of_logits_than_one_launch_takes(gemm):
    """A launch is of fewer than 2^32 threads: 2^23 rows of 512. Two equal logits: the first for numbers under a half."""
    rows = (1 << 23) + 3
    x, u = torch.zeros(rows, 2, device=DEV), torch.rand(rows, device=DEV)
    k = torch.zeros(rows, dtype=torch.int32, device=DEV)
    k[::5] = 1
    tokens, logprobs = gemm.sample_tokens(x, u, top_k=k)
    want = (u >= 0.5).int()
    want[::5] = 0
    assert torch.equal(tokens, want)
    assert (logprobs[::5] == 0).all() and ((logprobs + 0.6931472).abs() < 1e-6)[k == 0].all()


def test_more_heads_than_one_launch_takes(gemm):
    tokens, dim = (1 << 28) + 1, 64
    q = torch.zeros(1, 1, dim, dtype=BF, device=DEV).expand(tokens, 4, dim)
    with pytest.raises(abi.Unsupported):
        gemm.norm_rotate(q, q_out=q)
    k = q[:, :1]
    slots = torch.full((tokens,), -1, dtype=torch.int32, device=DEV)
    cache = sq.PagedCache(*(torch.zeros(1, 16, 1, dim, dtype=BF, device=DEV) for _ in "kv"))
    table = torch.zeros(1, dim, device=DEV)
    for append in (gemm.append_kv, gemm.norm_append_kv):
        with pytest.raises(abi.Unsupported):
            append(q, k, k, cache, slots, slots, table, q_out=q)


def test_more_prompts_than_one_launch_takes(gemm):
    """A tile of each kv head for every sequence, were none empty."""
    q, k = torch.zeros(4, 8, 64, dtype=BF, device=DEV), torch.zeros(4, 8, 64, dtype=BF, device=DEV)
    with pytest.raises(abi.Unsupported):
        gemm.prompt_attention(q, k, k, torch.zeros((1 << 21) + 2, dtype=torch.int32, device=DEV))
