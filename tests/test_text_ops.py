"""The text decoder operators' host checks, which answer without touching a GPU."""
import ctypes

import pytest
import torch

import siliconed_amd as sq
from siliconed_amd import _abi as abi


def test_null_contexts_are_refused():
    lib = abi.load()
    assert lib.sq8_add_norm_quantized(None, None, 1, 0, None, 0, 0, None, 0, None, 0.0, None, 4, 0, None, 0, 1, 1) == abi.EINVAL
    assert lib.sq8_quantize_groups(None, None, 1, 0, 1, 1, None, 0, None, 0) == abi.EINVAL
    assert lib.sq8_linear_f8(None, None, 0, None, 0, None, 0, None, 0, None, 0, None, 1, 0, 1, 1, 1, None) == abi.EINVAL
    assert lib.sq8_linear_f8_quantized(None, None, 9, 0, None, 0, None, 0, None, 0, None, 1, 0, 1, 1, 1,
                                       None) == abi.EUNSUPPORTED
    cache = abi.PagedCacheArgs()
    assert lib.sq8_append_kv(None, None, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, ctypes.byref(cache), None, None, None, 0,
                             0, 0, 0, 1, 1) == abi.EINVAL
    assert lib.sq8_paged_attention(None, None, 0, 0, ctypes.byref(cache), None, 0, 1, None, 1.0, 0.0, 0, None, 0, 0, 1,
                                   1) == abi.EINVAL


def test_the_cache_argument_is_the_header_s_struct():
    """Two pointers, six strides, two pointers, five ints."""
    assert ctypes.sizeof(abi.PagedCacheArgs) == 2 * 8 + 6 * 8 + 2 * 8 + 6 * 4  # padded to a multiple of 8
    assert abi.PagedCacheArgs.dtype.offset == 80


def test_tensors_off_the_gpu_are_refused():
    pool = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        sq.PagedCache(pool, pool)
