"""Tensors on another GPU than the context's are refused before the library is called. There is one GPU here: the entries
are replaced by stand-ins that say the context is on another and note what reaches them."""
import ctypes

import pytest
import torch

import siliconed_amd as sq
from siliconed_amd import _abi as abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
F8 = torch.float8_e4m3fn


@pytest.fixture
def elsewhere(gemm):
    """Calls bound to a context on "cuda:1"; yields the list of entries reached."""
    lib, reached = abi.load(), []
    kept = []

    def stand_in(name):
        restype, argtypes = abi.SIGNATURES[name]

        def entry(*_):
            if name == "sq8_device":
                return 1
            reached.append(name)
            return abi.EINVAL
        kept.append(ctypes.CFUNCTYPE(restype, *argtypes)(entry))
        return ctypes.cast(kept[-1], ctypes.c_void_p).value

    abi.text.bind(*(stand_in(name) for name in abi.TEXT_ENTRIES))
    yield reached
    abi.text.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in abi.TEXT_ENTRIES))


def test_tensors_on_another_gpu_are_refused(gemm, elsewhere):
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    cache = sq.PagedCache(z(2, 16, 2, 64), z(2, 16, 2, 64))
    for call in (lambda: gemm.add_norm_quantized(z(2, 128), f32(128)),
                 lambda: gemm.add_norm_quantized(z(2, 128), f32(128), residual=f32(2, 128), dtype=torch.int8),
                 lambda: gemm.quantize_groups(z(2, 128)),
                 lambda: gemm.product_f8(z(2, 128, dtype=F8), f32(2, 1), z(4, 128, dtype=F8), f32(1, 1)),
                 lambda: gemm.product_f8_quantized(z(2, 128), z(4, 128, dtype=F8), f32(1, 1), bias=f32(4)),
                 lambda: gemm.append_kv(z(3, 4, 64), z(3, 2, 64), z(3, 2, 64), cache, i32(3), i32(3), f32(9, 64)),
                 lambda: gemm.paged_attention(z(3, 4, 64), cache, i32(3, 2), i32(3))):
        with pytest.raises(ValueError, match="context's GPU"):
            call()
    assert not elsewhere


def test_the_context_s_own_gpu_is_not(gemm):
    assert abi.load().sq8_device(gemm._h) == 0 and abi.load().sq8_device(None) == -1
    codes, scales = gemm.quantize_groups(torch.ones(2, 128, device=DEV))
    assert (codes.float() == 448).all()


def test_a_cache_on_another_gpu_is_refused():
    pool = torch.zeros(2, 16, 1, 64, dtype=BF, device=DEV)
    cache = sq.PagedCache(pool, pool.clone())
    other = sq.TensorGEMM(None, 1)  # no context: what the cache's check has to come before
    q, i32 = torch.zeros(1, 1, 64, dtype=BF, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="context's GPU"):
        other.paged_attention(q, cache, i32, i32[0])
    with pytest.raises(ValueError, match="context's GPU"):
        other.append_kv(q, q, q, cache, i32[0], i32[0], torch.zeros(1, 64, device=DEV))
    with pytest.raises(ValueError):
        sq.PagedCache(pool.to(F8), pool.to(F8), torch.ones(1), None)  # a scale off the pools' GPU
