"""The native calls' own checks (text_bind.cpp), which answer before anything reaches the library."""
import pytest
import torch

from siliconed_amd import _abi as abi


@pytest.fixture
def text():
    abi.load()
    return abi.text


def test_counts_and_kinds_of_arguments(text):
    x = torch.zeros(2, 128)
    with pytest.raises(TypeError):
        text.quantize_groups(None, x, None)
    with pytest.raises(TypeError):
        text.quantize_groups(None, [1.0, 2.0], None, None)
    with pytest.raises(TypeError):
        text.quantize_groups(7, x, None, None)  # not a context's handle
    with pytest.raises(TypeError):
        text.append_kv(None, x, x, x, b"short", x, x, x, None, False)  # not a cache's description
    with pytest.raises(TypeError):
        text.bind(1, 2)
    with pytest.raises(ValueError):
        text.bind(*([0] * len(abi.TEXT_ENTRIES)))


def test_tensors_off_the_gpu_are_refused(text):
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    codes = x.to(torch.float8_e4m3fn)
    s = torch.ones(2, 1)
    for call in (lambda: text.quantize_groups(None, x, None, None),
                 lambda: text.add_norm_quantized(None, x, torch.ones(128), 1e-6, None, None, False, None, None),
                 lambda: text.product_f8(None, codes, s, codes, s[:1], None, False, None, False, False),
                 lambda: text.product_f8(None, x, None, codes, s[:1], None, False, None, False, False)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_numbers_must_be_numbers(text):
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        text.add_norm_quantized(None, x, torch.ones(128), "small", None, None, False, None, None)
