"""ctypes binding of the C ABI (include/siliconed_q8.h) in libsiliconed_q8.so.

The library is loaded from this package's directory only; a missing library is an error, never a
fallback: there is no CPU path behind these functions.
"""
from __future__ import annotations

import ctypes
import os

PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG, "libsiliconed_q8.so")

# Values of include/siliconed_q8.h.
OK, EINVAL, EUNSUPPORTED, ENODEVICE, ECAPACITY = 0, 1, 2, 3, 4
BF16, F32, INT8, FP8_E4M3, F16 = 1, 2, 3, 4, 5
KN, NK, PACKED, PACKED_GLU = 0, 1, 2, 3
SCALE_TENSOR, SCALE_COLUMNS, SCALE_BLOCKS, SCALE_ROWS = 0, 1, 2, 3
EPI_NONE, EPI_GELU_TANH, EPI_SILU_GLU, EPI_SITU_GLU = 0, 1, 2, 3

# Every symbol the header declares, with (restype, argtypes).
_P, _I, _I64, _D = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_double


class PagedCacheArgs(ctypes.Structure):
    """struct sq8_paged_cache."""

    _fields_ = [("k", _P), ("v", _P),
                *((name, _I64) for name in ("k_page", "k_token", "k_head", "v_page", "v_token", "v_head")),
                ("k_scale", _P), ("v_scale", _P),
                *((name, _I) for name in ("dtype", "pages", "page", "kv_heads", "dim"))]


SIGNATURES = {
    "sq8_create": (_I, [_I, _P, ctypes.POINTER(_P)]),
    "sq8_destroy": (_I, [_P]),
    "sq8_set_stream": (_I, [_P, _P]),
    "sq8_supports": (_I, [_P, _I, _I, _I, _I, _I, _I]),
    "sq8_linear": (_I, [_P, _P, _I, _I64, _P, _I, _I, _I64, _P, _I, _P, _I, _P, _I, _I64, _I, _I, _I,
                        ctypes.POINTER(_D)]),
    "sq8_linear_qkv": (_I, [_P, _P, _I, _I64, _P, _I, _I, _I64, _P, _I, _P, _P, _P, _P, _I, _I64, _I, _I, _I, _I,
                            ctypes.POINTER(_D)]),
    "sq8_linear_rotated": (_I, [_P, _P, _I, _I64, _I, _P, _I, _I, _I64, _P, _I, _P, _I, _P, _I, _I64, _I, _I, _I,
                                ctypes.POINTER(_D)]),
    "sq8_rotate_groups": (_I, [_P, _P, _I, _I64, _P, _I, _I64, _I, _I, _I]),
    "sq8_dequantize_rotated": (_I, [_P, _P, _I64, _I, _I, _I, _P, _I, _I, _P, _I64]),
    "sq8_quantize_rows": (_I, [_P, _P, _I, _I64, _I, _I, _I, _P, _I64, _P]),
    "sq8_linear_w8a8": (_I, [_P, _P, _I64, _P, _P, _I, _I64, _P, _I, _P, _I, _P, _I, _I64, _I, _I, _I,
                             ctypes.POINTER(_D)]),
    "sq8_linear_quantized": (_I, [_P, _P, _I, _I64, _I, _P, _I, _I64, _P, _I, _P, _I, _P, _I, _I64, _I, _I, _I,
                                  ctypes.POINTER(_D)]),
    "sq8_linear_quantized_static": (_I, [_P, _P, _I, _I64, _I, _P, _I, _I64, _P, _I, _P, _I, _P, _I, _I64, _I, _I,
                                         _I, ctypes.POINTER(_D)]),
    "sq8_static_scratch_bytes": (_I64, []),
    "sq8_linear_w8a8_qkv": (_I, [_P, _P, _I64, _P, _P, _I, _I64, _P, _I, _P, _P, _P, _P, _I, _I64, _I, _I, _I, _I,
                                 ctypes.POINTER(_D)]),
    "sq8_norm_modulate_rotated": (_I, [_P, _P, _I64, _P, _P, _P, ctypes.c_float, _I, _P, _I64, _P, _I64, _I, _I]),
    "sq8_norm_modulate_quantized": (_I, [_P, _P, _I64, _P, _P, _P, ctypes.c_float, _I, _P, _I64, _P, _P, _I64, _I, _I]),
    "sq8_linear_residual": (_I, [_P, _P, _I, _I64, _P, _I, _I, _I64, _P, _I, _P, _P, _P, _I64, _I, _I, _I,
                                 ctypes.POINTER(_D)]),
    "sq8_linear_w8a8_residual": (_I, [_P, _P, _I64, _P, _P, _I, _I64, _P, _I, _P, _P, _P, _I64, _I, _I, _I,
                                      ctypes.POINTER(_D)]),
    "sq8_packed_bytes": (_I64, [_I, _I, _I]),
    "sq8_pack_weight": (_I, [_P, _P, _I, _I64, _I, _I, _I, _P]),
    "sq8_linear_f32": (_I, [_P, _P, _I64, _I, _P, _I, _I, _I64, _P, _I, _I, _I, _P, _I, _P, _I, _I64, _I, _I, _I,
                            ctypes.POINTER(ctypes.c_double)]),
    "sq8_linear_bf16_weight": (_I, [_P, _P, _I, _I64, _P, _I, _I64, _P, _I64, _I, _I, _I, ctypes.POINTER(_D)]),
    "sq8_linear_blocks": (_I, [_P, _P, _I, _I64, _P, _I, _I64, _P, _I, _I, _P, _I, _P, _I, _I64, _I, _I, _I,
                               ctypes.POINTER(ctypes.c_double)]),
    "sq8_packed_blocks_bytes": (_I64, [_I, _I, _I]),
    "sq8_pack_blocks": (_I, [_P, _P, _I, _I64, _P, _I, _I, _I, _I, _I, _P]),
    "sq8_dequantize": (_I, [_P, _P, _I, _I64, _I64, _P, _I, _I, _I64, _I64, _P]),
    "sq8_round_bf16": (_I, [_P, _P, _P, _I64]),
    "sq8_norm_modulate": (_I, [_P, _P, _I64, _P, _P, _P, ctypes.c_float, _P, _I64, _I, _I]),
    "sq8_rms_rows": (_I, [_P, _P, _I64, _I64, _I, _P, ctypes.c_float]),
    "sq8_gated_residual": (_I, [_P, _P, _I64, _P, _I, _I64, _P, _I64, _I]),
    "sq8_add_norm_quantized": (_I, [_P, _P, _I, _I64, _P, _I, _I64, _P, _I64, _P, ctypes.c_float, _P, _I, _I64, _P, _I64,
                                    _I, _I]),
    "sq8_quantize_groups": (_I, [_P, _P, _I, _I64, _I, _I, _P, _I64, _P, _I64]),
    "sq8_linear_f8": (_I, [_P, _P, _I64, _P, _I64, _P, _I64, _P, _I64, _P, _I, _P, _I, _I64, _I, _I, _I,
                           ctypes.POINTER(_D)]),
    "sq8_linear_f8_quantized": (_I, [_P, _P, _I, _I64, _P, _I64, _P, _I64, _P, _I, _P, _I, _I64, _I, _I, _I,
                                     ctypes.POINTER(_D)]),
    "sq8_append_kv": (_I, [_P, _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64,
                           ctypes.POINTER(PagedCacheArgs), _P, _P, _P, _I64, _I, _I, _I, _I, _I]),
    "sq8_paged_attention": (_I, [_P, _P, _I64, _I64, ctypes.POINTER(PagedCacheArgs), _P, _I64, _I, _P, ctypes.c_float,
                                 ctypes.c_float, _I, _P, _I64, _I64, _I, _I]),
    "sq8_device": (_I, [_P]),
    "sq8_synchronize": (_I, [_P]),
    "sq8_status_string": (ctypes.c_char_p, [_I]),
    "sq8_abi_version": (_I, []),
}

# The entries that text_bind.cpp calls, in the order of its Entries.
TEXT_ENTRIES = ("sq8_add_norm_quantized", "sq8_quantize_groups", "sq8_linear_f8", "sq8_linear_f8_quantized",
                "sq8_append_kv", "sq8_paged_attention", "sq8_device")

_lib = None


class SQ8Error(RuntimeError):
    """A call the library refused (status > 0) or a HIP error (status < 0)."""

    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {status_string(status)} (status {status})")


class Unsupported(SQ8Error):
    """The library does not run this configuration: the caller keeps its widened route."""


def load() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is not built: run `python -c 'import __graft_entry__ as g; g.build()'`")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def __getattr__(name: str):
    """`text`: the text decoder's operators' native calls (text_bind.cpp), loaded when they are first asked for. The rest
    of the library does without that module, which is built against one version of torch."""
    if name != "text":
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    lib = load()
    import torch  # noqa: F401  (the libraries that the module is linked against)

    try:
        from . import _text_bind
    except ImportError as e:
        raise ImportError(f"the text operators' host module does not load ({e}): build it again with "
                          "`python -c 'import __graft_entry__ as g; g.build()'`") from e
    _text_bind.bind(*(ctypes.cast(getattr(lib, entry), _P).value for entry in TEXT_ENTRIES))
    globals()["text"] = _text_bind
    return _text_bind


def status_string(status: int) -> str:
    return load().sq8_status_string(status).decode()


def check(status: int, what: str) -> None:
    if status == OK:
        return
    if status in (EUNSUPPORTED, ENODEVICE):
        raise Unsupported(status, what)
    raise SQ8Error(status, what)
