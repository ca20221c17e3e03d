"""fp8 weights by 128×128 blocks (`weight_scale_inv`) out of a safetensors file: what they stand for, what is refused, and the
product of a staged one. The recognizer still refuses their files, as the reference does, and says who reads them."""
import numpy as np
import pytest

from siliconed_amd.safetensors_q8 import Refused, Safetensors, block_operands, recognize, stage_blocks
from test_safetensors_q8 import _bf16, _f32, _write


def layer(n, k, seed):
    r = np.random.default_rng(seed)
    codes = r.integers(0, 127, (n, k)).astype(np.uint8)
    return codes, r.uniform(1e-3, 2e-3, (-(-n // 128), -(-k // 128))).astype(np.float32)


def tensors(name, codes, scale):
    return {name: ("F8_E4M3", list(codes.shape), codes.tobytes()), name + "_scale_inv": ("F32", list(scale.shape), _f32(scale))}


def test_operands_are_the_published_bytes(tmp_path):
    a, sa = layer(300, 200, 1)
    b, sb = layer(128, 128, 2)
    half = sb.view(np.uint32) >> 16  # a bf16 scale: the fp32 one's upper half
    t = {**tensors("a.weight", a, sa), "b.weight": ("F8_E4M3", [128, 128], b.tobytes()),
         "b.weight_scale_inv": ("BF16", [1, 1], _bf16(sb))}
    st = Safetensors(_write(tmp_path, "w.safetensors", t))
    q, s = block_operands(st, "a.weight")
    assert np.array_equal(q, a) and np.array_equal(s, sa) and s.dtype == np.float32
    q, s = block_operands(st, "b.weight")
    assert np.array_equal(q, b) and np.array_equal(s.view(np.uint32), half << 16)
    with pytest.raises(Refused, match="stage_blocks"):
        recognize(st)


def test_refusals(tmp_path):
    a, sa = layer(300, 200, 1)
    st = Safetensors(_write(tmp_path, "w.safetensors", {
        **tensors("ok.weight", a, sa),
        "lone.weight": ("F8_E4M3", [300, 200], a.tobytes()),
        "wide.weight": ("F8_E4M3", [300, 200], a.tobytes()), "wide.weight_scale_inv": ("F32", [2, 2], _f32(sa[:2])),
        "int.weight": ("I8", [300, 200], a.tobytes()), "int.weight_scale_inv": ("F32", [3, 2], _f32(sa)),
        "odd.weight": ("F8_E4M3", [300, 200], a.tobytes()), "odd.weight_scale_inv": ("I32", [3, 2], bytes(24)),
        "flat.weight": ("F8_E4M3", [60000], a.tobytes()), "flat.weight_scale_inv": ("F32", [469], bytes(1876))}))
    block_operands(st, "ok.weight")
    for name, why in (("none.weight", "no such tensor"), ("lone.weight", "no such tensor"), ("wide.weight", r"\[3, 2\] blocks"),
                      ("int.weight", "I8"), ("odd.weight", "type I32"), ("flat.weight", "not an fp8")):
        with pytest.raises(Refused, match=why):
            block_operands(st, name)
    with pytest.raises(ValueError):
        stage_blocks(st)


@pytest.mark.gpu
def test_staged_weights_give_their_products(gemm, tmp_path):
    import torch
    from f8_shapes import product
    k = 400
    one, gate, up = layer(200, k, 3), layer(300, k, 4), layer(300, k, 5)
    st = Safetensors(_write(tmp_path, "w.safetensors", {**tensors("o.weight", *one), **tensors("g.weight", *gate),
                                                        **tensors("u.weight", *up)}))
    x = torch.randn(9, k, device="cuda").to(torch.bfloat16)
    codes, sx = gemm.quantize_groups(x)
    for names, parts, glu in ((("o.weight",), (one,), False), (("g.weight", "u.weight"), (gate, up), True)):
        w, scale = stage_blocks(st, *names)
        for t, i in ((w.view(torch.uint8), 0), (scale, 1)):
            assert torch.equal(t.cpu(), torch.from_numpy(np.concatenate([p[i] for p in parts])))
        got = gemm.product_f8_quantized(x, w, scale, epilogue="silu_glu" if glu else None, out_dtype=torch.float32)
        want, bound = product(codes, sx, w, scale, None, glu, torch.float32)
        assert ((got.double() - want).abs() <= bound).all()
    with pytest.raises(Refused, match="halves"):
        stage_blocks(st, "o.weight", "u.weight")
