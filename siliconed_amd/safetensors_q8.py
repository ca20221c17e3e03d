"""Published 8-bit weights in safetensors files, recognized and handed to the product.

Restates two parts of the reference's forge:
  * the safetensors reader's bounds (Tests/SiliconedTests/HostileFilesTests.swift:43-95 — a file
    shorter than its length field, a header length past the file or past 100 MB, data offsets out of
    order or past the data, a shape that is not a size, bytes that do not match the shape);
  * `QuantizedLayouts.recognize` (Sources/Siliconed/Forge/Quantization.swift:297-347, 430-720) for the
    layouts whose weight this library multiplies — the 8-bit ones kept as published, `w = q · s`:
    ComfyUI "scaled" and `comfy_quant` (`<l>.weight` F8_E4M3 or I8 with `<l>.weight_scale` or
    `<l>.scale_weight`, one for the tensor or one per row; `int8_tensorwise` with `convrot`), torchao
    (`<l>._weight_qdata` + `<l>._weight_scale`, described in the metadata), SDNQ (`<l>.weight` I8 +
    `<l>.scale` [N, 1]), and a plain fp8 cast. Refused, the whole file with it, as there: a 4-bit
    layer, mxfp8, fp8 E5M2, fp8 by 128×128 blocks (`weight_scale_inv`), an asymmetric int8, a scale
    of another shape, a scale whose products could be subnormal. Siliconed's own SQ files are read at
    their 8-bit tier (SQ8: per-row int8 codes of the weight rotated by groups of 256); GGUF's blocks
    are another container, not read here.

A recognized weight is `[N, K]` (published rows = outputs): `product_operands` gives the codes and
the fp32 scale (per output, or one) ready for `TensorGEMM.pack(..., layout="nk")` and
`TensorGEMM.product(..., rotation=group)`, and `stage` puts them on the device; `to_map` writes
them as a `.silicon` map ([K, N], the scale after the values).

A text decoder's fp8 checkpoint by 128×128 blocks has no such weight (the reference refuses the file): its layers are
read one by one, `stage_blocks`, for `TensorGEMM.product_f8`.
"""
from __future__ import annotations

import json
import os
import struct
from dataclasses import dataclass, field
from typing import Optional

import numpy as np

INT64_MAX = (1 << 63) - 1
_DTYPE_SIZES = {"F64": 8, "F32": 4, "F16": 2, "BF16": 2, "I64": 8, "I32": 4, "I16": 2, "I8": 1, "U8": 1,
                "BOOL": 1, "F8_E4M3": 1, "F8_E5M2": 1, "F8_E8M0": 1, "U16": 2, "U32": 4, "U64": 8}


def _int_list(v) -> bool:
    return isinstance(v, list) and all(isinstance(d, int) and not isinstance(d, bool) for d in v)
FOUR_BIT_FORMATS = ("nvfp4", "mxfp4", "int4", "uint4", "fp4", "nf4")


class SafetensorsError(Exception):
    """A safetensors file refused by its header (Safetensors.Failure.badHeader)."""


class Refused(Exception):
    """A file whose 8-bit layout this reader refuses, with the reference's reason."""


@dataclass
class Entry:
    name: str
    dtype: str
    shape: list
    begin: int
    end: int

    @property
    def bytes(self) -> int:
        return self.end - self.begin

    @property
    def count(self) -> int:
        c = 1
        for d in self.shape:
            c *= d
        return c


class Safetensors:
    """A safetensors file: its entries (in the order of their bytes), metadata and tensor bytes
    (memory-mapped). Safetensors.init (Sources/Siliconed/Safetensors.swift:60-137): every number
    of the header bounded before it is used."""

    MAXIMUM_HEADER = 100_000_000

    def __init__(self, path: str):
        self.path = path
        size = os.path.getsize(path)
        if size <= 8:
            raise SafetensorsError(f"{path}: {size} bytes cannot hold a safetensors header (an 8-byte length and JSON)")
        with open(path, "rb") as f:
            n = struct.unpack("<Q", f.read(8))[0]
            if n > INT64_MAX or n > self.MAXIMUM_HEADER or n > size - 8:
                raise SafetensorsError(f"header length {n} is out of bounds (a file of {size} bytes; headers hold up to "
                                       f"{self.MAXIMUM_HEADER} bytes)")
            try:
                header = json.loads(f.read(n))
            except (ValueError, UnicodeDecodeError):
                raise SafetensorsError("not a JSON object") from None
        if not isinstance(header, dict):
            raise SafetensorsError("not a JSON object")
        self.data_start = 8 + n
        data = size - self.data_start
        meta = header.pop("__metadata__", None)
        self.metadata = ({str(k): v if isinstance(v, str) else json.dumps(v) for k, v in meta.items()}
                         if isinstance(meta, dict) else {})
        entries = []
        for name, e in header.items():
            dtype = e.get("dtype") if isinstance(e, dict) else None
            shape = e.get("shape") if isinstance(e, dict) else None
            offs = e.get("data_offsets") if isinstance(e, dict) else None
            if (not isinstance(dtype, str) or not _int_list(shape) or not _int_list(offs) or len(offs) != 2):
                raise SafetensorsError(f"{name} is incomplete")
            if dtype not in _DTYPE_SIZES:
                raise SafetensorsError(f"safetensors: {name} has an unknown dtype {dtype}")
            if not (0 <= offs[0] <= offs[1] <= data):
                raise SafetensorsError(f"{name}: data_offsets {offs} outside the {data} bytes of data")
            expected = _DTYPE_SIZES[dtype]
            for d in shape:
                expected = expected * d if d >= 0 else -1
                if expected < 0 or expected > INT64_MAX:
                    raise SafetensorsError(f"{name}: shape {shape} as {dtype} is not a size")
            if offs[1] - offs[0] != expected:
                raise SafetensorsError(f"{name}: {offs[1] - offs[0]} bytes for {shape} as {dtype}")
            entries.append(Entry(name, dtype, list(shape), offs[0], offs[1]))
        entries.sort(key=lambda e: e.begin)
        self.entries = {e.name: e for e in entries}
        self.order = [e.name for e in entries]
        self._data = (np.memmap(path, dtype=np.uint8, mode="r", offset=self.data_start) if data > 0
                      else np.zeros(0, np.uint8))

    def raw(self, name: str) -> np.ndarray:
        e = self.entries[name]
        return self._data[e.begin:e.end]

    def array(self, name: str) -> np.ndarray:
        """The tensor's values (bf16 and fp16 widened to fp32 exactly; 8-bit codes as int8 / uint8)."""
        e = self.entries[name]
        b = np.array(self.raw(name))
        if e.dtype == "F32":
            v = b.view(np.float32)
        elif e.dtype == "BF16":
            v = (b.view(np.uint16).astype(np.uint32) << 16).view(np.float32)
        elif e.dtype == "F16":
            v = b.view(np.float16).astype(np.float32)
        elif e.dtype == "I8":
            v = b.view(np.int8)
        else:
            v = b
        return v.reshape(e.shape)


@dataclass
class QuantizedGroup:
    """An 8-bit weight as published (Forge/Quantization.swift's QuantizedGroup): the values' entry
    [N, K], its kind (int8 / float8_e4m3), its scale's entry (None: a plain fp8 cast), one scale per
    row (output) or one for the tensor, the convrot group (0: none), the publisher's format."""
    values: str
    kind: str
    scale: Optional[str]
    per_row: bool
    format: str
    rotation: int = 0


@dataclass
class Recognized:
    groups: dict = field(default_factory=dict)
    consumed: set = field(default_factory=set)
    notes: list = field(default_factory=list)


def _scale_type(dtype: str) -> Optional[str]:
    return {"F32": "float32", "BF16": "bfloat16", "F16": "float16"}.get(dtype)


def _number(v) -> Optional[int]:
    """A JSON number read as an integer, as Foundation's NSNumber bridging reads it (bool: 0/1)."""
    if isinstance(v, bool):
        return int(v)
    if isinstance(v, int):
        return v
    if isinstance(v, float) and v == int(v):
        return int(v)
    return None


def _flag(v) -> bool:
    return bool(_number(v)) if v is not None else False


def _convrot_group(js: dict, layer: str) -> int:
    """QuantizedLayouts.convrotGroup (Quantization.swift:369-379): 0 without `convrot`, else its group
    (256 by default), the flag and the size read at the top level or under `params`."""
    params = js.get("params") if isinstance(js.get("params"), dict) else {}
    if not _flag(js["convrot"] if "convrot" in js else params.get("convrot")):
        return 0
    size = js["convrot_groupsize"] if "convrot_groupsize" in js else params.get("convrot_groupsize")
    g = 256 if size is None else _number(size)
    if g not in (4, 16, 64, 256):
        raise Refused(f"{layer}: convrot group {size} — only a power of 4 up to 256 is read")
    return g


def _check_subnormal(st: Safetensors, scale: str, kind: str, rotation: int = 0) -> None:
    """QuantizedLayouts.checkSubnormal (Quantization.swift:387-403): no product below 2^-126. The
    smallest nonzero |code| is 1 (int8) or 2^-9 (e4m3's smallest subnormal), 1/sqrt(G) once rotated."""
    smallest = np.float32(1.0 if kind == "int8" else 2.0 ** -9) / np.sqrt(np.float32(rotation or 1))
    v = st.array(scale).astype(np.float32).reshape(-1)
    bad = (v != 0) & (np.abs(v) * smallest < np.float32(2.0 ** -126))
    if bad.any():
        raise Refused(f"{scale}: the scale {v[bad][0]} times the smallest code is a subnormal fp32 number, which "
                      f"the device and the host may round differently; the layout is refused")


def _json_bytes(st: Safetensors, name: str):
    try:
        js = json.loads(bytes(st.raw(name)))
    except (ValueError, UnicodeDecodeError):
        return None
    return js if isinstance(js, dict) else None


def recognize(st: Safetensors) -> Recognized:
    """The file's 8-bit weights, QuantizedLayouts.recognize (Quantization.swift:430-720) without its
    GGUF branches: groups by the weight's name, the names consumed, notes. Siliconed's own SQ files
    are read at their 8-bit tier only (SQ8, Quantization.swift:449-487); SQ4 / SQ5 codes are 4- and
    5-bit weights, outside this library's product: Refused, as is every layout the reference refuses."""
    r = Recognized()
    order, raw = st.order, st.entries
    # Siliconed's SQ: `<l>.sq.codes`, `.sq.scale`, the tier of each layer in the metadata.
    tiers = None
    if any(n.endswith(".sq.codes") for n in order):
        try:
            tiers = json.loads(st.metadata.get("tiers", ""))
        except ValueError:
            tiers = None
    if isinstance(tiers, dict):
        for name in order:
            if not name.endswith(".sq.codes"):
                continue
            layer = name[: -len(".sq.codes")]
            tier = tiers.get(layer)
            bits = int(tier[2:]) if isinstance(tier, str) and tier[:2] == "SQ" and tier[2:] in ("4", "5", "8") else None
            if bits is None:
                raise Refused(f"{name}: the metadata names no SQ tier (SQ4, SQ5 or SQ8) for these codes")
            codes, sname = raw[name], layer + ".sq.scale"
            sc = raw.get(sname)
            if (sc is None or sc.dtype != "F32" or len(sc.shape) != 1 or len(codes.shape) != 2
                    or codes.shape[0] != sc.shape[0]):
                raise Refused(f"{name}: the SQ{bits} codes come with no fp32 row scales")
            if bits != 8:
                raise Refused(f"{name}: SQ{bits} holds {bits}-bit codes; only the 8-bit tier has a product here")
            if codes.dtype != "I8" or codes.shape[1] % 256 != 0:
                raise Refused(f"{name}: SQ8 {codes.dtype} {codes.shape}")
            _check_subnormal(st, sname, "int8", 256)
            r.consumed.update({name, sname})
            r.groups[layer + ".weight"] = QuantizedGroup(name, "int8", sname, True, "Siliconed SQ8", 256)
            if layer + ".weight" in raw:
                r.consumed.add(layer + ".weight")
    # ComfyUI's per-layer formats: `comfy_quant` tensors, or the metadata's table.
    comfy, rotations = {}, {}
    try:
        table = json.loads(st.metadata.get("_quantization_metadata", ""))
    except ValueError:
        table = None
    if isinstance(table, dict) and isinstance(table.get("layers"), dict):
        comfy.update({k: v for k, v in table["layers"].items() if isinstance(v, dict)})
    for name in order:
        if name.endswith(".comfy_quant"):
            js = _json_bytes(st, name)
            if js is None:
                raise Refused(f"{name}: the `comfy_quant` record does not parse as JSON")
            comfy[name[: -len(".comfy_quant")]] = js
            r.consumed.add(name)
    # ComfyUI's attention preference (`{"attention": "comfy_kitchen_int8"}`): recognized by its exact
    # content and ignored; any other content stays an unknown U8, refused below.
    preferences = 0
    for name in order:
        if name.endswith(".comfy_attention.config") and raw[name].dtype == "U8":
            js = _json_bytes(st, name)
            if js is not None and len(js) == 1 and js.get("attention") == "comfy_kitchen_int8":
                r.consumed.add(name)
                preferences += 1
    if preferences:
        r.notes.append(f"{preferences} ComfyUI attention setting(s) skipped (`comfy_attention.config`, "
                       f"comfy_kitchen_int8): attention is computed in fp32")
    # What is refused before anything is accepted: one 4-bit layer refuses the file.
    for name in order:
        e = raw[name]
        if name.endswith(".weight_scale_2"):
            raise Refused(f"{name} carries a second-level scale (nvfp4, a 4-bit layer); files with any 4-bit layer are refused whole")
        if e.dtype == "U8" and not name.endswith(".comfy_quant") and name not in r.consumed:
            raise Refused(f"{name}: uint8 codes (packed 4-bit or zero-pointed 8-bit) have no product here")
        if e.dtype == "F8_E8M0":
            raise Refused(f"{name}: E8M0 block exponents (mxfp8) have no product here")
        if e.dtype == "F8_E5M2":
            raise Refused(f"{name}: fp8 in E5M2; the product reads E4M3 codes only")
        if name.endswith(".weight_scale_inv"):
            raise Refused(f"{name}: `weight_scale_inv` scales fp8 by 128×128 blocks, which the products of a recognized "
                          f"weight do not take; `stage_blocks` reads such a weight for `product_f8`")
    for layer in sorted(comfy):
        f = comfy[layer].get("format")
        fmt = (f if isinstance(f, str) else "").lower()
        if any(x in fmt for x in FOUR_BIT_FORMATS):
            raise Refused(f"{layer} is a 4-bit layer ({fmt}); files with any 4-bit layer are refused whole")
        if "mxfp8" in fmt:
            raise Refused(f"{layer}: mxfp8 has no product here")
        if fmt not in ("float8_e4m3fn", "int8_tensorwise"):
            raise Refused(f'{layer}: the ComfyUI format "{fmt}" is not one this reader knows')
        g = _convrot_group(comfy[layer], layer)
        if g:
            if fmt != "int8_tensorwise":
                raise Refused(f'{layer}: `convrot` asked of "{fmt}", but ComfyUI applies the rotation to int8_tensorwise weights alone')
            rotations[layer] = g
    if "scaled_fp8" in raw:
        r.consumed.add("scaled_fp8")
    # torchao: `_weight_qdata`, described in the metadata under the weight's name.
    activations_noted = False
    for name in order:
        if not name.endswith("._weight_qdata"):
            continue
        base = name[: -len("._weight_qdata")]
        logical = base + ".weight"
        try:
            js = json.loads(st.metadata[logical])
        except (KeyError, ValueError):
            js = None
        if (not isinstance(js, dict) or not isinstance(js.get("_type"), str)
                or not isinstance(js.get("_data"), dict)):
            raise Refused(f"{name}: torchao parts whose tensor description is missing from the metadata")
        typ, d = js["_type"], js["_data"]
        names = js.get("_tensor_data_names")
        parts = set(names) if isinstance(names, list) and all(isinstance(x, str) for x in names) else set()
        kind = {("Float8Tensor", "F8_E4M3"): "float8_e4m3", ("Int8Tensor", "I8"): "int8"}.get((typ, raw[name].dtype))
        if kind is None:
            raise Refused(f"{logical}: a torchao {typ} of {raw[name].dtype} has no product here")
        if not parts <= {"qdata", "scale", "zero_point"} or "scale" not in parts:
            raise Refused(f"{logical}: torchao parts {sorted(parts)} include some beyond qdata, scale and zero_point")
        f8 = d.get("float8_dtype")
        dt = f8.get("_data") if isinstance(f8, dict) else None
        if kind == "float8_e4m3" and isinstance(dt, str) and dt != "float8_e4m3fn":
            raise Refused(f"{logical}: torchao stores its float8 as {dt}; e4m3fn is the one read")
        sname = base + "._weight_scale"
        if sname not in raw or _scale_type(raw[sname].dtype) is None:
            raise Refused(f"{logical}: the torchao scale is absent or of a type that cannot be read")
        shape = raw[name].shape
        block = d.get("block_size") if _int_list(d.get("block_size")) else []
        if len(shape) == 2 and block == [1, shape[1]] and raw[sname].count == shape[0]:
            per_row = True
        elif block == shape and raw[sname].count == 1:
            per_row = False
        else:
            raise Refused(f"{logical}: torchao block {block} on {shape} is neither a row nor the whole tensor")
        # An Int8Tensor's zero point: all zeros for torchao's symmetric weights; checked, not assumed.
        zname = base + "._weight_zero_point"
        if zname in raw:
            z = raw[zname]
            if z.dtype != "I8" or z.count != raw[sname].count:
                raise Refused(f"{logical}: a zero point of {z.dtype} {z.shape} cannot be read")
            zp = np.array(st.raw(zname)).view(np.int8)
            if zp.any():
                i = int(np.argmax(zp != 0))
                raise Refused(f"{logical}: row {i} has zero point {int(zp[i])}; q − z then needs 9 bits, so "
                              f"asymmetric int8 is refused")
            r.consumed.add(zname)
        elif "zero_point" in parts:
            raise Refused(f"{logical}: a zero point is declared and no tensor holds it")
        if isinstance(d.get("act_quant_kwargs"), dict) and not activations_noted:
            activations_noted = True
            r.notes.append("`act_quant_kwargs` (torchao's activation quantization) skipped: the activations stay bf16")
        _check_subnormal(st, sname, kind)
        r.consumed.update({name, sname})
        r.groups[logical] = QuantizedGroup(name, kind, sname, per_row, f"torchao {typ}")
    stray = next((n for n in order if "._weight_" in n and n not in r.consumed), None)
    if stray:
        raise Refused(f"{stray}: this torchao component belongs to no weight that is read")
    # ComfyUI, SDNQ, plain fp8: the values under the weight's own name.
    input_scales = 0
    for name in order:
        e = raw[name]
        # An empty 8-bit tensor (ComfyUI's `scaled_fp8` marker) carries no weight.
        if e.dtype not in ("F8_E4M3", "I8") or e.count == 0 or name in r.consumed:
            continue
        base = name[: -len(".weight")] if name.endswith(".weight") else name
        kind = "int8" if e.dtype == "I8" else "float8_e4m3"
        for extra in (".zero_point", ".svd_up", ".svd_down"):
            if base + extra in raw:
                raise Refused(f"{name}: SDNQ's `{extra[1:]}` has no product here (symmetric int8 is read)")
        # SDNQ's `<l>.scale` only beside a `<l>.weight` (`prenorm.scale` and the like are norms).
        cands = [".weight_scale", ".scale_weight"] + ([".scale"] if name.endswith(".weight") else [])
        found = [base + c for c in cands if base + c in raw]
        if len(found) > 1:
            raise Refused(f"{name}: two scales name this weight")
        scale = found[0] if found else None
        declared = comfy.get(base)
        if declared is not None:
            fmt = declared.get("format") if isinstance(declared.get("format"), str) else ""
            if (fmt == "float8_e4m3fn") != (kind == "float8_e4m3"):
                raise Refused(f'{name}: {e.dtype} declared as "{fmt}"')
        if scale is None and kind != "float8_e4m3":
            raise Refused(f"{name}: int8 codes and no scale for them")
        if scale is None and declared is not None:
            raise Refused(f'{name}: ComfyUI says "float8_e4m3fn" yet ships no `weight_scale`; a plain cast would '
                          f"be guessing the scale")
        per_row = False
        if scale is not None:
            s = raw[scale]
            if _scale_type(s.dtype) is None:
                raise Refused(f"{scale}: a scale of type {s.dtype}")
            n = e.shape[0] if e.shape else 1
            if s.count == 1:
                per_row = False
            elif s.count == n and (s.shape == [n, 1] or s.shape == [n]):
                per_row = True
            else:
                raise Refused(f"{scale}: scale of shape {s.shape} for a weight of {e.shape}: one value, or one per "
                              f"row, is what is read")
            _check_subnormal(st, scale, kind)
            r.consumed.add(scale)
        rot = rotations.get(base, 0)
        if rot:
            if not (kind == "int8" and per_row and len(e.shape) == 2 and e.shape[1] % rot == 0):
                raise Refused(f"{name}: convrot (group {rot}) on {e.dtype} {e.shape} "
                              f"with {'a scale per row' if per_row else 'one scale'}; the rotation applies to per-row int8 whose "
                              f"input length is a multiple of the group")
            _check_subnormal(st, scale, kind, rot)
        if declared is not None:
            f = declared.get("format") if isinstance(declared.get("format"), str) else ""
            fmt = f"ComfyUI {f}" + (" convrot" if rot else "")
        else:
            fmt = "SDNQ" if scale is not None and scale.endswith(".scale") else ("fp8 cast" if scale is None
                                                                                 else "ComfyUI scaled")
        r.groups[name] = QuantizedGroup(name, kind, scale, per_row, fmt, rot)
    for name in order:
        if name in r.consumed:
            continue
        if name == "scaled_fp8":
            r.consumed.add(name)
        elif name.endswith(".input_scale") or name.endswith(".scale_input"):
            input_scales += 1
            r.consumed.add(name)
        elif name.endswith(".weight_scale") or name.endswith(".scale_weight"):
            r.consumed.add(name)
            r.notes.append(f"{name}: skipped, a scale with no 8-bit weight beside it")
    if input_scales:
        r.notes.append(f"{input_scales} `input_scale` skipped: the product takes its activations in bf16")
    return r


def product_operands(st: Safetensors, g: QuantizedGroup):
    """The group's codes [N, K] (int8, or uint8 e4m3 codes) and fp32 scale ([N], or [1]; 1 for a plain
    fp8 cast) for `TensorGEMM.pack(..., layout="nk")` and `product(..., rotation=g.rotation)`."""
    q = st.array(g.values)
    if g.scale is None:
        s = np.ones(1, np.float32)
    else:
        s = st.array(g.scale).astype(np.float32).reshape(-1)
    return np.ascontiguousarray(q), np.ascontiguousarray(s)


def stage(st: Safetensors, g: QuantizedGroup, ctx=None, device: int = 0):
    """The group on the device, ready for `TensorGEMM.product(x, packed, scale, rotation=group)`: codes
    packed from the published [N, K], fp32 scale per output (or one)."""
    import torch
    from .artifact import StagedWeight
    from .tensor_gemm import context
    q, s = product_operands(st, g)
    if q.ndim != 2:
        raise ValueError(f"{g.values}: {q.shape} is not an [N, K] weight")
    ctx = ctx or context(device)
    dev = torch.device("cuda", device)
    codes = torch.from_numpy(q).to(dev)
    w = codes.view(torch.int8) if g.kind == "int8" else codes.view(torch.float8_e4m3fn)
    packed = ctx.pack(w, layout="nk")
    n, k = q.shape
    return StagedWeight(name=g.values, packed=packed, scale=torch.from_numpy(s).to(dev), k=k, n=n,
                        group=g.rotation, dtype=g.kind)


BLOCK = 128


def block_operands(st: Safetensors, name: str):
    """An fp8 weight by 128×128 blocks as published, w = code · scale of its block: `<l>.weight` F8_E4M3 [N, K] with
    `<l>.weight_scale_inv` (F32, BF16 or F16) [⌈N/128⌉, ⌈K/128⌉]. The codes as uint8, the scales as fp32."""
    scale = name + "_scale_inv"
    w, s = st.entries.get(name), st.entries.get(scale)
    if w is None or w.dtype != "F8_E4M3" or len(w.shape) != 2:
        raise Refused(f"{name}: {'no such tensor' if w is None else f'{w.dtype} {w.shape}'} is not an fp8 [N, K] weight")
    if s is None or _scale_type(s.dtype) is None:
        raise Refused(f"{scale}: {'no such tensor' if s is None else f'a scale of type {s.dtype}'}")
    want = [-(-d // BLOCK) for d in w.shape]
    if s.shape != want:
        raise Refused(f"{scale}: scales of shape {s.shape} for a weight of {w.shape}, which has {want} blocks of 128×128")
    return np.ascontiguousarray(st.array(name)), np.ascontiguousarray(st.array(scale), dtype=np.float32)


def stage_blocks(st: Safetensors, *names: str, device: int = 0):
    """`product_f8`'s weight on the device, (codes float8_e4m3fn [N, K], scale fp32): one published weight, or a GLU's gate
    and up, whose halves are blocked each by itself (`product_f8(..., epilogue="silu_glu")`)."""
    import torch
    if len(names) not in (1, 2):
        raise ValueError("one weight, or a gate and an up")
    parts = [block_operands(st, name) for name in names]
    if any(q.shape != parts[0][0].shape for q, _ in parts):
        raise Refused(f"{names[0]} and {names[1]}: {parts[0][0].shape} and {parts[1][0].shape} are not the halves of a GLU")
    dev = torch.device("cuda", device)
    codes, scale = (torch.from_numpy(np.concatenate(p)).to(dev) for p in zip(*parts))
    return codes.view(torch.float8_e4m3fn), scale


def to_map(st: Safetensors, r: Recognized, path: str, page: int = 16384) -> None:
    """Writes the recognized 8-bit weights as a `.silicon` map: each `[K, N]` (the published [N, K]
    transposed, the map's `Linear` layout), its fp32 scale after the values, its rotation."""
    from .artifact import MapTensor, write_map
    tensors = {}
    for name, g in r.groups.items():
        q, s = product_operands(st, g)
        scale = s if g.per_row else np.array(s[0], np.float32)
        tensors[name] = MapTensor(np.ascontiguousarray(q.T), scale=scale, rotation=g.rotation)
    write_map(path, tensors, page=page)
