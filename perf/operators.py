"""The operators of a text decoder's layer on block-scaled fp8 weights, as measured cases.

A text encoder or a prompt writer beside the image model is a decoder: per layer a norm that adds the
residual stream and writes the next product's 8-bit operand, products of e4m3 codes with a scale per 128
of K, the new keys and values appended to a paged cache with the position rotation, and attention of each
sequence's new token over that cache. One token of one sequence is where latency counts; a batch of
sequences decoding together is the ordinary case; a prompt of thousands of tokens, or a context of a
hundred thousand, the large one. `listed` holds these for each operator; `draw` spreads sizes, types and
options over the ranges they stand for.

`run` computes the plain form (elementary torch operations in 32 bits, rounded once at the end) or, where
`own` is true, calls the library.
"""
from __future__ import annotations

import math

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": F8, "int8": torch.int8}
SIZE = {"bf16": 2, "f32": 4, "e4m3": 1, "int8": 1}
EPS = 1e-6
GROUP = 128  # values of K that share a scale

# The most a drawn case may take, as the largest listed ones: multiply-adds, values normed, tokens appended, cache bytes.
MOST_MACS = 8192 * 4096 * 24576
MOST_VALUES = 8192 * 4096
MOST_CACHE = 2 * 2 * 131072 * 8 * 128 * 2


def listed():
    return [
        # A decoding step's norm: one row, the smallest call there is.
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 4096, "x": "bf16", "residual": "bf16", "codes": "e4m3"},
        # The norm before a prompt's fused projection, the stream in bf16.
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "cols": 4096, "x": "bf16", "residual": "bf16",
         "codes": "e4m3"},
        # A ragged prompt on an int8 checkpoint, an fp32 stream, a width that is not whole groups.
        {"name": "norm_ragged_int8", "kind": "norm", "rows": 333, "cols": 2760, "x": "bf16", "residual": "f32",
         "codes": "int8"},
        # One token through the fused query, key and value projection: the weight's bytes.
        {"name": "product_token", "kind": "product", "m": 1, "k": 4096, "n": 6144, "a": "codes", "epilogue": "none",
         "bias": False, "out": "bf16"},
        # Forty-eight sequences through a gate and up projection, the activation quantized on the way.
        {"name": "product_batch", "kind": "product", "m": 48, "k": 4096, "n": 24576, "a": "bf16", "epilogue": "silu_glu",
         "bias": False, "out": "bf16"},
        # A ragged prompt, a K that ends inside a group, columns that end inside a block, fp32 out.
        {"name": "product_ragged", "kind": "product", "m": 333, "k": 2496, "n": 2112, "a": "codes", "epilogue": "none",
         "bias": True, "out": "f32"},
        # A long prompt through a gate and up projection (the most work of one product).
        {"name": "product_prompt", "kind": "product", "m": 8192, "k": 4096, "n": 24576, "a": "codes",
         "epilogue": "silu_glu", "bias": False, "out": "bf16"},
        # A decoding batch's new keys and values into an 8-bit cache, its last rows idle.
        {"name": "append_batch", "kind": "append", "tokens": 48, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "rot_dim": 128, "interleaved": False, "page": 16, "cache": "e4m3", "idle": 3},
        # A prompt's, into a bf16 cache.
        {"name": "append_prompt", "kind": "append", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "rot_dim": 128, "interleaved": False, "page": 64, "cache": "bf16", "idle": 0},
        # One sequence of a short context: latency.
        {"name": "attention_token", "kind": "attention", "batch": 1, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "length": 777, "ragged": False, "page": 16, "cache": "bf16", "window": 0, "softcap": 0.0},
        # A batch of ragged contexts over an 8-bit cache.
        {"name": "attention_batch", "kind": "attention", "batch": 48, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "length": 8192, "ragged": True, "page": 64, "cache": "e4m3", "window": 0, "softcap": 0.0},
        # Two long contexts.
        {"name": "attention_long", "kind": "attention", "batch": 2, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "length": 131072, "ragged": False, "page": 64, "cache": "bf16", "window": 0, "softcap": 0.0},
    ]


def draw(rng):
    """A case of the same kinds: 1 to 8192 rows, widths whole and ragged, every type, contexts of 1 to 131072."""
    kind = rng.choice(["norm", "product", "product", "append", "attention", "attention"])

    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    if kind == "norm":
        rows = log_int(1, 8192)
        step = rng.choice([1, 8, 128, 128])
        cols = max(1, round(log_int(512, 16384) / step)) * step
        while rows * cols > MOST_VALUES:
            rows = max(1, rows // 2)
        return {"kind": "norm", "rows": rows, "cols": cols, "x": rng.choice(["bf16", "bf16", "f32"]),
                "residual": rng.choice(["bf16", "bf16", "f32", "none"]), "codes": rng.choice(["e4m3", "e4m3", "int8"])}
    if kind == "product":
        m = log_int(1, 8192)
        k = max(1, round(log_int(512, 16384) / 128)) * 128
        n = max(1, round(log_int(512, 24576) / 128)) * 128
        ragged = rng.random() < 0.35
        if ragged:
            k, n = k - 16 * rng.randrange(8), n - rng.randrange(64)
        epilogue = rng.choice(["none", "none", "silu_glu"])
        if epilogue == "silu_glu":
            n += n % 2
        while m * k * n > MOST_MACS:
            m = max(1, m // 2)
        return {"kind": "product", "m": m, "k": k, "n": n, "a": rng.choice(["codes", "codes", "bf16"]),
                "epilogue": epilogue, "bias": rng.random() < 0.3, "out": rng.choice(["bf16", "bf16", "f32"])}
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    q = kv * rng.choice([1, 2, 4, 4, 5, 8])
    dim = rng.choice([64, 96, 128, 128, 256])
    page = rng.choice([1, 16, 16, 24, 32, 64, 128])
    cache = rng.choice(["bf16", "e4m3"])
    if kind == "append":
        tokens = log_int(1, 8192)
        while tokens * (q + 2 * kv) * dim > 8192 * 48 * 128:
            tokens = max(1, tokens // 2)
        return {"kind": "append", "tokens": tokens, "q_heads": q, "kv_heads": kv, "head_dim": dim,
                "rot_dim": dim if rng.random() < 0.7 else dim // 2, "interleaved": rng.random() < 0.3, "page": page,
                "cache": cache, "idle": min(tokens - 1, rng.choice([0, 0, 3]))}
    batch, length = log_int(1, 128), log_int(1, 131072)
    while 2 * batch * length * kv * dim * SIZE[cache] > MOST_CACHE:
        batch, length = max(1, batch // 2), length if batch > 1 else length // 2
    return {"kind": "attention", "batch": batch, "q_heads": q, "kv_heads": kv, "head_dim": dim, "length": length,
            "ragged": rng.random() < 0.6, "page": page, "cache": cache,
            "window": rng.choice([0, 0, 0, 1024]), "softcap": rng.choice([0.0, 0.0, 30.0])}


# ---- inputs ----------------------------------------------------------------------------------------------------


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _ceil(count, size):
    return -(-count // size)


def _groups(k):
    return _ceil(k, GROUP)


def _spread(scales, k):
    """A scale per group of 128, for each of the k values."""
    return scales.repeat_interleave(GROUP, dim=1)[:, :k]


def _halves(case):
    """The weight's rows in the parts that are blocked by themselves: a GLU's gate and up halves."""
    return [case["n"] // 2] * 2 if case["epilogue"] == "silu_glu" else [case["n"]]


def _row_blocks(case):
    """For each weight row, the row of its block scale."""
    at, found = 0, []
    for rows in _halves(case):
        found.append(at + torch.arange(rows, device="cuda") // GROUP)
        at += _groups(rows)
    return torch.cat(found)


def _lengths(case):
    """The batch's context lengths: all alike, or a sixteenth of the longest up to it, one sequence in a batch idle."""
    batch, length = case["batch"], case["length"]
    if not case["ragged"] or batch == 1:
        return [length] * batch
    found = [max(1, length * ((7 * i + 15) % 16 + 1) // 16) for i in range(batch)]
    if batch >= 4:
        found[2] = 0
    return found


def _inputs(case, seed):
    """Activations N(0, 1) (a norm's or projection's rows), weights N(0, 0.02) quantized per block of 128 x 128, keys and
    values N(0, 1) scattered over the pool's pages as a server that has run for a while leaves them."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]
    if kind == "norm":
        rows, cols = case["rows"], case["cols"]
        s = {"x": _normal(g, rows, cols).to(TYPES[case["x"]]), "w": 1.0 + 0.1 * _normal(g, cols), "residual": None}
        if case["residual"] != "none":
            s["residual"] = (2.0 * _normal(g, rows, cols)).to(TYPES[case["residual"]])
        return s
    if kind == "product":
        m, k, n = case["m"], case["k"], case["n"]
        row_block = _row_blocks(case)
        x = _normal(g, m, k).to(torch.bfloat16)
        w = 0.02 * _normal(g, n, k)
        amax = []
        for part in w.abs().split(_halves(case)):
            part = torch.nn.functional.pad(part, (0, -k % GROUP, 0, -part.shape[0] % GROUP))
            amax.append(part.view(-1, GROUP, _groups(k), GROUP).amax(dim=(1, 3)))
        scale = torch.cat(amax) / 448.0
        s = {"scale": scale, "w": (w / _spread(scale, k)[row_block]).to(F8), "bias": None}
        if case["bias"]:
            s["bias"] = 0.02 * _normal(g, n)
        if case["a"] == "codes":
            s["a"], s["sx"] = _quantized(x.float())
        else:
            s["x"] = x
        return s
    kv, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    if kind == "append":
        tokens = case["tokens"]
        pages = _ceil(tokens, page) + 5
        qkv = _normal(g, tokens, (case["q_heads"] + 2 * kv) * dim).to(torch.bfloat16)
        half = case["rot_dim"] // 2
        angle = torch.arange(tokens + 100, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, device="cuda") / half)
        slots = torch.randperm(pages, device="cuda", generator=g)[:, None] * page + torch.arange(page, device="cuda")
        slots = slots.reshape(-1)[:tokens].to(torch.int32)
        if case["idle"]:
            slots[-case["idle"]:] = -1
        s = {"qkv": qkv, "table": torch.cat([angle.cos(), angle.sin()], dim=1).contiguous(), "slots": slots,
             "positions": (torch.arange(tokens, device="cuda") + int(seed) % 100).to(torch.int32)}
    else:
        lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
        lengths = lengths[torch.randperm(case["batch"], device="cuda", generator=g)]
        each = _ceil(case["length"], page)
        pages = case["batch"] * each + 3
        order = torch.randperm(pages, device="cuda", generator=g)[:case["batch"] * each]
        s = {"q": _normal(g, case["batch"], case["q_heads"], dim).to(torch.bfloat16), "lengths": lengths,
             "pages": order.view(case["batch"], each).to(torch.int32)}
    for name in ("k", "v"):
        s[name + "_scale"] = None
        pool = torch.empty(pages, page, kv, dim, device="cuda", dtype=TYPES[case["cache"]])
        if case["cache"] == "e4m3":
            s[name + "_scale"] = 0.02 * (1.0 + torch.rand(kv, device="cuda", generator=g))
        for part in pool.split(max(1, (1 << 26) // (page * kv * dim))):
            values = _normal(g, *part.shape)
            part.copy_(values / s[name + "_scale"][:, None] if s[name + "_scale"] is not None else values)
        s[name + "_cache"] = pool
    return s


def _heads(case, s):
    """The query, key and value heads in a fused projection's rows."""
    rows, nq, nkv, dim = s["qkv"].shape[0], case["q_heads"], case["kv_heads"], case["head_dim"]
    return [t.view(rows, -1, dim) for t in s["qkv"].split([nq * dim, nkv * dim, nkv * dim], dim=1)]


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import siliconed_amd as sq

        s["ctx"] = sq.context(0)
        kind = case["kind"]
        if kind == "norm":
            s["out"] = torch.empty_like(s["residual"]) if s["residual"] is not None else None
        elif kind == "product":
            width = case["n"] // 2 if case["epilogue"] == "silu_glu" else case["n"]
            s["out"] = torch.empty(case["m"], width, device="cuda", dtype=TYPES[case["out"]])
        elif kind == "append":
            s["heads"] = _heads(case, s)
            s["out"] = torch.empty(case["tokens"], case["q_heads"], case["head_dim"], device="cuda", dtype=torch.bfloat16)
        else:
            s["out"] = torch.empty_like(s["q"])
        if kind in ("append", "attention"):
            s["cache"] = sq.PagedCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


def _run_own(case, s):
    ctx, kind = s["ctx"], case["kind"]
    if kind == "norm":
        codes, scales, stream = ctx.add_norm_quantized(s["x"], s["w"], EPS, residual=s["residual"], residual_out=s["out"],
                                                       dtype=TYPES[case["codes"]])
        return _norm_outputs(codes, scales, stream)
    if kind == "product":
        if case["a"] == "codes":
            return ctx.product_f8(s["a"], s["sx"], s["w"], s["scale"], bias=s["bias"], epilogue=case["epilogue"], out=s["out"])
        return ctx.product_f8_quantized(s["x"], s["w"], s["scale"], bias=s["bias"], epilogue=case["epilogue"], out=s["out"])
    if kind == "append":
        q, k, v = s["heads"]
        out = ctx.append_kv(q, k, v, s["cache"], s["positions"], s["slots"], s["table"], q_out=s["out"],
                            interleaved=case["interleaved"])
        return {"q": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return ctx.paged_attention(s["q"], s["cache"], s["pages"], s["lengths"], softcap=case["softcap"],
                               window=case["window"], out=s["out"])


def _norm_outputs(codes, scales, stream):
    """The codes as the values they stand for: e4m3 is a type of its own, an int8 code is exact in bf16."""
    found = {"codes": codes.to(torch.bfloat16) if codes.dtype == torch.int8 else codes, "scales": scales}
    if stream is not None:
        found["residual"] = stream
    return found


def _quantized(y):
    """e4m3 codes and a scale per group of 128 of each row."""
    rows, k = y.shape
    padded = torch.nn.functional.pad(y, (0, _groups(k) * GROUP - k)) if k % GROUP else y
    amax = padded.view(rows, -1, GROUP).abs().amax(dim=2)
    scales = (amax / 448.0).clamp_min(1e-30)
    return (y / _spread(scales, k)).to(F8), scales


def _run_plain(case, s):
    kind = case["kind"]
    if kind == "norm":
        x = s["x"].float()
        stream = None
        if s["residual"] is not None:
            x = x + s["residual"].float()
            stream = x.to(s["residual"].dtype)
        y = x * (1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPS)) * s["w"]
        if case["codes"] == "e4m3":
            return _norm_outputs(*_quantized(y), stream)
        scales = (y.abs().amax(dim=1) / 127.0).clamp_min(1e-30)
        return _norm_outputs(torch.round(y / scales[:, None]).clamp(-128, 127).to(torch.int8), scales, stream)
    if kind == "product":
        a, sx = (s["a"], s["sx"]) if case["a"] == "codes" else _quantized(s["x"].float())
        k = case["k"]
        row_block = _row_blocks(case)
        w = s["w"].float() * _spread(s["scale"], k)[row_block]
        c = (a.float() * _spread(sx, k)) @ w.t()
        if s["bias"] is not None:
            c = c + s["bias"]
        if case["epilogue"] == "silu_glu":
            gate, up = c.chunk(2, dim=1)
            c = gate / (1.0 + torch.exp(-gate)) * up
        return c.to(TYPES[case["out"]])
    if kind == "append":
        q, k, v = (t.float() for t in _heads(case, s))
        rows = s["table"][s["positions"].long()]
        cos, sin = (t[:, None] for t in rows.chunk(2, dim=1))
        q, k = (_rotated(t, cos, sin, case["interleaved"]) for t in (q, k))
        live = s["slots"] >= 0
        slots = s["slots"][live].long()
        for name, t in (("k", k), ("v", v)):
            pool = s[name + "_cache"]
            if s[name + "_scale"] is not None:
                t = (t / s[name + "_scale"][:, None]).clamp(-448.0, 448.0)
            flat = pool.view(-1, *pool.shape[2:])
            flat.view(torch.uint8)[slots] = t[live].to(pool.dtype).view(torch.uint8)
        return {"q": q.to(torch.bfloat16), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    k, v = (_gathered(s[n + "_cache"], s["pages"], s[n + "_scale"]) for n in ("k", "v"))
    batch, length, kv, dim = k.shape
    q = s["q"].float().view(batch, kv, -1, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(dim))
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    at, end = torch.arange(length, device="cuda"), s["lengths"].long()[:, None]
    seen = at < end
    if case["window"]:
        seen = seen & (at >= end - case["window"])
    scores = torch.where(seen[:, None, None], scores, torch.full_like(scores, -math.inf))
    top = scores.amax(dim=3, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=3, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
    return o.view(batch, -1, dim).to(torch.bfloat16)


def _rotated(t, cos, sin, interleaved):
    """The first values of each head turned by their position's angles: the pairs (i, i + half), or (2i, 2i + 1)."""
    rot = 2 * cos.shape[-1]
    a, b = (t[..., 0:rot:2], t[..., 1:rot:2]) if interleaved else (t[..., :rot // 2], t[..., rot // 2:rot])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([c, d], dim=-1).flatten(-2) if interleaved else torch.cat([c, d], dim=-1)
    return torch.cat([turned, t[..., rot:]], dim=-1)


def _gathered(pool, pages, scale):
    """A batch's keys or values [batch, tokens, heads, dim] out of the pool's pages."""
    batch = pages.shape[0]
    t = pool.view(torch.uint8)[pages.long()].view(pool.dtype).float()
    if scale is not None:
        t = t * scale[:, None]
    return t.view(batch, -1, *pool.shape[2:])


# ---- the definition in 64 bits -------------------------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        x = s["x"].double()
        found = {}
        if s["residual"] is not None:
            x = x + s["residual"].double()
            found["residual"] = x
        y = x / torch.sqrt(x.pow(2).mean(dim=1, keepdim=True) + EPS) * s["w"].double()
        top, width = (448.0, GROUP) if case["codes"] == "e4m3" else (127.0, case["cols"])
        parts = y.split(width, dim=1)
        scales = [(p.abs().amax(dim=1) / top).clamp_min(1e-30) for p in parts]
        # The codes' values before their rounding to 8 bits.
        found["codes"] = torch.cat([p / t[:, None] for p, t in zip(parts, scales)], dim=1)
        found["scales"] = torch.stack(scales, dim=1) if case["codes"] == "e4m3" else scales[0]
        return found
    if kind == "product":
        k = case["k"]
        if case["a"] == "codes":
            a, sx = s["a"].double(), s["sx"].double()
        else:
            parts = s["x"].double().split(GROUP, dim=1)
            sx = torch.stack([(p.abs().amax(dim=1) / 448.0).clamp_min(1e-30) for p in parts], dim=1)
            a = torch.cat([p / sx[:, i:i + 1] for i, p in enumerate(parts)], dim=1).float().to(F8).double()
        row_block = _row_blocks(case)
        c = torch.zeros(case["m"], case["n"], device="cuda", dtype=torch.float64)
        for b, at in enumerate(range(0, k, GROUP)):
            part = a[:, at:at + GROUP] @ s["w"][:, at:at + GROUP].double().t()
            c += part * sx[:, b:b + 1] * s["scale"][row_block, b].double()
        if s["bias"] is not None:
            c += s["bias"].double()
        if case["epilogue"] == "silu_glu":
            h = case["n"] // 2
            c = c[:, :h] * torch.sigmoid(c[:, :h]) * c[:, h:]
        return c
    if kind == "append":
        q, k, v = (t.double() for t in _heads(case, s))
        half = case["rot_dim"] // 2
        angles = s["table"].double()[s["positions"].long()]
        turn = torch.complex(angles[:, :half], angles[:, half:])[:, None]

        def rotated(t):
            t = t.clone()
            first, second = (t[..., 0:2 * half:2], t[..., 1:2 * half:2]) if case["interleaved"] else (t[..., :half], t[..., half:2 * half])
            z = torch.complex(first.contiguous(), second.contiguous()) * turn
            first.copy_(z.real)
            second.copy_(z.imag)
            return t

        found = {"q": rotated(q)}
        for name, t in (("k", rotated(k)), ("v", v)):
            pool = s[name + "_cache"].double()
            if s[name + "_scale"] is not None:
                t = (t / s[name + "_scale"].double()[:, None]).clamp(-448.0, 448.0)
            for i, slot in enumerate(s["slots"].tolist()):
                if slot >= 0:
                    pool[slot // case["page"], slot % case["page"]] = t[i]
            found[name + "_cache"] = pool
        return found
    dim, kv = case["head_dim"], case["kv_heads"]
    o = torch.zeros(case["batch"], kv, case["q_heads"] // kv, dim, device="cuda", dtype=torch.float64)
    for b, n in enumerate(s["lengths"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n, device="cuda")
        page, row = s["pages"][b].long()[at // case["page"]], at % case["page"]
        for h in range(kv):
            k, v = (s[c][:, :, h].contiguous().view(torch.uint8)[page, row].view(s[c].dtype).double()
                    for c in ("k_cache", "v_cache"))
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            t = k @ s["q"].double().view(case["batch"], kv, -1, dim)[b, h].t() / math.sqrt(dim)
            if case["softcap"]:
                t = case["softcap"] * torch.tanh(t / case["softcap"])
            o[b, h] = torch.softmax(t, dim=0).t() @ v
    return o.view(case["batch"], -1, dim)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "norm":
        values = case["rows"] * case["cols"]
        stream = 0 if case["residual"] == "none" else 2 * SIZE[case["residual"]]
        scales = case["rows"] * (_groups(case["cols"]) if case["codes"] == "e4m3" else 1)
        return {"bytes": values * (SIZE[case["x"]] + stream + 1) + 4 * scales + 4 * case["cols"], "flops": 8 * values}
    if kind == "product":
        m, k, n = case["m"], case["k"], case["n"]
        width = n // 2 if case["epilogue"] == "silu_glu" else n
        a = m * k + 4 * m * _groups(k) if case["a"] == "codes" else 2 * m * k
        blocks = sum(_groups(r) for r in _halves(case))
        return {"bytes": a + n * k + 4 * blocks * _groups(k) + m * width * SIZE[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * m * k * n}
    nq, nkv, dim, size = case["q_heads"], case["kv_heads"], case["head_dim"], SIZE[case["cache"]]
    if kind == "append":
        tokens = case["tokens"]
        live = tokens - case["idle"]
        return {"bytes": tokens * (nq * dim * 4 + 4 * case["rot_dim"] + 8) + live * 2 * nkv * dim * (2 + size),
                "flops": 3 * tokens * (nq + nkv) * case["rot_dim"]}
    seen = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
    return {"bytes": 2 * seen * nkv * dim * size + 2 * case["batch"] * nq * dim * 2, "flops": 4 * seen * nq * dim}
