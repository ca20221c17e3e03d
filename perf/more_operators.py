"""What a decoder does with whole prompts, chunks of them and its logits, as measured cases.

`perf/operators.py` has a decoder's step of one token a sequence. Beside it stand: the norm of every query and key
head with the position rotation in the same pass (into a paged cache, or in place of the heads as an image model
takes them), attention of whole packed prompts, attention of a chunk of new tokens (a draft to verify, a piece of a
long prompt) over a paged cache, and the draw of the next token from the logits. The smallest calls are where latency
counts, the largest a prompt of thousands of tokens; `draw` spreads sizes, types and options between them.

`run` computes the plain form (elementary torch operations in 32 bits, in 64 where a border or a long sum needs them,
rounded once at the end) or, where `own` is true, calls the library.
"""
from __future__ import annotations

import math

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": F8}
SIZE = {"bf16": 2, "f32": 4, "e4m3": 1}
EPS = 1e-6

# The most a drawn case may take, as the largest listed ones: values of heads, scores of a batch padded to its longest (of
# heads of 128; fewer of larger ones), values of a padded batch's keys, logits.
MOST_VALUES = 8192 * 48 * 128
MOST_SCORES = 2048 * 31700 * 32
MOST_KEYS = 32 * 8192 * 8 * 128
MOST_LOGITS = 128 * 128000


def listed():
    return [
        # A decoding step's heads: one token's queries and keys normed, turned and kept.
        {"name": "heads_token", "kind": "heads", "tokens": 1, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "rot_dim": 128,
         "interleaved": False, "cache": "bf16", "page": 16, "idle": 0},
        # A prompt's, into an 8-bit cache.
        {"name": "heads_prompt", "kind": "heads", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "rot_dim": 128,
         "interleaved": False, "cache": "e4m3", "page": 64, "idle": 0},
        # An image block's tokens (text and image together), no cache, pairs side by side.
        {"name": "heads_image", "kind": "heads", "tokens": 4608, "q_heads": 24, "kv_heads": 24, "head_dim": 128, "rot_dim": 128,
         "interleaved": True, "cache": "none", "page": 0, "idle": 0},
        # A short prompt by itself: latency.
        {"name": "prompt_short", "kind": "prompt", "sequences": 1, "longest": 100, "spare": 0, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "causal": True, "window": 0, "softcap": 0.0},
        # A server's batch of prompts of different lengths, the buffer's last rows unused.
        {"name": "prompt_packed", "kind": "prompt", "sequences": 12, "longest": 2048, "spare": 5, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "causal": True, "window": 0, "softcap": 0.0},
        # An image block's joint attention: no mask, every head its own keys.
        {"name": "prompt_image", "kind": "prompt", "sequences": 1, "longest": 4608, "spare": 0, "q_heads": 24, "kv_heads": 24,
         "head_dim": 128, "causal": False, "window": 0, "softcap": 0.0},
        # A long prompt.
        {"name": "prompt_long", "kind": "prompt", "sequences": 1, "longest": 8192, "spare": 0, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "causal": True, "window": 0, "softcap": 0.0},
        # Sixteen tokens of one sequence over a short cache: latency.
        {"name": "chunk_one", "kind": "chunk", "batch": 1, "new": 16, "mixed": False, "length": 500, "ragged": False, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "cache": "bf16", "window": 0, "softcap": 0.0},
        # Drafts of four tokens to verify, a batch of ragged contexts in an 8-bit cache: the cache's bytes.
        {"name": "chunk_draft", "kind": "chunk", "batch": 32, "new": 4, "mixed": False, "length": 8192, "ragged": True, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "cache": "e4m3", "window": 0, "softcap": 0.0},
        # A piece of a long prompt behind what is cached of it (the most work of one call).
        {"name": "chunk_long", "kind": "chunk", "batch": 1, "new": 2048, "mixed": False, "length": 32768, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "cache": "bf16", "window": 0, "softcap": 0.0},
        # One sequence's next token, nucleus of a small vocabulary.
        {"name": "sample_one", "kind": "sample", "batch": 1, "vocab": 32000, "logits": "f32", "top_k": 0, "top_p": True, "min_p": False},
        # A batch's, every option set for each row by itself, some rows greedy.
        {"name": "sample_batch", "kind": "sample", "batch": 128, "vocab": 128000, "logits": "f32", "top_k": 100, "top_p": True,
         "min_p": True},
    ]


def draw(rng):
    """A case of the same kinds: 1 to 8192 tokens, heads of 64 to 256, contexts of 1 to 131072, 1000 to 262144 logits a row."""
    kind = rng.choice(["heads", "prompt", "prompt", "chunk", "chunk", "sample"])

    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    if kind == "sample":
        batch, vocab = log_int(1, 256), log_int(1000, 262144)
        while batch * vocab > MOST_LOGITS:
            batch = max(1, batch // 2)
        return {"kind": "sample", "batch": batch, "vocab": vocab, "logits": rng.choice(["f32", "bf16"]),
                "top_k": rng.choice([0, 0, 1, 50, 1000]), "top_p": rng.random() < 0.6, "min_p": rng.random() < 0.4}
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    q = kv * rng.choice([1, 2, 4, 4, 5, 8])
    dim = rng.choice([64, 96, 128, 128, 128, 256])
    if kind == "heads":
        tokens = log_int(1, 8192)
        dim = rng.choice([dim, dim, 80])
        while tokens * (q + 2 * kv) * dim > MOST_VALUES:
            tokens = max(1, tokens // 2)
        cache = rng.choice(["bf16", "e4m3", "none"])
        return {"kind": "heads", "tokens": tokens, "q_heads": q, "kv_heads": kv, "head_dim": dim,
                "rot_dim": dim if rng.random() < 0.7 else dim // 2, "interleaved": rng.random() < 0.4, "cache": cache,
                "page": 0 if cache == "none" else rng.choice([1, 16, 16, 24, 64, 128]),
                "idle": 0 if cache == "none" else min(tokens - 1, rng.choice([0, 0, 3]))}
    window, softcap = rng.choice([0, 0, 0, 1024]), rng.choice([0.0, 0.0, 0.0, 30.0])
    if kind == "prompt":
        count, longest = log_int(1, 32), log_int(1, 8192)
        while count * longest * longest * q * max(dim, 128) > MOST_SCORES * 128 or count * longest * (q + 2 * kv) * dim > MOST_VALUES:
            count, longest = max(1, count // 2), longest if count > 1 else longest // 2
        causal = rng.random() < 0.8
        return {"kind": "prompt", "sequences": count, "longest": longest, "spare": rng.choice([0, 0, 7]), "q_heads": q, "kv_heads": kv,
                "head_dim": dim, "causal": causal, "window": window if causal else 0, "softcap": softcap}
    batch, new, length = log_int(1, 64), log_int(1, 2048), log_int(1, 131072)
    new = min(new, length)
    while (batch * new * length * q * max(dim, 128) > MOST_SCORES * 128 or batch * length * kv * dim > MOST_KEYS or
           batch * new * q * dim > MOST_VALUES):
        if batch > 1:
            batch = batch // 2
        elif new > 16:
            new = new // 2
        else:
            length = length // 2
            new = min(new, length)
    return {"kind": "chunk", "batch": batch, "new": new, "mixed": rng.random() < 0.4, "length": length, "ragged": rng.random() < 0.6,
            "q_heads": q, "kv_heads": kv, "head_dim": dim, "page": rng.choice([1, 16, 16, 24, 64, 128]),
            "cache": rng.choice(["bf16", "e4m3"]), "window": window, "softcap": softcap}


# ---- inputs ----------------------------------------------------------------------------------------------------


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _prompt_lengths(case):
    """The packed prompts' lengths: the longest, and sixteenths of it; one of many is empty."""
    count, longest = case["sequences"], case["longest"]
    found = [max(1, longest * ((7 * i + 15) % 16 + 1) // 16) for i in range(count)]
    if count >= 4:
        found[2] = 0
    return found


def _chunks(case):
    """(new tokens, cached tokens with them) of each sequence. `mixed`: the first sequence a prompt's piece, the others one
    token each; one of many is idle. `ragged`: contexts of a sixteenth of the longest up to it."""
    batch, new, length = case["batch"], case["new"], case["length"]
    found = []
    for i in range(batch):
        count = new if i == 0 or not case["mixed"] else 1
        held = max(count, length * ((7 * i + 15) % 16 + 1) // 16 if case["ragged"] else length)
        found.append((count, held))
    if case["mixed"] and batch >= 4:
        found[2] = (0, found[2][1])
    return found


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _pool(case, s, g, name, pages):
    """A pool of keys or values N(0, 1), in 8 bits with a scale per head."""
    kv, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    scale = None
    if case["cache"] == "e4m3":
        scale = 0.02 * (1.0 + torch.rand(kv, device="cuda", generator=g))
    pool = torch.empty(pages, page, kv, dim, device="cuda", dtype=TYPES[case["cache"]])
    for part in pool.split(max(1, (1 << 26) // (page * kv * dim))):
        values = _normal(g, *part.shape)
        part.copy_(values / scale[:, None] if scale is not None else values)
    s[name + "_cache"], s[name + "_scale"] = pool, scale


def _inputs(case, seed):
    """A fused projection's rows N(0, 1); queries a little larger, so that attention has its peaks; keys and values scattered
    over the pool's pages; logits whose softmax has the heavy head of a language model's (a sixty-fourth of them forbidden)."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]
    if kind == "sample":
        batch, vocab = case["batch"], case["vocab"]
        x = _normal(g, batch, vocab) + 1.5 * torch.empty(batch, vocab, device="cuda").exponential_(generator=g)
        x[:, torch.randperm(vocab, device="cuda", generator=g)[:vocab // 64]] = -math.inf

        def rows(low, high):
            return low + (high - low) * torch.rand(batch, device="cuda", generator=g)

        t = rows(0.5, 1.3)
        if batch >= 8:
            t[::8] = 0.0
        s = {"x": x.to(TYPES[case["logits"]]), "temperature": t, "u": torch.rand(batch, device="cuda", generator=g),
             "top_k": None, "top_p": rows(0.8, 1.0) if case["top_p"] else None, "min_p": rows(0.0, 0.1) if case["min_p"] else None}
        if case["top_k"]:
            s["top_k"] = torch.randint(1, case["top_k"] + 1, (batch,), device="cuda", generator=g, dtype=torch.int32)
        return s
    nq, kv, dim = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "heads":
        tokens, page = case["tokens"], case["page"]
        half = case["rot_dim"] // 2
        angle = torch.arange(tokens + 100, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, device="cuda") / half)
        s = {"qkv": _normal(g, tokens, (nq + 2 * kv) * dim).to(torch.bfloat16), "q_norm": 1.0 + 0.1 * _normal(g, dim),
             "k_norm": 1.0 + 0.1 * _normal(g, dim), "table": torch.cat([angle.cos(), angle.sin()], dim=1).contiguous(),
             "positions": (torch.arange(tokens, device="cuda") + int(seed) % 100).to(torch.int32)}
        if case["cache"] != "none":
            pages = -(-tokens // page) + 5
            slots = torch.randperm(pages, device="cuda", generator=g)[:, None] * page + torch.arange(page, device="cuda")
            s["slots"] = slots.reshape(-1)[:tokens].to(torch.int32)
            if case["idle"]:
                s["slots"][-case["idle"]:] = -1
            _pool(case, s, g, "k", pages)
            _pool(case, s, g, "v", pages)
        return s
    if kind == "prompt":
        at = _starts(_prompt_lengths(case))
        rows = at[-1] + case["spare"]
        qkv = _normal(g, rows, nq + 2 * kv, dim)
        qkv[:, :nq] *= 1.5
        return {"qkv": qkv.to(torch.bfloat16), "starts": torch.tensor(at, device="cuda", dtype=torch.int32)}
    counts, held = zip(*_chunks(case))
    at, page = _starts(counts), case["page"]
    each = -(-max(held) // page)
    pages = case["batch"] * each + 3
    s = {"q": (1.5 * _normal(g, at[-1], nq, dim)).to(torch.bfloat16), "starts": torch.tensor(at, device="cuda", dtype=torch.int32),
         "lengths": torch.tensor(held, device="cuda", dtype=torch.int32),
         "pages": torch.randperm(pages, device="cuda", generator=g)[:case["batch"] * each].view(case["batch"], each).to(torch.int32)}
    _pool(case, s, g, "k", pages)
    _pool(case, s, g, "v", pages)
    return s


def _heads(case, s):
    """The query, key and value heads in a fused projection's rows: [rows, heads, dim] each."""
    nq, kv = case["q_heads"], case["kv_heads"]
    return s["qkv"].view(-1, nq + 2 * kv, case["head_dim"]).split([nq, kv, kv], dim=1)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    bf16 = dict(device="cuda", dtype=torch.bfloat16)
    if case["kind"] == "heads":
        s["q_out"] = torch.empty(case["tokens"], case["q_heads"], case["head_dim"], **bf16)
        s["k_out"] = torch.empty(case["tokens"], case["kv_heads"], case["head_dim"], **bf16)
    elif case["kind"] == "prompt":
        s["out"] = torch.zeros(s["qkv"].shape[0], case["q_heads"], case["head_dim"], **bf16)
    elif case["kind"] == "chunk":
        s["out"] = torch.empty_like(s["q"])
    if own:
        import siliconed_amd as sq

        s["ctx"] = sq.context(0)
        if "k_cache" in s:
            s["cache"] = sq.PagedCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


def _run_own(case, s):
    ctx, kind = s["ctx"], case["kind"]
    if kind == "heads":
        q, k, v = _heads(case, s)
        if case["cache"] == "none":
            q, k = ctx.norm_rotate(q, k, s["positions"], s["table"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                                   q_out=s["q_out"], k_out=s["k_out"], interleaved=case["interleaved"])
            return {"q": q, "k": k}
        q = ctx.norm_append_kv(q, k, v, s["cache"], s["positions"], s["slots"], s["table"], q_norm=s["q_norm"],
                               k_norm=s["k_norm"], eps=EPS, q_out=s["q_out"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if kind == "prompt":
        q, k, v = _heads(case, s)
        return ctx.prompt_attention(q, k, v, s["starts"], causal=case["causal"], softcap=case["softcap"], window=case["window"],
                                    out=s["out"])
    if kind == "chunk":
        return ctx.chunk_attention(s["q"], s["cache"], s["pages"], s["lengths"], s["starts"], softcap=case["softcap"],
                                   window=case["window"], out=s["out"])
    tokens, logprobs = ctx.sample_tokens(s["x"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                         min_p=s["min_p"])
    return {"tokens": tokens, "logprobs": logprobs}


def _run_plain(case, s):
    kind = case["kind"]
    if kind == "heads":
        return _heads_plain(case, s)
    if kind == "prompt":
        q, k, v = (t.float() for t in _heads(case, s))
        start = s["starts"].long()
        count = start[1:] - start[:-1]
        step = torch.arange(case["longest"], device="cuda")
        rows = (start[:-1, None] + step).clamp(max=q.shape[0] - 1)  # of the batch padded to its longest
        o = _attended(case, q[rows], k[rows], v[rows], step.expand_as(rows), count)
        live = step < count[:, None]
        s["out"][rows[live]] = o[live].to(torch.bfloat16)
        return s["out"]
    if kind == "chunk":
        start, held = s["starts"].long(), s["lengths"].long()
        count = start[1:] - start[:-1]
        step = torch.arange(case["new"], device="cuda")
        rows = (start[:-1, None] + step).clamp(max=s["q"].shape[0] - 1)
        k, v = (_gathered(s[n + "_cache"], s["pages"], s[n + "_scale"]) for n in ("k", "v"))
        o = _attended(case, s["q"].float()[rows], k, v, (held - count)[:, None] + step, held)
        live = step < count[:, None]
        s["out"][rows[live]] = o[live].to(torch.bfloat16)
        return s["out"]
    return _sampled(s)


def _heads_plain(case, s):
    q, k, v = (t.float() for t in _heads(case, s))
    q, k = (t * (1.0 / torch.sqrt((t * t).mean(dim=2, keepdim=True) + EPS)) * s[n] for t, n in ((q, "q_norm"), (k, "k_norm")))
    cos, sin = (t[:, None] for t in s["table"][s["positions"].long()].chunk(2, dim=1))
    q, k = (_rotated(t, cos, sin, case["interleaved"]) for t in (q, k))
    if case["cache"] == "none":
        return {"q": q.to(torch.bfloat16), "k": k.to(torch.bfloat16)}
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    for name, t in (("k", k), ("v", v)):
        pool = s[name + "_cache"]
        if s[name + "_scale"] is not None:
            t = (t / s[name + "_scale"][:, None]).clamp(-448.0, 448.0)
        flat = pool.view(-1, *pool.shape[2:])
        flat.view(torch.uint8)[slots] = t[live].to(pool.dtype).view(torch.uint8)
    return {"q": q.to(torch.bfloat16), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _rotated(t, cos, sin, interleaved):
    """The first values of each head turned by their position's angles: the pairs (i, i + half), or (2i, 2i + 1)."""
    rot = 2 * cos.shape[-1]
    a, b = (t[..., 0:rot:2], t[..., 1:rot:2]) if interleaved else (t[..., :rot // 2], t[..., rot // 2:rot])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([c, d], dim=-1).flatten(-2) if interleaved else torch.cat([c, d], dim=-1)
    return torch.cat([turned, t[..., rot:]], dim=-1)


def _gathered(pool, pages, scale):
    """A batch's keys or values [batch, tokens, heads, dim] out of the pool's pages."""
    t = pool.view(torch.uint8)[pages.long()].view(pool.dtype).float()
    if scale is not None:
        t = t * scale[:, None]
    return t.view(pages.shape[0], -1, *pool.shape[2:])


def _attended(case, q, k, v, at, end):
    """Attention of a padded batch: q [batch, n, heads, dim] at positions `at` [batch, n] over k, v [batch, m, kv heads, dim], of
    which a sequence has `end` [batch]."""
    batch, n, heads, dim = q.shape
    kv, m = k.shape[2], k.shape[1]
    q = q.view(batch, n, kv, -1, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, -1, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).mul_(1.0 / math.sqrt(dim)).view(batch, kv, -1, n, m)
    if case["softcap"]:
        scores = scores.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    t = torch.arange(m, device="cuda")
    seen = (t < end[:, None])[:, None]
    if case.get("causal", True):
        seen = seen & (t <= at[..., None])
        if case["window"]:
            seen = seen & (t > at[..., None] - case["window"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=4, keepdim=True)
    p = scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(dim=4, keepdim=True)
    o = torch.matmul(p.view(batch, kv, -1, m), v.permute(0, 2, 1, 3).contiguous()).view(batch, kv, -1, n, dim)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(batch, n, heads, dim)


def _sampled(s):
    """The next token of each row and the log of the probability it was drawn with: of the tokens by falling logit (equal ones by
    index) the first top_k, of these the fewest that hold top_p of their sum, of these the ones of at least min_p times the
    first's probability; then, by index, the first whose running sum passes u of the whole."""
    x = s["x"].double()
    greedy = s["temperature"] == 0.0
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None])
    rank = torch.arange(x.shape[1], device="cuda")
    most = torch.where(greedy, 1, s["top_k"] if s["top_k"] is not None else x.shape[1])
    w = torch.where(rank < most[:, None], w, torch.zeros_like(w))
    if s["top_p"] is not None:
        upto = w.cumsum(dim=1)
        w = torch.where(upto - w < s["top_p"].double()[:, None] * upto[:, -1:], w, torch.zeros_like(w))
    if s["min_p"] is not None:
        w = torch.where(w >= s["min_p"].double()[:, None], w, torch.zeros_like(w))
    kept = torch.zeros_like(w).scatter_(1, order, w)
    upto = kept.cumsum(dim=1)
    total = upto[:, -1:]
    tokens = (upto > s["u"].double()[:, None] * total).to(torch.int32).argmax(dim=1)
    logprobs = torch.log(kept.gather(1, tokens[:, None]) / total)[:, 0]
    return {"tokens": tokens.to(torch.int32), "logprobs": logprobs.float()}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "heads":
        return _heads_exact(case, s)
    if kind == "sample":
        return _sampled_exact(case, s)
    dim, kv = case["head_dim"], case["kv_heads"]
    if kind == "prompt":
        q, k, v = (t.double() for t in _heads(case, s))
        found = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    else:
        q = s["q"].double()
        found = torch.zeros_like(q)
    at = s["starts"].tolist()
    for b, (lo, hi) in enumerate(zip(at[:-1], at[1:])):
        if lo == hi:
            continue
        held = hi - lo if kind == "prompt" else int(s["lengths"][b])
        t = torch.arange(held, device="cuda")
        place = torch.arange(lo, hi, device="cuda") - hi + held
        hidden = torch.zeros(hi - lo, held, device="cuda", dtype=torch.bool)
        if case.get("causal", True):
            ahead = t[None] - place[:, None]
            hidden = ahead > 0
            if case["window"]:
                hidden |= ahead <= -case["window"]
        for h in range(case["q_heads"]):
            g = h // (case["q_heads"] // kv)
            if kind == "prompt":
                kh, vh = k[lo:hi, g], v[lo:hi, g]
            else:
                page, row = s["pages"][b].long()[t // case["page"]], t % case["page"]
                kh, vh = (s[c][:, :, g].contiguous().view(torch.uint8)[page, row].view(s[c].dtype).double() for c in ("k_cache", "v_cache"))
                if s["k_scale"] is not None:
                    kh, vh = kh * s["k_scale"][g].double(), vh * s["v_scale"][g].double()
            e = q[lo:hi, h] @ kh.t() / math.sqrt(dim)
            if case["softcap"]:
                e = case["softcap"] * torch.tanh(e / case["softcap"])
            found[lo:hi, h] = torch.softmax(e.masked_fill_(hidden, -math.inf), dim=1) @ vh
    return found


def _heads_exact(case, s):
    q, k, v = (t.double() for t in _heads(case, s))
    half = case["rot_dim"] // 2
    angles = s["table"].double()[s["positions"].long()]
    turn = torch.complex(angles[:, :half], angles[:, half:])[:, None]

    def turned(t, w):
        t = t / torch.sqrt(t.pow(2).mean(dim=2, keepdim=True) + EPS) * w.double()
        first, second = (t[..., 0:2 * half:2], t[..., 1:2 * half:2]) if case["interleaved"] else (t[..., :half], t[..., half:2 * half])
        z = torch.complex(first.contiguous(), second.contiguous()) * turn
        first.copy_(z.real)
        second.copy_(z.imag)
        return t

    found = {"q": turned(q, s["q_norm"])}
    k = turned(k, s["k_norm"])
    if case["cache"] == "none":
        found["k"] = k
        return found
    live = s["slots"] >= 0
    page = torch.div(s["slots"][live], case["page"], rounding_mode="floor").long()
    row = s["slots"][live].long() - page * case["page"]
    for name, t in (("k", k), ("v", v)):
        pool = s[name + "_cache"].double()
        if s[name + "_scale"] is not None:
            t = (t / s[name + "_scale"].double()[:, None]).clamp(-448.0, 448.0)
        pool.index_put_((page, row), t[live])
        found[name + "_cache"] = pool
    return found


def _sampled_exact(case, s):
    tokens, logprobs = [], []
    value = lambda name, b, none: none if s[name] is None else s[name][b].item()  # noqa: E731
    for b in range(case["batch"]):
        x, t = s["x"][b].double(), s["temperature"][b].item()
        if t == 0.0:
            tokens.append(int((x == x.max()).nonzero()[0, 0]))
            logprobs.append(0.0)
            continue
        p = torch.exp((x - x.max()) / t)
        by = torch.sort(-x, stable=True).indices[:value("top_k", b, case["vocab"])]
        p = p[by]
        before = torch.cat([p.new_zeros(1), p.cumsum(0)])
        keep = (before[:-1] < value("top_p", b, 1.0) * before[-1]) & (p >= value("min_p", b, 0.0))
        by, back = torch.sort(by[keep])
        p = p[keep][back]
        upto = p.cumsum(0)
        i = int((upto <= s["u"][b].item() * upto[-1]).sum())
        tokens.append(int(by[i]))
        logprobs.append(math.log(p[i].item() / upto[-1].item()))
    return {"tokens": torch.tensor(tokens, device="cuda", dtype=torch.int32),
            "logprobs": torch.tensor(logprobs, device="cuda", dtype=torch.float64)}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def _pairs(count, held, case):
    """The (query, key) pairs of `count` tokens at the end of `held`."""
    if not case.get("causal", True):
        return count * held
    first, w = held - count, case["window"]
    if not w:
        return count * held - count * (count - 1) // 2
    return sum(min(w, first + i + 1) for i in range(count))


def work(case):
    kind = case["kind"]
    if kind == "sample":
        values = case["batch"] * case["vocab"]
        return {"bytes": values * SIZE[case["logits"]] + 24 * case["batch"], "flops": 4 * values}
    nq, kv, dim = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "heads":
        tokens, live = case["tokens"], case["tokens"] - case["idle"]
        held = 2 * live * kv * dim * (2 + SIZE[case["cache"]]) if case["cache"] != "none" else tokens * kv * dim * 4
        return {"bytes": tokens * (nq * dim * 4 + 4 * case["rot_dim"] + 8) + held,
                "flops": tokens * (nq + kv) * (4 * dim + 3 * case["rot_dim"])}
    if kind == "prompt":
        lengths = _prompt_lengths(case)
        return {"bytes": 2 * sum(lengths) * (2 * nq + 2 * kv) * dim, "flops": 4 * sum(_pairs(n, n, case) for n in lengths) * nq * dim}
    chunks = _chunks(case)
    seen = sum(0 if n == 0 else min(held, case["window"] + n - 1) if case["window"] else held for n, held in chunks)
    return {"bytes": 2 * seen * kv * dim * SIZE[case["cache"]] + 4 * sum(n for n, _ in chunks) * nq * dim,
            "flops": 4 * sum(_pairs(n, held, case) for n, held in chunks) * nq * dim}
