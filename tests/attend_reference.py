"""Attention of prompts and chunks in 64 bits, for the tests: one sequence at a time, each row over the tokens it sees.

The tolerance of an output o = Σ p v / Σ p (bf16): its own rounding, 2^-8 of it; the probabilities' rounding to bf16, 2^-8 of
each at most, so 2^-8 of A = Σ p |v| / Σ p; and what fp32 puts on an exponent: a score of `dim` products is off by dim · 2^-24 of
Σ |q k|, its scaling, the subtraction of the maximum and the exponential by 4 · 2^-24 of the largest exponent (in units of
log2), a cap by another 3e-7 of the cap's, each again relative to p, so to A."""
import math

import torch

U = 2.0 ** -8


def attended(q, k, v, first, *, scale=None, softcap=0.0, window=0, causal=True, dead=None):
    """q [n, heads, dim] at places first, first + 1, ... over k, v [m, kv heads, dim] (any types): (o, tolerance) in 64 bits.
    `dead`: [m] tokens that count as masked. A row that sees nothing gives zeros."""
    n, heads, dim = q.shape
    m, kv = k.shape[0], k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    t, at = torch.arange(m, device=q.device), first + torch.arange(n, device=q.device)[:, None]
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        seen = t <= at
        if window:
            seen &= t > at - window
    if dead is not None:
        seen &= ~dead
    o = torch.zeros(n, heads, dim, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for h in range(heads):
        g = h // (heads // kv)
        qh, kh, vh = q[:, h].double(), k[:, g].double(), v[:, g].double()
        used = seen.any(0)
        kh, vh = torch.where(used[:, None], kh, 0.0), torch.where(used[:, None], vh, 0.0)
        s = qh @ kh.T * scale
        off = dim * 2.0 ** -24 * abs(scale) * (qh.abs() @ kh.abs().T)
        if softcap and not math.isinf(softcap):
            s = softcap * torch.tanh(s / softcap)
            off = off + 3e-7 * softcap
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(1, keepdim=True) if m else s.new_full((n, 1), -math.inf)
        top = torch.where(top == -math.inf, 0.0, top)
        p = torch.exp(s - top)
        total = p.sum(1, keepdim=True)
        total = torch.where(total > 0, total, 1.0)
        size = torch.where(seen, s.abs(), 0.0).amax(1, keepdim=True) if m else torch.zeros(n, 1, device=q.device)
        off = torch.where(seen, off, 0.0).amax(1, keepdim=True) if m else torch.zeros(n, 1, device=q.device)
        o[:, h] = p @ vh / total
        a = p @ vh.abs() / total
        tol[:, h] = U * o[:, h].abs() + (U + 2 * off + 8 * 1.45 * 2.0 ** -24 * (1 + size)) * 1.01 * a
    return o, tol


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max())}, at "
                           f"{bad.nonzero()[0].tolist()}: {float(got[bad][0])} for {float(want[bad][0])} +- {float(tol[bad][0])}")
