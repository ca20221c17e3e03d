"""That the tolerance of chunks of few rows tells probabilities of two bf16 parts from rounded ones: both planted in the formula, on the
CPU."""
import math

import pytest
import torch

from attend_reference import attended, within
from narrow_chunks import attended_narrow

BF = torch.bfloat16


def planted(q, k, v, parts):
    """One head's output from probabilities of so many bf16 parts, rounded once."""
    s = q.double() @ k.double().T / math.sqrt(q.shape[1])
    p = torch.exp(s - s.amax(1, keepdim=True)).float()
    if parts == 1:
        used = p.to(BF).double()
    else:
        first = (p.view(torch.int32) & -65536).view(torch.float32)
        used = first.double() + (p - first).to(BF).double()
    return (used @ v.double() / p.double().sum(1, keepdim=True)).to(BF)


@pytest.mark.parametrize("tokens", [40, 700])
def test_parts_of_probabilities(tokens):
    g = torch.Generator().manual_seed(tokens)
    q, k, v = (torch.randn(n, 1, 64, generator=g).to(BF) for n in (16, tokens, tokens))
    want, tight = attended_narrow(q, k, v, 0, causal=False)
    _, wide = attended(q, k, v, 0, causal=False)
    one, two = (planted(q[:, 0], k[:, 0], v[:, 0], parts)[:, None] for parts in (1, 2))
    within(two, want, tight, "two parts")
    within(one, want, wide, "one part")
    with pytest.raises(AssertionError):
        within(one, want, tight, "one part")
