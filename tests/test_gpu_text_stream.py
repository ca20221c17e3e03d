"""A decoder layer under another stream than its context's: everything it queues goes to torch's current stream."""
import pytest
import torch

import siliconed_amd as sq

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def run(tb, block):
    """A prompt of 70 tokens and three steps after it."""
    d, page, most = block.d, 16, 8
    g = torch.Generator(device=DEV).manual_seed(9)
    cache = block.cache(most, page)
    pages = torch.arange(most, dtype=torch.int32, device=DEV).flip(0)
    table = tb.rotation_table(80, block.dim)

    def slots(at):
        return pages[at // page] * page + at.to(torch.int32) % page

    at = torch.arange(70, device=DEV)
    y = torch.randn(70, d, generator=g, device=DEV).to(torch.bfloat16)
    found = list(block.prompt(y, torch.zeros(70, d, device=DEV), cache, at.to(torch.int32), slots(at), pages, table))
    for t in range(70, 73):
        at = torch.tensor([t], device=DEV)
        y = torch.randn(1, d, generator=g, device=DEV).to(torch.bfloat16)
        found += block.step(y, torch.zeros(1, d, device=DEV), cache, at.to(torch.int32), slots(at), pages[None],
                            (at + 1).to(torch.int32), table)
    return found


def test_a_layer_follows_torch_s_current_stream(monkeypatch):
    from siliconed_amd import text_block as tb
    ctx = sq.TensorGEMM.make(0)
    block = tb.TextBlock(256, 4, 2, 64, 384, seed=6, ctx=ctx)
    want = run(tb, block)
    torch.cuda.synchronize()
    asked = []
    move = ctx.set_stream
    monkeypatch.setattr(ctx, "set_stream", lambda s: (asked.append(s.cuda_stream), move(s))[1])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run(tb, block)
    assert asked == [side.cuda_stream] * 4
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # Back on the first stream, and on the side one again after another context's user moved it away.
    assert all(torch.equal(a, b) for a, b in zip(run(tb, block), want))
    with torch.cuda.stream(side):
        got = run(tb, block)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    ctx.close()
