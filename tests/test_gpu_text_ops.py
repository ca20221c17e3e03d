"""A text decoder's operators against their formulas in 64 bits (on the CPU).

Tolerances: u = 2^-8 is the most a rounding to bf16 moves a value by, relative to it; an e4m3 code (4 significant
bits, smallest step 2^-9) is within max(2^-4 |v|, 2^-10) of the value it rounds; an fp32 sum of n terms within
n · 2^-24 of the sum of their sizes."""
import math

import pytest
import torch

import siliconed_amd as sq
from siliconed_amd import _abi as abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
BF = torch.bfloat16
U = 2.0 ** -8


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g)


def wide(t, extra, offset):
    """`t` on the GPU as a view into a wider buffer, `offset` values in: rows that are not aligned or contiguous."""
    rows, cols = t.shape
    buffer = torch.zeros(rows * (cols + extra) + offset, dtype=t.dtype, device=DEV)
    if buffer.dtype == F8:
        buffer = buffer.view(torch.uint8)
        view = buffer[offset:].view(rows, cols + extra)[:, :cols]
        view.copy_(t.view(torch.uint8))
        return view.view(F8)
    view = buffer[offset:].view(rows, cols + extra)[:, :cols]
    view.copy_(t)
    return view


def groups(k):
    return -(-k // 128)


def within(got, want, tol, what):
    got, want = got.double().cpu(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((got - want).abs().max())} (tolerance there {float(tol.max())})")


def norm_oracle(x, r, w, eps):
    s = x.double() if r is None else x.double() + r.double()
    return s, s / torch.sqrt(s.pow(2).mean(1, keepdim=True) + eps) * w.double()


def check_codes(codes, scales, y, int8):
    """Codes and scales against y in 64 bits. The norm's fp32 arithmetic moves y by less than 2e-6 of it: the sum of
    squares (in runs of at most 32 values a lane and a tree, under 40 roundings of positive terms), its mean, square root
    and reciprocal, two products: under 45 · 2^-24."""
    y = y.double()
    slack = 4e-6
    if int8:
        top = (y.abs().amax(1) / 127).clamp_min(1e-30)
        within(scales, top, slack * top, "scales")
        within(codes, y / top[:, None], 0.5 + 127 * 2 * slack, "codes")
        return
    k = y.shape[1]
    padded = torch.nn.functional.pad(y, (0, -k % 128)).view(y.shape[0], -1, 128)
    top = (padded.abs().amax(2) / 448).clamp_min(1e-30)
    within(scales, top, slack * top, "scales")
    v = y / top.repeat_interleave(128, 1)[:, :k]
    within(codes.float(), v, (v.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) * (1 + 1e-4) + v.abs() * 2 * slack, "codes")


NORM_SHAPES = [(1, 8), (3, 1), (2, 127), (5, 128), (1, 129), (4, 1000), (33, 2760), (2, 4096), (7, 5120), (2, 8200),
               (3, 16384), (2, 20001), (1, 32768), (9000, 24), (2500, 1032)]


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [F8, torch.int8], ids=["e4m3", "int8"])
def test_add_norm(gemm, rows, cols, dtype):
    g = gen(rows * 31 + cols)
    for xt, rt in ((BF, BF), (torch.float32, BF), (BF, torch.float32), (BF, None)):
        print(f"norm {rows} x {cols} x {xt} residual {rt} {dtype}", flush=True)
        x, w = normal(g, rows, cols).to(xt), 1 + 0.2 * normal(g, cols)
        r = None if rt is None else (3 * normal(g, rows, cols)).to(rt)
        s, y = norm_oracle(x, r, w, 1e-6)
        rd = None if r is None else r.to(DEV)
        codes, scales, out = gemm.add_norm_quantized(x.to(DEV), w.to(DEV), 1e-6, residual=rd, dtype=dtype)
        check_codes(codes, scales, y, dtype == torch.int8)
        if r is None:
            assert out is None
        else:
            assert out is rd  # in place
            within(out, s, s.abs() * (U if rt == BF else 2.0 ** -23), "stream")


@pytest.mark.parametrize("dtype", [F8, torch.int8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("extra,offset", [(8, 8), (3, 0), (0, 1), (5, 3)])
def test_add_norm_strided_and_unaligned(gemm, dtype, extra, offset):
    g = gen(5)
    for rows, cols in ((3, 256), (2, 1111)):
        x, r, w = normal(g, rows, cols).to(BF), normal(g, rows, cols), 1 + 0.2 * normal(g, cols)
        s, y = norm_oracle(x, r, w, 1e-5)
        out = wide(torch.zeros(rows, cols), extra, offset)
        codes = wide(torch.zeros(rows, cols).to(dtype), extra, offset)
        before = r.to(DEV)
        got, scales, back = gemm.add_norm_quantized(wide(x, extra, offset), w.to(DEV), 1e-5, residual=wide(before, extra, offset),
                                                    residual_out=out, dtype=dtype, codes=codes)
        assert got is codes and back is out
        check_codes(codes, scales, y, dtype == torch.int8)
        within(out, s, s.abs() * 2.0 ** -23, "stream")


def test_add_norm_of_nothing_and_of_values_past_all(gemm):
    x = torch.zeros(4, 256, dtype=BF, device=DEV)
    x[1, 3] = math.inf
    x[2, 200] = math.nan
    x[3] = 1e-30
    w = torch.ones(256, device=DEV)
    codes, scales, _ = gemm.add_norm_quantized(x, w, 1e-6)
    c, t = codes.float().cpu(), scales.cpu()
    assert (c[0] == 0).all() and (t[0] == torch.tensor(1e-30)).all()
    assert torch.isnan(c[1, 3])  # inf / inf; the others of the row are 0
    assert torch.isnan(c[2]).all()  # the row's mean is NaN
    assert (t[3] > 0).all() and torch.isfinite(t[3]).all() and (c[3] == 448).all()
    codes, scales, _ = gemm.add_norm_quantized(x[:1], w, 1e-6, dtype=torch.int8)
    assert (codes == 0).all() and float(scales[0]) == pytest.approx(1e-30)
    for shape in ((0, 256), (3, 0)):
        codes, scales, _ = gemm.add_norm_quantized(torch.zeros(shape, device=DEV), torch.ones(shape[1], device=DEV))
        assert codes.shape == shape


def test_add_norm_int8_feeds_the_w8a8_product(gemm):
    """The int8 codes are what quantize_rows writes from the norm's row in fp32: rows whose mean square is a power of four
    and weights of 1 make the norm exact, so the two must agree bit for bit."""
    x = torch.zeros(3, 256, device=DEV)
    x[:, ::4] = torch.randint(0, 2, (3, 64), device=DEV) * 2.0 - 1.0  # 64 of 256: mean square 1/4
    x[:, 1::4] = 0.0
    codes, scales, _ = gemm.add_norm_quantized(x, torch.ones(256, device=DEV), 0.0, dtype=torch.int8)
    want, t = gemm.quantize_rows(2 * x)
    assert torch.equal(codes, want) and torch.equal(scales, t)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 128), (2, 130), (17, 1000), (5, 4096), (300, 264)])
@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "f32"])
def test_quantize_groups(gemm, rows, cols, dtype):
    g = gen(cols)
    x = (normal(g, rows, cols) * torch.exp(3 * normal(g, rows, 1))).to(dtype)
    codes, scales = gemm.quantize_groups(x.to(DEV))
    check_codes(codes, scales, x, False)
    codes, scales = gemm.quantize_groups(wide(x, 3, 1), codes=wide(torch.zeros(rows, cols).to(F8), 1, 1))
    check_codes(codes, scales, x, False)


# ---- the product -----------------------------------------------------------------------------------------------


def operands(g, m, k, n, glu):
    a, w = normal(g, m, k).mul(60).to(F8), normal(g, n, k).mul(100).clamp(-448, 448).to(F8)
    blocks = 2 * groups(n // 2) if glu else groups(n)
    sx = torch.rand(m, groups(k), generator=g) * 0.02 + 1e-3
    sw = torch.rand(blocks, groups(k), generator=g) * 2e-3 + 1e-4
    return a, sx, w, sw


def alignment(ad, wd):
    """What the e4m3 matrix instructions may drop for a bf16 C: of each 8 consecutive K, seven products up to 2^-13 of
    the largest one's power of two, summed over K."""
    m, k = ad.shape
    a, w = (torch.nn.functional.pad(t.abs(), (0, -k % 8)).view(t.shape[0], -1, 8) for t in (ad, wd))
    found = torch.zeros(m, w.shape[0], dtype=torch.float64)
    for i in range(m):
        found[i] = (a[i] * w).amax(2).sum(1)
    return 7 * 2.0 ** -13 * found


def product_oracle(a, sx, w, sw, bias, glu, out):
    """(C, the tolerance): each block's 128 exact products summed in fp32 (a bf16 C: but for their alignment), the
    blocks' sums in fp32."""
    m, k = a.shape
    n = w.shape[0]
    h = n // 2 if glu else n
    at = torch.arange(h) // 128
    rows = torch.cat([at, at + groups(h)]) if glu else at
    sxk = sx.double().repeat_interleave(128, 1)[:, :k]
    swk = sw.double().repeat_interleave(128, 1)[:, :k][rows]
    ad, wd = a.double() * sxk, w.double() * swk
    c = ad @ wd.t()
    err = (128 + groups(k) + 4) * 2.0 ** -24 * (ad.abs() @ wd.abs().t())
    if out == BF:
        err = err + alignment(ad, wd)
    if bias is not None:
        c = c + bias.double()
        err = err + 2.0 ** -24 * c.abs()
    if glu:
        gate, up = c[:, :h], c[:, h:]
        sig = torch.sigmoid(gate)
        # silu has slope under 1.1; its exponential's argument is rounded: |gate| · 2^-23 of the result.
        err = 1.1 * err[:, :h] * up.abs() + (gate * sig).abs() * err[:, h:] + (gate * sig * up).abs() * (gate.abs() + 8) * 2.0 ** -22
        c = gate * sig * up
    return c, err + (c.abs() + err) * (U if out == BF else 2.0 ** -23) + 1e-37


def run_product(gemm, m, k, n, glu, bias, out, seed=0, a_view=None, w_view=None):
    g = gen(m * 7 + k * 3 + n + seed)
    a, sx, w, sw = operands(g, m, k, n, glu)
    b = normal(g, n) if bias else None
    want, tol = product_oracle(a, sx, w, sw, b, glu, out)
    print(f"f8 product {m} x {k} x {n} glu {glu} bias {bias} {out}", flush=True)
    got = gemm.product_f8((a_view or (lambda t: t.to(DEV)))(a), sx.to(DEV), (w_view or (lambda t: t.to(DEV)))(w), sw.to(DEV),
                          bias=None if b is None else b.to(DEV), epilogue="silu_glu" if glu else None, out_dtype=out)
    assert got.dtype == out and tuple(got.shape) == (m, n // 2 if glu else n)
    within(got, want, tol, "product")


PRODUCT_SHAPES = [(1, 128, 16), (1, 16, 1), (3, 144, 7), (16, 1024, 130), (17, 256, 200), (33, 2496, 96), (64, 640, 256),
                  (65, 128, 384), (100, 4096, 64), (129, 512, 300), (257, 384, 520), (300, 1152, 1030), (513, 256, 257)]


@pytest.mark.parametrize("m,k,n", PRODUCT_SHAPES)
@pytest.mark.parametrize("out", [BF, torch.float32], ids=["bf16", "f32"])
def test_product_f8(gemm, m, k, n, out):
    run_product(gemm, m, k, n, False, False, out)
    run_product(gemm, m, k, n, False, True, out)
    run_product(gemm, m, k, 2 * n, True, m % 2 == 0, out)


@pytest.mark.parametrize("m,k,n", [(48, 8192, 40), (64, 9216 + 48, 130), (300, 12288, 96), (20, 16384 + 16, 64), (700, 2560, 1100),
                                   (1537, 640, 2570), (2049, 1296, 1300), (3000, 256, 4100)])
@pytest.mark.parametrize("out", [BF, torch.float32], ids=["bf16", "f32"])
def test_product_f8_large(gemm, m, k, n, out):
    """Long sums split over workgroups, more than 64 blocks of K, and each of the tiles: rows, columns and K that end
    inside them. Checked at rows and columns taken from all over, and the edges."""
    for glu in (False, True):
        g = gen(m + k + n)
        a, sx, w, sw = operands(g, m, k, 2 * n if glu else n, glu)
        rows = torch.unique(torch.cat([torch.randint(0, m, (40,), generator=g), torch.arange(max(0, m - 18), m), torch.arange(min(18, m))]))
        print(f"f8 product {m} x {k} x {n} glu {glu} {out}", flush=True)
        want, tol = product_oracle(a[rows], sx[rows], w, sw, None, glu, out)
        got = gemm.product_f8(a.to(DEV), sx.to(DEV), w.to(DEV), sw.to(DEV), epilogue="silu_glu" if glu else None, out_dtype=out)
        within(got[rows.to(DEV)], want, tol, "product")


@pytest.mark.parametrize("k", [1, 8, 17, 100, 130, 1001])
@pytest.mark.parametrize("m", [2, 70])
def test_product_f8_ragged_k(gemm, m, k):
    run_product(gemm, m, k, 72, False, True, torch.float32)
    run_product(gemm, m, k, 72, True, False, BF)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_product_f8_strided_and_unaligned(gemm, m):
    for extra, offset in ((16, 16), (1, 0), (0, 5)):
        view = lambda t: wide(t, extra, offset)  # noqa: E731
        run_product(gemm, m, 256, 136, False, False, BF, a_view=view)
        run_product(gemm, m, 256, 136, False, True, torch.float32, w_view=view)
    # The output's rows apart, an odd distance; scales' rows apart.
    g = gen(m)
    a, sx, w, sw = operands(g, m, 384, 75, False)
    want, tol = product_oracle(a, sx, w, sw, None, False, torch.float32)
    buffer = torch.full((m, 99), 7.0, device=DEV)
    gemm.product_f8(a.to(DEV), wide(sx, 2, 1), w.to(DEV), wide(sw, 4, 3), out=buffer[:, 3:78])
    within(buffer[:, 3:78], want, tol, "product")
    assert (buffer[:, :3] == 7).all() and (buffer[:, 78:] == 7).all()


def test_product_f8_edges(gemm):
    a, sx, w, sw = (t.to(DEV) for t in operands(gen(1), 5, 256, 40, False))
    assert gemm.product_f8(a[:0], sx[:0], w, sw).shape == (0, 40)
    assert gemm.product_f8(a, sx, w[:0], sw[:0]).shape == (5, 0)
    bias = torch.arange(40, dtype=torch.float32, device=DEV)
    none = gemm.product_f8(a[:, :0].contiguous(), sx[:, :0].contiguous(), w[:, :0].contiguous(), sw[:, :0].contiguous(),
                           bias=bias, out_dtype=torch.float32)
    assert torch.equal(none, bias.expand(5, 40))
    # A NaN code makes its row, or its column, NaN and nothing else.
    bad = a.clone()
    bad.view(torch.uint8)[2, 77] = 0x7F
    worse = w.clone()
    worse.view(torch.uint8)[9, 200] = 0xFF
    got = torch.isnan(gemm.product_f8(bad, sx, worse, sw)).cpu()
    want = torch.zeros(5, 40, dtype=torch.bool)
    want[2], want[:, 9] = True, True
    assert torch.equal(got, want)
    # gpu seconds
    out, seconds = gemm.product_f8(a, sx, w, sw, timed=True)
    assert seconds > 0 and torch.equal(out, gemm.product_f8(a, sx, w, sw))


@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (48, 1000, 200), (200, 640, 384)])
@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "f32"])
def test_product_f8_quantized_is_both_steps(gemm, m, k, n, dtype):
    g = gen(m)
    x = normal(g, m, k).to(dtype).to(DEV)
    _, _, w, sw = (t.to(DEV) for t in operands(g, 1, k, n, True))
    codes, sx = gemm.quantize_groups(x)
    for epilogue in (None, "silu_glu"):
        s = sw if epilogue else sw[:groups(n)]
        got = gemm.product_f8_quantized(x, w, s, epilogue=epilogue)
        assert torch.equal(got, gemm.product_f8(codes, sx, w, s, epilogue=epilogue))


def test_product_f8_past_32_bits(gemm):
    """Rows so far apart that their offsets pass 32 bits."""
    a, sx, w, sw = operands(gen(3), 20, 256, 40, False)
    want, tol = product_oracle(a, sx, w, sw, None, False, torch.float32)
    far = 240 << 20
    buffer = torch.empty(far * 19 + 256, dtype=torch.uint8, device=DEV)
    view = buffer.as_strided((20, 256), (far, 1))
    view.copy_(a.view(torch.uint8))
    within(gemm.product_f8(view.view(F8), sx.to(DEV), w.to(DEV), sw.to(DEV), out_dtype=torch.float32), want, tol, "product")


# ---- the cache -----------------------------------------------------------------------------------------------------


def rotated(t, angles, interleaved):
    half = angles.shape[1] // 2
    t, c, s = t.double().clone(), angles[:, None, :half].double(), angles[:, None, half:].double()
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = t[..., i].clone(), t[..., j].clone()
    t[..., i], t[..., j] = a * c - b * s, b * c + a * s
    return t


def code_tolerance(v):
    return (v.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) * (1 + 1e-4)


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,qh,kvh,dim,rot,page", [(1, 1, 1, 2, 2, 1), (5, 4, 2, 128, 128, 16), (130, 8, 8, 64, 32, 24),
                                                        (7, 5, 1, 96, 48, 5), (3, 6, 3, 40, 36, 64), (33, 40, 8, 256, 0, 16),
                                                        (11, 3, 3, 18, 10, 7)])
def test_append(gemm, dtype, interleaved, tokens, qh, kvh, dim, rot, page):
    g = gen(tokens + dim)
    row = (qh + 2 * kvh) * dim
    qkv = normal(g, tokens, row).to(BF)
    angles = 6.3 * torch.rand(50, rot // 2, generator=g)
    table = torch.cat([angles.cos(), angles.sin()], 1)
    positions = torch.randint(0, 50, (tokens,), generator=g, dtype=torch.int32)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    if tokens > 4:
        slots[1], slots[3] = -1, pages * page  # neither is written
    scales = [0.01 + 0.02 * torch.rand(kvh, generator=g) for _ in range(2)] if dtype == F8 else [None, None]
    fill = torch.full((pages, page, kvh, dim), 3.0)
    pools = [fill.to(dtype).to(DEV) for _ in range(2)]
    cache = sq.PagedCache(*pools, *(None if s is None else s.to(DEV) for s in scales))
    dev = qkv.to(DEV)
    q, k, v = (t.view(tokens, -1, dim) for t in dev.split([qh * dim, kvh * dim, kvh * dim], 1))
    out = gemm.append_kv(q, k, v, cache, positions.to(DEV), slots.to(DEV), table.to(DEV), interleaved=interleaved)
    assert torch.equal(dev.cpu(), qkv)
    cq, ck, cv = (t.view(tokens, -1, dim) for t in qkv.split([qh * dim, kvh * dim, kvh * dim], 1))
    at = table[positions.long()]
    size = lambda t: t.double().abs().amax(-1, keepdim=True) * 2  # noqa: E731
    want = rotated(cq, at, interleaved)
    within(out, want, want.abs() * U + size(cq) * 2.0 ** -22, "q")
    for pool, t, s in zip(pools, (rotated(ck, at, interleaved), cv.double()), scales):
        expect = fill.double()
        tol = torch.zeros_like(expect)
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                w = t[i] if s is None else (t[i] / s[:, None].double()).clamp(-448, 448)
                expect[slot // page, slot % page] = w
                slack = (2.0 ** -22 * size(t[i]) / (1 if s is None else s[:, None].double())).expand_as(w)
                tol[slot // page, slot % page] = (w.abs() * U if s is None else code_tolerance(w)) + slack
        within(pool.float(), expect, tol, "pool")
    # In place, from contiguous heads, to a pool laid out head by head.
    headed = [fill.to(dtype).to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for _ in range(2)]
    cache = sq.PagedCache(*headed, cache.k_scale, cache.v_scale)
    same = cq.contiguous().to(DEV)
    back = gemm.append_kv(same, ck.contiguous().to(DEV), cv.contiguous().to(DEV), cache, positions.to(DEV), slots.to(DEV),
                          table.to(DEV), q_out=same, interleaved=interleaved)
    assert back is same and torch.equal(same, out)
    for a, b in zip(headed, pools):
        assert torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))


def test_append_saturates_and_clamps_positions(gemm):
    pools = [torch.zeros(1, 16, 1, 16, device=DEV).to(F8) for _ in range(2)]
    scale = torch.tensor([0.5], device=DEV)
    cache = sq.PagedCache(*pools, scale, scale)
    x = torch.full((2, 1, 16), 1000.0, dtype=BF, device=DEV)
    x[1] = -1000.0
    x[1, 0, 3] = math.nan
    table = torch.cat([torch.ones(4, 8), torch.zeros(4, 8)], 1).to(DEV)
    table[3, :8] = 0.5  # the last row, which positions outside the table take
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    q = gemm.append_kv(x, x, x, cache, i32(-5, 900), i32(0, 1), table)
    assert (q[0] == 500).all()
    v = pools[1].float().cpu()[0, :2, 0]
    assert (v[0] == 448).all() and torch.isnan(v[1, 3]) and (v[1][torch.arange(16) != 3] == -448).all()


def attention_oracle(q, k, v, first, last, scale, softcap):
    """One sequence in 64 bits: q [heads, dim], k, v [tokens, kv_heads, dim]; (o, the tolerance)."""
    heads, dim = q.shape
    kvh = k.shape[1]
    o, tol = torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64)
    if last <= first:
        return o, tol
    k, v = k[first:last].double(), v[first:last].double()
    for h in range(heads):
        kk, vv = k[:, h // (heads // kvh)], v[:, h // (heads // kvh)]
        s = kk @ q[h].double() * scale
        # dim products' sum, the scale and the softmax's base change in fp32; tanh is within 1e-6 of its size.
        off = (dim + 8) * 2.0 ** -24 * (kk.abs() @ q[h].double().abs()).max() * abs(scale) + 4e-6 * (1 + s.abs().max())
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        p = torch.softmax(s, 0)
        o[h] = p @ vv
        tol[h] = (U + 2 * off) * (p @ vv.abs()) + U * o[h].abs() + 1e-6 * vv.abs().max()
    return o, tol


def run_attention(gemm, lengths, qh, kvh, dim, page, dtype, window=0, softcap=0.0, scale=None, by_head=False, extra_pages=2,
                  seed=0, bad=()):
    """Random pages in random order, everything that no sequence holds set to NaN. `bad`: (sequence, page number, index) of
    page table entries replaced by an index outside the pools: those tokens count as masked."""
    g = gen(seed + sum(lengths) + dim + qh)
    print(f"attention lengths {lengths[:6]} heads {qh}/{kvh} dim {dim} page {page} {dtype} window {window} cap {softcap}", flush=True)
    batch = len(lengths)
    each = max(1, max(-(-n // page) for n in lengths)) + 1
    total = sum(-(-n // page) for n in lengths) + extra_pages
    order = torch.randperm(total, generator=g)
    table = torch.full((batch, each), -7, dtype=torch.int32)
    pools = [torch.full((total, page, kvh, dim), math.nan) for _ in range(2)]
    scales = [0.5 + torch.rand(kvh, generator=g) for _ in range(2)] if dtype == F8 else [None, None]
    values, at = [], 0
    for b, n in enumerate(lengths):
        count = -(-n // page)
        table[b, :count] = order[at:at + count].to(torch.int32)
        at += count
        kv = [normal(g, n, kvh, dim).to(dtype).float() for _ in range(2)]
        for pool, t in zip(pools, kv):
            for i in range(count):
                rows = t[i * page:(i + 1) * page]
                pool[table[b, i], :rows.shape[0]] = rows
        values.append([t if s is None else t * s[:, None] for t, s in zip(kv, scales)])
    dead = {}
    for b, i, index in bad:
        table[b, i] = index
        dead.setdefault(b, []).append(i)
    pools = [p.to(dtype).to(DEV) for p in pools]
    if by_head:
        pools = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in pools]
    cache = sq.PagedCache(*pools, *(None if s is None else s.to(DEV) for s in scales))
    q = normal(g, batch, qh, dim).to(BF)
    got = gemm.paged_attention(q.to(DEV), cache, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=scale,
                               softcap=softcap, window=window).cpu()
    for b, n in enumerate(lengths):
        k, v = values[b]
        first, last = max(0, n - window) if window else 0, n
        if b in dead:
            keep = torch.tensor([t for t in range(first, last) if t // page not in dead[b]], dtype=torch.long)
            k, v, first, last = k[keep], v[keep], 0, len(keep)
        want, tol = attention_oracle(q[b], k, v, first, last, 1 / math.sqrt(dim) if scale is None else scale, softcap)
        within(got[b], want, tol, f"sequence {b} of length {n}")
    return got


LENGTHS = [0, 1, 15, 16, 17, 31, 32, 33, 100, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64])
def test_attention_lengths_and_pages(gemm, dtype, page):
    run_attention(gemm, LENGTHS, 8, 2, 128, page, dtype)


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("qh,kvh,dim", [(1, 1, 64), (8, 8, 128), (5, 1, 96), (40, 8, 128), (32, 1, 128), (20, 1, 64), (6, 2, 256),
                                        (3, 3, 16), (4, 2, 80), (4, 1, 192), (12, 4, 48)])
def test_attention_heads_and_dims(gemm, dtype, qh, kvh, dim):
    for page in (16, 7):
        run_attention(gemm, [3, 200, 0, 65], qh, kvh, dim, page, dtype, by_head=page == 7)


@pytest.mark.parametrize("dim", [8, 24, 40, 72, 120])
def test_attention_narrow_dims_in_bf16(gemm, dim):
    run_attention(gemm, [90, 4], 4, 2, dim, 16, BF)


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("window", [1, 16, 50, 128, 500, 5000])
def test_attention_window(gemm, dtype, window):
    run_attention(gemm, [0, 1, 49, 50, 51, 700, 1400], 8, 2, 64, 16, dtype, window=window)
    run_attention(gemm, [129, 260], 4, 4, 128, 3, dtype, window=window)


@pytest.mark.parametrize("softcap", [0.5, 30.0])
def test_attention_softcap_and_scale(gemm, softcap):
    run_attention(gemm, [1, 140, 500], 8, 2, 128, 16, BF, softcap=softcap)
    run_attention(gemm, [1, 140, 500], 8, 2, 128, 16, F8, softcap=softcap, scale=1.0)
    run_attention(gemm, [140], 8, 2, 64, 16, BF, scale=-0.3)
    run_attention(gemm, [140], 8, 2, 64, 16, BF, scale=0.0)


@pytest.mark.parametrize("dtype", [BF, F8], ids=["bf16", "e4m3"])
def test_attention_split_over_workgroups(gemm, dtype):
    run_attention(gemm, [9001], 4, 1, 128, 16, dtype)
    run_attention(gemm, [5000, 0, 3, 8000, 130], 16, 2, 64, 32, dtype)
    run_attention(gemm, [3000, 1500], 2, 2, 256, 9, dtype)


def test_attention_of_many_sequences(gemm):
    lengths = [(37 * i) % 290 for i in range(150)]
    lengths[64:70] = [0] * 6
    run_attention(gemm, lengths, 4, 2, 64, 16, BF)
    run_attention(gemm, [0] * 130 + [5], 4, 2, 64, 16, F8)
    run_attention(gemm, [0, 0, 0], 4, 2, 64, 16, BF)


def test_attention_masks_pages_outside_the_pools(gemm):
    for page in (16, 5):
        run_attention(gemm, [200, 64], 4, 2, 64, page, BF, bad=[(0, 1, -1), (0, 3, 1 << 30), (1, 0, 99999)])
    got = run_attention(gemm, [16, 40], 4, 2, 64, 16, BF, bad=[(0, 0, -1)])
    assert (got[0] == 0).all()


def test_attention_cuts_lengths_to_the_table(gemm):
    g = gen(9)
    k, v = (normal(g, 3, 16, 1, 64).to(BF).to(DEV) for _ in range(2))
    cache = sq.PagedCache(k, v)
    q = normal(g, 3, 2, 64).to(BF).to(DEV)
    table = torch.tensor([[2, 0], [1, 2], [0, 1]], dtype=torch.int32, device=DEV)
    lengths = lambda *n: torch.tensor(n, dtype=torch.int32, device=DEV)  # noqa: E731
    got = gemm.paged_attention(q, cache, table, lengths(1 << 30, -4, 32))
    want = gemm.paged_attention(q, cache, table, lengths(32, 0, 32))
    assert torch.equal(got, want) and (got[1] == 0).all()
    assert gemm.paged_attention(q[:0], cache, table[:0], lengths()).shape == (0, 2, 64)
    none = gemm.paged_attention(q, cache, table[:, :0], lengths(5, 5, 5))
    assert (none == 0).all()


def test_attention_of_infinite_and_nan_values(gemm):
    """A NaN or an infinity that a sequence holds is its own; a key of -inf scores hides its token."""
    g = gen(4)
    k, v = (normal(g, 2, 64, 1, 64).to(BF) for _ in range(2))
    q = torch.ones(2, 1, 64, dtype=BF)
    k[0, 5] = -math.inf
    v[1, 7] = math.nan
    cache = sq.PagedCache(k.to(DEV), v.to(DEV))
    table = torch.tensor([[0], [1]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([60, 60], dtype=torch.int32, device=DEV)
    got = gemm.paged_attention(q.to(DEV), cache, table, lengths).cpu()
    keep = [t for t in range(60) if t != 5]
    want, tol = attention_oracle(q[0], k[0, keep], v[0, keep], 0, 59, 1 / 8, 0.0)
    within(got[0], want, tol, "a hidden token")
    assert torch.isnan(got[1]).all()
    k[0, :60] = -math.inf  # every score of the row the lowest there is
    got = gemm.paged_attention(q.to(DEV), sq.PagedCache(k.to(DEV), v.to(DEV)), table, lengths).cpu()
    assert (got[0] == 0).all()


def test_cache_past_32_bits(gemm):
    """Pages so far apart that offsets in the pools pass 32 bits, appended to and read."""
    g = gen(11)
    far = 300 << 20
    pools = []
    for _ in range(2):
        buffer = torch.empty(far * 16 + 16 * 2 * 64, dtype=torch.uint8, device=DEV).view(F8)
        pools.append(buffer.as_strided((17, 16, 2, 64), (far, 128, 64, 1)))
    cache = sq.PagedCache(*pools)
    n = 40
    x = [normal(g, n, 2, 64).to(F8).to(BF) for _ in range(2)]
    slots = torch.tensor([(16, 3, 15)[t // 16] * 16 + t % 16 for t in range(n)], dtype=torch.int32)
    table = torch.cat([torch.ones(1, 32), torch.zeros(1, 32)], 1)
    q = normal(g, n, 4, 64).to(BF)
    zeros = torch.zeros(n, dtype=torch.int32, device=DEV)
    out = gemm.append_kv(q.to(DEV), x[0].to(DEV), x[1].to(DEV), cache, zeros, slots.to(DEV), table.to(DEV))
    assert torch.equal(out.cpu(), q)
    pages = torch.tensor([[16, 3, 15]], dtype=torch.int32, device=DEV)
    got = gemm.paged_attention(out[:1], cache, pages, torch.tensor([n], dtype=torch.int32, device=DEV)).cpu()
    want, tol = attention_oracle(q[0], x[0].float(), x[1].float(), 0, n, 1 / 8, 0.0)
    within(got[0], want, tol, "attention")


def test_attention_is_the_same_each_time(gemm):
    a = run_attention(gemm, [9001, 40, 2000], 8, 2, 128, 16, BF)
    b = run_attention(gemm, [9001, 40, 2000], 8, 2, 128, 16, BF)
    assert torch.equal(a, b)


def test_step_in_a_graph(gemm):
    """Append and attention captured once; the replays follow the positions, slots and lengths written between them."""
    g = gen(21)
    pools = [torch.zeros(40, 16, 2, 64, dtype=BF, device=DEV) for _ in range(2)]
    angles = 6.3 * torch.rand(600, 32, generator=g)
    table = torch.cat([angles.cos(), angles.sin()], 1).to(DEV)
    pages = torch.randperm(40, generator=g)[:36].view(1, 36).to(torch.int32).to(DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = sq.TensorGEMM.make(0, stream)
        cache = sq.PagedCache(*pools)
        q, k, v = (normal(g, 1, h, 64).to(BF).to(DEV) for h in (4, 2, 2))
        where = [torch.zeros(1, dtype=torch.int32, device=DEV) for _ in range(3)]
        qo, out = torch.empty_like(q), torch.empty_like(q)

        def step():
            ctx.append_kv(q, k, v, cache, where[0], where[1], table, q_out=qo)
            ctx.paged_attention(qo, cache, pages, where[2], out=out)

        def place(t):
            where[0].fill_(t)
            where[1].copy_(pages[0, t // 16:t // 16 + 1] * 16 + t % 16)
            where[2].fill_(t + 1)

        place(0)
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for t in range(560):
            for x in (q, k, v):
                x.copy_(normal(g, *x.shape).to(BF))
            place(t)
            graph.replay()
            if t % 111 == 0 or t == 559:
                got = out.clone(), [p.clone() for p in pools]
                step()
                stream.synchronize()
                assert torch.equal(got[0], out)
                assert all(torch.equal(a, b) for a, b in zip(got[1], pools))
        stream.synchronize()
        del graph
        ctx.close()


# ---- refusals -----------------------------------------------------------------------------------------------------


def test_refusals(gemm):
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    w = torch.ones(64, device=DEV)
    for call in (lambda: gemm.add_norm_quantized(z(2, 64).half(), w), lambda: gemm.add_norm_quantized(z(2, 64), w[:63]),
                 lambda: gemm.add_norm_quantized(z(2, 64), w, dtype=torch.float16),
                 lambda: gemm.add_norm_quantized(z(2, 64), w, residual=z(2, 63)),
                 lambda: gemm.add_norm_quantized(z(2, 64), w, residual_out=z(2, 64)),
                 lambda: gemm.add_norm_quantized(z(2, 64).cpu(), w), lambda: gemm.add_norm_quantized(z(64, 2).t(), w),
                 lambda: gemm.quantize_groups(z(2, 64).half()),
                 lambda: gemm.product_f8(z(2, 128), z(2, 1, dtype=torch.float32), z(4, 128, dtype=F8), z(1, 1, dtype=torch.float32)),
                 lambda: gemm.product_f8(z(2, 128, dtype=F8), z(2, 2, dtype=torch.float32), z(4, 128, dtype=F8), z(1, 1, dtype=torch.float32)),
                 lambda: gemm.product_f8_quantized(z(2, 128), z(4, 120, dtype=F8), z(1, 1, dtype=torch.float32)),
                 lambda: gemm.product_f8_quantized(z(2, 128), z(4, 128, dtype=F8), z(1, 1, dtype=torch.float32), epilogue="gelu"),
                 lambda: gemm.product_f8_quantized(z(2, 128), z(5, 128, dtype=F8), z(2, 1, dtype=torch.float32), epilogue="silu_glu"),
                 lambda: sq.PagedCache(z(2, 16, 1, 64), z(2, 16, 1, 64, dtype=F8)), lambda: sq.PagedCache(z(2, 16, 64), z(2, 16, 64)),
                 lambda: sq.PagedCache(z(2, 16, 1, 64), z(2, 16, 1, 64), w[:1], w[:1])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(abi.Unsupported):
        gemm.add_norm_quantized(z(1, 32776), torch.ones(32776, device=DEV))
    cache = sq.PagedCache(z(2, 16, 2, 64), z(2, 16, 2, 64))
    table = z(9, 64, dtype=torch.float32)
    q, kv = z(3, 4, 64), z(3, 2, 64)
    for call in (lambda: gemm.append_kv(q, kv, z(3, 1, 64), cache, i32(3), i32(3), table),
                 lambda: gemm.append_kv(q, kv, kv, cache, i32(2), i32(3), table),
                 lambda: gemm.append_kv(q, kv, kv, cache, i32(3).long(), i32(3), table),
                 lambda: gemm.append_kv(q.float(), kv, kv, cache, i32(3), i32(3), table),
                 lambda: gemm.paged_attention(z(3, 4, 32), cache, i32(3, 2), i32(3)),
                 lambda: gemm.paged_attention(q, cache, i32(2, 2), i32(3)),
                 lambda: gemm.paged_attention(q, cache, i32(3, 2), i32(2))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(abi.SQ8Error):  # more rotated values than a head has
        gemm.append_kv(q, kv, kv, cache, i32(3), i32(3), z(9, 66, dtype=torch.float32))
    with pytest.raises(abi.Unsupported):  # pairs of an odd number
        gemm.append_kv(q, kv, kv, cache, i32(3), i32(3), z(9, 3, dtype=torch.float32))
    with pytest.raises(abi.SQ8Error):  # heads that do not divide
        gemm.paged_attention(z(3, 5, 64), cache, i32(3, 2), i32(3))
    with pytest.raises(abi.SQ8Error):
        gemm.paged_attention(q, cache, i32(3, 2), i32(3), window=-1)
    with pytest.raises(abi.SQ8Error):
        gemm.paged_attention(q, cache, i32(3, 2), i32(3), softcap=math.nan)
    for dim in (4, 264):
        odd = sq.PagedCache(z(2, 16, 1, dim), z(2, 16, 1, dim))
        with pytest.raises(abi.Unsupported):
            gemm.paged_attention(z(3, 1, dim), odd, i32(3, 2), i32(3))
    with pytest.raises(abi.Unsupported):  # rows that are not 16-byte aligned
        gemm.paged_attention(z(3, 4, 65)[:, :, 1:], cache, i32(3, 2), i32(3))
