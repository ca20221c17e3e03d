"""Block-scaled products' shapes, the kernel and parts of K that each takes on 256 CUs (test_text_plan.py asks the rule, without
a GPU), and the formula in 64 bits that the GPU tests of them share."""
import torch

F8 = torch.float8_e4m3fn

# (rows, K, N, GLU) of codes, up to 16 rows: waves of one block, of several at once and of several rounds; K that ends inside one.
FEW = [((1, 4096, 200, False), "short/1"), ((16, 4224, 200, False), "short/1"), ((4, 12304, 200, False), "short/1"),
       ((9, 8192, 75, False), "short/1"), ((1, 8192, 400, True), "short/1"), ((8, 12304, 400, True), "short/1"),
       ((1, 12304, 6149, False), "short wide/1"), ((4, 4224, 6149, False), "short wide/1"), ((16, 8192, 6149, False), "short wide/1"),
       ((9, 8192, 12298, True), "short wide/1"), ((16, 4224, 12298, True), "short wide/1")]

# (rows, K, N) of values, quantized on the way where their groups of 128 are at most 128: under, at and over.
VALUES = [((1, 16256, 6149), "staged wide/1"), ((1, 16384, 200), "staged/1"), ((1, 16400, 200), "short/1"), ((1, 12288, 4096), "staged/1"),
          ((1, 7424, 6149), "staged wide/1"), ((2, 8192, 4200), "staged wide/1"), ((2, 12288, 200), "short/1"), ((3, 5376, 200), "staged/1"),
          ((4, 4096, 6149), "staged wide/1"), ((8, 2048, 200), "staged/1"), ((9, 1792, 75), "staged/1"), ((9, 1920, 200), "short/1"),
          ((13, 1200, 200), "short/1"), ((16, 1008, 200), "staged/1"), ((16, 1024, 6149), "staged wide/1")]

# (rows, K, N, GLU), the choices for a bf16 and for an fp32 C: more than 64, and than 128, blocks of K in one workgroup; tiles
# of 64 x 128 and of 64 x 64 whose K is split.
LONG = [((2048, 12288, 4096, False), "128/1", "128/1"), ((1024, 12288, 8192, True), "128/1", "128/1"),
        ((4096, 8336, 8200, False), "256/1", "128/1"), ((1000, 16512, 4000, False), "128 one/1", "128 one/1"),
        ((1000, 16528, 4002, True), "128 one/1", "128 one/1"), ((300, 8320, 8200, False), "64x128/1", "64x128/1"),
        ((100, 12288, 4096, False), "64x128/4", "64x128/6"), ((128, 12304, 4098, True), "64x128/4", "64x128/7"),
        ((600, 9216, 1300, False), "64x128/3", "64x128/4"), ((33, 4096, 65, False), "64/4", "64/8")]


def formula(a, sx, w, sw):
    """The sums, the sizes of their terms, and the sizes of the largest of each eight, over K, in 64 bits."""
    y = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device=a.device)
    size, largest = torch.zeros_like(y), torch.zeros_like(y)
    for b in range(-(-a.shape[1] // 128)):
        at = slice(128 * b, min(a.shape[1], 128 * b + 128))
        scale = sx[:, b, None].double() * sw[:, b].double().repeat_interleave(128)[: w.shape[0]]
        x, z = a[:, at].double(), w[:, at].double()
        y += scale * (x @ z.T.contiguous())
        size += scale * (x.abs() @ z.abs().T.contiguous())
        for c in range(0, x.shape[1], 8):
            largest += scale * (x[:, None, c:c + 8].float() * z[None, :, c:c + 8].float()).abs().amax(-1)
    return y, size, largest


def product(a, sx, w, sw, bias, glu, out):
    """(C, its bound). A sum in fp32 of a block's four instructions, of K / 128 scaled blocks and of up to eight parts rounds
    at most K / 128 + 16 times, each by 2^-24 of the terms' sizes summed (doubled: an instruction's own sum may round more
    than once); the instructions of a bf16 C also drop what is under 2^-13 of the largest of eight products, at most 7 of
    them. A gate's error reaches the output by the slope of SiLU, under 1.1, times up, an up's by SiLU(gate), and their
    product; SiLU itself and its product are within 2^-20 of theirs. A bf16 C is then rounded by 2^-8 at most."""
    n, k = w.shape
    h = n // 2 if glu else n
    rows = -(-h // 128)

    def half(part):
        at = slice(part * h, part * h + h)
        y, size, largest = formula(a, sx, w[at], sw[part * rows:part * rows + rows])
        if bias is not None:
            y += bias[at].double()
            size = size + bias[at].double().abs()
        off = 2 * (k / 128 + 16) * 2.0 ** -24 * size
        return y, off + 7 * 2.0 ** -13 * largest if out == torch.bfloat16 else off

    y, bound = half(0)
    if glu:
        u, up = half(1)
        s = torch.nn.functional.silu(y)
        y, bound = s * u, 1.1 * bound * u.abs() + s.abs() * up + 1.1 * bound * up + 2.0 ** -20 * (s * u).abs()
    if out == torch.bfloat16:
        bound = bound + 2.0 ** -8 * (y.abs() + bound)
    return y, bound


def operands(m, k, n, glu, seed, device="cuda"):
    """Codes and scales, a weight's block scales a power of two apart between blocks of K that are 64 apart."""
    g = torch.Generator(device=device).manual_seed(seed)
    blocks, rows = -(-k // 128), 2 * -(-(n // 2) // 128) if glu else -(-n // 128)
    a = (torch.randn(m, k, generator=g, device=device) * 60).to(F8)
    w = (torch.randn(n, k, generator=g, device=device) * 60).to(F8)
    sx = torch.rand(m, blocks, generator=g, device=device) * 2e-2 + 1e-3
    sw = torch.rand(rows, blocks, generator=g, device=device) * 1e-3 + 1e-4
    sw *= 4.0 ** -(torch.arange(blocks, device=device) // 64)
    sx *= 4.0 ** (torch.arange(blocks, device=device) // 64 % 2)  # so that late blocks still count
    return a, sx, w, sw, torch.randn(n, generator=g, device=device)
