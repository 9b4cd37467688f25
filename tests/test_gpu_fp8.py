"""8-bit floating point on the GPU against plain 64-bit formulas: matrices in blocks, products with block scales, a layer's training step.

Codes and scales are compared for equality (the definition leaves no choice).  A product may be off by what its sums in 32-bit floats lose:
128 products in a block, the blocks and four roundings for the scales, a step of 2^-23 each (sums may be cut off, not rounded) relative to the sum
of magnitudes, and half a step of the result's type."""
import math

import pytest

pytestmark = pytest.mark.gpu

CODES = {"e4m3": ("float8_e4m3fn", 3, -6, 448.0), "e5m2": ("float8_e5m2", 2, -14, 57344.0)}
BLOCKS = {"rows": (1, 128), "columns": (128, 1), "square": (128, 128)}


@pytest.fixture(scope="module")
def ctx():
    from lancelot_b200 import cabi

    return cabi.Context(12, cabi.coeff_modulus_create(1 << 12, [40, 40]), 1)


def gen(seed):
    import torch

    return torch.Generator("cuda").manual_seed(seed)


def same(x, y):
    import torch

    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())


def spread(scales, rows, cols, block):
    s = scales.repeat_interleave(128, 0)[:rows] if block[0] == 128 else scales
    return s.repeat_interleave(128, 1)[:, :cols] if block[1] == 128 else s


def nearest(q, code):
    """the type's value nearest to q (64 bits), ties to even"""
    import torch

    _, bits, least, most = CODES[code]
    step = torch.exp2(((torch.frexp(q)[1] - 1).clamp(min=least) - bits).double())
    return ((q / step).round() * step).clamp(-most, most)


def quantized(v, block, code):
    """v [rows][cols] float32 -> the codes' values (64 bits) and the scales, from the definition"""
    import torch

    rows, cols = v.shape
    h, w = block
    t = torch.nn.functional.pad(v, (0, -cols % w, 0, -rows % h))
    most = t.reshape(t.shape[0] // h, h, t.shape[1] // w, w).abs().amax((1, 3))
    scales = torch.where(most.isfinite(), most / torch.full_like(most, CODES[code][3]), torch.full_like(most, math.nan))
    each = spread(scales, rows, cols, block).double()
    codes = nearest(v.double() / each, code)
    return torch.where(each > 0, codes, torch.zeros_like(codes)), scales


def dt(name):
    import torch

    return getattr(torch, name)


SIZES = [(1, 1), (1, 4096), (3, 130), (128, 128), (129, 257), (300, 16), (777, 1000), (5, 1003), (260, 384)]


@pytest.mark.parametrize("code", sorted(CODES))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_matrices_in_blocks(ctx, dtype, code, rows, cols):
    import torch

    g = gen(rows * cols)
    v = (torch.randn(rows, cols, generator=g, device="cuda") * torch.rand(1, cols, generator=g, device="cuda").mul(6).exp()).to(dt(dtype))
    v[:, ::7] = 0
    kind = dt(CODES[code][0])
    found = {}
    for name, block in BLOCKS.items():
        codes, scales = ctx.quantize_fp8(v, block, dtype=kind)
        want, want_scales = quantized(v.float(), block, code)
        assert codes.dtype == kind and torch.equal(scales, want_scales), name
        assert torch.equal(codes.double(), want), name
        found[name] = (codes, scales)
        for out in (torch.float32, torch.bfloat16, torch.float16):
            back = ctx.dequantize_fp8(codes, scales, dtype=out)
            assert same(back, (codes.float() * spread(scales, rows, cols, block)).to(out)), name
    both = ctx.quantize_fp8_both(v, dtype=kind)
    for got, want in zip(both, found["rows"] + found["columns"]):
        assert torch.equal(got.float(), want.float())


@pytest.mark.parametrize("code", sorted(CODES))
@pytest.mark.parametrize("block", sorted(BLOCKS))
def test_borders_between_codes_are_decided_exactly(ctx, code, block):
    """values on, and one step of 32 bits next to, what lies half way between two codes, among the codes below the normal numbers too"""
    import torch

    _, bits, least, most = CODES[code]
    levels = [math.ldexp(f, least - bits) for f in range(1 << bits)]
    levels += [math.ldexp((1 << bits) + f, e + least - bits) for e in range(40) for f in range(1 << bits)]
    levels = torch.tensor([x for x in levels if x <= most], dtype=torch.float64, device="cuda")
    half = (levels[1:] + levels[:-1]) / 2
    g = gen(3)
    rows, cols = 256, 512
    top = torch.rand(rows, cols, generator=g, device="cuda") * 10 + 0.1
    h, w = BLOCKS[block]
    top = top[: -(-rows // h), : -(-cols // w)]
    s = spread((top / torch.full_like(top, most)), rows, cols, (h, w)).double()
    pick = half[torch.randint(0, len(half), (rows, cols), generator=g, device="cuda")]
    v = (pick * s).float()
    step = torch.randint(-1, 2, (rows, cols), generator=g, device="cuda", dtype=torch.int32)
    v = (v.view(torch.int32) + step).view(torch.float32)
    v[::h, ::w] = top  # the largest of each block
    codes, scales = ctx.quantize_fp8(v, (h, w), dtype=dt(CODES[code][0]))
    want, want_scales = quantized(v, (h, w), code)
    assert torch.equal(scales, want_scales)
    assert torch.equal(codes.double(), want)


@pytest.mark.parametrize("code", sorted(CODES))
@pytest.mark.parametrize("block", sorted(BLOCKS))
def test_values_at_and_beside_every_code_and_every_border(ctx, code, block):
    """up to two steps of 32 bits beside, under many scales; the quotient that decides may itself be two steps off"""
    import torch

    _, bits, least, most = CODES[code]
    levels = [math.ldexp(f, least - bits) for f in range(1 << bits)]
    levels += [math.ldexp((1 << bits) + f, e + least - bits) for e in range(40) for f in range(1 << bits)]
    levels = torch.tensor([x for x in levels if x <= most], dtype=torch.float64, device="cuda")
    every = torch.cat([levels, (levels[1:] + levels[:-1]) / 2])
    every = torch.cat([every, every[(every >= 2.0 ** (least - 1)) & (every <= 2.0 ** (least + 1))].repeat(8)])  # around the least normal number
    h, w = BLOCKS[block]
    rows, cols = {"rows": (4096, 1024), "columns": (1024, 4096), "square": (6400, 6400)}[block]
    for seed in range(2):
        g = gen(30 + seed)
        top = torch.rand(-(-rows // h), -(-cols // w), generator=g, device="cuda") * 10 + 0.1
        s = spread(top / torch.full_like(top, most), rows, cols, (h, w))
        v = (every[torch.randint(0, len(every), (rows, cols), generator=g, device="cuda")] * s.double()).float()
        step = torch.randint(-2, 3, (rows, cols), generator=g, device="cuda", dtype=torch.int32)
        v = (v.view(torch.int32) + step).clamp(min=0).view(torch.float32)
        v = torch.minimum(v, s * most)
        v[::h, ::w] = top  # the largest of each block
        codes, scales = ctx.quantize_fp8(v, (h, w), dtype=dt(CODES[code][0]))
        want, want_scales = quantized(v, (h, w), code)
        assert torch.equal(scales, want_scales)
        wrong = (codes.double() != want).sum().item()
        assert wrong == 0, (wrong, v.numel())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("code", sorted(CODES))
def test_16_bit_values_at_the_least_normal_number(ctx, dtype, code):
    """every significand of a block's largest value, against the values of its type next to the least normal number times the scale; among them 41/1024 beside 1148 in
    16 bits, whose quotient is 2^-6"""
    import torch

    _, bits, least, most = CODES[code]
    kind = dt(dtype)
    n = 1024 if dtype == "float16" else 128
    top = ((1 + torch.arange(n, device="cuda").double() / n) * 1024).to(kind)
    s = (top.float() / torch.full((n,), most, device="cuda")).double()
    v = torch.zeros(n, 128, dtype=kind, device="cuda")
    near = (s * 2.0 ** least).to(kind)
    for i, step in enumerate(range(-3, 4)):
        v[:, i] = (near.view(torch.int16) + step).view(kind)
        v[:, 8 + i] = -v[:, i]
    v[:, 127] = top
    codes, scales = ctx.quantize_fp8(v, dtype=dt(CODES[code][0]))
    want, want_scales = quantized(v.float(), (1, 128), code)
    assert torch.equal(scales, want_scales) and torch.equal(codes.double(), want)
    if dtype == "float16" and code == "e4m3":
        x = torch.zeros(1, 128, dtype=kind, device="cuda")
        x[0, 0], x[0, 1] = 1148, 41 / 1024
        assert ctx.quantize_fp8(x)[0][0, 1].item() == 2.0 ** -6


@pytest.mark.parametrize("code", sorted(CODES))
@pytest.mark.parametrize("block", sorted(BLOCKS))
def test_blocks_of_zeros_tiny_huge_and_values_that_are_not_finite(ctx, code, block):
    import torch

    g = gen(9)
    v = torch.randn(384, 640, generator=g, device="cuda")
    v[:128, :128] = 0
    v[0, 200] = math.inf
    v[130, 128 + 7] = -math.inf
    v[140, 300] = math.nan
    v[256:, :128] *= 1e-38  # scales below the normal numbers
    v[256:, 128:256] *= 1e-43
    v[256:, 256:384] *= 1e37
    v[256:, 384:512] = 2.0 ** -149
    v[256:, 512:] *= 1e-30
    v[300, 600] = 3.4028234663852886e38
    block = BLOCKS[block]
    codes, scales = ctx.quantize_fp8(v, block, dtype=dt(CODES[code][0]))
    want, want_scales = quantized(v, block, code)
    assert same(scales, want_scales)
    assert torch.equal(codes.double(), want)
    back = ctx.dequantize_fp8(codes, scales)
    assert same(back, codes.float() * spread(scales, 384, 640, block))
    x = torch.zeros(2, 130, device="cuda")
    x[1, 129] = math.nan
    assert ctx.dequantize_fp8(*ctx.quantize_fp8(x)).isnan().sum() == 2


@pytest.mark.parametrize("code", sorted(CODES))
@pytest.mark.parametrize("block", sorted(BLOCKS))
def test_scales_that_round_to_zero(ctx, code, block):
    """blocks whose largest value is so small that no scale is left have codes 0, whatever the blocks beside them are"""
    import torch

    h, w = BLOCKS[block]
    rows, cols = 256, 512
    for e in range(-149, -125):
        top = torch.full((-(-rows // h), -(-cols // w)), 2.0 ** e, dtype=torch.float64, device="cuda").float()
        for beside in (None, 2.0 ** -120, 1.0, math.inf):
            if beside is not None:
                top.view(-1)[1::2] = beside
            v = spread(top, rows, cols, (h, w)).contiguous()
            v[1::2] *= -1
            codes, scales = ctx.quantize_fp8(v, (h, w), dtype=dt(CODES[code][0]))
            want, want_scales = quantized(v, (h, w), code)
            assert same(scales, want_scales) and torch.equal(codes.double(), want), (e, beside)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shift,pitch", [(0, 520), (1, 520), (0, 517), (3, 515), (8, 528)])
def test_strided_values_and_given_results(ctx, dtype, shift, pitch):
    """rows off their alignment, results in the middle of other memory, which is left as it was"""
    import torch

    rows, cols = 150, 501
    g = gen(shift + pitch)
    store = torch.randn(rows * pitch + 64, generator=g, device="cuda").to(dt(dtype))
    v = store[shift:shift + rows * pitch].view(rows, pitch)[:, :cols]
    for name, block in BLOCKS.items():
        for at, step in ((0, 512), (16, 528), (5, 509)):
            held = torch.full((rows * step + 64,), 0x11, dtype=torch.uint8, device="cuda")
            codes = held[at:at + rows * step].view(rows, step)[:, :cols].view(torch.float8_e4m3fn)
            shape = (rows if block[0] == 1 else 2, cols if block[1] == 1 else 4)
            room = torch.full((shape[0] + 1, shape[1] + 2), 7.0, device="cuda")
            scales = room[1:, 1:1 + shape[1]]
            got = ctx.quantize_fp8(v, block, codes=codes, scales=scales)
            assert got[0].data_ptr() == codes.data_ptr() and got[1].data_ptr() == scales.data_ptr()
            want, want_scales = quantized(v.float(), block, "e4m3")
            assert torch.equal(codes.double(), want) and torch.equal(scales, want_scales), (name, at)
            held[at:at + rows * step].view(rows, step)[:, :cols] = 0x11
            assert bool((held == 0x11).all())
            room[1:, 1:1 + shape[1]] = 7.0
            assert bool((room == 7.0).all())
        codes, scales = ctx.quantize_fp8(v, block)
        wide = torch.full((rows, cols + 3), 5.0, dtype=dt(dtype), device="cuda")
        back = ctx.dequantize_fp8(codes, scales, out=wide[:, 1:1 + cols])
        assert torch.equal(back, ctx.dequantize_fp8(codes, scales, dtype=dt(dtype)))
        assert bool((wide[:, 0] == 5).all() and (wide[:, 1 + cols:] == 5).all())


def test_matrices_past_32_bit_offsets(ctx):
    import torch

    rows, cols = 66000, 33000
    v = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    g = gen(1)
    tail = torch.randn(300, cols, generator=g, device="cuda").to(torch.bfloat16)
    v[-300:] = tail
    for block in BLOCKS.values():
        codes, scales = ctx.quantize_fp8(v, block)
        back = ctx.dequantize_fp8(codes, scales, dtype=torch.bfloat16)
        first = (rows - 300) // 128 * 128
        want, want_scales = quantized(v[first:].float(), block, "e4m3")
        assert torch.equal(codes[first:].double(), want)
        assert same(back[first:], (want.float() * spread(want_scales, rows - first, cols, block)).to(torch.bfloat16))
        assert not back[:first:999].any()
        del codes, scales, back, want


# ---- products ------------------------------------------------------------------------------------------------------------


def operand(g, rows, k, code, block, across, pitch=None, shift=0):
    """codes [rows][k], scales, and what they stand for in 64 bits; stored with k across the rows if `across`"""
    import torch

    kind, _, _, most = CODES[code]
    r, c = (k, rows) if across else (rows, k)
    pitch = pitch or max(16, -(-c // 16) * 16)
    held = torch.zeros(shift + r * pitch + 16, dtype=torch.uint8, device="cuda").fill_(0x7f)  # NaN in e4m3: what lies between the rows must not be read
    codes = held[shift:shift + r * pitch].view(r, pitch)[:, :c].view(dt(kind))
    v = (torch.randn(r, c, generator=g, device="cuda") * most / 4).clamp(-most, most).to(dt(kind))
    codes.view(torch.uint8).copy_(v.view(torch.uint8))
    b = block[::-1] if across else block
    scales = torch.rand(-(-r // 128) if b[0] == 128 else r, -(-c // 128) if b[1] == 128 else c, generator=g, device="cuda") + 0.1
    value = codes.double() * spread(scales, r, c, b).double()
    return (codes.t(), scales.t(), value.t()) if across else (codes, scales, value)


def check_product(out, a, b, k):
    import torch

    want = a @ b.t()
    size = a.abs() @ b.abs().t()
    bound = (128 + -(-k // 128) + 4) * 2.0 ** -23 * size + torch.finfo(out.dtype).eps / 2 * 1.001 * want.abs() + 1e-30
    if out.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step below its normal numbers
    off = (out.double() - want).abs() - bound
    assert not out.isnan().any() and off.max().item() <= 0, (off.max().item(), size.max().item())


FORMS = {"forward": ((1, 128), (128, 128), False, False), "input": ((1, 128), (128, 128), False, True), "weight": ((1, 128), (1, 128), True, True),
         "factors": ((1, 128), (1, 128), False, False), "turned": ((128, 128), (1, 128), True, False), "squares": ((128, 128), (128, 128), False, False)}
PRODUCTS = [(1, 64, 64), (1, 1, 1), (7, 33, 129), (32, 200, 1000), (33, 65, 31), (64, 64, 128), (100, 300, 200), (128, 128, 128), (129, 257, 385), (333, 1111, 511),
            (200, 640, 2048), (1000, 1500, 640), (2, 4096, 300), (700, 3, 260), (1100, 5003, 390), (3001, 1300, 130)]


@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products(ctx, form, m, n, k):
    import torch

    block_a, block_b, across_a, across_b = FORMS[form]
    for i, (dtype, ca, cb) in enumerate((("bfloat16", "e4m3", "e4m3"), ("float32", "e5m2", "e4m3"), ("float16", "e4m3", "e5m2"))):
        g = gen(m * n + k + i)
        a, sa, va = operand(g, m, k, ca, block_a, across_a)
        b, sb, vb = operand(g, n, k, cb, block_b, across_b)
        sa, va, sb, vb = (t * (1.0 / CODES[c][3]) for t, c in ((sa, ca), (va, ca), (sb, cb), (vb, cb)))
        va, vb = a.double() * spread(sa, m, k, block_a).double(), b.double() * spread(sb, n, k, block_b).double()
        out = ctx.fp8_matmul(a, sa, b, sb, dtype=dt(dtype))
        check_product(out, va, vb, k)


@pytest.mark.parametrize("form", ["forward", "input", "weight"])
@pytest.mark.parametrize("m,n,k", [(20, 333, 500), (150, 333, 500)])
def test_products_of_operands_off_their_alignment(ctx, form, m, n, k):
    """codes that start on any byte, results in rows that end anywhere: nothing behind a row's end is read or written"""
    import torch

    block_a, block_b, across_a, across_b = FORMS[form]
    for shift, more in ((1, 0), (0, 3), (15, 17), (8, 8)):
        g = gen(shift)
        a, sa, va = operand(g, m, k, "e4m3", block_a, across_a, pitch=(m if across_a else k) + more, shift=shift)
        b, sb, vb = operand(g, n, k, "e4m3", block_b, across_b, pitch=(n if across_b else k) + more, shift=shift)
        for dtype in ("float32", "bfloat16"):
            for at, step in ((0, n), (1, n + 1), (4, n + 11)):
                held = torch.full((at + m * step + 8,), 3.0, dtype=dt(dtype), device="cuda")
                out = held[at:at + m * step].view(m, step)[:, :n]
                ctx.fp8_matmul(a, sa, b, sb, out=out)
                check_product(out, va, vb, k)
                out.fill_(3.0)
                assert bool((held == 3.0).all())


# Exponents of the scales of a and b, the largest code (of 8 bits), and how many scales are of ordinary size: the product of two scales, and that of a block's sum and
# a's scale, are up to the ends of the normal numbers; the block's sum times b's scale need not be in range
APART = [(-62, -62, 127, 0.3), (64, 63, 1, 0.3), (-20, 110, 127, 0.0), (-100, 126, 127, 0.0), (-140, 20, 127, 0.0), (-70, 70, 127, 0.3), (70, -70, 1, 0.3),
         (110, -20, 1, 0.3)]


@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("m,n,k", [(3, 200, 300), (200, 3, 300), (40, 200, 300), (129, 65, 2100), (1300, 2500, 400), (1301, 2501, 400)])
def test_scales_far_apart(ctx, form, m, n, k):
    """Scales of ordinary size beside others in the same tile.  The bound is that of check_product; a term may lose half a step of the subnormal numbers
    twice beside it, once before it is multiplied by b's scale"""
    import torch

    block_a, block_b, across_a, across_b = FORMS[form]
    for i, (ea, eb, top, ordinary) in enumerate(APART):
        g = gen(m + n + i)
        a, sa, _ = operand(g, m, k, "e4m3", block_a, across_a)
        b, sb, _ = operand(g, n, k, "e4m3", block_b, across_b)
        if top == 1:  # zeros and 2^-9
            for t in (a, b):
                t.view(torch.uint8).copy_(torch.randint(0, 2, t.shape, generator=g, device="cuda"))
            a.view(torch.uint8)[::5] = 0
            b.view(torch.uint8)[1::3] = 0
        for s, e in ((sa, ea), (sb, eb)):
            s.clamp_(0.5, 1.0).mul_(torch.where(torch.rand(s.shape, generator=g, device="cuda") < ordinary, 1.0, 2.0 ** (e // 2)))
            s.mul_(torch.where(s > 1.5, 2.0 ** (e - e // 2), 1.0) if e > 0 else torch.where(s < 0.4, 2.0 ** (e - e // 2), 1.0))
        va, vb = a.double() * spread(sa, m, k, block_a).double(), b.double() * spread(sb, n, k, block_b).double()
        out = ctx.fp8_matmul(a, sa, b, sb, dtype=torch.float32)
        want, size = va @ vb.t(), va.abs() @ vb.abs().t()
        blocks = -(-k // 128)
        bound = (128 + blocks + 4) * 2.0 ** -23 * size + 2.0 ** -24 * want.abs() + blocks * 2.0 ** -149 * (1 + sb.max().item())
        off = (out.double() - want).abs() - bound
        assert not out.isnan().any() and off.max().item() <= 0, (ea, eb, off.max().item())


def test_scales_that_are_not_finite_or_zero_in_products(ctx):
    import torch

    g = gen(2)
    m, n, k = 140, 300, 400
    a, sa, va = operand(g, m, k, "e4m3", (1, 128), False)
    b, sb, vb = operand(g, n, k, "e4m3", (128, 128), False)
    sa[3, 1], sb[2, 3] = math.nan, math.inf
    sa[5] = 0
    a.view(torch.uint8)[3, 128:256] = 0
    out = ctx.fp8_matmul(a, sa, b, sb, dtype=torch.float32)
    assert bool(out[3].isnan().all()) and not bool(out[:, 256:].isfinite().any())
    assert bool((out[5, :256] == 0).all())
    keep = [i for i in range(m) if i != 3]
    va = a.double() * spread(sa, m, k, (1, 128)).double()
    check_product(out[keep][:, :256], va[keep], vb[:256], k)
    # codes that are not finite
    c = torch.zeros(4, 64, dtype=torch.float8_e5m2, device="cuda")
    c.view(torch.uint8)[1, 5], c.view(torch.uint8)[2, 6] = 0x7c, 0x7f
    ones = torch.ones(40, 64, device="cuda").to(torch.float8_e5m2)
    out = ctx.fp8_matmul(c, torch.ones(4, 1, device="cuda"), ones, torch.ones(40, 1, device="cuda"), dtype=torch.float32)
    assert bool((out[1] == math.inf).all()) and bool(out[2].isnan().all()) and not out[0].any() and not out[3].any()


@pytest.mark.parametrize("form", ["forward", "weight", "squares"])
@pytest.mark.parametrize("m,n,k", [(300, 1100, 1300), (2500, 2300, 2100), (129, 65, 4000)])
def test_products_among_others_are_the_same_every_time(ctx, form, m, n, k):
    """two streams at once, so that the warps that take sums out wait in ever other turns; whole tiles, and rows that end within one"""
    import torch

    g = gen(m)
    block_a, block_b, across_a, across_b = FORMS[form]
    a, sa, va = operand(g, m, k, "e4m3", block_a, across_a)
    b, sb, vb = operand(g, n, k, "e4m3", block_b, across_b)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ctx.fp8_matmul(a, sa, b, sb, dtype=torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs)
    check_product(outs[0], va, vb, k)
    ctx.check_status()


def test_empty_products_and_scales_of_any_stride(ctx):
    import torch

    e = lambda *s: torch.empty(*s, dtype=torch.float8_e4m3fn, device="cuda")  # noqa: E731
    f = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
    out = torch.full((5, 9), 7.0, device="cuda")
    ctx.fp8_matmul(e(5, 0), f(5, 0), e(9, 0), f(1, 0), out=out[:, :9])
    assert not out.any()
    assert ctx.fp8_matmul(e(0, 7), f(0, 1), e(9, 7), f(9, 1)).shape == (0, 9)
    assert ctx.fp8_matmul(e(3, 7), f(3, 1), e(0, 7), f(0, 1)).shape == (3, 0)
    assert ctx.quantize_fp8(f(0, 5))[0].shape == (0, 5) and ctx.quantize_fp8(f(5, 0))[1].shape == (5, 0)
    g = gen(8)
    a, sa, va = operand(g, 70, 300, "e4m3", (1, 128), False)
    b, sb, vb = operand(g, 90, 300, "e4m3", (1, 128), False)
    one = torch.full((1, 1), 0.5, device="cuda").expand(70, 3)  # one scale for all
    wide = torch.zeros(90, 9, device="cuda")
    wide[:, ::3] = sb
    out = ctx.fp8_matmul(a, one, b, wide[:, ::3], dtype=torch.float32)
    check_product(out, a.double() * 0.5, vb, 300)


def test_two_streams_and_a_captured_graph(ctx):
    """products that need a workspace, on two streams at once and replayed with other inputs"""
    import torch

    g = gen(11)
    pairs = []
    for shift in (1, 3):
        a, sa, va = operand(g, 300, 700, "e4m3", (1, 128), False, pitch=701, shift=shift)
        b, sb, vb = operand(g, 500, 700, "e4m3", (128, 128), True, pitch=507, shift=shift)
        pairs.append((a, sa, b, sb, va, vb))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pairs]
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ctx.fp8_matmul(*pairs[i][:4], dtype=torch.float32))
    torch.cuda.synchronize()
    for i in range(2):
        check_product(outs[i][0], *pairs[i][4:], 700)
        assert all(torch.equal(outs[i][0], o) for o in outs[i])
    x = torch.randn(130, 260, generator=g, device="cuda")
    w = torch.randn(150, 260, generator=g, device="cuda")

    def chain():
        x8, xs, xd, xds = ctx.quantize_fp8_both(x)
        w8, ws = ctx.quantize_fp8(w, (128, 128))
        return ctx.fp8_matmul(x8, xs, w8, ws, dtype=torch.float32), ctx.fp8_matmul(xd.t(), xds.t(), xd.t(), xds.t(), dtype=torch.float32), ctx.clip_updates([[x, w]], 3.0)

    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for seed in (1, 2):
        x.copy_(torch.randn(130, 260, generator=gen(seed), device="cuda"))
        w.copy_(torch.randn(150, 260, generator=gen(seed + 5), device="cuda"))
        kept = x.clone(), w.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got] + [x.clone(), w.clone()]
        x.copy_(kept[0])
        w.copy_(kept[1])
        for p, q in zip(replayed, list(chain()) + [x, w]):
            assert torch.equal(p, q)
    ctx.check_status()


# ---- a training step ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape,n,grad", [((50, 784), 200, "e4m3"), ((3, 7, 130), 65, "e5m2"), ((260,), 33, "e4m3"), ((1, 1), 1, "e4m3")])
def test_a_layers_step(ctx, dtype, shape, n, grad):
    import torch

    from lancelot_b200 import updates

    g = gen(n)
    x = torch.randn(*shape, generator=g, device="cuda").to(dt(dtype)).requires_grad_()
    w = (torch.randn(n, shape[-1], generator=g, device="cuda") * 0.1).to(dt(dtype)).requires_grad_()
    y = updates.fp8_linear(ctx, x, w, grad_dtype=dt(CODES[grad][0]))
    assert y.shape == (*shape[:-1], n) and y.dtype == x.dtype
    dy = torch.randn(y.shape, generator=g, device="cuda").to(y.dtype)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dx.shape == x.shape and dx.dtype == x.dtype and dw.shape == w.shape and dw.dtype == w.dtype
    flat, d = x.detach().reshape(-1, shape[-1]), dy.reshape(-1, n)
    m, k = flat.shape

    def held(t, block, code):
        codes, scales = quantized(t.detach().float(), block, code)
        return codes * spread(scales, *t.shape, block).double()

    w8 = held(w, (128, 128), "e4m3")
    check_product(y.detach().reshape(m, n), held(flat, (1, 128), "e4m3"), w8, k)
    check_product(dx.reshape(m, k), held(d, (1, 128), grad), w8.t(), n)
    check_product(dw, held(d, (128, 1), grad).t(), held(flat, (128, 1), "e4m3").t(), m)
    # only one of the two gradients, and a gradient that is one value for all
    y = updates.fp8_linear(ctx, x.detach(), w)
    y.float().sum().backward()
    ones = torch.ones(m, n, device="cuda")
    check_product(w.grad, held(ones, (128, 1), "e4m3").t(), held(flat, (128, 1), "e4m3").t(), m)
    y = updates.fp8_linear(ctx, x, w.detach())
    y.float().sum().backward()
    check_product(x.grad.reshape(m, k), held(ones, (1, 128), "e4m3"), w8.t(), n)


def test_a_layers_step_on_an_empty_batch_and_on_transposed_operands(ctx):
    import torch

    from lancelot_b200 import updates

    g = gen(12)
    w = torch.randn(200, 64, generator=g, device="cuda").t().requires_grad_()  # [64][200], its rows not dense
    x = torch.zeros(0, 200, device="cuda", requires_grad=True)
    y = updates.fp8_linear(ctx, x, w)
    assert y.shape == (0, 64)
    dx, dw = torch.autograd.grad(y, (x, w), y.detach())
    assert dx.shape == (0, 200) and dw.shape == (64, 200) and not dw.any()
    x = torch.randn(200, 30, generator=g, device="cuda").t()
    assert torch.equal(updates.fp8_linear(ctx, x, w), updates.fp8_linear(ctx, x.contiguous(), w.detach().contiguous()))
    one = torch.randn(200, generator=g, device="cuda")
    # one value for several rows; the sums of 12 rows and those of one are formed in other orders, so both are held to the formula
    codes, scales = quantized(one[None], (1, 128), "e4m3")
    x8 = codes * spread(scales, 1, 200, (1, 128)).double()
    codes, scales = quantized(w.detach().contiguous(), (128, 128), "e4m3")
    w8 = codes * spread(scales, 64, 200, (128, 128)).double()
    check_product(updates.fp8_linear(ctx, one.expand(4, 3, 200), w).detach().reshape(12, 64), x8.expand(12, 200), w8, 200)
    check_product(updates.fp8_linear(ctx, one, w).detach()[None], x8, w8, 200)
    # what is kept for the backward pass are codes: the layer's operands may change in between
    x = torch.randn(20, 200, generator=g, device="cuda").requires_grad_()
    y = updates.fp8_linear(ctx, x, w)
    want = torch.autograd.grad(y, (x, w), torch.ones_like(y), retain_graph=True)
    with torch.no_grad():
        w.zero_()
        x.zero_()
    for p, q in zip(torch.autograd.grad(y, (x, w), torch.ones_like(y)), want):
        assert torch.equal(p, q)


def test_gradients_of_gradients_and_a_context_closed_in_between():
    import torch

    from lancelot_b200 import cabi, updates

    c = cabi.Context(12, cabi.coeff_modulus_create(1 << 12, [40, 40]), 1)
    g = gen(14)
    x = torch.randn(20, 150, generator=g, device="cuda").requires_grad_()
    w = torch.randn(30, 150, generator=g, device="cuda").requires_grad_()
    dx, dw = torch.autograd.grad(updates.fp8_linear(c, x, w).square().sum(), (x, w), create_graph=True)
    want = torch.autograd.grad(updates.fp8_linear(c, x, w).square().sum(), (x, w))
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    with pytest.raises(RuntimeError, match="not differentiable"):
        (dx.sum() + dw.sum()).backward()
    y = updates.fp8_linear(c, x, w)
    with torch.no_grad():
        assert not updates.fp8_linear(c, x, w).requires_grad
    c.close()
    with pytest.raises(ValueError):
        y.sum().backward()
    with pytest.raises(ValueError):
        updates.fp8_linear(c, x, w)


def test_a_backward_pass_on_another_stream(ctx):
    import torch

    from lancelot_b200 import updates

    g = gen(15)
    x = torch.randn(200, 300, generator=g, device="cuda").requires_grad_()
    w = torch.randn(100, 300, generator=g, device="cuda").requires_grad_()
    dy = torch.randn(200, 100, generator=g, device="cuda")
    want = torch.autograd.grad(updates.fp8_linear(ctx, x, w), (x, w), dy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(side):
            y = updates.fp8_linear(ctx, x, w)
            got = torch.autograd.grad(y, (x, w), dy)
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_a_captured_step(ctx):
    """forward and gradients replayed with other inputs, in two graphs at once that share the operands"""
    import torch

    from lancelot_b200 import updates

    g = gen(13)
    x = torch.randn(70, 200, generator=g, device="cuda").requires_grad_()
    w = torch.randn(90, 200, generator=g, device="cuda").requires_grad_()
    dy = torch.randn(70, 90, generator=g, device="cuda")

    def step():
        y = updates.fp8_linear(ctx, x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    got = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            got.append(step())
    with torch.no_grad():
        x.normal_(generator=g)
        w.normal_(generator=g)
        dy.normal_(generator=g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for want, *replayed in zip(step(), *got):
        for r in replayed:
            assert torch.equal(r, want)
    ctx.check_status()


def test_gradients_against_differences(ctx):
    """Values that 8 bits hold exactly: multiples of 1/4 up to 1.25 and, in every block, 1.75, whose scale is 2^-8.  All sums are then exact in 32 bits
    (multiples of 2^-4, below 2^20), and the change of the loss along a direction is what the gradient says, without a tolerance"""
    import torch

    from lancelot_b200 import updates

    g = gen(4)
    m, n, k = 150, 70, 200

    def quarters(rows, cols, most):  # multiples of most / 4
        v = torch.randint(-4, 5, (rows, cols), generator=g, device="cuda") * (most / 4)
        return v

    def marks(rows, cols):
        return (torch.arange(rows, device="cuda")[:, None] + torch.arange(cols, device="cuda")) % 8 == 0

    x, w, c = (torch.where(marks(r, q), torch.full((), 1.75, device="cuda"), quarters(r, q, 1.0)) for r, q in ((m, k), (n, k), (m, n)))
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(updates.fp8_linear(ctx, x, w), (x, w), c)
    with torch.no_grad():
        for t, grad, y in ((x, dx, lambda t: updates.fp8_linear(ctx, t, w)), (w, dw, lambda t: updates.fp8_linear(ctx, x, t))):
            d = torch.where(marks(*t.shape), torch.zeros((), device="cuda"), torch.randint(-1, 2, t.shape, generator=g, device="cuda") * 0.25)
            found = ((y(t + d).double() - y(t - d).double()) * c).sum() / 2
            said = (grad.double() * d).sum()
            assert said != 0 and found == said


def test_what_is_written_counts_as_changed(ctx):
    """autograd notices that a tensor which it saved was overwritten; a call that is refused changes nothing"""
    import torch

    from lancelot_b200 import updates
    from lancelot_b200._lib import InvalidArgument

    g = gen(16)
    x = torch.randn(64, 256, generator=g, device="cuda")
    x8, xs, xd, xds = ctx.quantize_fp8_both(x)
    y = torch.zeros(64, 64, device="cuda")
    wide, rows = torch.zeros(64, 256, device="cuda"), torch.zeros(2, 256, device="cuda")
    i8, i8s = torch.zeros(64, 256, dtype=torch.int8, device="cuda"), torch.zeros(64, 1, device="cuda")
    res = torch.zeros(64, 256, device="cuda")
    a, b = torch.ones(256, device="cuda"), torch.ones(256, device="cuda")
    for call, written in ((lambda: ctx.quantize_fp8(x, codes=x8, scales=xs), (x8, xs)),
                          (lambda: ctx.quantize_fp8(x, (128, 1), codes=xd, scales=xds), (xd, xds)),
                          (lambda: ctx.dequantize_fp8(x8, xs, out=wide), (wide,)),
                          (lambda: ctx.fp8_matmul(x8, xs, x8, xs, out=y), (y,)),
                          (lambda: ctx.clip_updates([[a], [b]], 1.0, out=rows), (rows,)),
                          (lambda: ctx.clip_updates([[a], [b]], 1.0), (a, b)),
                          (lambda: ctx.clip_updates(rows, 1.0), (rows,)),
                          (lambda: ctx.quantize_rows(x, i8, i8s, residual=res, residual_out=res), (i8, i8s, res)),
                          (lambda: ctx.dequantize_rows(i8, i8s, 256, out=wide), (wide,)),
                          (lambda: ctx.int8_matmul(i8, i8, i8s.view(-1), i8s.view(-1), out=y), (y,))):
        before = [t._version for t in written]
        others = [(t, t._version) for t in (x, x8, xs, xd, xds, y, wide, rows, i8, i8s, res, a, b) if not any(t is u for u in written)]
        call()
        assert all(t._version > v for t, v in zip(written, before))
        assert all(t._version == v for t, v in others)
    for call, kept in ((lambda: ctx.clip_updates([[a], [a]], 1.0), a), (lambda: ctx.clip_updates([[a, b[:3]], [b]], 1.0), a),
                       (lambda: ctx.clip_updates([[rows[0]], [a]], 1.0, out=rows.view(2, 256).flip(0)[:, :255]), rows)):
        before = kept._version
        with pytest.raises(InvalidArgument):
            call()
        assert kept._version == before
    # nothing is read for the norms alone, and a saved result that a later call overwrites is found out
    before = a._version
    ctx.clip_updates([[a], [b]])
    assert a._version == before
    p = torch.ones(64, 64, device="cuda", requires_grad=True)
    z = (p * y).sum()
    ctx.fp8_matmul(x8, xs, x8, xs, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.inference_mode():
        t = torch.zeros(64, 64, device="cuda")
        ctx.fp8_matmul(x8, xs, x8, xs, out=t)
        ctx.clip_updates([[t]], 1.0)


def test_updates_of_low_rank_from_8_bit_floats(ctx):
    import torch

    from lancelot_b200 import updates

    g = gen(6)
    factors, want, ints = [], [], []
    for rows, cols, rank in ((100, 64, 16), (33, 257, 5), (8, 8, 1)):
        b, a = torch.randn(rows, rank, generator=g, device="cuda"), torch.randn(cols, rank, generator=g, device="cuda")
        factors.append((*ctx.quantize_fp8(b), *ctx.quantize_fp8(a)))
        ints.append((*updates.quantize_matrix(ctx, b), *updates.quantize_matrix(ctx, a)))
        want.append((ctx.dequantize_fp8(*factors[-1][:2]).double(), ctx.dequantize_fp8(*factors[-1][2:]).double(), rank))
    flat = updates.low_rank_update(ctx, factors)
    at = 0
    for b, a, rank in want:
        size = b.shape[0] * a.shape[0]
        check_product(flat[at:at + size].view(b.shape[0], a.shape[0]), b, a, rank)
        at += size
    assert at == flat.numel()
    mixed = updates.low_rank_update(ctx, [factors[0], ints[1], factors[2]])
    assert torch.equal(mixed[: 6400], flat[: 6400]) and torch.equal(mixed[6400 + 33 * 257:], flat[6400 + 33 * 257:])
    assert torch.equal(mixed[6400: 6400 + 33 * 257], updates.low_rank_update(ctx, ints)[6400: 6400 + 33 * 257])


def test_what_the_calls_refuse(ctx):
    import torch

    from lancelot_b200 import updates
    from lancelot_b200._lib import InvalidArgument

    x = torch.randn(64, 256, device="cuda")
    codes, scales = ctx.quantize_fp8(x)
    wide = torch.empty(64, 512, device="cuda")
    for call in (lambda: ctx.quantize_fp8(x.double()),
                 lambda: ctx.quantize_fp8(x.cpu()),
                 lambda: ctx.quantize_fp8(x[0]),
                 lambda: ctx.quantize_fp8(x.t()),
                 lambda: ctx.quantize_fp8(x, (64, 128)),
                 lambda: ctx.quantize_fp8(x, 128),
                 lambda: ctx.quantize_fp8(x, dtype=torch.int8),
                 lambda: ctx.quantize_fp8(x[:1].expand(64, 256)),
                 lambda: ctx.quantize_fp8(x, codes=codes[:, :128]),
                 lambda: ctx.quantize_fp8(x, codes=codes.view(torch.uint8)),
                 lambda: ctx.quantize_fp8(x, scales=scales[:, :1]),
                 lambda: ctx.quantize_fp8_both(x, dtype=torch.float16),
                 lambda: ctx.dequantize_fp8(codes, scales[:, :1]),
                 lambda: ctx.dequantize_fp8(codes.view(torch.uint8), scales),
                 lambda: ctx.dequantize_fp8(codes, scales, dtype=torch.float64),
                 lambda: ctx.dequantize_fp8(codes, scales, out=wide),
                 lambda: ctx.fp8_matmul(codes, scales, codes[:, :128], scales[:, :1]),
                 lambda: ctx.fp8_matmul(codes, scales[:, :1], codes, scales),
                 lambda: ctx.fp8_matmul(codes, scales[:3], codes, scales),
                 lambda: ctx.fp8_matmul(codes[:, ::2], scales[:, :1], codes[:, :128], scales[:, :1]),
                 lambda: ctx.fp8_matmul(codes, scales.double(), codes, scales),
                 lambda: ctx.fp8_matmul(codes.view(torch.int8), scales, codes, scales),
                 lambda: ctx.fp8_matmul(codes, scales, codes, scales, dtype=torch.float64),
                 lambda: ctx.fp8_matmul(codes, scales, codes, scales, out=wide),
                 lambda: ctx.fp8_matmul(codes[:1].expand(64, 256), scales, codes, scales),
                 lambda: ctx.fp8_matmul(codes.cpu(), scales, codes, scales)):
        with pytest.raises(InvalidArgument):
            call()
    for call in (lambda: updates.fp8_linear(ctx, x, x[:, :128]), lambda: updates.fp8_linear(ctx, x, x[0]),
                 lambda: updates.fp8_linear(ctx, x, x, grad_dtype=torch.float16)):
        with pytest.raises(ValueError):
            call()
    ctx.check_status()


def test_a_closed_context_is_refused():
    import torch

    from lancelot_b200 import cabi
    from lancelot_b200._lib import InvalidArgument

    c = cabi.Context(12, cabi.coeff_modulus_create(1 << 12, [40, 40]), 1)
    x = torch.randn(64, 256, device="cuda")
    codes, scales = c.quantize_fp8(x)
    c.close()
    for call in (lambda: c.quantize_fp8(x), lambda: c.dequantize_fp8(codes, scales), lambda: c.fp8_matmul(codes, scales, codes, scales),
                 lambda: c.clip_updates([[x]], 1.0)):
        with pytest.raises(InvalidArgument):
            call()
