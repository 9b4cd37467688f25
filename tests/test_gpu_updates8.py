"""8-bit updates on the GPU against plain 64-bit formulas: cache rows written and read back, the 8-bit matrix product, pair distances.

Codes, scales and residuals are compared for equality (the definition leaves no choice); a product may be off by the roundings it
makes: the integer sum to 32 bits, two products by a scale, the result's type.  Distances are sums of 64-bit floats."""
import math

import pytest

pytestmark = pytest.mark.gpu

F32, F64 = 2.0 ** -24, 2.0 ** -53  # half a step, relative


@pytest.fixture(scope="module")
def ctx():
    from lancelot_b200 import cabi

    return cabi.Context(12, cabi.coeff_modulus_create(1 << 12, [40, 40]), 1)


def gen(seed):
    import torch

    return torch.Generator("cuda").manual_seed(seed)


def quantized(t, page, group):
    """t [rows][cols] float32 -> codes [rows * pages][page], scales, lost [rows][cols], from the definition with 64-bit quotients"""
    import torch

    rows, cols = t.shape
    pages = -(-cols // page)
    size = group if 0 < group < page else page
    groups = -(-page // size)
    x = torch.zeros(rows, pages * page, device=t.device)
    x[:, :cols] = t
    x = x.view(rows * pages, page)
    x = torch.nn.functional.pad(x, (0, groups * size - page)).view(rows * pages, groups, size)
    most = x.abs().amax(2)
    scale = torch.where(most.isfinite(), most / torch.full_like(most, 127), torch.full_like(most, math.nan))
    s = scale.double()[:, :, None]
    code = (x.double() / s).round().clamp(-127, 127)
    code = torch.where(s > 0, code, torch.zeros_like(code))
    lost = torch.where(s.isnan(), torch.zeros_like(s), x.double() - code * s.nan_to_num())
    assert torch.equal(lost, lost.float().double())  # what is lost fits 32 bits
    codes = code.view(rows * pages, -1)[:, :page].to(torch.int8)
    lost = lost.float().view(rows * pages, -1)[:, :page].reshape(rows, -1)[:, :cols]
    return codes, scale, lost


def same(x, y):
    import torch

    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num()) if x.is_floating_point() else torch.equal(x, y)


def expanded(codes, scales, group):
    page = codes.shape[1]
    return codes.float() * scales.repeat_interleave(group if 0 < group < page else page, 1)[:, :page]


GROUPS = [0, 32, 64, 128, 256, 512, 1024, 4096, 65536]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols,page", [(1, 1, 16), (3, 33, 48), (5, 1000, 1008), (2, 5000, 2048), (3, 70001, 32768), (2, 100000, 98304), (3, 140003, 65536),
                                            (2, 3001, 4096), (2, 20005, 16384)])
def test_rows_written_and_read_back(ctx, dtype, rows, cols, page):
    import torch

    dt = getattr(torch, dtype)
    for group in GROUPS:
        g = gen(rows * cols + group)
        v = (torch.randn(rows, cols, generator=g, device="cuda") * torch.rand(rows, 1, generator=g, device="cuda")).to(dt)
        v[:, ::7] = 0
        pages, groups = -(-cols // page), -(-page // group) if 0 < group < page else 1
        codes = torch.full((rows * pages, page), 99, dtype=torch.int8, device="cuda")
        scales = torch.full((rows * pages, groups), 99.0, device="cuda")
        lost = torch.empty(rows, cols, device="cuda")
        ctx.quantize_rows(v, codes, scales, group=group, residual_out=lost)
        want_codes, want_scales, want_lost = quantized(v.float(), page, group)
        assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales) and torch.equal(lost, want_lost), group
        back = ctx.dequantize_rows(codes, scales, cols, group=group, dtype=dt)
        want = expanded(codes, scales, group).view(rows, pages * page)[:, :cols].to(dt)
        assert torch.equal(back, want), group


def test_borders_between_codes_are_decided_exactly(ctx):
    """values on and next to the half steps of the scale, where a 32-bit quotient rounds to the wrong side"""
    import torch

    g = gen(5)
    rows, cols = 64, 4096
    most = torch.rand(rows, 1, generator=g, device="cuda") * 10 + 0.1
    s = most / torch.full_like(most, 127)
    half = (torch.randint(-126, 126, (rows, cols), generator=g, device="cuda") + 0.5).double() * s.double()
    v = half.float()
    step = torch.randint(-1, 2, (rows, cols), generator=g, device="cuda", dtype=torch.int32)
    v = (v.view(torch.int32) + step).view(torch.float32)
    v[:, :1] = most
    codes = torch.empty(rows, cols, dtype=torch.int8, device="cuda")
    scales = torch.empty(rows, 1, device="cuda")
    lost = torch.empty(rows, cols, device="cuda")
    ctx.quantize_rows(v, codes, scales, residual_out=lost)
    want = quantized(v, cols, 0)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1]) and torch.equal(lost, want[2])
    # exact ties go to the even code: a scale of 2^-5 and odd multiples of 2^-6
    v = (torch.arange(-253, 254, device="cuda") / 64.0).view(1, -1)
    v[0, 0] = 127 / 32
    codes, scales = torch.empty(1, 512, dtype=torch.int8, device="cuda"), torch.empty(1, 1, device="cuda")
    ctx.quantize_rows(v, codes, scales)
    assert float(scales) == 1 / 32 and torch.equal(codes[0, 1:507].float(), (v[0, 1:] * 32).round())


@pytest.mark.parametrize("group", [0, 64, 1024])
def test_infinities_nan_and_tiny_values(ctx, group):
    import torch

    v = torch.randn(9, 4096, generator=gen(1), device="cuda")
    v[0, 5] = math.inf
    v[1, 4095] = -math.inf
    v[2, 1024] = math.nan
    v[3] *= 2.0 ** -130  # the scales of these rows are below the normal range
    v[4] *= 2.0 ** -148
    v[5] = 0
    v[6] = -0.0
    v[7] *= 1e38
    v[8] = torch.finfo(torch.float32).max
    n = 4096 // group if group else 1
    codes, scales, lost = torch.empty(9, 4096, dtype=torch.int8, device="cuda"), torch.empty(9, n, device="cuda"), torch.empty(9, 4096, device="cuda")
    v.clamp_(-torch.finfo(torch.float32).max, torch.finfo(torch.float32).max)[0, 5] = math.inf
    v[1, 4095] = -math.inf
    ctx.quantize_rows(v, codes, scales, group=group, residual_out=lost)
    want = quantized(v, 4096, group)
    assert torch.equal(codes, want[0]) and same(scales, want[1]) and torch.equal(lost, want[2])
    back = ctx.dequantize_rows(codes, scales, 4096, group=group)
    assert same(back, expanded(codes, scales, group))
    assert back[0].isnan().any() and back[2].isnan().any() and not back[3:].isnan().any()


@pytest.mark.parametrize("group", [0, 128])
def test_lengths_slots_residual_and_strides(ctx, group):
    """ragged rows (empty ones among them), slots in any order with some outside the cache, strided rows off their alignment, the residual in
    place; what a call does not own stays as it was"""
    import torch

    g = gen(3)
    rows, cols, page = 7, 1003, 512
    pages, groups = 2, page // group if group else 1
    wide = torch.randn(rows, 1100, generator=g, device="cuda")
    v = wide[:, 13:13 + cols]
    res_wide = torch.randn(rows, 1050, generator=g, device="cuda") * 0.01
    res = res_wide[:, 5:5 + cols]
    lengths = torch.tensor([0, 1, 512, 513, 1003, 5000, -4], dtype=torch.int32, device="cuda")
    slots = torch.randperm(20, generator=g, device="cuda")[: rows * pages].to(torch.int32).view(rows, pages)
    slots[2, 1], slots[4, 0] = -1, 20
    codes = torch.full((20, page + 16), 77, dtype=torch.int8, device="cuda")[:, :page]
    scales = torch.full((20, groups), 77.0, device="cuda")
    before, res_before = res_wide.clone(), res.clone()
    ctx.quantize_rows(v, codes, scales, group=group, slots=slots, lengths=lengths, residual=res, residual_out=res)
    inside = torch.arange(cols, device="cuda") < lengths[:, None]
    t = torch.where(inside, v + res_before, torch.zeros(()).cuda())
    want_codes, want_scales, want_lost = quantized(t, page, group)
    written = torch.zeros(20, dtype=torch.bool, device="cuda")
    for i in range(rows):
        for p in range(pages):
            s, lo, hi = int(slots[i, p]), p * page, min((p + 1) * page, cols)
            if 0 <= s < 20:
                written[s] = True
                assert torch.equal(codes[s], want_codes[i * pages + p]) and torch.equal(scales[s], want_scales[i * pages + p])
                want = torch.where(inside[i, lo:hi], want_lost[i, lo:hi], res_before[i, lo:hi])
                assert torch.equal(res[i, lo:hi], want)
            else:
                assert torch.equal(res[i, lo:hi], res_before[i, lo:hi])
    assert bool((codes[~written] == 77).all()) and bool((scales[~written] == 77).all())
    res_wide[:, 5:5 + cols] = 0
    before[:, 5:5 + cols] = 0
    assert torch.equal(res_wide, before)
    out = torch.full((rows, 1111), 5.0, device="cuda")
    back = ctx.dequantize_rows(codes, scales, cols, group=group, slots=slots, out=out[:, 3:3 + cols])
    full = torch.zeros(rows, pages, page, device="cuda")
    for i in range(rows):
        for p in range(pages):
            s = int(slots[i, p])
            if 0 <= s < 20:
                full[i, p] = expanded(codes[s:s + 1], scales[s:s + 1], group)[0]
    assert torch.equal(back, full.view(rows, -1)[:, :cols])
    assert bool((out[:, :3] == 5).all()) and bool((out[:, 3 + cols:] == 5).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("cols", [509, 510, 511, 512, 513, 1021, 1022, 1023])
def test_rows_that_end_next_to_a_run_of_512_columns(ctx, dtype, cols):
    """at every offset from an aligned piece, written and read back, with nothing touched beside the rows"""
    import torch

    dt = getattr(torch, dtype)
    for group in (0, 32, 256):
        for shift in range(4):
            g = gen(cols * 4 + shift)
            wide = torch.randn(3, cols + 1 + shift, generator=g, device="cuda").to(dt)
            base = torch.full((3, cols + 5), 7.0, device="cuda")
            v, lost = wide[:, shift:shift + cols], base[:, shift:shift + cols]
            codes = torch.empty(6, 1008, dtype=torch.int8, device="cuda")[: 3 * -(-cols // 1008)]
            scales = torch.empty(codes.shape[0], -(-1008 // group) if group else 1, device="cuda")
            ctx.quantize_rows(v, codes, scales, group=group, residual_out=lost)
            want_codes, want_scales, want_lost = quantized(v.float(), 1008, group)
            assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales) and torch.equal(lost, want_lost), (group, shift)
            out = torch.full((3, cols + 5), 7.0, dtype=dt, device="cuda")
            ctx.dequantize_rows(codes, scales, cols, group=group, out=out[:, shift:shift + cols])
            want = torch.full_like(out, 7.0)
            want[:, shift:shift + cols] = expanded(codes, scales, group).view(3, -1)[:, :cols].to(dt)
            assert torch.equal(out, want), (group, shift)
            assert (base[:, :shift] == 7).all() and (base[:, shift + cols:] == 7).all()


def test_error_feedback_over_rounds_loses_nothing(ctx):
    """sum of what was sent plus the residual left = sum of the updates (to the roundings of the 32-bit sums t)"""
    import torch

    g = gen(8)
    res = torch.zeros(2, 3000, device="cuda")
    sent, total, slack = torch.zeros(2, 3000, dtype=torch.float64, device="cuda"), torch.zeros(2, 3000, dtype=torch.float64, device="cuda"), 0.0
    codes, scales = torch.empty(2, 3008, dtype=torch.int8, device="cuda"), torch.empty(2, 47, device="cuda")
    for _ in range(5):
        v = torch.randn(2, 3000, generator=g, device="cuda")
        slack += F32 * float((v + res).abs().max())
        ctx.quantize_rows(v, codes, scales, group=64, residual=res, residual_out=res)
        sent += (codes.double() * scales.double().repeat_interleave(64, 1))[:, :3000]
        total += v.double()
    assert float((sent + res.double() - total).abs().max()) <= slack


PRODUCTS = [(1, 1, 1), (1, 4096, 4096), (8, 64, 16), (9, 100, 33), (17, 130, 64), (32, 77, 1000), (300, 5, 260), (33, 33, 128), (128, 256, 128),
            (129, 257, 129), (64, 1000, 16), (200, 300, 8), (333, 1111, 2047), (1024, 2048, 512), (2500, 2600, 384), (256, 512, 4160), (40, 48, 131071),
            (5, 48, 131071), (50, 60, 0), (3, 4, 0)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(ctx, m, n, k, dtype):
    import torch

    dt = getattr(torch, dtype)
    g = gen(m * n + k)
    a = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sa = torch.rand(m, generator=g, device="cuda") * 1e-2 / math.sqrt(k + 1)
    sb = torch.rand(n, generator=g, device="cuda") * 1e-2
    got = ctx.int8_matmul(a, b, sa, sb, dtype=dt)
    ctx.check_status()
    check_product(got, a, b, sa, sb)


def check_product(got, a, b, sa, sb):
    import torch

    want = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    # sum, two products, and the type; numbers below the type's normal range are off by half of its smallest step
    rel = 3 * F32 + (0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2)
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps / 2
    assert bool(((got.double() - want).abs() <= want.abs() * rel * (1 + 1e-6) + tiny).all())


def test_product_of_the_largest_sums(ctx):
    """all codes at the ends of their range: the sums need all 32 bits"""
    import torch

    for m, n in [(3, 40), (64, 70)]:
        for x, y in [(-128, -128), (127, -128), (127, 127)]:
            a = torch.full((m, 131071), x, dtype=torch.int8, device="cuda")
            b = torch.full((n, 131071), y, dtype=torch.int8, device="cuda")
            one = torch.ones(max(m, n), device="cuda")
            got = ctx.int8_matmul(a, b, one[:m].contiguous(), one[:n].contiguous(), dtype=torch.float32)
            assert bool((got == float(torch.tensor(x * y * 131071).float())).all())


@pytest.mark.parametrize("m,n,k", [(1, 300, 256), (20, 40, 96), (150, 500, 256), (300, 300, 100)])
def test_product_of_strided_rows(ctx, m, n, k):
    """operands and results that are columns of wider matrices, at every alignment; what lies beside them stays as it was"""
    import torch

    g = gen(k)
    for off, pad in [(0, 16), (16, 0), (1, 15), (4, 3), (7, 0)]:
        a = torch.randint(-127, 128, (m, off + k + pad), generator=g, device="cuda", dtype=torch.int8)[:, off:off + k]
        b = torch.randint(-127, 128, (n, off + k + 2 * pad), generator=g, device="cuda", dtype=torch.int8)[:, off:off + k]
        sa, sb = torch.rand(m + 1, generator=g, device="cuda")[1:], torch.rand(n + 3, generator=g, device="cuda")[3:]
        for dt in (torch.float32, torch.bfloat16):
            wide = torch.full((m, off + n + pad), 7.0, dtype=dt, device="cuda")
            got = ctx.int8_matmul(a, b, sa, sb, out=wide[:, off:off + n])
            check_product(got, a, b, sa, sb)
            assert bool((wide[:, :off] == 7).all()) and bool((wide[:, off + n:] == 7).all())


@pytest.mark.parametrize("k", [16, 240, 2048])
@pytest.mark.parametrize("n", [33, 36, 41, 44, 45, 130, 257, 260, 300])
def test_product_into_aligned_rows_with_room_behind_them(ctx, n, k):
    """rows of the result start on 16-byte boundaries and end between two: what lies behind their ends stays as it was"""
    import torch

    g = gen(n + k)
    m = 70
    a = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sa, sb = torch.rand(m, generator=g, device="cuda") * 1e-3, torch.rand(n, generator=g, device="cuda")
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        wide = torch.full((m + 1, -(-n // 16) * 16 + 16), 7.0, dtype=dt, device="cuda")
        check_product(ctx.int8_matmul(a, b, sa, sb, out=wide[:m, :n]), a, b, sa, sb)
        assert bool((wide[:m, n:] == 7).all()) and bool((wide[m] == 7).all())


def distances(codes, scales, slots, group):
    """from differences, in 64 bits, and how far sums of 64-bit floats may be off"""
    import torch

    n, pages = slots.shape
    page = codes.shape[1]
    x = torch.zeros(n, pages, page, dtype=torch.float64, device="cuda")
    wide = codes.double() * scales.double().repeat_interleave(group if 0 < group < page else page, 1)[:, :page]
    there = (slots >= 0) & (slots < codes.shape[0])
    x[there] = wide[slots[there].long()]
    x = x.view(n, -1)
    want = torch.stack([(x - x[i]).square().sum(1) for i in range(n)])
    norm = x.square().sum(1)
    return want, (norm[:, None] + norm) * F64 * (x.shape[1] + 8)


@pytest.mark.parametrize("n,pages,page", [(1, 1, 16), (2, 1, 32), (4, 7, 8192), (9, 3, 1008), (17, 2, 2048), (20, 5, 4096), (32, 1, 48), (33, 2, 512),
                                          (70, 3, 1040), (100, 2, 4096), (5, 40, 8192), (64, 4, 2048), (97, 1, 1200), (100, 30, 8192), (70, 33, 8192), (40, 70, 8192), (56, 70, 8192), (20, 150, 8192), (128, 2, 1024), (130, 2, 1040),
                                          (200, 1, 2048)])
@pytest.mark.parametrize("group", [0, 32, 64, 128, 1024])
def test_pair_distances(ctx, n, pages, page, group):
    import torch

    g = gen(n * page + group)
    groups = -(-page // group) if 0 < group < page else 1
    codes = torch.randint(-127, 128, (n * pages + 2, page), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand(n * pages + 2, groups, generator=g, device="cuda")
    slots = torch.randperm(n * pages + 2, generator=g, device="cuda")[: n * pages].to(torch.int32).view(n, pages)
    if n > 2:
        slots[1] = slots[2]  # two rows that are the same
        slots[0, 0] = -1     # a page that is not there
    got = ctx.int8_distances(codes, scales, slots, group=group)
    want, slack = distances(codes, scales, slots, group)
    assert bool(((got - want).abs() <= slack).all())
    assert torch.equal(got, got.T) and bool((got.diagonal() == 0).all())
    if n > 2:
        assert float(got[1, 2]) == 0.0 and torch.equal(got[1], got[2])


def test_the_c_entry_takes_pages_in_order_where_no_slots_are_given(ctx):
    import ctypes as C

    import torch

    from lancelot_b200._lib import check, lib

    for n in (3, 40, 130):
        pages, page = 3, 1024
        codes = torch.randint(-127, 128, (n * pages, page), generator=gen(n), device="cuda", dtype=torch.int8)
        scales = torch.rand(n * pages, 8, generator=gen(n + 1), device="cuda")
        out, i, p = torch.empty(n, n, dtype=torch.float64, device="cuda"), C.c_int64, C.c_void_p
        lib.lb_int8_distances_workspace_bytes.restype = C.c_size_t
        need = lib.lb_int8_distances_workspace_bytes(ctx.h, i(n), i(pages), i(page))
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        call = lambda size: lib.lb_int8_distances(ctx.h, p(codes.data_ptr()), i(page), p(scales.data_ptr()), i(8), i(n * pages), i(page), i(128), None, i(n),  # noqa: E731
                                                  i(pages), p(out.data_ptr()), p(ws.data_ptr()), C.c_size_t(size), ctx._stream())
        check(call(need))
        slots = torch.arange(n * pages, dtype=torch.int32, device="cuda").view(n, pages)
        assert torch.equal(out, ctx.int8_distances(codes, scales, slots, group=128))
        assert call(need - 1) == 1 and b"workspace" in lib.lb_last_error()


def test_offsets_past_32_bits(ctx):
    """slots, rows and results more than 2^32 bytes or elements from the start of their memory"""
    import torch

    g = gen(11)
    page, cols = 32768, 40001
    codes = torch.empty(140000, page, dtype=torch.int8, device="cuda")
    scales = torch.empty(140000, page // 128, device="cuda")
    slots = (torch.randperm(2000, generator=g, device="cuda")[:80] + 138000).int()
    for n in (3, 40):
        t = slots[: n * 2].view(n, 2)
        v = torch.randn(n, cols, generator=g, device="cuda")
        ctx.quantize_rows(v, codes, scales, group=128, slots=t)
        want_codes, want_scales, _ = quantized(v, page, 128)
        at = t.view(-1).long()
        assert torch.equal(codes[at], want_codes) and torch.equal(scales[at], want_scales)
        x = expanded(want_codes, want_scales, 128).view(n, -1)[:, :cols]
        assert torch.equal(ctx.dequantize_rows(codes, scales, cols, group=128, slots=t), x)
        want, tol = distances(want_codes, want_scales, torch.arange(2 * n, device="cuda", dtype=torch.int32).view(n, 2), 128)
        assert bool(((ctx.int8_distances(codes, scales, t, group=128) - want).abs() <= tol).all())
    del codes, scales
    wide = torch.empty(40, 1 << 27, dtype=torch.bfloat16, device="cuda")
    v = wide[::39, -cols:]
    v.copy_(torch.randn(2, cols, generator=g, device="cuda"))
    codes, scales = torch.empty(4, page, dtype=torch.int8, device="cuda"), torch.empty(4, 1, device="cuda")
    ctx.quantize_rows(v, codes, scales)
    want_codes, want_scales, _ = quantized(v.float(), page, 0)
    assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales)
    ctx.dequantize_rows(codes, scales, cols, out=v)
    assert torch.equal(v, expanded(codes, scales, 0).view(2, -1)[:, :cols].to(torch.bfloat16))
    a = torch.randint(-127, 128, (40, 64), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-127, 128, (301, 64), generator=g, device="cuda", dtype=torch.int8)
    sa, sb = torch.rand(40, generator=g, device="cuda"), torch.rand(301, generator=g, device="cuda")
    check_product(ctx.int8_matmul(a, b, sa, sb, out=wide[:, -304:-3]), a, b, sa, sb)
    check_product(ctx.int8_matmul(a[:9], b, sa[:9], sb, out=wide[-9:, -304:-3]), a[:9], b, sa[:9], sb)


def test_two_streams_at_once(ctx):
    """calls of one context on two streams share no scratch: each gives what it gives alone"""
    import torch

    n, page = 40, 4096
    sets = []
    for k in range(2):
        codes = torch.randint(-127, 128, (n, page), generator=gen(k), device="cuda", dtype=torch.int8)
        sets.append((codes, torch.rand(n, 32, generator=gen(9 + k), device="cuda"), torch.rand(n, generator=gen(20 + k), device="cuda")))
    slots = torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1)
    odd = [c[:, :1001] for c, _, _ in sets]

    def work(k):
        codes, scales, s = sets[k]
        return ctx.int8_distances(codes, scales, slots, group=128), ctx.int8_matmul(odd[k], odd[k], s, s, dtype=torch.float32)

    alone = [work(k) for k in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(work(k))
        torch.cuda.synchronize()
        for x, y in zip(got, alone):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_distances_of_a_row_that_is_not_a_number(ctx):
    import torch

    codes = torch.randint(-127, 128, (5, 256), generator=gen(2), device="cuda", dtype=torch.int8)
    scales = torch.rand(5, 2, generator=gen(3), device="cuda")
    scales[3, 1] = math.nan
    d = ctx.int8_distances(codes, scales, torch.arange(5, dtype=torch.int32, device="cuda").view(5, 1), group=128)
    others = [i for i in range(5) if i != 3]
    assert bool(d[3, others].isnan().all()) and bool(d[others, 3].isnan().all()) and not d[others][:, others].isnan().any()
    assert float(d[3, 3]) == 0.0


def test_a_chain_is_captured_and_replayed(ctx):
    """write, read back, distances and a product of the written codes in one CUDA graph, on values that change between replays"""
    import torch

    n, cols, page = 6, 2000, 1024
    v = torch.zeros(n, cols, device="cuda")
    codes, scales = torch.zeros(2 * n, page, dtype=torch.int8, device="cuda"), torch.zeros(2 * n, 8, device="cuda")
    slots = torch.arange(2 * n, dtype=torch.int32, device="cuda").view(n, 2)
    whole, whole_scale = torch.zeros(n, 2000, dtype=torch.int8, device="cuda"), torch.zeros(n, 1, device="cuda")
    weight = torch.randint(-127, 128, (200, 2000), generator=gen(1), device="cuda", dtype=torch.int8)
    weight_scale = torch.rand(200, generator=gen(2), device="cuda")

    def work():
        ctx.quantize_rows(v, codes, scales, group=128, slots=slots)
        ctx.quantize_rows(v, whole, whole_scale)
        return (ctx.dequantize_rows(codes, scales, cols, group=128, slots=slots), ctx.int8_distances(codes, scales, slots, group=128),
                ctx.int8_matmul(whole, weight, whole_scale.view(-1), weight_scale, dtype=torch.float32))

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for seed in range(3):
        v.copy_(torch.randn(n, cols, generator=gen(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        for x, y in zip(replayed, work()):
            assert torch.equal(x, y)


def test_calls_on_another_stream(ctx):
    import torch

    v = torch.randn(3, 40000, generator=gen(4), device="cuda")
    side = torch.cuda.Stream()
    codes, scales = torch.zeros(3, 40000, dtype=torch.int8, device="cuda"), torch.zeros(3, 1, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ctx.quantize_rows(v, codes, scales)
        back = ctx.dequantize_rows(codes, scales, 40000)
    side.synchronize()
    want = quantized(v, 40000, 0)
    assert torch.equal(codes, want[0]) and torch.equal(back, expanded(codes, scales, 0))


def test_refusals(ctx):
    import torch

    from lancelot_b200._lib import InvalidArgument

    v = torch.zeros(2, 64, device="cuda")
    codes, scales = torch.zeros(2, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 1, device="cuda")
    bad = [lambda: ctx.quantize_rows(v.double(), codes, scales), lambda: ctx.quantize_rows(v.cpu(), codes, scales),
           lambda: ctx.quantize_rows(v, codes, scales, group=48), lambda: ctx.quantize_rows(v, codes, scales, group=16),
           lambda: ctx.quantize_rows(v, codes, scales, group=-32), lambda: ctx.quantize_rows(v, codes, scales, group=32),  # two scales a slot
           lambda: ctx.quantize_rows(v, codes[:, :60], scales), lambda: ctx.quantize_rows(v, codes[:1], scales),
           lambda: ctx.quantize_rows(v, codes, scales[:1]), lambda: ctx.quantize_rows(v, codes, scales, lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
           lambda: ctx.quantize_rows(v, codes, scales, slots=torch.zeros(3, dtype=torch.int32, device="cuda")),
           lambda: ctx.quantize_rows(v, codes, scales, slots=torch.zeros(2, dtype=torch.int64, device="cuda")),
           lambda: ctx.quantize_rows(v, codes, scales, residual=torch.zeros(2, 63, device="cuda")),
           lambda: ctx.quantize_rows(v.t()[:2], codes, scales), lambda: ctx.quantize_rows(v[:1].expand(2, 64), codes, scales),
           lambda: ctx.dequantize_rows(codes, scales, 64, dtype=torch.float64), lambda: ctx.dequantize_rows(codes, scales, 64, n_rows=3),
           lambda: ctx.dequantize_rows(codes, scales, 64, out=torch.zeros(2, 65, device="cuda")),
           lambda: ctx.int8_matmul(codes, codes[:, :32], v[0, :2], v[0, :2]), lambda: ctx.int8_matmul(codes, codes, v[0, :3], v[0, :2]),
           lambda: ctx.int8_matmul(codes, codes, v[0, :2], v[0, :2], dtype=torch.int32), lambda: ctx.int8_matmul(codes.to(torch.uint8), codes, v[0, :2], v[0, :2]),
           lambda: ctx.int8_matmul(*[torch.zeros(1, 131072, dtype=torch.int8, device="cuda")] * 2, v[0, :1], v[0, :1]),
           lambda: ctx.int8_distances(codes, scales, torch.zeros(2, dtype=torch.int32, device="cuda")),
           lambda: ctx.int8_distances(codes, scales, torch.zeros(5000, 1, dtype=torch.int32, device="cuda"))]
    for i, call in enumerate(bad):
        with pytest.raises(InvalidArgument):
            call()
            pytest.fail("call %d was not refused" % i)
    assert not codes.any() and not scales.any()
    # rows of no columns and no rows at all are served
    ctx.quantize_rows(v[:0], codes, scales)
    ctx.quantize_rows(v[:, :0], codes, scales)
    assert ctx.dequantize_rows(codes, scales, 0, n_rows=2).shape == (2, 0)
    assert ctx.int8_matmul(codes[:0], codes, v[0, :0], v[0, :2]).shape == (0, 2)
    assert ctx.int8_distances(codes, scales, torch.zeros(0, 1, dtype=torch.int32, device="cuda")).shape == (0, 0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(4000, 4096, 16), (4001, 4096, 128), (2337, 4104, 48), (300, 40000, 16), (1100, 20000, 1024)])
def test_product_whose_last_rows_fill_part_of_a_tile(ctx, m, n, k, dtype):
    """several tiles a block, of which some lie partly behind the last row: no result that is still on its way out is written over"""
    import torch

    g = gen(m + n + k)
    a = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sa, sb = torch.rand(m, generator=g, device="cuda") * 1e-3 + 1e-4, torch.rand(n, generator=g, device="cuda") + 0.1
    out = torch.empty(m, n, dtype=getattr(torch, dtype), device="cuda")
    first = ctx.int8_matmul(a, b, sa, sb, out=out).clone()
    check_product(first, a, b, sa, sb)
    for _ in range(30):
        out.fill_(math.nan)
        ctx.int8_matmul(a, b, sa, sb, out=out)
        assert torch.equal(out, first)
    ctx.check_status()


def test_a_single_row_or_slot_has_no_stride(ctx):
    """one row of a wider matrix beside a dense one, one slot of wider slots: how far the next row would lie does not matter"""
    import torch

    g = gen(6)
    cols = 1003
    v = torch.randn(1, cols + 7, generator=g, device="cuda")[:, 3:3 + cols]
    res = torch.randn(1, 1050, generator=g, device="cuda")[:, :cols] * 0.01
    res = torch.cat([res, torch.zeros(1, 47, device="cuda")], 1)[:, :cols]
    assert res.stride(0) == 1050
    lost = torch.empty(1, cols, device="cuda")
    wide = torch.full((3, 1025), 9, dtype=torch.int8, device="cuda")
    codes, scales = wide[:1, :1008], torch.empty(1, 9, device="cuda")[:, :8]
    ctx.quantize_rows(v, codes, scales, group=128, residual=res, residual_out=lost)
    want_codes, want_scales, want_lost = quantized(v + res, 1008, 128)
    assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales) and torch.equal(lost, want_lost)
    assert bool((wide[0, 1008:] == 9).all()) and bool((wide[1:] == 9).all())
    assert torch.equal(ctx.dequantize_rows(codes, scales, cols, group=128), expanded(codes, scales, 128)[:, :cols])
    assert float(ctx.int8_distances(codes, scales, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), group=128).abs().max()) == 0
    # the residual that is kept in a row of another width, the other way round
    kept = torch.full((2, 1050), 5.0, device="cuda")
    ctx.quantize_rows(v, codes, scales, group=128, residual=res.contiguous(), residual_out=kept[1:, :cols])
    assert torch.equal(kept[1:, :cols], want_lost) and bool((kept[0] == 5).all()) and bool((kept[1, cols:] == 5).all())


@pytest.mark.parametrize("group", [32, 0])
def test_residuals_in_the_gaps_of_one_another(ctx, group):
    """residual and residual_out are memory apart where their rows take turns; rows that share an element are refused"""
    import torch

    from lancelot_b200._lib import InvalidArgument

    g = gen(12)
    n, cols = 5, 1003
    v = torch.randn(n, cols, generator=g, device="cuda")
    codes, scales = torch.empty(n, 1008, dtype=torch.int8, device="cuda"), torch.empty(n, -(-1008 // group) if group else 1, device="cuda")
    for gap in (0, 1, 5):
        both = torch.randn(n, 2 * cols + gap, generator=g, device="cuda") * 0.01
        for x, y in ((0, cols + gap), (cols + gap, 0)):
            before = both.clone()
            res, lost = both[:, x:x + cols], both[:, y:y + cols]
            ctx.quantize_rows(v, codes, scales, group=group, residual=res, residual_out=lost)
            want_codes, want_scales, want_lost = quantized(v + before[:, x:x + cols], 1008, group)
            assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales) and torch.equal(lost, want_lost)
            before[:, y:y + cols] = want_lost
            assert torch.equal(both, before)
    wide = torch.zeros(n + 1, 2 * cols, device="cuda")
    for res, lost in ((wide[:n, :cols], wide[:n, 1:1 + cols]), (wide[:n, :cols], wide[:n, cols - 1:-1]), (wide[:n, :cols], wide[1:, :cols]),
                      (wide[1:, 2:2 + cols], wide[:n, :cols]), (wide[:n, 1:1 + cols], wide[:n, :cols]), (wide[:1, :cols], wide[:1, 1:1 + cols])):
        with pytest.raises(InvalidArgument, match="apart"):
            ctx.quantize_rows(v[: len(res)], codes, scales, group=group, residual=res, residual_out=lost)
    assert not wide.any()


THREADS = """
import ctypes as C, threading, torch
from lancelot_b200 import cabi
from lancelot_b200._lib import lib
ctx = cabi.Context(12, cabi.coeff_modulus_create(1 << 12, [40, 40]), 1)
lib.lb_int8_distances_workspace_bytes.restype = C.c_size_t
i, p = C.c_int64, lambda t: C.c_void_p(t.data_ptr())
g = torch.Generator("cuda").manual_seed(1)
codes = torch.randint(-127, 128, (40, 1024), generator=g, device="cuda", dtype=torch.int8)
scale = torch.rand(40, generator=g, device="cuda")
want = (codes.double() @ codes.double().T) * scale.double()[:, None] * scale.double()
need = lib.lb_int8_distances_workspace_bytes(ctx.h, i(40), i(1), i(1024))
n, results = 8, []
for _ in range(n):
    results.append((torch.empty(40, 40, device="cuda"), torch.empty(40, 40, dtype=torch.float64, device="cuda"), torch.empty(need, dtype=torch.uint8, device="cuda"),
                    torch.cuda.Stream(), [None, None]))
torch.cuda.synchronize()
start = threading.Barrier(n)
def call(product, distances, ws, stream, codes_of):  # the C entries themselves: ctypes lets the threads run side by side
    start.wait()
    s = C.c_void_p(stream.cuda_stream)
    codes_of[0] = lib.lb_int8_matmul(ctx.h, i(40), i(40), i(1024), p(codes), i(1024), p(scale), p(codes), i(1024), p(scale), p(product), 1, i(40), None, C.c_size_t(0), s)
    codes_of[1] = lib.lb_int8_distances(ctx.h, p(codes), i(1024), p(scale), i(1), i(40), i(1024), i(0), None, i(40), i(1), p(distances), p(ws), C.c_size_t(need), s)
threads = [threading.Thread(target=call, args=r) for r in results]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
d = want.diagonal()[:, None] + want.diagonal() - 2 * want
for product, distances, _, _, codes_of in results:
    assert codes_of == [0, 0]
    assert bool(((product.double() - want).abs() <= want.abs() * 3.1 * 2.0 ** -24).all())
    assert bool(((distances - d).abs() <= (want.diagonal()[:, None] + want.diagonal()) * 2.0 ** -53 * 1032 * 2).all())
print("threads agree")
"""


def test_threads_that_make_the_first_calls_at_once():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", THREADS], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "threads agree" in r.stdout, r.stderr


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,n,k", [(3, 200, 64), (20, 70, 1001), (140, 300, 128), (140, 301, 2048), (200, 256, 100)])
def test_product_with_scales_that_are_not_finite(ctx, m, n, k, dtype):
    """they reach their own row or column of the result and no other: a sum of 0 times an infinity is NaN, any other one infinite"""
    import torch

    g = gen(m + k)
    a = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    b = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    a[m // 2] = 0  # a row of sums that are 0
    sa, sb = torch.rand(m, generator=g, device="cuda") + 0.5, torch.rand(n, generator=g, device="cuda") + 0.5
    clean = ctx.int8_matmul(a, b, sa, sb, dtype=getattr(torch, dtype))
    sa[0], sa[m - 1], sb[1], sb[n - 1] = math.inf, math.nan, -math.inf, math.nan
    got = ctx.int8_matmul(a, b, sa, sb, dtype=getattr(torch, dtype))
    total = (a.double() @ b.double().T).float()  # 64 bits hold the sum exactly; rounded once, as defined
    want = (total * sa[:, None] * sb).to(got.dtype)
    fine = torch.ones(m, n, dtype=torch.bool, device="cuda")
    fine[0] = fine[m - 1] = False
    fine[:, 1] = fine[:, n - 1] = False
    assert torch.equal(got[fine], clean[fine]) and bool(got[fine].isfinite().all())
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~fine].nan_to_num(0.0), want[~fine].nan_to_num(0.0))
    assert bool(got[m // 2, 1].isnan()) and bool(got[m - 1].isnan().all()) and bool(got[:, n - 1].isnan().all())
    assert got[0].isinf().any()


@pytest.mark.parametrize("n", [5, 20, 40, 130])
def test_distances_of_a_row_with_an_infinite_scale(ctx, n):
    """they are not finite (64-bit terms that are infinite cancel to NaN); those of all other pairs are what they were"""
    import torch

    codes = torch.randint(1, 128, (n, 512), generator=gen(n), device="cuda", dtype=torch.int8)
    scales = torch.rand(n, 4, generator=gen(n + 1), device="cuda") + 0.5
    slots = torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1)
    before = ctx.int8_distances(codes, scales, slots, group=128)
    scales[2, 1] = math.inf
    got = ctx.int8_distances(codes, scales, slots, group=128)
    others = [i for i in range(n) if i != 2]
    assert torch.equal(got[others][:, others], before[others][:, others])
    assert not bool(got[2, others].isfinite().any()) and torch.equal(got[2].isnan(), got[:, 2].isnan()) and float(got[2, 2]) == 0.0


@pytest.mark.parametrize("n,pages,page", [(129, 5, 1040), (160, 3, 4096), (200, 6, 2048), (257, 2, 1008)])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_pair_distances_of_many_clients_over_several_pages(ctx, n, pages, page, group):
    import torch

    g = gen(n * pages + group)
    groups = -(-page // group) if 0 < group < page else 1
    codes = torch.randint(-127, 128, (n * pages + 2, page), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand(n * pages + 2, groups, generator=g, device="cuda")
    slots = torch.randperm(n * pages + 2, generator=g, device="cuda")[: n * pages].to(torch.int32).view(n, pages)
    slots[n - 1] = slots[0]                        # two rows that are the same, in blocks of clients far apart
    slots[1, pages - 1], slots[40, 0] = -1, 1 << 30  # pages that are not there
    got = ctx.int8_distances(codes, scales, slots, group=group)
    want, slack = distances(codes, scales, slots, group)
    assert bool(((got - want).abs() <= slack).all())
    assert torch.equal(got, got.T) and bool((got.diagonal() == 0).all()) and float(got[0, n - 1]) == 0.0
    assert torch.equal(got, ctx.int8_distances(codes, scales, slots, group=group))
