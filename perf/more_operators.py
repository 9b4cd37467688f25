"""Operators that form a client's update in 8-bit floating point and bound it, taken through ``cabi.Context`` and ``updates``.

  quantize  a matrix is brought to 8-bit floating point with a scale for each block (``quantize_fp8``) and read back
            (``dequantize_fp8``).  Blocks: 128 columns of a row ("rows"), 128 rows of a column ("columns"), 128 x 128 ("square"), or
            both of the first two in one call ("both", ``quantize_fp8_both``): one for products over columns, one for products over rows
  product   matrix product of such operands (``fp8_matmul``), out = a b^T with a scale for each block of 128 of the summed axis.
            "forward": a [m][k] in rows, b [n][k] in squares; "input": the gradient of the first operand, b lies [k][n] in squares;
            "weight": the gradient of the second one, a [k][m] and b [k][n] lie with the summed axis first, both in columns;
            "factors": a [m][k] and b [n][k] in rows, a short summed axis: an update of low rank from its factors
  clip      the norm of every client's update over all of its tensors, and the tensors, scaled down to a largest norm, as one flat row a
            client (``clip_updates``)
  step      y = x w^T and, from the gradient of y, the gradients of x and w, with all three products in 8-bit floating point
            (``updates.fp8_linear``)

A block whose largest magnitude is m has the scale m / M (rounded to 32 bits), M the type's largest value (448 for e4m3, 57344 for e5m2); a code
is the type's value nearest to value / scale, ties to even, at most M in magnitude.
"""
import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
BLOCK = 128


def listed():
    return [
        # one row of activations, the smallest call, where latency counts
        {"name": "quantize_row_4096", "kind": "quantize", "rows": 1, "cols": 4096, "block": "rows", "dtype": "bfloat16", "code": "e4m3"},
        # a weight matrix odd in both directions
        {"name": "quantize_777x1000_square", "kind": "quantize", "rows": 777, "cols": 1000, "block": "square", "dtype": "float32", "code": "e4m3"},
        # the activations of a training step, for the product and for its gradient
        {"name": "quantize_8192x4096_both", "kind": "quantize", "rows": 8192, "cols": 4096, "block": "both", "dtype": "bfloat16", "code": "e4m3"},
        # one row against a square weight matrix: bound by the weights' bytes
        {"name": "product_1x4096x4096", "kind": "product", "form": "forward", "m": 1, "n": 4096, "k": 4096, "dtype": "bfloat16", "code": "e4m3"},
        # the gradient of the first operand, odd in every direction
        {"name": "product_input_333x1111x2047", "kind": "product", "form": "input", "m": 333, "n": 1111, "k": 2047, "dtype": "float16", "code": "e4m3"},
        # the gradient of a weight matrix, in the 32 bits that updates have
        {"name": "product_weight_4096x11008x4096", "kind": "product", "form": "weight", "m": 4096, "n": 11008, "k": 4096, "dtype": "float32", "code": "e5m2"},
        # a large square product, bound by the tensor cores
        {"name": "product_8192", "kind": "product", "form": "forward", "m": 8192, "n": 8192, "k": 8192, "dtype": "bfloat16", "code": "e4m3"},
        # a small federation with a small model
        {"name": "clip_4x50k", "kind": "clip", "clients": 4, "tensors": 8, "dim": 50890, "dtype": "float32", "into": "float32"},
        # one client's gradients of a model of 11 million parameters
        {"name": "clip_1x11m", "kind": "clip", "clients": 1, "tensors": 62, "dim": 11173962, "dtype": "bfloat16", "into": "float32"},
        # all updates of the 20-client federation
        {"name": "clip_20x11m", "kind": "clip", "clients": 20, "tensors": 62, "dim": 11173962, "dtype": "float32", "into": "float32"},
        # a training step of a small layer on a small, odd batch
        {"name": "step_50x784x200", "kind": "step", "m": 50, "n": 200, "k": 784, "dtype": "float32"},
        # a training step of a large layer
        {"name": "step_2048x4096x11008", "kind": "step", "m": 2048, "n": 11008, "k": 4096, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(lo * (hi / lo) ** rng.random() + 0.5)


def draw(rng):
    kind = rng.choice(["quantize", "product", "clip", "step"])
    dtype = rng.choice(sorted(TYPES))
    code = rng.choice(sorted(CODES))
    if kind == "quantize":
        cols = _log(rng, 30, 12000)
        rows = min(_log(rng, 1, 12000), 33000000 // cols)
        return {"kind": kind, "rows": rows, "cols": cols, "block": rng.choice(["rows", "columns", "square", "both"]), "dtype": dtype, "code": code}
    if kind == "product":
        form = rng.choice(["forward", "input", "weight", "factors"])
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 8, 300) if form == "factors" else _log(rng, 64, 8192)
        if rng.random() < 0.5:
            n, k = n + -n % 16, k + -k % 16
        return {"kind": kind, "form": form, "m": m, "n": n, "k": k, "dtype": dtype, "code": code if form in ("input", "weight") else "e4m3"}
    if kind == "clip":
        dim = _log(rng, 3000, 11000000)
        clients = max(1, min(_log(rng, 1, 100), 200000000 // dim))
        return {"kind": kind, "clients": clients, "tensors": _log(rng, 2, 150), "dim": dim, "dtype": dtype, "into": rng.choice(["float32", dtype])}
    return {"kind": kind, "m": _log(rng, 8, 4096), "n": _log(rng, 64, 8192), "k": _log(rng, 64, 4096), "dtype": dtype}


def _values(g, rows, cols):
    """small values around zero; columns differ in spread, as features do, and a few entries stand out"""
    v = torch.randn(rows, cols, generator=g, device="cuda")
    v.mul_(torch.rand(cols, generator=g, device="cuda").mul_(3).exp_().mul_(0.02))
    return v.mul_(torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 1e-4, 30.0, 1.0))


def _blocks(n):
    return -(-n // BLOCK)


def _operand(g, rows, cols, tall, wide, code):
    """codes and scales as quantised values have them: the largest of a block is near the type's largest value.  tall, wide: whether a
    block spans 128 rows, 128 columns"""
    codes = torch.randn(rows, cols, generator=g, device="cuda").mul_(torch.finfo(CODES[code]).max / 4).clamp_(-torch.finfo(CODES[code]).max, torch.finfo(CODES[code]).max)
    scales = torch.rand(_blocks(rows) if tall else rows, _blocks(cols) if wide else cols, generator=g, device="cuda").add_(0.1).mul_(1 / torch.finfo(CODES[code]).max)
    pitch = cols + -cols % 16  # rows start on 16-byte boundaries, as quantised matrices have them
    held = torch.zeros(rows, pitch, dtype=CODES[code], device="cuda")
    held[:, :cols] = codes.to(CODES[code])
    return held[:, :cols], scales


def _sizes(dim, tensors):
    """a model's tensors: small vectors between weights that grow with depth, so that few start on a 16-byte boundary of the flat row"""
    small = max(1, int(math.sqrt(dim / tensors)) // 2)
    sizes = [small + i % 3 if i % 2 else 0 for i in range(tensors)]
    weights = range(0, tensors, 2)
    left, parts = dim - sum(sizes), sum(i + 1 for i in weights)
    for i in weights:
        sizes[i] = left * (i + 1) // parts
    sizes[weights[-1]] += dim - sum(sizes)
    return sizes


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["kind"] == "quantize":
        s["values"] = _values(g, case["rows"], case["cols"]).to(TYPES[case["dtype"]])
    elif case["kind"] == "product":
        m, n, k, form = case["m"], case["n"], case["k"], case["form"]
        if form == "weight":  # the gradient of the outputs and the inputs, both with their rows summed over
            s["a"], s["a_scale"] = _operand(g, k, m, True, False, case["code"])
            s["b"], s["b_scale"] = _operand(g, k, n, True, False, "e4m3")
        else:
            s["a"], s["a_scale"] = _operand(g, m, k, False, True, case["code"])
            s["b"], s["b_scale"] = _operand(g, k, n, True, True, "e4m3") if form == "input" else _operand(g, n, k, form == "forward", True, "e4m3")
    elif case["kind"] == "clip":
        sizes, kind = _sizes(case["dim"], case["tensors"]), TYPES[case["dtype"]]
        spread = random.Random(seed)
        # updates of different length; some are over the bound, one by far where there are several
        scale = [0.01 * 2 ** spread.uniform(-1, 1) * (50 if i == 2 else 1) for i in range(case["clients"])]
        s["updates"] = [[(torch.randn(n, generator=g, device="cuda") * c).to(kind) for n in sizes] for c in scale]
        s["max_norm"] = 0.01 * math.sqrt(case["dim"])
        s["out"] = torch.zeros(case["clients"], case["dim"], dtype=TYPES[case["into"]], device="cuda")
    else:
        kind = TYPES[case["dtype"]]
        s["x"] = _values(g, case["m"], case["k"]).to(kind).requires_grad_()
        s["w"] = (torch.randn(case["n"], case["k"], generator=g, device="cuda") * case["k"] ** -0.5).to(kind).requires_grad_()
        s["g"] = (torch.randn(case["m"], case["n"], generator=g, device="cuda") * 0.01).to(kind)
    return s


_contexts = {}


def _context():
    """the handle that a program keeps"""
    from lancelot_b200 import cabi

    device = torch.cuda.current_device()
    if device not in _contexts:
        _contexts[device] = cabi.Context(12, cabi.coeff_modulus_create(1 << 12, [40, 40]), 1, device=device)
    return _contexts[device]


def run(state):
    if own:
        return _own(state)
    return {"quantize": _quantize, "product": _product, "clip": _clip, "step": _step}[state["kind"]](state)


SHAPES = {"rows": (1, BLOCK), "columns": (BLOCK, 1), "square": (BLOCK, BLOCK)}


def _own(s):
    ctx = _context()
    if s["kind"] == "quantize":
        values, code = s["values"], CODES[s["code"]]
        if s["block"] == "both":
            codes, scales, codes_down, scales_down = ctx.quantize_fp8_both(values, dtype=code)
            return {"values": ctx.dequantize_fp8(codes, scales, dtype=values.dtype), "scales": scales,
                    "values_down": ctx.dequantize_fp8(codes_down, scales_down, dtype=values.dtype), "scales_down": scales_down}
        codes, scales = ctx.quantize_fp8(values, block=SHAPES[s["block"]], dtype=code)
        return {"values": ctx.dequantize_fp8(codes, scales, dtype=values.dtype), "scales": scales}
    if s["kind"] == "product":
        a, a_scale, b, b_scale = s["a"], s["a_scale"], s["b"], s["b_scale"]
        if s["form"] == "weight":
            a, a_scale = a.t(), a_scale.t()
        if s["form"] in ("weight", "input"):
            b, b_scale = b.t(), b_scale.t()
        return ctx.fp8_matmul(a, a_scale, b, b_scale, dtype=TYPES[s["dtype"]])
    if s["kind"] == "clip":
        norms = ctx.clip_updates(s["updates"], s["max_norm"], out=s["out"])
        return {"norms": norms, "rows": s["out"]}
    from lancelot_b200 import updates

    y = updates.fp8_linear(ctx, s["x"], s["w"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["g"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def _spread(scales, rows, cols, tall, wide):
    """a scale for every value"""
    scales = scales.repeat_interleave(BLOCK, 0)[:rows] if tall else scales
    return scales.repeat_interleave(BLOCK, 1)[:, :cols] if wide else scales


def _round(q, code):
    """the code type's value nearest to q (64 bits), ties to even"""
    bits, least = (3, -6) if code == "e4m3" else (2, -14)
    step = torch.exp2((torch.frexp(q)[1] - 1).clamp_min_(least).double() - bits)
    most = torch.finfo(CODES[code]).max
    return (q / step).round_().mul_(step).clamp_(-most, most)


def _coded(v, tall, wide, code):
    """values (32 bits) -> the values that their codes stand for, before the scale (64 bits), and the scales"""
    rows, cols = v.shape
    high, broad = BLOCK if tall else 1, BLOCK if wide else 1
    t = torch.nn.functional.pad(v, (0, -cols % broad, 0, -rows % high))
    most = t.view(t.shape[0] // high, high, t.shape[1] // broad, broad).abs().amax((1, 3))
    scales = torch.where(most.isfinite(), most / torch.full_like(most, torch.finfo(CODES[code]).max), float("nan"))
    each = _spread(scales, rows, cols, tall, wide)
    # next to a border between two codes 32 bits of the quotient decide wrongly
    codes = _round(v.double() / each.double(), code)
    return torch.where(each > 0, codes, 0.0), scales


def _held(v, tall, wide, code):
    """the values that codes and scales stand for, in 32 bits, and the scales"""
    codes, scales = _coded(v, tall, wide, code)
    return codes.float() * _spread(scales, *v.shape, tall, wide), scales


def _quantize(s):
    v, block, code = s["values"].float(), s["block"], s["code"]
    kind = s["values"].dtype
    held, scales = _held(v, block in ("columns", "square"), block != "columns", code)
    if block != "both":
        return {"values": held.to(kind), "scales": scales}
    down, scales_down = _held(v, True, False, code)
    return {"values": held.to(kind), "scales": scales, "values_down": down.to(kind), "scales_down": scales_down}


def _product(s):
    m, n, k, form = s["m"], s["n"], s["k"], s["form"]
    if form == "weight":
        a = (s["a"].float() * _spread(s["a_scale"], k, m, True, False)).T
    else:
        a = s["a"].float() * _spread(s["a_scale"], m, k, False, True)
    if form in ("weight", "input"):
        b = s["b"].float() * _spread(s["b_scale"], k, n, True, form == "input")
    else:
        b = (s["b"].float() * _spread(s["b_scale"], n, k, form == "forward", True)).T
    return (a @ b).to(TYPES[s["dtype"]])


def _clip(s):
    flat = torch.stack([torch.cat([t.float() for t in tensors]) for tensors in s["updates"]])
    norms = torch.stack([row.double().square().sum().sqrt() for row in flat])
    factor = torch.where(norms > s["max_norm"], s["max_norm"] / norms, 1.0)
    s["out"].copy_(flat * torch.where(norms.isfinite(), factor, float("nan")).float()[:, None])
    return {"norms": norms, "rows": s["out"]}


def _step(s):
    x, w, g = s["x"].detach().float(), s["w"].detach().float(), s["g"].float()
    kind = s["x"].dtype
    w8 = _held(w, True, True, "e4m3")[0]
    y = _held(x, False, True, "e4m3")[0] @ w8.T
    dx = _held(g, False, True, "e4m3")[0] @ w8
    dw = _held(g, True, False, "e4m3")[0].T @ _held(x, True, False, "e4m3")[0]
    return {"y": y.to(kind), "dx": dx.to(kind), "dw": dw.to(kind)}


def work(case):
    if case["kind"] == "quantize":
        rows, cols, item = case["rows"], case["cols"], TYPES[case["dtype"]].itemsize
        scales = {"rows": rows * _blocks(cols), "columns": _blocks(rows) * cols, "square": _blocks(rows) * _blocks(cols)}
        scales["both"] = scales["rows"] + scales["columns"]
        # values in; codes and scales out; the values read back
        times = 2 if case["block"] == "both" else 1
        return {"bytes": rows * cols * (item + times * (1 + item)) + 4 * scales[case["block"]], "flops": 4 * times * rows * cols}
    if case["kind"] == "clip":
        n = case["clients"] * case["dim"]
        return {"bytes": n * (TYPES[case["dtype"]].itemsize + TYPES[case["into"]].itemsize) + 8 * case["clients"], "flops": 3 * n}
    m, n, k = case["m"], case["n"], case["k"]
    item = TYPES[case["dtype"]].itemsize
    if case["kind"] == "product":
        scales = {"forward": m * _blocks(k) + _blocks(n) * _blocks(k), "input": m * _blocks(k) + _blocks(n) * _blocks(k),
                  "weight": (m + n) * _blocks(k), "factors": (m + n) * _blocks(k)}
        return {"bytes": m * k + n * k + 4 * scales[case["form"]] + item * m * n, "flops": 2 * m * n * k}
    # x, w and the gradient of y in; y and the gradients of x and w out
    return {"bytes": 2 * item * (m * k + n * k + m * n), "flops": 6 * m * n * k}


def _levels(code):
    """the magnitudes of an 8-bit type in order, and what lies half way between neighbours"""
    bits, least, most = (3, -6, 448.0) if code == "e4m3" else (2, -14, 57344.0)
    found = [0.0]
    for i in range(1, 128):
        e, f = divmod(i, 1 << bits)
        v = math.ldexp(f, least - bits) if e == 0 else math.ldexp((1 << bits) + f, e - 1 + least - bits)
        if v <= most:
            found.append(v)
    values = torch.tensor(found, dtype=torch.float64, device="cuda")
    return values, (values[1:] + values[:-1]) / 2


def _exact_held(v, tall, wide, code):
    """what the blocks of v (64 bits) are held as, and their scales, both in 64 bits: by blocks, and by place in the list of magnitudes"""
    values, between = _levels(code)
    high, broad = BLOCK if tall else 1, BLOCK if wide else 1
    rows, cols = v.shape
    i = torch.arange(rows, device="cuda") // high
    j = torch.arange(cols, device="cuda") // broad
    across = torch.zeros(rows, int(j[-1]) + 1, dtype=torch.float64, device="cuda").scatter_reduce_(1, j.expand(rows, cols), v.abs(), "amax")
    scales = torch.zeros(int(i[-1]) + 1, across.shape[1], dtype=torch.float64, device="cuda").scatter_reduce_(0, i[:, None].expand(across.shape), across, "amax")
    scales = scales / values[-1]
    held = scales.float().double()  # 32 bits of it are held
    out = torch.empty_like(v)
    for at in range(0, rows, 1024):
        each = held[i[at:at + 1024]][:, j]
        q = torch.where(each > 0, v[at:at + 1024].abs() / each, 0.0)
        low, high_ = torch.bucketize(q, between), torch.bucketize(q, between, right=True)
        place = torch.where(low % 2 == 0, low, high_)  # they differ half way between two values, where the even one is taken
        out[at:at + 1024] = torch.where(low == high_, values[low], values[place]) * v[at:at + 1024].sign() * each
    return out, scales


def exact(case, seed):
    """from the definitions, in 64 bits"""
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        v, block, code = s["values"].double(), case["block"], case["code"]
        held, scales = _exact_held(v, block in ("columns", "square"), block != "columns", code)
        if block != "both":
            return {"values": held, "scales": scales}
        down, scales_down = _exact_held(v, True, False, code)
        return {"values": held, "scales": scales, "values_down": down, "scales_down": scales_down}
    if case["kind"] == "product":
        m, n, k, form = case["m"], case["n"], case["k"], case["form"]
        out = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        of = torch.arange(max(m, n), device="cuda") // BLOCK
        for p in range(_blocks(k)):  # a block of the summed axis at a time
            at = slice(p * BLOCK, min(k, (p + 1) * BLOCK))
            if form == "weight":
                a, b = s["a"][at].double() * s["a_scale"][p].double(), s["b"][at].double() * s["b_scale"][p].double()
                out += torch.einsum("km,kn->mn", a, b)
                continue
            a = s["a"][:, at].double() * s["a_scale"][:, p, None].double()
            if form == "input":
                out += torch.einsum("mk,kn->mn", a, s["b"][at].double() * s["b_scale"][p].double()[of[:n]])
            else:
                each = s["b_scale"][:, p].double()
                out += torch.einsum("mk,nk->mn", a, s["b"][:, at].double() * (each[of[:n]] if form == "forward" else each)[:, None])
        return out
    if case["kind"] == "clip":
        norms = torch.zeros(case["clients"], dtype=torch.float64, device="cuda")
        rows = torch.empty(case["clients"], case["dim"], dtype=torch.float64, device="cuda")
        for i, tensors in enumerate(s["updates"]):
            at = 0
            for t in tensors:
                rows[i, at:at + t.numel()] = t.double()
                at += t.numel()
            norms[i] = torch.linalg.vector_norm(rows[i])
            if norms[i] > case["dim"] ** 0.5 * 0.01:
                rows[i] *= case["dim"] ** 0.5 * 0.01 / norms[i]
        return {"norms": norms, "rows": rows}
    x, w, g = s["x"].detach().double(), s["w"].detach().double(), s["g"].double()
    w8 = _exact_held(w, True, True, "e4m3")[0]
    y = torch.einsum("mk,nk->mn", _exact_held(x, False, True, "e4m3")[0], w8)
    dx = torch.einsum("mn,nk->mk", _exact_held(g, False, True, "e4m3")[0], w8)
    dw = torch.einsum("mn,mk->nk", _exact_held(g, True, False, "e4m3")[0], _exact_held(x, True, False, "e4m3")[0])
    return {"y": y, "dx": dx, "dw": dw}
