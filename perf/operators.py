"""Operators on the 8-bit updates of a federation's clients, taken through ``cabi.Context``.

  cache      values are written into slots of an 8-bit cache (``quantize_rows``: a scale per group of columns, what the rounding
             lost handed on as a residual) and read back by slot (``dequantize_rows``).  A row of ``cols`` values covers
             ceil(cols / page) slots; rows may be shorter than ``cols`` (``ragged``), also empty
  product    matrix product of 8-bit integers with a scale per row of a and per row of b (``int8_matmul``): out = (a b^T) * sa * sb
  distances  squared distances between all pairs of cached updates (``int8_distances``), read through a table of slots

Scales are 32-bit floats, codes lie in [-127, 127].  A group whose largest magnitude is m has the scale m / 127 (rounded to 32
bits); a code is the integer nearest to value / scale, ties to even.
"""
import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one row of a bfloat16 matrix: the smallest write, where latency counts
        {"name": "cache_row_4096", "kind": "cache", "rows": 1, "cols": 4096, "page": 4096, "group": 128, "dtype": "bfloat16", "residual": False, "ragged": False},
        # rows of an odd width with lengths of their own, some empty; one scale a row (the operand of an 8-bit product)
        {"name": "cache_777x1000_rows", "kind": "cache", "rows": 777, "cols": 1000, "page": 1008, "group": 0, "dtype": "float16", "residual": False, "ragged": True},
        # one client's update of odd length in pages of 32768 slots, with the error feedback of 8-bit uploads
        {"name": "cache_upload_1.6m", "kind": "cache", "rows": 1, "cols": 1663370, "page": 32768, "group": 128, "dtype": "float32", "residual": True, "ragged": False},
        # all updates of the 20-client federation, one scale a page, the largest write
        {"name": "cache_20x11m", "kind": "cache", "rows": 20, "cols": 11173962, "page": 32768, "group": 0, "dtype": "float32", "residual": True, "ragged": False},
        # one row against a square weight matrix: bound by the weights' bytes
        {"name": "product_1x4096x4096", "kind": "product", "m": 1, "n": 4096, "k": 4096, "dtype": "bfloat16"},
        # a low-rank update formed from its two factors of rank 16: bound by the 32-bit result
        {"name": "product_4096x4096x16", "kind": "product", "m": 4096, "n": 4096, "k": 16, "dtype": "float32"},
        # odd in every direction: rows that start on no 16-byte boundary
        {"name": "product_333x1111x2047", "kind": "product", "m": 333, "n": 1111, "k": 2047, "dtype": "float16"},
        # a large square product, bound by the tensor cores
        {"name": "product_8192", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "dtype": "bfloat16"},
        # a small federation with a small model, pages of a 2^14 ring
        {"name": "distances_4x50k", "kind": "distances", "clients": 4, "cols": 50890, "page": 8192, "group": 128},
        # ten clients of a 1.6 million parameter model, one scale a page
        {"name": "distances_10x1.6m", "kind": "distances", "clients": 10, "cols": 1663370, "page": 16384, "group": 0},
        # the 20-client round, a scale for every 128 values
        {"name": "distances_20x11m", "kind": "distances", "clients": 20, "cols": 11173962, "page": 32768, "group": 128},
        # many clients of the smaller model
        {"name": "distances_100x1.6m", "kind": "distances", "clients": 100, "cols": 1663370, "page": 32768, "group": 64},
    ]


def _log(rng, lo, hi):
    return int(lo * (hi / lo) ** rng.random() + 0.5)


def draw(rng):
    kind = rng.choice(["cache", "product", "distances"])
    group = rng.choice([0, 32, 64, 128, 256, 512, 1024])
    if kind == "cache":
        cols = _log(rng, 100, 10000000)
        rows = min(_log(rng, 1, 4000), 200000000 // cols)
        page = max(32, cols + -cols % 16) if cols < 20000 else rng.choice([4096, 8192, 16384, 32768])
        return {"kind": kind, "rows": max(1, rows), "cols": cols, "page": page, "group": group, "dtype": rng.choice(sorted(TYPES)),
                "residual": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    if kind == "product":
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 8, 8192)
        if rng.random() < 0.5:
            n, k = n + -n % 16, k + -k % 16
        return {"kind": kind, "m": m, "n": n, "k": k, "dtype": rng.choice(sorted(TYPES))}
    cols = _log(rng, 3000, 10000000)
    clients = min(_log(rng, 2, 100), 160000000 // cols)
    return {"kind": kind, "clients": max(2, clients), "cols": cols, "page": rng.choice([4096, 8192, 16384, 32768]), "group": group}


def _groups(page, group):
    return -(-page // group) if group else 1


def _values(g, rows, cols):
    """updates: small values around zero whose spread differs between runs of columns, as between layers"""
    v = torch.randn(rows, cols, generator=g, device="cuda")
    spread = torch.rand(-(-cols // 1000), generator=g, device="cuda").mul_(3).exp_().mul_(1e-3)
    return v.mul_(spread.repeat_interleave(1000)[:cols])


def _codes(g, rows, cols):
    """what quantised normal values look like: the largest of a group is 127"""
    return torch.randn(rows, cols, generator=g, device="cuda").mul_(36).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["kind"] == "product":
        s["a"], s["b"] = _codes(g, case["m"], case["k"]), _codes(g, case["n"], case["k"])
        s["sa"] = torch.rand(case["m"], generator=g, device="cuda") * 0.01 + 0.001
        s["sb"] = torch.rand(case["n"], generator=g, device="cuda") * 0.001 + 0.0001
        return s
    page, rows = case["page"], case.get("rows") or case["clients"]
    pages, groups = -(-case["cols"] // page), _groups(page, case["group"])
    # the cache has a few slots more than are used, and its slots are handed out in any order
    slots = rows * pages + 3
    s["slots"] = torch.randperm(slots, generator=g, device="cuda")[: rows * pages].view(rows, pages).to(torch.int32)
    if case["kind"] == "distances":
        s["codes"], s["scales"] = _codes(g, slots, page), torch.rand(slots, groups, generator=g, device="cuda") * 1e-4 + 1e-5
        short = pages * page - case["cols"]
        if short:  # behind the end of an update lie zeros
            s["codes"][s["slots"][:, -1].long(), page - short:] = 0
        return s
    s["codes"] = torch.zeros(slots, page, dtype=torch.int8, device="cuda")
    s["scales"] = torch.zeros(slots, groups, device="cuda")
    s["values"] = _values(g, rows, case["cols"]).to(TYPES[case["dtype"]])
    s["residual"] = s["residual_out"] = s["lengths"] = None
    if case["residual"]:
        s["residual"] = _values(g, rows, case["cols"]).mul_(0.01)
        s["residual_out"] = torch.zeros_like(s["residual"])
    if case["ragged"]:
        lengths = torch.randint(0, case["cols"] + 1, (rows,), generator=g, device="cuda")
        s["lengths"] = (lengths * (torch.rand(rows, generator=g, device="cuda") > 0.1)).to(torch.int32)
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
    return {"cache": _cache, "product": _product, "distances": _distances}[state["kind"]](state)


def _own(s):
    ctx = _context()
    if s["kind"] == "product":
        return ctx.int8_matmul(s["a"], s["b"], s["sa"], s["sb"], dtype=TYPES[s["dtype"]])
    if s["kind"] == "distances":
        return ctx.int8_distances(s["codes"], s["scales"], s["slots"], group=s["group"])
    ctx.quantize_rows(s["values"], s["codes"], s["scales"], group=s["group"], slots=s["slots"], lengths=s["lengths"],
                      residual=s["residual"], residual_out=s["residual_out"])
    out = ctx.dequantize_rows(s["codes"], s["scales"], s["cols"], group=s["group"], slots=s["slots"], dtype=TYPES[s["dtype"]])
    return {"values": out, "scales": s["scales"]} if s["residual"] is None else {"values": out, "scales": s["scales"], "residual": s["residual_out"]}


def _spread(scales, page, group):
    """a scale for every column"""
    return scales.repeat_interleave(group or page, 1)[:, :page]


def _cache(s):
    rows, cols, page, group = s["rows"], s["cols"], s["page"], s["group"]
    pages, groups = -(-cols // page), _groups(page, group)
    t = s["values"].float()
    if s["residual"] is not None:
        t = t + s["residual"]
    if s["lengths"] is not None:
        inside = torch.arange(cols, device=t.device) < s["lengths"][:, None]
        t = torch.where(inside, t, 0.0)
    t = torch.nn.functional.pad(t, (0, pages * page - cols)).view(rows * pages, page)
    t = torch.nn.functional.pad(t, (0, groups * (group or page) - page)).view(rows * pages, groups, group or page)
    most = t.abs().amax(2)
    scale = torch.where(most.isfinite(), most / torch.full_like(most, 127.0), float("nan"))
    # next to a border between two codes 32 bits of the quotient decide wrongly
    code = (t.double() / scale.double()[:, :, None]).round().clamp(-127, 127)
    code = torch.where(scale[:, :, None] > 0, code, 0.0)
    lost = (t.double() - code * scale.double()[:, :, None]).float()
    at = s["slots"].view(-1).long()
    s["codes"][at] = code.view(rows * pages, -1)[:, :page].to(torch.int8)
    s["scales"][at] = scale
    back = s["codes"][at].float() * _spread(s["scales"][at], page, group)
    out = {"values": back.view(rows, pages * page)[:, :cols].to(s["values"].dtype), "scales": s["scales"]}
    if s["residual"] is not None:
        lost = lost.view(rows * pages, -1)[:, :page].reshape(rows, pages * page)[:, :cols]
        out["residual"] = lost if s["lengths"] is None else torch.where(inside, lost, s["residual_out"])
        s["residual_out"].copy_(out["residual"])
    return out


def _product(s):
    # the partial sums of such codes stay below 2^24, where 32 bits hold them exactly
    total = s["a"].float() @ s["b"].float().T
    return (total * s["sa"][:, None] * s["sb"]).to(TYPES[s["dtype"]])


def _distances(s):
    at = s["slots"].view(-1).long()
    x = s["codes"][at].double() * _spread(s["scales"][at].double(), s["page"], s["group"])
    x = x.view(s["clients"], -1)
    dot = x @ x.T
    norm = dot.diagonal()
    return (norm[:, None] + norm - 2 * dot).clamp_min_(0).fill_diagonal_(0)


def work(case):
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + TYPES[case["dtype"]].itemsize * m * n, "flops": 2 * m * n * k}
    rows, cols = case.get("rows") or case["clients"], case["cols"]
    pages = -(-cols // case["page"])
    scales = 4 * rows * pages * _groups(case["page"], case["group"])
    if case["kind"] == "distances":
        return {"bytes": rows * cols + scales + 8 * rows * rows, "flops": rows * (rows + 1) * cols}
    # values in and, rounded, out again; their codes and scales into the cache; the residual in and out.  Ragged rows are half full
    # on average, of the values and the residual that are read as of the residual that is written
    item, full = TYPES[case["dtype"]].itemsize, 0.45 if case["ragged"] else 1.0
    size = full * item + item + 1 + (full * 8 if case["residual"] else 0)
    return {"bytes": rows * cols * size + scales, "flops": 4 * rows * cols}


def exact(case, seed):
    """from the definitions, in 64 bits; row by row where that is another way"""
    s = prepare(case, seed)
    if case["kind"] == "product":
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        b = s["b"].double() * s["sb"].double()[:, None]
        for i in range(0, case["m"], 1024):
            out[i:i + 1024] = torch.einsum("mk,nk->mn", s["a"][i:i + 1024].double() * s["sa"][i:i + 1024].double()[:, None], b)
        return out
    page = case["page"]
    size = case["group"] or page
    if case["kind"] == "distances":
        n = case["clients"]
        out = torch.zeros(n, n, dtype=torch.float64, device="cuda")
        column = torch.arange(page, device="cuda") // size
        for p in range(s["slots"].shape[1]):
            at = s["slots"][:, p].long()
            x = s["codes"][at].double() * s["scales"][at].double()[:, column]
            for i in range(n):
                out[i] += (x - x[i]).square().sum(1)
        return out
    rows, cols = case["rows"], case["cols"]
    values = torch.empty(rows, cols, dtype=torch.float64, device="cuda")
    scales = torch.zeros(s["scales"].shape, dtype=torch.float64, device="cuda")
    residual = torch.zeros(rows, cols, dtype=torch.float64, device="cuda")
    lengths = [cols] * rows if s["lengths"] is None else s["lengths"].tolist()
    for i in range(rows):
        t = s["values"][i].double()
        if s["residual"] is not None:  # the sum that is quantised is a 32-bit number
            t = (t + s["residual"][i].double()).float().double()
        t[lengths[i]:] = 0
        column = torch.arange(cols, device="cuda")
        column = column // page * _groups(page, case["group"]) + column % page // size
        most = torch.zeros(s["scales"].shape[1] * s["slots"].shape[1], dtype=torch.float64, device="cuda")
        most.scatter_reduce_(0, column, t.abs(), "amax")
        scale = most / torch.full_like(most, 127.0)
        scales[s["slots"][i].long()] = scale.view(s["slots"].shape[1], -1)
        held = scale.float().double()[column]  # the cache holds 32 bits of it
        code = torch.where(held > 0, (t / held).round(), 0.0)
        values[i] = code * held
        residual[i] = t - code * held
    return {"values": values, "scales": scales} if s["residual"] is None else {"values": values, "scales": scales, "residual": residual}
