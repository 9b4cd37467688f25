"""Norms and clipping on the GPU against plain formulas in 64 bits.

The squares of 32-bit floats are exact in 64 bits, so a norm is off by the roundings of its sum alone: at most n steps of 2^-53 in the sum, and
half of that in the root.  A result is value * factor, both in 32 bits: compared for equality with a factor from the call's own norm."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from lancelot_b200 import cabi

    return cabi.Context(12, cabi.coeff_modulus_create(1 << 12, [40, 40]), 1)


def gen(seed):
    import torch

    return torch.Generator("cuda").manual_seed(seed)


def dt(name):
    import torch

    return getattr(torch, name)


def same(x, y):
    import torch

    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())


def norm_of(tensors):
    import torch

    return torch.cat([t.double().reshape(-1) for t in tensors] + [torch.zeros(1, dtype=torch.float64, device="cuda")]).square().sum().sqrt()


def check_norms(norms, updates):
    for got, tensors in zip(norms.tolist(), updates):
        want = norm_of(tensors).item()
        assert abs(got - want) <= want * 2.0 ** -53 * (sum(t.numel() for t in tensors) + 4)


def factor(norm, most):
    """as the definition has it: in 64 bits, rounded to 32"""
    import numpy as np

    return float(np.float32(most / norm)) if norm > most else 1.0 if math.isfinite(norm) else math.nan


def clipped(t, f, dtype=None):
    return (t.float() * f).to(dtype or t.dtype)


def make(g, sizes, dtype, scale=1.0):
    import torch

    return [(torch.randn(n, generator=g, device="cuda") * scale).to(dt(dtype)) for n in sizes]


LAYOUTS = [[[1]], [[0]], [[5, 0, 3]], [[1000, 17, 4096, 1], [1, 4096, 17, 1000]], [[40000, 3, 70001]] * 3, [[300001]], [[12, 50000]] * 40]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("into", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("case", range(len(LAYOUTS)))
def test_norms_and_rows(ctx, dtype, into, case):
    import torch

    g = gen(case)
    updates = [make(g, sizes, dtype, 0.5 + i) for i, sizes in enumerate(LAYOUTS[case])]
    dim = sum(LAYOUTS[case][0])
    kept = [[t.clone() for t in tensors] for tensors in updates]
    norms = ctx.clip_updates(updates)
    assert norms.dtype == torch.float64 and norms.shape == (len(updates),)
    check_norms(norms, updates)
    for most in (norms.max().item() * 0.4, norms.max().item() * 2, 0.0, math.inf, None):
        room = torch.full((len(updates), dim + 3), 9.0, dtype=dt(into), device="cuda")
        out = room[:, 1:1 + dim]
        again = ctx.clip_updates(updates, most, out=out)
        assert torch.equal(norms, again)
        for i, tensors in enumerate(updates):
            f = factor(norms[i].item(), math.inf if most is None else most)
            want = torch.cat([clipped(t, f, dt(into)) for t in tensors])
            assert same(out[i], want), (most, i)
        assert bool((room[:, 0] == 9).all() and (room[:, 1 + dim:] == 9).all())
    for tensors, before in zip(updates, kept):
        assert all(torch.equal(t, b) for t, b in zip(tensors, before))
    most = norms.max().item() * 0.5
    ctx.clip_updates(updates, most)
    for i, (tensors, before) in enumerate(zip(updates, kept)):
        f = factor(norms[i].item(), most)
        assert all(torch.equal(t, clipped(b, f)) for t, b in zip(tensors, before))


def test_a_matrix_of_updates_and_tensors_of_several_types(ctx):
    import torch

    g = gen(1)
    m = torch.randn(7, 5003, generator=g, device="cuda")
    rows = m[:, 1:5002]
    norms = ctx.clip_updates(rows)
    check_norms(norms, [[r] for r in rows])
    before = m.clone()
    ctx.clip_updates(rows, norms[3].item() * 0.7)
    for i in range(7):
        assert torch.equal(rows[i], clipped(before[i, 1:5002], factor(norms[i].item(), norms[3].item() * 0.7)))
    assert torch.equal(m[:, 0], before[:, 0]) and torch.equal(m[:, 5002:], before[:, 5002:])
    mixed = [make(g, [1000], "float32") + make(g, [33, 4000], "bfloat16") + make(g, [77], "float16")]
    mixed[0].append(torch.randn(30, 40, generator=g, device="cuda").t())  # dense in another order
    mixed[0].append(torch.randn(4, 3, 8, 8, generator=g, device="cuda").to(memory_format=torch.channels_last))
    before = [t.clone() for t in mixed[0]]
    norms = ctx.clip_updates(mixed, 10.0)
    check_norms(norms, [before])
    f = factor(norms[0].item(), 10.0)
    assert f < 1 and all(torch.equal(t, clipped(b, f)) for t, b in zip(mixed[0], before))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_tensors_off_their_alignment(ctx, dtype):
    import torch

    g = gen(2)
    for a in range(5):
        store = [torch.randn(n + 16, generator=g, device="cuda").to(dt(dtype)) for n in (2049, 70007, 13)]
        tensors = [s[a:a + n] for s, n in zip(store, (2049, 70007, 13))]
        before = [s.clone() for s in store]
        norms = ctx.clip_updates([tensors], 5.0)
        check_norms(norms, [[b[a:a + n] for b, n in zip(before, (2049, 70007, 13))]])
        f = factor(norms[0].item(), 5.0)
        for s, b, n in zip(store, before, (2049, 70007, 13)):
            b[a:a + n] = clipped(b[a:a + n], f)
            assert torch.equal(s, b)


def test_clients_without_values_and_without_tensors(ctx):
    import torch

    z, x, y = torch.zeros(0, device="cuda"), torch.ones(16, device="cuda"), torch.ones(16, device="cuda")
    assert ctx.clip_updates([]).shape == (0,)
    assert ctx.clip_updates([[], [x], [z], [z, y, z], []], 1.0).tolist() == [0, 4, 0, 4, 0]
    assert bool((x == 0.25).all() and (y == 0.25).all())
    assert ctx.clip_updates(torch.zeros(3, 0, device="cuda"), 1.0).tolist() == [0, 0, 0]


def test_updates_that_are_made_on_access(ctx):
    """nobody but the call holds the tensors: their memory is not for its scratch and its results"""
    import torch

    class Made:
        def __init__(self, make, n):
            self.make, self.n = make, n

        def __len__(self):
            return self.n

        def __getitem__(self, i):
            if i >= self.n:
                raise IndexError(i)
            return self.make(i)

    sizes = [3, 64, 40, 70001]  # some of the size of the norms and the scratch
    base = [torch.randn(sum(sizes), generator=gen(20 + c), device="cuda") for c in range(8)]
    at = [sum(sizes[:i]) for i in range(5)]
    plain = [[b[x:y] for x, y in zip(at, at[1:])] for b in base]
    box = []

    def refill(c):  # the same list for every client
        box[:] = [t.clone() for t in plain[c]]
        return box

    for updates in (Made(lambda c: Made(lambda i: plain[c][i] * 1, 4), 8), Made(refill, 8)):
        norms = ctx.clip_updates(updates)
        assert torch.equal(norms, ctx.clip_updates(plain))
        out = torch.empty(8, sum(sizes), device="cuda")
        assert torch.equal(ctx.clip_updates(updates, 200.0, out=out), norms)
        for o, b, norm in zip(out, base, norms.tolist()):
            assert torch.equal(o, clipped(b, factor(norm, 200.0)))


def test_values_that_are_not_finite_large_and_small(ctx):
    import torch

    big = torch.full((5000,), 3e38, device="cuda")
    small = torch.full((5000,), 2.0 ** -149, device="cuda")
    bad = torch.ones(5000, device="cuda")
    bad[77] = math.nan
    worse = torch.ones(5000, device="cuda")
    worse[4999] = -math.inf
    fine = torch.full((5000,), 0.5, device="cuda")
    zero = torch.zeros(5000, device="cuda")
    updates = [[big], [small], [bad, fine.clone()], [worse, fine.clone()], [fine], [zero]]
    before = [[t.clone() for t in tensors] for tensors in updates]
    norms = ctx.clip_updates(updates, 1.0)
    check_norms(norms[[0, 1, 4, 5]], [before[i] for i in (0, 1, 4, 5)])
    assert math.isnan(norms[2].item()) and norms[3].item() == math.inf
    assert all(bool(t.isnan().all()) for i in (2, 3) for t in updates[i])  # throughout: the other tensors of the client too
    for i in (0, 1, 4, 5):
        assert torch.equal(updates[i][0], clipped(before[i][0], factor(norms[i].item(), 1.0)))
    assert updates[0][0].isfinite().all() and updates[0][0][0] > 0


def test_more_tensors_than_one_launch_holds(ctx):
    import torch

    g = gen(3)
    updates = [make(g, [1 + (i * 7 + c) % 50 for i in range(211)], "float32", 1 + c) for c in range(9)]
    updates.append(make(g, [2000] * 1000, "bfloat16"))
    before = [[t.clone() for t in tensors] for tensors in updates]
    norms = ctx.clip_updates(updates, 100.0)
    check_norms(norms, before)
    for i in range(10):
        f = factor(norms[i].item(), 100.0)
        assert all(torch.equal(t, clipped(b, f)) for t, b in zip(updates[i], before[i]))


ROUNDS = {"by count": (5, [3 + i * 37 % 91 for i in range(150)], "float32"), "by count, 16 bits": (7, [1 + i * 53 % 701 for i in range(201)], "bfloat16"),
          "by bytes": (4, [9999999, 1, 77, 123457], "float32"), "by bytes, 16 bits": (5, [17000003, 5, 2999], "float16"),
          "one client a round": (3, [26000001, 13], "float32"), "clients of more tensors than a launch holds": (3, [5 + i % 7 for i in range(700)], "float32")}


@pytest.mark.parametrize("case", sorted(ROUNDS))
@pytest.mark.parametrize("bad", [None, 2])
def test_several_rounds_of_clients(ctx, case, bad):
    """results of some clients are written while the next ones are summed up: in place, as rows of either width, norms alone"""
    import torch

    clients, sizes, dtype = ROUNDS[case]
    g = gen(40)
    base = [make(g, sizes, dtype, 0.01 * (1 + c)) for c in range(clients)]
    if bad is not None:
        base[bad][len(sizes) // 2][0] = math.inf
    # every tensor lies somewhere else between two boundaries of 16 bytes, in memory that is otherwise left as it was
    pads = [[(i + c) % 9 for i in range(len(sizes))] for c in range(clients)]

    def laid_out():
        held = [[torch.full((n + 16,), 3.0, dtype=dt(dtype), device="cuda") for n in sizes] for _ in range(clients)]
        views = [[h[p:p + n] for h, p, n in zip(hs, ps, sizes)] for hs, ps in zip(held, pads)]
        for vs, bs in zip(views, base):
            for v, b in zip(vs, bs):
                v.copy_(b)
        return held, views

    held, views = laid_out()
    norms = ctx.clip_updates(views)
    good = [c for c in range(clients) if c != bad]
    check_norms(norms[good], [base[c] for c in good])
    assert bad is None or norms[bad].item() == math.inf
    most = norms[good].median().item()
    factors = [math.nan if c == bad else factor(norms[c].item(), most) for c in range(clients)]
    dim = sum(sizes)
    for into in ("float32", dtype):
        want = torch.stack([torch.cat([clipped(b, f, dt(into)) for b in bs]) for bs, f in zip(base, factors)])
        for _ in range(3):
            room = torch.full((clients, dim + 5), 9.0, dtype=dt(into), device="cuda")
            assert torch.equal(ctx.clip_updates(views, most, out=room[:, 2:2 + dim]), norms)
            assert same(room[:, 2:2 + dim], want)
            assert bool((room[:, :2] == 9).all() and (room[:, 2 + dim:] == 9).all())
        del want, room
    for _ in range(2):
        assert torch.equal(ctx.clip_updates(views, most), norms)
        for vs, hs, bs, ps, f in zip(views, held, base, pads, factors):
            for v, h, b, p in zip(vs, hs, bs, ps):
                assert same(v, clipped(b, f))
                assert bool((h[:p] == 3).all() and (h[p + v.numel():] == 3).all())
        held, views = laid_out()


def test_rounds_in_a_captured_graph(ctx):
    import torch

    clients, sizes, dtype = ROUNDS["by count"]
    g = gen(41)
    updates = [make(g, sizes, dtype, 1 + c) for c in range(clients)]
    out = torch.empty(clients, sum(sizes), device="cuda")
    ctx.clip_updates(updates, 100.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = ctx.clip_updates(updates, 100.0, out=out)
    for seed in (1, 2):
        for ts in updates:
            for t in ts:
                t.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), norms.clone()
        want = torch.empty_like(out)
        assert torch.equal(ctx.clip_updates(updates, 100.0, out=want), got[1]) and torch.equal(got[0], want)


def test_norms_of_more_clients_than_one_launch_holds(ctx):
    import torch

    m = torch.randn(4321, 37, generator=gen(42), device="cuda")
    norms = ctx.clip_updates(m)
    want = m.double().square().sum(1).sqrt()
    assert bool(((norms - want).abs() <= want * 2.0 ** -53 * 41).all())
    out = torch.empty_like(m)
    assert torch.equal(ctx.clip_updates(m, 6.0, out=out), norms)
    f = torch.where(norms > 6.0, 6.0 / norms, torch.ones_like(norms)).float()
    assert torch.equal(out, m * f[:, None])


def test_the_same_result_every_time_and_on_two_streams(ctx):
    import torch

    g = gen(4)
    updates = [make(g, [11, 300000, 1000001], "float32", 1 + i) for i in range(5)]
    outs, norms = [], []
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            out = torch.empty(5, 1300012, device="cuda")
            norms.append(ctx.clip_updates(updates, 700.0, out=out))
            outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(norms[0], n) for n in norms) and all(torch.equal(outs[0], o) for o in outs)


def test_updates_past_32_bit_sizes(ctx):
    import torch

    n = (1 << 31) + 12345
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[-3:] = 4.0
    t[0] = 4.0
    norms = ctx.clip_updates([[t]], 1.0)
    assert norms.item() == 8.0
    assert t[-3:].tolist() == [0.5] * 3 and t[0].item() == 0.5 and not t[1:-3].any()


def test_what_the_call_refuses(ctx):
    import torch

    from lancelot_b200._lib import InvalidArgument

    x, y = torch.ones(40, device="cuda"), torch.ones(2, 40, device="cuda")
    out = torch.empty(2, 40, device="cuda")
    for call in (lambda: ctx.clip_updates([x]),
                 lambda: ctx.clip_updates([[1.0]]),
                 lambda: ctx.clip_updates(5),
                 lambda: ctx.clip_updates([[x.double()]]),
                 lambda: ctx.clip_updates([[x.cpu()]]),
                 lambda: ctx.clip_updates([[x]], -1.0),
                 lambda: ctx.clip_updates([[x]], math.nan),
                 lambda: ctx.clip_updates([[x[::2]]], 1.0),
                 lambda: ctx.clip_updates([[x], [x]], 1.0),
                 lambda: ctx.clip_updates([[x[:30], x[20:]]], 1.0),
                 lambda: ctx.clip_updates([[x]], 1.0, out=out),
                 lambda: ctx.clip_updates([[x], [x[:39]]], 1.0, out=out),
                 lambda: ctx.clip_updates([[x], []], 1.0, out=out),
                 lambda: ctx.clip_updates([[x], [x]], 1.0, out=out.double()),
                 lambda: ctx.clip_updates([[x], [x]], 1.0, out=out[0]),
                 lambda: ctx.clip_updates([[x], [x]], 1.0, out=out[:1].expand(2, 40)),
                 lambda: ctx.clip_updates([[y.t()], [y.t()]], 1.0, out=torch.empty(2, 80, device="cuda")),
                 lambda: ctx.clip_updates([[out[1]], [x]], 1.0, out=out),
                 lambda: ctx.clip_updates(y[:1].expand(2, 40), 1.0)):
        with pytest.raises(InvalidArgument):
            call()
    assert bool((x == 1).all())
    # what is only read may come twice, and an update may lie in its own row of the result
    assert torch.equal(ctx.clip_updates([[x], [x, x]]), torch.tensor([40.0, 80.0], dtype=torch.float64, device="cuda").sqrt())
    ctx.clip_updates([[x], [x]], 1.0, out=out)
    kept = out.clone()
    ctx.clip_updates([[out[0]], [out[1]]], 0.5, out=out)
    assert torch.equal(out, clipped(kept, factor(norm_of([kept[0]]).item(), 0.5)))


def test_a_federation_from_training_to_selection(ctx):
    """clients train a layer in 8-bit floating point, their gradients become bounded rows, the rows are cached in 8 bits and compared"""
    import torch

    from lancelot_b200 import updates
    from lancelot_b200.krum import plaintext_krum

    g = gen(5)
    w0, bias0 = torch.randn(40, 120, generator=g, device="cuda") * 0.1, torch.zeros(40, device="cuda")
    data = torch.randn(6, 64, 120, generator=g, device="cuda")
    target = torch.randn(40, 120, generator=g, device="cuda") * 0.1
    found = []
    for c in range(6):
        w, bias = w0.clone().requires_grad_(), bias0.clone().requires_grad_()
        loss = (updates.fp8_linear(ctx, data[c], w) + bias - data[c] @ target.t()).square().mean()
        found.append(list(torch.autograd.grad(loss, (w, bias))))
    found[4] = [t * -1000 for t in found[4]]  # an attacker
    flat, norms = updates.flat_updates(ctx, found, max_norm=2 * sorted(norm_of(f).item() for f in found)[2])
    check_norms(norms, found)
    assert flat.shape == (6, 40 * 121) and flat.dtype == torch.float32
    assert norm_of([flat[4]]).item() <= 2 * sorted(norms.tolist())[2] * (1 + 1e-6)
    cache = updates.UpdateCache(ctx, 6, flat.shape[1], page=4096)
    cache.write(flat)
    plain, cached = plaintext_krum(flat), plaintext_krum(cache)
    assert int(plain[1][-1]) == int(cached[1][-1]) == 4
