"""The encrypted and the plaintext driver on 8-bit updates: a run of cache, product, distances and encryption as a program uses them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SLOTS = 12


@pytest.fixture(scope="module")
def ek():
    from lancelot_b200.krum import EncryptedKrum

    return EncryptedKrum(log_slots=SLOTS, seed=7, encrypt_batch=16)


def updates(n, dim, seed):
    import torch

    return torch.randn(n, dim, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * 1e-2


@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("dim", [3 << SLOTS, (3 << SLOTS) + 77, 100])
def test_a_round_on_cached_updates_is_the_round_on_what_the_cache_holds(ek, dim, group):
    import torch

    from lancelot_b200.krum import plaintext_krum

    n = 5
    x = updates(n, dim, dim + group)
    cache = ek.update_cache(n, dim, group=group)
    cache.write(x[:3], clients=slice(0, 3))
    cache.write(x[3], clients=3)
    cache.write(x[4].double(), clients=4)
    held = cache.read()
    assert held.shape == x.shape
    # every value is held to half a step of its group's scale
    assert float((held - x).abs().max()) <= float(cache.scales.max()) * 0.5 * (1 + 2.0 ** -20)
    got, order = ek.round(cache)
    want, want_order = ek.round(held)
    assert got == want and np.array_equal(order, want_order)  # the same seeds: the same ciphertexts
    d, plain_order = plaintext_krum(cache)
    p, _ = plaintext_krum(held.cpu())
    # codes times a 32-bit scale are rounded to 32 bits in what is read, not in the distances
    assert np.allclose(d, p, rtol=1e-6) and np.array_equal(plain_order, np.argsort(p))
    cts = ek.encrypt_slices(cache, 0, ek.n_chunks(dim))
    assert torch.equal(cts, ek.encrypt_slices(held, 0, ek.n_chunks(dim)))
    if dim > 2 << SLOTS:
        assert torch.equal(ek.encrypt_slices(cache, 1, 3), ek.encrypt_slices(held, 1, 3))


def test_smaller_pages_and_the_point_to_point_feed(ek):
    import torch

    from lancelot_b200.updates import UpdateCache

    dim = (2 << SLOTS) + 1000
    x = updates(3, dim, 1)
    cache = UpdateCache(ek.lb, 3, dim, page=1 << (SLOTS - 2), group=64)
    cache.write(x)
    assert torch.equal(ek.encrypt_slices(cache, 0, 3), ek.encrypt_slices(cache.read(), 0, 3))
    for c, u in ek.staged(cache, [2, 0]):
        assert torch.equal(u, cache.read(c)[0])
    other = UpdateCache(ek.lb, 3, dim, page=96, group=32)
    other.write(x)
    with pytest.raises(ValueError):
        ek.encrypt_slices(other, 0, 3)
    for call in (lambda: cache.read(3), lambda: cache.read(0, 8, 2), lambda: cache.write(x[:2]), lambda: cache.write(x[0, :-1], clients=0)):
        with pytest.raises(ValueError):
            call()


def test_error_feedback_follows_the_sum_of_the_updates(ek):
    import torch

    dim, n = 5000, 2
    cache = ek.update_cache(n, dim)
    residual = torch.zeros(n, dim, device="cuda")
    sent, total = torch.zeros(n, dim, dtype=torch.float64, device="cuda"), torch.zeros(n, dim, dtype=torch.float64, device="cuda")
    for r in range(6):
        x = updates(n, dim, 40 + r)
        cache.write(x, residual=residual, residual_out=residual)
        sent += cache.read().double()
        total += x.double()
    # what was sent and what is still to be sent make up the updates, to the 32-bit roundings of six sums and six values read
    assert float((sent + residual.double() - total).abs().max()) <= 12 * 2.0 ** -24 * 0.1


@pytest.mark.parametrize("rank", [1, 8, 33])
def test_low_rank_updates_are_formed_and_encrypted(ek, rank):
    import torch

    from lancelot_b200.updates import low_rank_update, quantize_matrix

    gen = torch.Generator("cuda").manual_seed(rank)
    factors, want = [], []
    for rows, cols in [(64, 100), (33, 7), (1, 300), (130, 70)]:
        b = torch.randn(rows, rank, generator=gen, device="cuda").to(torch.bfloat16)
        a = torch.randn(cols, rank, generator=gen, device="cuda") * 0.1
        (qb, sb), (qa, sa) = quantize_matrix(ek.lb, b), quantize_matrix(ek.lb, a)
        factors.append((qb, sb, qa, sa))
        # (the integer sum first: scaled terms that cancel to 0 leave 64-bit rounding noise, against which no relative bound holds)
        want.append(((qb.double() @ qa.double().T) * sb.double()[:, None] * sa.double()).reshape(-1))
    got, want = low_rank_update(ek.lb, factors), torch.cat(want)
    assert bool(((got.double() - want).abs() <= want.abs() * 3.1 * 2.0 ** -24).all())
    cts = ek.encrypt_low_rank(factors, client=2)
    assert torch.equal(cts, ek.encrypt_client(got, client=2))
    ek.lb.check_status()
    with pytest.raises(ValueError):
        low_rank_update(ek.lb, factors, out=torch.empty(3, device="cuda"))


def test_factors_without_columns(ek):
    """rank 0: rows of zeros, whatever their memory held before"""
    import torch

    from lancelot_b200.updates import low_rank_update, quantize_matrix

    for dtype in (torch.float32, torch.bfloat16):
        stale = torch.full((1 << 16,), float("nan"), device="cuda")
        del stale
        (qb, sb), (qa, sa) = [quantize_matrix(ek.lb, torch.empty(rows, 0, dtype=dtype, device="cuda")) for rows in (70, 300)]
        assert qb.shape == (70, 0) and qa.shape == (300, 0) and not sb.any() and not sa.any()
        update = low_rank_update(ek.lb, [(qb, sb, qa, sa)])
        assert update.shape == (70 * 300,) and not update.any()
    codes, scales = quantize_matrix(ek.lb, torch.empty(0, 8, device="cuda"))
    assert codes.shape == (0, 8) and scales.shape == (0,)
