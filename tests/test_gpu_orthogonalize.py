"""Accuracy of optim.orthogonalize on the spectra that updates have, against the same iteration in 64 bits.

Limits.  The kernel holds every operand in 22 bits where float32 has 24: four times the rounding, and it rounds both operands of a
product and drops a product of their remainders where float32 rounds the result (three in quadrature, less than twice).
The iteration amplifies either's errors alike: at most 8 times what the plain form loses in float32 (or 8 half steps of 22 bits).
A result x^ that is off by d is rounded to the nearest bf16, so |round(x^) - x^| <= |round(x) - x^| and with that
|round(x^) - x| <= |round(x) - x| + 2 d: no more than the exact result's own rounding and twice the float32 error."""
import pytest
import torch

from _dvae_pkg import dvae_amd
from test_gpu_muon import off, plain

O = dvae_amd.optim
pytestmark = pytest.mark.gpu


def matrix(shape, kind, seed):
    """on the device, float32: `kind` is how the singular values lie"""
    m, n = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    noise = torch.randn(m, n, generator=g, device="cuda")
    if isinstance(kind, int):  # four directions that many times above the noise
        u, v = (torch.linalg.qr(torch.randn(k, min(4, m, n), generator=g, device="cuda"))[0] for k in shape)
        return noise + kind * (m ** 0.5 + n ** 0.5) * (u @ v.t())
    least = min(m, n)
    u, v = (torch.linalg.qr(torch.randn(k, least, generator=g, device="cuda", dtype=torch.float64))[0] for k in shape)
    k = torch.arange(1, least + 1, device="cuda", dtype=torch.float64)
    s = {"equal": torch.ones_like(k), "falling": k ** -0.5, "two": torch.where(k <= least // 2, 1.0, 1 / 300)}[kind]
    return ((u * s) @ v.t()).float()


def float32_error(m, want):
    return max(off(plain(m, dtype=torch.float32), want.cpu()), 2.0 ** -22)


def within_rounding(got, m, what):
    want = plain(m)
    limit = off(want.to(got.dtype), want.cpu()) + 2 * 8 * float32_error(m, want)
    assert off(got, want.cpu()) <= limit, (what, off(got, want.cpu()), limit)


@pytest.mark.parametrize("shape", [(512, 512), (600, 640), (700, 520), (1400, 1500), (2300, 2500)])
@pytest.mark.parametrize("kind", [30, "equal", "falling", "two"])
def test_large_bf16_matrices_have_float32_accuracy(shape, kind):
    """unless the caller asks for less"""
    if isinstance(kind, str) and max(shape) > 1000:
        shape = (shape[0] // 2, shape[1] // 2)
    m = matrix(shape, kind, 1).bfloat16()
    within_rounding(O.orthogonalize(m), m, "alone")


def test_accuracy_does_not_depend_on_the_other_matrices_or_their_order():
    mats = [matrix((600, 640), "equal", k).bfloat16() for k in range(2)] + [matrix((40, 700), 0, 2).bfloat16()] * 33
    for order in (mats, mats[::-1], mats[:2]):
        for m, o in zip(order, O.orthogonalize(order)):
            if m.shape[0] == 600:
                within_rounding(o, m, len(order))


@pytest.mark.parametrize("shape", [(512, 512), (900, 640), (640, 900), (2300, 2500), (3200, 3205), (4096, 4096), (5600, 5630)])
@pytest.mark.parametrize("times", [0, 30, 300])
def test_half_products_keep_the_small_directions(shape, times):
    """Limit as derived for one plane in test_orthogonalize_large: five steps of 8 times the rounding of 11 bits (r.m.s.) and the
    result's rounding.  Were the second plane of X lost, directions of 30 times the noise would cost 8.7e-3 and of 300 3.7e-2."""
    m = matrix(shape, times, 3).bfloat16()
    want = plain(m)
    got = O.orthogonalize(m, products="half")
    assert float((got.double() - want).norm() / want.norm()) < 40 * 2.0 ** -12 / 3 ** 0.5 + 2.0 ** -9


def test_half_products_look_at_each_matrix_alone():
    """a small matrix among large ones keeps full products, and takes none from them; more than one launch group of either"""
    large, small = matrix((512, 530), 30, 4).bfloat16(), matrix((9, 1), 0, 5).bfloat16()
    alone = O.orthogonalize(large, products="half")
    mixed = O.orthogonalize([small, large] * 34, products="half")
    want = plain(large)
    for o in mixed[1::2]:
        assert off(o, want.cpu()) < 40 * 2.0 ** -12 / 3 ** 0.5 + 2.0 ** -9
    assert off(alone, want.cpu()) < 40 * 2.0 ** -12 / 3 ** 0.5 + 2.0 ** -9
    for o in mixed[::2]:
        within_rounding(o, small, "small")
    full = O.orthogonalize([small, large] * 34)
    assert all(torch.equal(a, b) for a, b in zip(mixed[::2][:32], O.orthogonalize([small] * 32)))
    for o in full[1::2]:
        within_rounding(o, large, "large")


def test_half_products_are_for_bf16_and_asked_for_by_name():
    m = torch.randn(520, 520, device="cuda")
    for bad in ((m, "half"), (m.half(), "half"), (m.bfloat16(), "fast"), (m, None)):
        with pytest.raises(ValueError, match="products"):
            O.orthogonalize(bad[0], products=bad[1])
    turned = m.bfloat16().t()
    assert torch.equal(O.orthogonalize(turned, products="half"), O.orthogonalize(turned.contiguous(), products="half"))


@pytest.mark.parametrize("shape", [(70, 100), (100, 70), (8, 33), (300, 200), (513, 600)])
@pytest.mark.parametrize("kind", ["scaled up", "scaled down", "rank one", "strided", "falling"])
def test_float32_accuracy_of_special_inputs(shape, kind):
    m = matrix(shape, "falling" if kind == "falling" else 0, 6)
    if kind == "rank one":
        m = torch.outer(m[:, 0], m[0])
    elif kind.startswith("scaled"):
        m = m * (1e30 if kind == "scaled up" else 1e-30)
    given = m
    if kind == "strided":
        hole = torch.zeros(shape[0] + 2, shape[1] + 5, device="cuda")
        hole[1:-1, 3:-2] = m
        given = hole[1:-1, 3:-2]
    want = plain(m)
    got = off(O.orthogonalize(given), want.cpu())
    assert got <= 8 * float32_error(m, want), (got, float32_error(m, want))
    one = plain(m, 1)
    got = off(O.orthogonalize(given, steps=1), one.cpu())
    assert got <= 8 * max(off(plain(m, 1, dtype=torch.float32), one.cpu()), 2.0 ** -22), got


def test_outputs_in_the_place_of_other_inputs():
    """more matrices than one launch group holds: what a later group reads is not overwritten by an earlier one's outputs"""
    g = torch.Generator().manual_seed(7)
    buffer = torch.randn(60, 20, 33, generator=g).cuda()
    want = O.orthogonalize([m.clone() for m in buffer])
    for shift in (0, 5, 59):
        mine = buffer.clone()
        O.orthogonalize(list(mine), out=[mine[(k + shift) % 60] for k in range(60)])
        assert torch.equal(mine, torch.stack([want[(k - shift) % 60] for k in range(60)])), shift
    mine = buffer[:40].clone().view(40 * 20, 33)  # rows of two matrices in turn, in one range of addresses
    pairs = [mine[40 * k + b:40 * k + 40:2] for k in range(20) for b in (0, 1)]
    want = O.orthogonalize([p.clone() for p in pairs])
    O.orthogonalize(pairs, out=pairs)
    assert all(torch.equal(a, b) for a, b in zip(pairs, want))
    large, small = torch.randn(512, 512, generator=g).bfloat16().cuda(), torch.randn(512, 511, generator=g).bfloat16().cuda()
    mine = torch.cat([large, small], 1)  # the small one's group is launched first, and writes where the large one begins
    want = O.orthogonalize([large, small], products="half")
    O.orthogonalize([mine[:, :512], mine[:, 512:]], out=[mine[:, 511:], mine[:, :511]], products="half")
    assert torch.equal(mine[:, 511:], want[0]) and torch.equal(mine[:, :511], want[1])


LARGE = [(1312, 1785), (619, 1766), (790, 578), (500, 542)]
LONG_SETS = [[(9, 1883)] + LARGE, [(9, 1883), (17, 690), (11, 267), (30, 1500), (8, 2048), (56, 501), (64, 2000), (100, 2000)] + LARGE,
             [(9, 20000), (40, 9000), (100, 20000), (300, 20000)] + LARGE, [(300, 8192)] * 32, [(250, 4000)] * 32,
             [(2048, 2048)] * 2 + [(9, 1883), (30, 2000), (2000, 9), (384, 3000), (385, 3000)], [(4096, 4096), (9, 1883)], [(9, 20000)], [(300, 20000)]]


@pytest.mark.parametrize("k", range(len(LONG_SETS)))
def test_few_rows_with_long_sums_keep_float32_accuracy_in_every_set(k):
    """An entry of X X^T is a sum over a whole row, and where there are few rows its rounding is not averaged over many: added up
    one by one in float32 it was up to 3.6 times as far off as the float32 iteration, in some sets.  Its parts are summed
    apart; half as much again as the float32 iteration loses is allowed, or 16 of its half steps."""
    for seed in range(2):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        for kind in ("noise", "spiked"):
            mats = [torch.randn(m, n, generator=g, device="cuda") for m, n in LONG_SETS[k]]
            if kind == "spiked":
                mats = [a + 3 * torch.randn(a.shape[0], 4, generator=g, device="cuda") @ torch.randn(4, a.shape[1], generator=g, device="cuda") for a in mats]
            for m, o in list(zip(mats, O.orthogonalize(mats)))[:8]:
                want = plain(m).cpu()
                got, mine = off(o, want), off(plain(m, dtype=torch.float32), want)
                assert got <= max(1.5 * mine, 2.0 ** -20), (kind, tuple(m.shape), got, mine)


@pytest.mark.parametrize("shape", [(1, 40), (3, 50), (8, 80), (9, 84), (16, 300), (64, 90), (65, 90), (600, 12)])
def test_few_rows_with_other_coefficients(shape):
    """B of up to 64 rows is held shifted, unless the coefficients leave no room for that (the last two sets, whose singular values
    stay below 1); limits as at the head of the file"""
    m = matrix(shape, 0, 8)
    for abc, steps in (((1.5, -0.5, 0.0), 3), ((2.0, -1.5, 0.5), 8), ([(3.4445, -4.7750, 2.0315), (2.0, -1.5, 0.5)], 2), ((1.0, 0.0, 0.0), 2),
                       ([(0.5, 0.0, 0.0), (3.8, -6.8, -1.3)], 2), ([(0.4, 0.0, 0.0), (1.36, 7.15, 2.38), (1.5, -0.5, 0.0)], 3)):
        want = plain(m, steps, abc).cpu()
        for given in ([m], [m] + [matrix((200, 300), 0, k) for k in range(9)]):  # by itself and on larger tiles
            got = O.orthogonalize(given, steps=steps, coefficients=abc)[0]
            assert off(got, want) <= 8 * max(off(plain(m, steps, abc, dtype=torch.float32), want), 2.0 ** -22), (abc, len(given))
