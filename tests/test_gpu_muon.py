"""Orthogonalised updates (optim.orthogonalize, optim.FlatMuon) against the same iteration in 64 bits.

Tolerances of the iteration.  Every product holds its operands in two fp16 planes (22 bits: 2^-22 of an entry of theirs),
drops 2^-22 and accumulates in fp32; a step has three of them, so that its own error is at most 16 * 2^-22 of |X| (Frobenius; A and
B are at most 4 and 2 |X|).  An error in X grows by at most sup |p'| <= 4 on [0, 1.2] a step: with five steps 341 times."""
import math

import pytest
import torch

from _dvae_pkg import dvae_amd

O = dvae_amd.optim
pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def plain(g, steps=5, abc=(3.4445, -4.7750, 2.0315), dtype=torch.float64):
    x = g.to(dtype)
    turned = x.shape[0] > x.shape[1]
    x = x.t() if turned else x
    x = x / (g.double().norm().to(dtype) if g.any() else 1.0)
    for t in range(steps):
        a, b, c = abc[t] if hasattr(abc[0], "__len__") else abc
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if turned else x


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


SETS = [[(1, 1)], [(1, 7)], [(9, 1)], [(5, 3), (64, 64), (65, 63)], [(501, 501)], [(56, 501), (501, 56), (8, 1002), (130, 300)],
        [(300, 40)] * 40, [(1100, 1300), (2000, 700), (64, 3000), (129, 128)]]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("k", range(len(SETS)))
def test_orthogonalize(dtype, k):
    dt, g = DT[dtype], gen(k)
    mats = [(torch.randn(m, n, generator=g) * 10.0 ** (i % 5 - 2)).to(dt) for i, (m, n) in enumerate(SETS[k])]
    outs = O.orthogonalize([m.cuda() for m in mats])
    for m, o in zip(mats, outs):
        want = plain(m)
        assert o.shape == m.shape and o.dtype == dt
        assert off(o, want) < 341 * 16 * 2.0 ** -22 + torch.finfo(dt).eps / 2, (m.shape, off(o, want))
        if dt == torch.float32 and min(m.shape) > 1:
            # 22 bits against 24: within four times of what the plain form loses in float32, or of a rounding of the result
            assert off(o, want) < 4 * max(off(plain(m, dtype=torch.float32), want), 2.0 ** -22)
    again = O.orthogonalize([m.cuda() for m in mats])
    assert all(torch.equal(a, b) for a, b in zip(outs, again))


def test_orthogonalize_makes_singular_values_near_one():
    m = torch.randn(200, 333, generator=gen(1)).cuda()
    s = torch.linalg.svdvals(O.orthogonalize(m).double().cpu())
    assert s.min() > 0.65 and s.max() < 1.25  # where five steps of these coefficients take [0.002, 1]


def test_orthogonalize_one_step_and_other_coefficients():
    m = torch.randn(150, 90, generator=gen(2))
    for abc, steps in (((1.5, -0.5, 0.0), 1), ((2.0, -1.5, 0.5), 12), ([(3.4445, -4.7750, 2.0315)] * 2 + [(2.0, -1.5, 0.5)] * 3, 5)):
        got, want = O.orthogonalize(m.cuda(), steps=steps, coefficients=abc), plain(m, steps, abc)
        growth = sum(4 ** i for i in range(steps)) if steps <= 5 else 341 * 16  # the convergent sets: sup |p'| <= 2, 1 near 1
        assert off(got, want) < growth * 16 * 2.0 ** -22


def test_orthogonalize_extremes():
    g = gen(3)
    base = torch.randn(70, 100, generator=g)
    want = plain(base)
    for scale in (1e-30, 1e30):  # no range of the input overflows or vanishes
        assert off(O.orthogonalize((base * scale).cuda()), plain(base * scale)) < 341 * 16 * 2.0 ** -22
    zero = O.orthogonalize([torch.zeros(70, 100).cuda(), base.cuda()])
    assert not zero[0].any() and off(zero[1], want) < 341 * 16 * 2.0 ** -22
    for bad in (float("nan"), float("inf")):
        m = base.clone()
        m[3, 5] = bad
        got = O.orthogonalize([m.cuda(), base.cuda()])
        assert torch.isnan(got[0]).all() and torch.equal(got[1], O.orthogonalize(base.cuda()))
    rank1 = torch.outer(torch.randn(300, generator=g), torch.randn(200, generator=g))
    assert off(O.orthogonalize(rank1.cuda()), plain(rank1)) < 341 * 16 * 2.0 ** -22


def test_orthogonalize_strides_and_outputs():
    g = gen(4)
    big = torch.randn(120, 400, generator=g).cuda()
    view, turned = big[3:90, 7:207], big.t()
    want = O.orthogonalize([view.contiguous(), turned.contiguous()])
    got = O.orthogonalize([view, turned])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    hole = torch.zeros(120, 400, device="cuda")
    back = O.orthogonalize(view, out=hole[3:90, 7:207])
    assert back.data_ptr() == hole[3:90, 7:207].data_ptr() and torch.equal(hole[3:90, 7:207], want[0])
    hole[3:90, 7:207] = 0
    assert not hole.any()  # nothing beside it was written
    mine = [view.clone(), view.clone() * 3]
    O.orthogonalize(mine, out=mine)
    assert torch.equal(mine[0], want[0])


def test_orthogonalize_captured_and_replayed():
    g = gen(5)
    mats = [torch.randn(s, generator=g).cuda() for s in ((130, 70), (200, 200), (3, 50))]
    O.orthogonalize(mats)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = O.orthogonalize(mats)
    for k in range(4):
        for m in mats:
            m.copy_(torch.randn(m.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, O.orthogonalize(mats))), k


def test_orthogonalize_on_two_streams_at_once():
    g = gen(6)
    jobs = [[torch.randn(300, 500, generator=g).cuda(), torch.randn(40, 30, generator=g).cuda()] for _ in range(2)]
    want = [O.orthogonalize(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [None, None]
    for _ in range(3):
        for k, j in enumerate(jobs):
            with torch.cuda.stream(streams[k]):
                got[k] = O.orthogonalize(j)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
