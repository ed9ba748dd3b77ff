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


BIG = [[(600, 640)], [(1400, 1500)], [(2300, 2500)], [(3200, 3205)], [(4000, 4096)], [(5600, 5630)], [(2305, 1000), (1000, 2305), (700, 3000)]]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("k", range(len(BIG)))
def test_orthogonalize_large(dtype, k):
    """every tile size and both numbers of planes.  bf16 matrices of these sizes are held in one plane: A, B and X are rounded by
    2^-12 / sqrt(3) (r.m.s., independent entries), of which A's counts |b + 2 c A| <= 5 times and B's twice: 8 a step relative
    to X, and relative errors do not grow where p is concave from 0 (s p'(s) <= p(s)): five steps, and the result's rounding."""
    dt, g = DT[dtype], torch.Generator(device="cuda")
    g.manual_seed(k)
    mats = [torch.randn(s, generator=g, device="cuda").to(dt) for s in BIG[k]]
    for m, o in zip(mats, O.orthogonalize(mats)):
        want = plain(m)  # in float64 on the device
        rel = float((o.double() - want).norm() / want.norm())
        assert rel < (341 * 16 * 2.0 ** -22 if dtype == "fp32" else 40 * 2.0 ** -12 / 3 ** 0.5 + 2.0 ** -9), (m.shape, rel)
        if dtype == "fp32":
            plain32 = plain(m, dtype=torch.float32).double()
            assert rel < 4 * max(float((plain32 - want).norm() / want.norm()), 2.0 ** -22), (m.shape, rel)


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


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(700, 901), (901, 700), (1500, 1300), (2600, 2801), (2801, 2600), (4001, 3901)])
def test_orthogonalize_rows_at_any_address(shape, dtype):
    """wide and tall, on every size of tile: rows of the result and of the input that begin at no multiple of 16 bytes"""
    m, n = shape
    g = torch.randn(m, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)).to(DT[dtype])
    want = O.orthogonalize(g)
    hole = torch.zeros(m + 2, n + 5, device="cuda", dtype=g.dtype)
    O.orthogonalize(g, out=hole[1:m + 1, 3:n + 3])
    assert torch.equal(hole[1:m + 1, 3:n + 3], want)
    hole[1:m + 1, 3:n + 3] = 0
    assert not hole.any()  # nothing beside it was written
    hole[1:m + 1, 3:n + 3] = g
    got = O.orthogonalize(hole[1:m + 1, 3:n + 3])
    # the norm is summed in another order: 2^-24 of a factor, which moves an entry of X by as much, and its rounding by a step
    assert float((got.double() - want.double()).norm() / want.double().norm()) < 341 * 16 * 2.0 ** -22 + torch.finfo(g.dtype).eps


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


# --------------------------------------------------------------------------------------------------------------- FlatMuon

def model_and_batch(bn=False, seed=0):
    import numpy as np
    torch.manual_seed(seed)
    cls = dvae_amd.DVAE_BN if bn else dvae_amd.DVAE
    model = cls(8, 8, 0, 1, hs=70, nz=16, bidirectional=True).cuda().train()
    rng = np.random.default_rng(seed)
    types = rng.integers(2, 8, (24, 8))
    types[:, 0], types[:, -1] = 0, 1
    adj = np.triu(rng.random((24, 8, 8)) < 0.4, 1)
    adj[:, np.arange(7), np.arange(1, 8)] = True
    ga = dvae_amd.GraphArrays.from_dense(types, adj, np.full(24, 8))
    return model, ga


def grads_of(model, ga, eps):
    batch = model._collate_fn(ga)
    mu, logvar = model.encode(batch)
    loss = model.loss(mu, logvar, batch, eps=eps)[0]
    loss.backward()
    return loss


@pytest.mark.parametrize("bn,nesterov,wd,fn", [(False, True, 0.0, "original"), (True, False, 0.1, "match_rms_adamw")])
def test_flat_muon_steps_against_the_formulas(bn, nesterov, wd, fn):
    model, ga = model_and_batch(bn)
    opt = O.FlatMuon(model, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=wd, adam_lr=1e-3, adjust_lr_fn=fn)
    r = opt.reducer
    assert opt.matrices and "grue_forward.weight_ih" not in opt.matrices and "add_edge.2.weight" not in opt.matrices
    assert ("gate_forward.0.weight" in opt.matrices) == (not bn)
    want = [p.detach().double().cpu().clone() for p in r.params]
    mom = [torch.zeros_like(w) for w in want]
    sq = [torch.zeros_like(w) for w in want]
    slack = [0.0] * len(want)  # what the orthogonalisation may be off by, times the step
    rounding = [0.0] * len(want)
    g = gen(9)
    for step in range(1, 4):
        opt.zero_grad()
        grads_of(model, ga, torch.randn(24, 16, generator=g))
        grads = [p.grad.double().cpu().clone() for p in r.params]
        opt.step()
        for i, (name, d) in enumerate(zip(r.names, grads)):
            if name in opt.matrices:
                mom[i] += (1 - 0.9) * (d - mom[i])
                u = d + 0.9 * (mom[i] - d) if nesterov else mom[i]
                rows, cols = d.shape
                f = max(1.0, rows / cols) ** 0.5 if fn == "original" else 0.2 * max(rows, cols) ** 0.5
                o = plain(u)
                want[i] = (1 - 0.02 * wd) * want[i] - 0.02 * f * o
                # + 8 u for the momentum in fp32, amplified like the iteration's own errors
                slack[i] += 0.02 * f * float(o.norm()) * 341 * (16 * 2.0 ** -22 + 8 * 2.0 ** -24)
            else:
                mom[i] += 0.1 * (d - mom[i])
                sq[i] = 0.999 * sq[i] + 0.001 * d * d
                want[i] = want[i] - 1e-3 / (1 - 0.9 ** step) * mom[i] / (sq[i].sqrt() / math.sqrt(1 - 0.999 ** step) + 1e-8)
                slack[i] += 1e-3 * math.sqrt(d.numel()) * 64 * 2.0 ** -24  # a dozen roundings of an update of at most ~1
            rounding[i] += 3 * 2.0 ** -24 * float(want[i].norm())
        for i, p in enumerate(r.params):
            assert float((p.detach().double().cpu() - want[i]).norm()) <= slack[i] + rounding[i], (step, r.names[i])
    assert not r.flat.any()  # the gradients were left zeroed for the next step


def test_flat_muon_checkpoint_continues_identically(tmp_path):
    model, ga = model_and_batch()
    opt = O.FlatMuon(model, lr=0.01, weight_decay=0.01)
    g = gen(10)
    eps = [torch.randn(24, 16, generator=g) for _ in range(4)]
    for e in eps[:2]:
        opt.zero_grad()
        grads_of(model, ga, e)
        opt.step()
    dvae_amd.harness.save_checkpoint(str(tmp_path), 2, model, opt)
    other, _ = model_and_batch(seed=5)
    opt2 = O.FlatMuon(other, lr=0.5)
    dvae_amd.harness.load_module_state(other, str(tmp_path / "model_checkpoint2.pth"))
    dvae_amd.harness.load_module_state(opt2, str(tmp_path / "optimizer_checkpoint2.pth"))
    assert opt2.steps == 2 and opt2.param_groups[0]["lr"] == 0.01 and opt2.param_groups[0]["weight_decay"] == 0.01
    assert torch.equal(opt.exp_avg, opt2.exp_avg)
    mats = torch.cat([torch.arange(o, o + p.numel()) for p, o, m in zip(opt.reducer.params, opt.reducer.offsets, opt.is_matrix) if not m])
    assert torch.equal(opt.exp_avg_sq.cpu()[mats], opt2.exp_avg_sq.cpu()[mats])
    for e in eps[2:]:
        for m, o in ((model, opt), (other, opt2)):
            o.zero_grad()
            grads_of(m, ga, e)
        opt2.reducer.flat.copy_(opt.reducer.flat)  # (the step's own gradients vary in the last bits: atomics)
        opt.step(), opt2.step()
    assert torch.equal(opt.flat_p, opt2.flat_p)
    with pytest.raises(ValueError, match="FlatMuon state"):
        opt.load_state_dict(O.FlatAdam(model_and_batch()[0]).state_dict())
    with pytest.raises(ValueError, match="choice of matrices"):
        opt.load_state_dict(O.FlatMuon(model_and_batch()[0], matrices=["fc3.weight"]).state_dict())


def test_flat_muon_trains_an_epoch_with_a_scheduler():
    import random
    model, ga = model_and_batch()
    opt = O.FlatMuon(model)
    sched = torch.optim.lr_scheduler.ReduceLROnPlateau(opt, "min", factor=0.1, patience=10)
    before = {k: p.detach().clone() for k, p in model.named_parameters()}
    import numpy as np
    for _ in range(2):
        sums = dvae_amd.harness.train_epoch(model, opt, (ga, np.zeros(24)), batch_size=8, rng=random.Random(0))
        assert all(math.isfinite(v) for v in sums)
        sched.step(sums[0])
    moved = {k for k, p in model.named_parameters() if not torch.equal(p, before[k])}
    assert set(opt.reducer.names) == moved


def test_flat_muon_refusals():
    model, _ = model_and_batch()
    for bad in (dict(adjust_lr_fn="none"), dict(momentum=1.0), dict(lr=-1.0), dict(matrices=["fc1.bias"]), dict(matrices=["nothing"])):
        with pytest.raises(ValueError):
            O.FlatMuon(model, **bad)
    with pytest.raises(ValueError, match="capturable"):
        dvae_amd.harness.GraphedTrainStep(model, O.FlatMuon(model))
    m = torch.randn(8, 8).cuda()
    for bad in ((m[0], {}), (m.double(), {}), ([m, m.half()], {}), (m[:0], {}), (m, dict(out=m[:4])), (m, dict(steps=0)), (m, dict(coefficients=(1.0, 2.0))),
                (m, dict(coefficients=())), (m.clone().requires_grad_(True), {}), ([m], dict(out=[])), (m, dict(out=m.t()[:, :4]))):
        with pytest.raises((ValueError, dvae_amd._lib.DvaeHipError)):
            O.orthogonalize(bad[0], **bad[1])
    with pytest.raises(dvae_amd._lib.DvaeHipError, match="singular values leave"):
        O.orthogonalize(m, coefficients=(4.0, 0.0, 0.0))
    assert O.orthogonalize([]) == []


def test_flat_muon_checkpoint_holds_the_iteration_and_the_factor(tmp_path):
    """resumed by an optimizer built with the defaults"""
    model, ga = model_and_batch()
    convergent = [(2.0, -1.5, 0.5)] * 7
    opt = O.FlatMuon(model, lr=0.01, ns_steps=7, ns_coefficients=convergent, adjust_lr_fn="match_rms_adamw", nesterov=False, momentum=0.8)
    g = gen(11)
    eps = [torch.randn(24, 16, generator=g) for _ in range(2)]
    opt.zero_grad()
    grads_of(model, ga, eps[0])
    opt.step()
    dvae_amd.harness.save_checkpoint(str(tmp_path), 1, model, opt)
    other, _ = model_and_batch(seed=5)
    opt2 = O.FlatMuon(other)
    dvae_amd.harness.load_module_state(other, str(tmp_path / "model_checkpoint1.pth"))
    dvae_amd.harness.load_module_state(opt2, str(tmp_path / "optimizer_checkpoint1.pth"))
    assert opt2.ns_steps == 7 and list(map(tuple, opt2.ns_coefficients)) == convergent
    for m, o in ((model, opt), (other, opt2)):
        o.zero_grad()
        grads_of(m, ga, eps[1])
    opt2.reducer.flat.copy_(opt.reducer.flat)  # (the step's own gradients vary in the last bits: atomics)
    opt.step(), opt2.step()
    assert torch.equal(opt.flat_p, opt2.flat_p) and torch.equal(opt.factor, opt2.factor)
    old = opt.state_dict()  # a state without these keys keeps what the optimizer was built with
    for k in ("ns_steps", "ns_coefficients", "adjust_lr_fn"):
        del old["param_groups"][0][k]
    opt3 = O.FlatMuon(model_and_batch()[0], ns_steps=3)
    opt3.load_state_dict(old)
    assert opt3.ns_steps == 3 and opt3.param_groups[0]["adjust_lr_fn"] == "original"
    old["param_groups"][0]["adjust_lr_fn"] = "none"
    before = opt3.exp_avg.clone()
    with pytest.raises(ValueError, match="adjust_lr_fn"):
        opt3.load_state_dict(old)
    assert torch.equal(before, opt3.exp_avg)


def test_flat_muon_refuses_an_iteration_before_anything_moves():
    model, ga = model_and_batch()
    for bad in (dict(ns_coefficients=(4.0, 0.0, 0.0)), dict(ns_coefficients=(1.0, 2.0)), dict(ns_steps=0), dict(ns_coefficients=[(1.5, -0.5, 0.0)] * 2)):
        with pytest.raises((ValueError, dvae_amd._lib.DvaeHipError)):
            O.FlatMuon(model_and_batch()[0], **bad)
    opt = O.FlatMuon(model)
    opt.zero_grad()
    grads_of(model, ga, torch.randn(24, 16, generator=gen(12)))
    opt.param_groups[0]["ns_coefficients"] = (4.0, 0.0, 0.0)
    kept = [t.clone() for t in (opt.flat_p, opt.exp_avg, opt.exp_avg_sq, opt.reducer.flat)]
    with pytest.raises(dvae_amd._lib.DvaeHipError, match="singular values leave"):
        opt.step()
    assert opt.steps == 0 and all(torch.equal(a, b) for a, b in zip(kept, (opt.flat_p, opt.exp_avg, opt.exp_avg_sq, opt.reducer.flat)))
    state = opt.state_dict()
    with pytest.raises(dvae_amd._lib.DvaeHipError, match="singular values leave"):
        O.FlatMuon(model_and_batch()[0]).load_state_dict(state)
    opt.param_groups[0]["ns_coefficients"] = O.QUINTIC
    opt.step()
    assert opt.steps == 1 and not torch.equal(kept[0], opt.flat_p)


def test_flat_muon_iteration_can_be_set_as_an_attribute():
    model, ga = model_and_batch()
    opt = O.FlatMuon(model)
    opt.ns_steps, opt.ns_coefficients = 2, (1.5, -0.5, 0.0)
    opt.zero_grad()
    grads_of(model, ga, torch.randn(24, 16, generator=gen(13)))
    before = [p.detach().double().cpu() for p in opt.reducer.params]
    grads = [p.grad.double().cpu().clone() for p in opt.reducer.params]
    opt.step()
    for name, p, b, d in zip(opt.reducer.names, opt.reducer.params, before, grads):
        if name in opt.matrices:
            rows, cols = d.shape
            f = 0.02 * max(1.0, rows / cols) ** 0.5
            o = plain(d + 0.95 * (0.05 * d - d), 2, (1.5, -0.5, 0.0))  # u = g + mu (m - g), m = (1 - mu) g
            # (sup |p'| is 1.5 here: 1 + 1.5 steps' errors; the momentum's and the update's roundings as above)
            slack = f * float(o.norm()) * 2.5 * (16 * 2.0 ** -22 + 8 * 2.0 ** -24) + 3 * 2.0 ** -24 * float(b.norm())
            assert float((p.detach().double().cpu() - (b - f * o)).norm()) <= slack, name
