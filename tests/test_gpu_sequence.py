"""The sequence operators (d-vae_amd/sequence.py) against plain implementations in 64 bits.

Tolerances: u = 2^-24 is half a step of float32, r = eps / 2 of the output's type; M bounds the values of x and h0 (and so
of every state, a convex combination of them).  A step of the recurrence rounds a few times (gate and its complement about
3 u each relative, two products, one sum: 8 u M together) and passes older errors on times z <= zmax, so they add up to at most
8 u M min(T, 1 / (1 - zmax)); the exponential's argument adds 16 u |g| / 10 relative to z (1 - z), which sums to 32 u M."""
import numpy as np
import pytest
import torch
import torch.utils.checkpoint

from _dvae_pkg import dvae_amd

S = dvae_amd.sequence
pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tol, what=""):
    """|got - want| <= tol + half a step of got's type, element by element (tol: number or array)"""
    got64 = got.detach().double().cpu()
    err = (got64 - want).abs()
    lim = tol + want.abs() * half_step(got.dtype) * (1 + 1e-6)
    if got.dtype == torch.float16:
        lim = lim + 2.0 ** -25  # half a step among its subnormal numbers
    assert torch.isfinite(got64).all(), what
    bad = err > lim
    assert not bad.any(), "%s: %d of %d off, worst %.3g where %.3g is allowed" % (
        what, int(bad.sum()), bad.numel(), float((err - lim).max() + lim.max()), float(lim.max()))


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------------------------------------------------------ embed

@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (5, 3, 7), (31, 8, 501), (33, 255, 64), (64, 256, 96), (257, 40, 1024), (1500, 70000, 33),
                                         (8192, 8, 130), (8193, 8, 130), (9001, 300, 256), (20011, 66000, 20), (70001, 5, 16)])
def test_embed_and_its_gradient(dtype, n, vocab, dim):
    dt, g = DT[dtype], gen(n + vocab)
    w = torch.randn(vocab, dim, generator=g).to(dt)
    ids = torch.randint(0, vocab, (n,), generator=g)
    ids[torch.rand(n, generator=g) < 0.3] = min(2, vocab - 1)  # a hot row
    ids[torch.rand(n, generator=g) < 0.1] = -1
    if n > 2:
        ids[1] = vocab
    dout = torch.randn(n, dim, generator=g).to(dt)
    scale = 2.5
    wd = w.cuda().requires_grad_(True)
    out = S.embed(wd, ids.to(torch.int32).cuda() if n % 2 else ids.cuda(), scale)
    ok = (ids >= 0) & (ids < vocab)
    want = w.double()[ids.clamp(0, vocab - 1)] * scale * ok[:, None]
    close(out, want, want.abs() * U, "out")  # one product in fp32, then the rounding to the type
    dw, = torch.autograd.grad(out, [wd], dout.cuda())
    want = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, ids[ok], dout.double()[ok])
    size = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, ids[ok], dout.double()[ok].abs())
    # additions on any one path: 32 in a chunk, the partials of a wave, the eight waves; each is off by u of a partial sum
    depth = 32 + (n // 32 // 8 + 2) + 8 + 2
    close(dw, want * scale, size * scale * depth * U, "dw")
    again, = torch.autograd.grad(S.embed(wd, ids.cuda(), scale), [wd], dout.cuda())
    assert torch.equal(dw, again)


def test_embed_many_tokens():
    """more tokens than one round of the sorting workgroups"""
    g = gen(30)
    n, V = 600_001, 300
    ids = torch.randint(-1, V, (n,), generator=g)
    w = torch.randn(V, 3, generator=g).cuda().requires_grad_(True)
    dout = torch.randn(n, 3, generator=g)
    dw, = torch.autograd.grad(S.embed(w, ids.cuda()), [w], dout.cuda())
    ok = ids >= 0
    want = torch.zeros(V, 3, dtype=torch.float64).index_add_(0, ids[ok], dout.double()[ok])
    size = torch.zeros(V, 3, dtype=torch.float64).index_add_(0, ids[ok], dout.double()[ok].abs())
    close(dw, want, size * (32 + 70 + 8 + 2) * U, "dw")  # 63 chunks or so per row


def test_offsets_past_32_bits():
    n, D = 2_200_000, 1024  # 2.25e9 elements
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    ids[-40:] = torch.arange(40, device="cuda", dtype=torch.int32) % 3
    w = torch.randn(3, D, device="cuda").bfloat16().requires_grad_(True)
    out = S.embed(w, ids)
    assert torch.equal(out[-40:], w[ids[-40:].long()]) and torch.equal(out[:3], w[:1].expand(3, D))
    dout = torch.zeros(n, D, device="cuda", dtype=torch.bfloat16)
    dout[-40:] = 1
    dw, = torch.autograd.grad(out, [w], dout)
    count = torch.bincount(ids[-40:].long(), minlength=3).bfloat16()
    assert torch.equal(dw, count[:, None].expand(3, D))
    del out, dout
    gate = torch.empty(n, D, device="cuda", dtype=torch.bfloat16).normal_()
    x = torch.empty(n, D, device="cuda", dtype=torch.bfloat16).normal_()
    off = torch.tensor([0, 1_100_000, n - 300, n], device="cuda")
    a, b = gate.requires_grad_(True), x.requires_grad_(True)
    h, last = S.gated_scan(a, b, off)
    dg, dx = torch.autograd.grad([h, last], [a, b], [torch.ones(1, 1, device="cuda", dtype=torch.bfloat16).expand(n, D), torch.ones_like(last)])
    h2, last2 = S.gated_scan(gate.detach()[-300:], x.detach()[-300:], torch.tensor([0, 300], device="cuda"))
    # other tiles, so the last sequence's sums are composed in another order: both are within their bound of the exact one
    tol = 2 * (8 * 300 + 32) * U * 6
    close(h[-300:], h2.double().cpu(), tol + 2.0 ** -8 * 6, "h")
    close(last[2], last2[0].double().cpu(), tol, "last")
    assert torch.isfinite(dg[-300:]).all() and dx[-300:].abs().sum() > 0 and torch.isfinite(dx[:300]).all()


def test_embed_shapes_strides_and_no_tokens():
    g = gen(1)
    big = torch.randn(9, 40, generator=g).cuda()
    w = big[:, 3:24].requires_grad_(True)  # rows of stride 40 that begin at an odd element
    ids = torch.randint(-1, 10, (4, 3, 2), generator=g).cuda()
    out = S.embed(w, ids, 1.0)
    assert out.shape == (4, 3, 2, 21)
    ok = ((ids >= 0) & (ids < 9))[..., None]
    assert torch.equal(out, w[ids.clamp(0, 8)] * ok)
    one = torch.ones(21, device="cuda").expand(4, 3, 2, 21)  # a gradient of stride 0, as sum() gives it
    dw, = torch.autograd.grad(out, [w], one)
    count = torch.stack([(ids == v).sum() for v in range(9)]).float()
    assert torch.equal(dw, count[:, None].expand(9, 21))
    out = S.embed(w, ids, 1.0)
    turned = torch.randn(21, 24, generator=g).cuda().t().reshape(4, 3, 2, 21)
    dw, = torch.autograd.grad(out, [w], turned)
    want = torch.zeros(9, 21, dtype=torch.float64)
    flat, t64 = ids.reshape(-1).cpu(), turned.reshape(-1, 21).double().cpu()
    for t in range(24):
        if 0 <= flat[t] < 9:
            want[flat[t]] += t64[t]
    close(dw, want, 24 * 24 * U, "dw of a turned gradient")
    none = S.embed(w, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert none.shape == (0, 21)
    dw, = torch.autograd.grad(none, [w], torch.empty(0, 21, device="cuda"))
    assert torch.equal(dw, torch.zeros(9, 21, device="cuda"))


def test_embed_padding_rows_do_not_spread_what_they_hold():
    w = torch.randn(4, 65).cuda().requires_grad_(True)
    ids = torch.tensor([1, -1, 3, 4, 1, -7], device="cuda")
    dout = torch.ones(6, 65, device="cuda")
    dout[1], dout[3], dout[5] = float("nan"), float("inf"), float("nan")
    dw, = torch.autograd.grad(S.embed(w, ids), [w], dout)
    assert torch.equal(dw, torch.tensor([0.0, 2.0, 0.0, 1.0], device="cuda")[:, None].expand(4, 65))
    all_pad = torch.full((70,), -1, device="cuda")
    dw, = torch.autograd.grad(S.embed(w, all_pad), [w], torch.full((70, 65), float("nan"), device="cuda"))
    assert torch.equal(dw, torch.zeros(4, 65, device="cuda"))


# ------------------------------------------------------------------------------------------------------------------- scan

def plain_scan(gate, x, off, h0, dh=None, dlast=None):
    """row by row in 64 bits; off: list of S + 1 row numbers"""
    N, D = x.shape
    Sn = len(off) - 1
    z = torch.sigmoid(gate)
    omz = torch.sigmoid(-gate)
    h, prev = torch.zeros(N, D, dtype=torch.float64), torch.zeros(N, D, dtype=torch.float64)
    init = torch.zeros(Sn, D, dtype=torch.float64) if h0 is None else h0
    last = init.clone()
    for s in range(Sn):
        for t in range(off[s], off[s + 1]):
            prev[t] = last[s]
            last[s] = z[t] * last[s] + omz[t] * x[t]
            h[t] = last[s]
    if dh is None:
        return h, last
    dg, dx, dh0, big = torch.zeros_like(h), torch.zeros_like(h), torch.zeros_like(last), 0.0
    for s in range(Sn):
        c = dlast[s].clone()
        for t in reversed(range(off[s], off[s + 1])):
            G = dh[t] + c
            big = max(big, float(G.abs().max()))
            dx[t] = omz[t] * G
            dg[t] = G * (prev[t] - x[t]) * z[t] * omz[t]
            c = z[t] * G
        dh0[s] = c
    return h, last, dg, dx, dh0, big


def offsets_of(lengths, front=0):
    return [front + int(v) for v in np.concatenate([[0], np.cumsum(lengths)])]


SHAPES = [  # (lengths, rows before the first sequence, rows behind the last)
    ([1], 0, 0), ([0], 0, 0), ([0, 0, 3], 0, 0), ([5, 0, 0, 1, 64, 65, 0], 0, 0), ([200], 0, 0), ([63, 1, 64, 128, 2], 7, 70),
    ([7] * 40, 0, 1), ([0, 0], 3, 0), ([700, 1, 1, 1000], 65, 0)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [1, 6, 64, 501, 516])
@pytest.mark.parametrize("k", range(len(SHAPES)))
def test_gated_scan_and_its_gradient(dtype, dim, k):
    lengths, front, behind = SHAPES[k]
    dt, g = DT[dtype], gen(100 * k + dim)
    off = offsets_of(lengths, front)
    N, Sn = off[-1] + behind, len(lengths)
    gate = (torch.randn(N, dim, generator=g) * 2 + 1).clamp(-5, 5).to(dt)
    x = torch.randn(N, dim, generator=g).clamp(-3, 3).to(dt)
    h0 = torch.randn(Sn, dim, generator=g).clamp(-3, 3) if k % 2 else None
    dh, dlast = torch.randn(N, dim, generator=g).to(dt), torch.randn(Sn, dim, generator=g)
    mem = min(max(lengths + [1]), 1 + np.exp(5.0))
    M = 3.0
    ref = plain_scan(gate.double(), x.double(), off, None if h0 is None else h0.double(), dh.double(), dlast.double())
    both = torch.cat([gate, x], 1).cuda()  # the two halves of one projection: rows of stride 2 D
    gd, xd = both[:, :dim].detach().requires_grad_(True), both[:, dim:].detach().requires_grad_(True)
    hd = None if h0 is None else h0.cuda().requires_grad_(True)
    o = torch.tensor(off, dtype=torch.int64 if k % 2 else torch.int32, device="cuda")
    h, last = S.gated_scan(gd, xd, o, hd)
    tol_h = (8 * mem + 32) * U * M
    close(h, ref[0], tol_h, "h")
    close(last, ref[1], tol_h, "last")
    got = torch.autograd.grad([h, last], [gd, xd] + ([hd] if h0 is not None else []), [dh.cuda(), dlast.cuda()])
    big = max(ref[5], 1.0)
    tol_G = (8 * mem + 32) * U * big
    close(got[1], ref[3], tol_G + 4 * U * big, "dx")
    # G, h_{t-1} - x (at most 2 M, off by tol_h) and z (1 - z) <= 1 / 4, each a few roundings of its own
    close(got[0], ref[2], (tol_G * 2 * M + big * tol_h + 32 * U * big * 2 * M) / 4, "dgate")
    if h0 is not None:
        close(got[2], ref[4], tol_G, "dh0")
    if behind:
        assert not h[off[-1]:].any() and not got[0][off[-1]:].any() and not got[1][off[-1]:].any()
    h2, last2 = S.gated_scan(gd, xd, o, hd)
    assert torch.equal(h, h2) and torch.equal(last, last2)


@pytest.mark.parametrize("dim", [5, 70, 516])
@pytest.mark.parametrize("lengths", [[64], [0, 60, 0, 4], [65, 0], [0, 128, 0], [129], [0] * 150 + [3, 0, 70] + [0] * 150, [1] * 64, [2] * 65])
def test_gated_scan_of_one_tile_and_just_more(lengths, dim):
    g = gen(len(lengths) * 1000 + dim)
    off = offsets_of(lengths)
    N, Sn = off[-1], len(lengths)
    gate = (torch.randn(N, dim, generator=g) * 2 + 1).clamp(-5, 5)
    x, h0 = torch.randn(N, dim, generator=g).clamp(-3, 3), torch.randn(Sn, dim, generator=g).clamp(-3, 3)
    dh, dlast = torch.randn(N, dim, generator=g), torch.randn(Sn, dim, generator=g)
    ref = plain_scan(gate.double(), x.double(), off, h0.double(), dh.double(), dlast.double())
    gd, xd, hd = (t.cuda().requires_grad_(True) for t in (gate, x, h0))
    h, last = S.gated_scan(gd, xd, torch.tensor(off, device="cuda"), hd)
    mem, big = min(max(lengths), 1 + np.exp(5.0)), max(ref[5], 1.0)
    tol_h, tol_G = (8 * mem + 32) * U * 3.0, (8 * mem + 32) * U * big  # as above
    close(h, ref[0], tol_h, "h")
    close(last, ref[1], tol_h, "last")
    got = torch.autograd.grad([h, last], [gd, xd, hd], [dh.cuda(), dlast.cuda()])
    close(got[0], ref[2], (tol_G * 6 + big * tol_h + 32 * U * big * 6) / 4, "dgate")
    close(got[1], ref[3], tol_G + 4 * U * big, "dx")
    close(got[2], ref[4], tol_G, "dh0")
    none = [k for k in range(Sn) if lengths[k] == 0]
    assert torch.equal(last[none], hd[none]) and torch.equal(got[2][none].cpu(), dlast[none])
    again = S.gated_scan(gd, xd, torch.tensor(off, device="cuda"), hd)
    assert torch.equal(h, again[0]) and torch.equal(last, again[1])


def test_gated_scan_gradient_against_differences():
    g = gen(5)
    off, D, N = [0, 3, 70, 75], 5, 75
    gate, x, h0 = torch.randn(N, D, generator=g) + 1, torch.randn(N, D, generator=g), torch.randn(3, D, generator=g)
    a, b = torch.randn(N, D, generator=g), torch.randn(3, D, generator=g)
    leaves = [t.cuda().requires_grad_(True) for t in (gate, x, h0)]
    h, last = S.gated_scan(leaves[0], leaves[1], torch.tensor(off).cuda(), leaves[2])
    got = torch.autograd.grad((h * a.cuda()).sum() + (last * b.cuda()).sum(), leaves)

    def loss(v):
        hh, ll = plain_scan(v[0], v[1], off, v[2])
        return float((hh * a.double()).sum() + (ll * b.double()).sum())

    for i in range(3):
        for _ in range(4):
            d = [torch.zeros_like(t).double() for t in (gate, x, h0)]
            d[i] = torch.randn(d[i].shape, generator=g).double()
            step = 1e-4
            up = [t.double() + step * e for t, e in zip((gate, x, h0), d)]
            down = [t.double() - step * e for t, e in zip((gate, x, h0), d)]
            diff = (loss(up) - loss(down)) / (2 * step)
            mine = float((got[i].double().cpu() * d[i]).sum())
            # differences: third derivatives times step^2 (below 1e-6 in all); the kernel: about 1e3 terms of fp32 accuracy
            assert abs(diff - mine) < 1e-6 * 100 + 1000 * 32 * U, (i, diff, mine)


def test_gated_scan_equal_lengths_and_layouts():
    g = gen(6)
    B, T, D = 3, 70, 36
    base = torch.randn(B, T, 2 * D, generator=g).cuda()
    gate, x = base[..., :D], base[..., D:]
    h, last = S.gated_scan(gate, x)
    off = torch.arange(0, B * T + 1, T).cuda()
    h2, last2 = S.gated_scan(gate.reshape(B * T, D), x.reshape(B * T, D), off)
    assert torch.equal(h.reshape(B * T, D), h2) and torch.equal(last, last2)
    for view in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        h3, last3 = S.gated_scan(view(gate), view(x))
        assert torch.equal(h, h3) and torch.equal(last, last3)
    one, last4 = S.gated_scan(gate[:, :1], x[:, :1])  # length one, rows of stride T 2 D
    assert torch.equal(one, h[:, :1]) and torch.equal(last4, h[:, 0])
    wide = torch.zeros(2, 1 << 18, D, device="cuda")  # rows 2^18 D elements apart
    wide[:, :1] = gate[:2, :1]
    far, _ = S.gated_scan(wide[:, :1], x[:2, :1])
    assert torch.equal(far, h[:2, :1])
    none, last5 = S.gated_scan(gate[:, :0], x[:, :0], h0=torch.ones(B, D, device="cuda"))
    assert none.shape == (B, 0, D) and torch.equal(last5, torch.ones(B, D, device="cuda"))
    gl, xl = gate.detach().requires_grad_(True), x.detach().requires_grad_(True)
    dg, dx = torch.autograd.grad(S.gated_scan(gl, xl)[0].sum(), [gl, xl])  # dh of stride 0, no dlast
    dg2, dx2 = torch.autograd.grad(S.gated_scan(gl, xl)[0], [gl, xl], torch.ones(B, T, D, device="cuda"))
    assert torch.equal(dg, dg2) and torch.equal(dx, dx2)
    h0 = torch.randn(B, D, generator=g).cuda().requires_grad_(True)
    dh0, = torch.autograd.grad(S.gated_scan(gl, xl, h0=h0)[1].sum(), [h0])  # dlast alone
    want = torch.sigmoid(gate.double()).prod(1)
    close(dh0, want.cpu(), 8 * T * U, "dh0 of the last state")


def test_gated_scan_extreme_gates():
    inf = float("inf")
    gate = torch.tensor([[inf, -inf, 200.0, -200.0, 100.0, 0.0]] * 3, device="cuda")
    x = torch.tensor([[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]] * 3, device="cuda")
    h0 = torch.full((1, 6), 7.0, device="cuda")
    h, last = S.gated_scan(gate[None], x[None], h0=h0)
    assert torch.equal(h[0, -1].cpu(), torch.tensor([7.0, 2.0, 7.0, 4.0, 7.0, 6.125]))
    bad = x.clone()
    bad[1, 0] = float("nan")  # a NaN stays in its own sequence and channel
    two = torch.cat([bad, x])
    h, _ = S.gated_scan(torch.zeros_like(two), two, torch.tensor([0, 3, 6]).cuda())
    assert torch.isnan(h[1:3, 0]).all() and torch.isfinite(h[3:]).all() and torch.isfinite(h[:, 1:]).all() and torch.isfinite(h[0]).all()


def test_gated_scan_keeps_nan_and_inf_in_their_sequence():
    """also where a sequence begins in the middle of a tile, at its first row, or many tiles later"""
    g = gen(7)
    off = [0, 130, 131, 300, 320, 1920, 1984, 2100]
    N, D = off[-1], 70
    gate, x = torch.randn(N, D, generator=g) * 3, torch.randn(N, D, generator=g)
    dh, dlast = torch.randn(N, D, generator=g).cuda(), torch.randn(len(off) - 1, D, generator=g).cuda()
    bad = x.clone()
    bad[5, 0], bad[140, 1], bad[330, 2], bad[1930, 3] = float("nan"), float("inf"), float("nan"), float("-inf")
    hit = {0: (0, 5), 1: (2, 140), 2: (4, 330), 3: (5, 1930)}  # channel -> (its sequence, the row)

    def run(xx):
        leaves = [gate.cuda().requires_grad_(True), xx.cuda().requires_grad_(True)]
        h, last = S.gated_scan(leaves[0], leaves[1], torch.tensor(off).cuda())
        return [h.detach(), last.detach()] + list(torch.autograd.grad([h, last], leaves, [dh, dlast]))

    good, got = run(x), run(bad)
    h, last, dg, dx = got
    for c in range(D):
        keep = torch.ones(N, dtype=torch.bool)
        if c in hit:
            s, row = hit[c]
            keep[off[s]:off[s + 1]] = False
            assert not torch.isfinite(h[row:off[s + 1], c]).any() and not torch.isfinite(last[s, c])
            assert torch.equal(h[off[s]:row, c], good[0][off[s]:row, c])
        assert torch.equal(h[keep, c], good[0][keep, c]) and torch.equal(dg[keep, c], good[2][keep, c])
    assert torch.equal(dx, good[3])  # dx does not depend on x


def test_gated_scan_offsets_outside_the_rows_count_as_the_nearer_end():
    g = gen(8)
    gate, x = torch.randn(90, 8, generator=g).cuda(), torch.randn(90, 8, generator=g).cuda()
    h, last = S.gated_scan(gate, x, torch.tensor([-5, 40, 200]).cuda())
    h2, last2 = S.gated_scan(gate, x, torch.tensor([0, 40, 90]).cuda())
    assert torch.equal(h, h2) and torch.equal(last, last2)


# ------------------------------------------------------------------------------------------------------------------- step

@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,pool,dim", [(1, 1, 1), (5, 9, 7), (64, 64, 501), (65, 300, 256), (300, 200, 68), (255, 50, 20), (256, 50, 20), (2500, 700, 40)])
def test_gated_step(dtype, rows, pool, dim):
    dt, g = DT[dtype], gen(rows + dim)
    gate, x = (torch.randn(rows, dim, generator=g) * 2).to(dt), torch.randn(rows, dim, generator=g).clamp(-3, 3).to(dt)
    state = torch.randn(pool, dim, generator=g).clamp(-3, 3)
    slots = torch.randint(-2, pool + 2, (rows,), generator=g)  # padding rows and repeated slots among them
    ref, want = state.double().clone(), torch.zeros(rows, dim, dtype=torch.float64)
    longest = 1
    for b in range(rows):
        k = int(slots[b])
        if 0 <= k < pool:
            z, omz = torch.sigmoid(gate[b].double()), torch.sigmoid(-gate[b].double())
            ref[k] = z * ref[k] + omz * x[b].double()
            want[b] = ref[k]
            longest = max(longest, int((slots == k).sum()))
    both, sd = torch.cat([gate, x], 1).cuda(), state.cuda()
    h = S.gated_step(both[:, :dim], both[:, dim:], sd, slots.cuda() if dim % 2 else slots.to(torch.int32).cuda())
    tol = (8 * longest + 32) * U * 3
    close(h, want, tol, "h")
    close(sd, ref, tol, "state")
    untouched = torch.ones(pool, dtype=torch.bool)
    untouched[slots[(slots >= 0) & (slots < pool)]] = False
    assert torch.equal(sd.cpu()[untouched], state[untouched])


def test_gated_step_continues_a_scan():
    """a prompt read in at once and then token by token gives what the scan over all of it gives"""
    g = gen(9)
    lengths, D, more = [5, 1, 130, 0], 96, 3
    Sn = len(lengths)
    full = [torch.randn(n + more, 2 * D, generator=g).cuda() for n in lengths]
    prompt = torch.cat([f[:n] for f, n in zip(full, lengths)])
    h, last = S.gated_scan(prompt[:, :D], prompt[:, D:], torch.tensor(offsets_of(lengths)).cuda())
    pool = torch.zeros(9, D, device="cuda")
    slots = torch.tensor([7, 0, 3, 4]).cuda()
    pool[slots] = last
    outs = [S.gated_step(t[:, :D], t[:, D:], pool, slots) for t in (torch.stack([f[n + i] for f, n in zip(full, lengths)]) for i in range(more))]
    allrows = torch.cat(full)
    off = offsets_of([n + more for n in lengths])
    ref, _ = plain_scan(allrows[:, :D].double().cpu(), allrows[:, D:].double().cpu(), off, None)
    tol = (8 * 133 + 32) * U * float(allrows.abs().max())
    for i in range(more):
        close(outs[i], torch.stack([ref[off[s] + lengths[s] + i] for s in range(Sn)]), tol, "token %d" % i)


# ------------------------------------------------------------------------------------------------------ streams and graphs

def test_sequence_operators_on_two_streams_at_once():
    g = gen(11)
    jobs = []
    for k in range(2):
        w = torch.randn(50, 64, generator=g).cuda().requires_grad_(True)
        ids = torch.randint(0, 50, (9000,), generator=g).cuda()
        gate, x = (torch.randn(9000, 64, generator=g).cuda().requires_grad_(True) for _ in range(2))
        off = torch.tensor([0, 10, 4000 + k, 9000]).cuda()
        jobs.append((w, ids, gate, x, off))

    def work(w, ids, gate, x, off):
        e = S.embed(w, ids, 2.0)
        h, last = S.gated_scan(gate, e, off)
        return [h.detach(), last.detach()] + list(torch.autograd.grad([h, last], [w, gate], [torch.ones_like(h), torch.ones_like(last)]))

    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [None, None]
    for _ in range(3):
        for k, j in enumerate(jobs):
            with torch.cuda.stream(streams[k]):
                got[k] = work(*j)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_sequence_operators_captured_and_replayed():
    g = gen(12)
    D, N = 72, 9000
    w = torch.randn(40, D, generator=g).cuda().requires_grad_(True)
    gate = torch.randn(N, D, generator=g).cuda().requires_grad_(True)
    ids, off = torch.randint(-1, 40, (N,), generator=g).cuda(), torch.tensor([0, 100, 100, 8000, N]).cuda()
    state, slots = torch.zeros(6, D, device="cuda"), torch.tensor([3, 1, 3]).cuda()

    def work():
        h, last = S.gated_scan(gate, S.embed(w, ids, 2.0), off)
        dw, dg = torch.autograd.grad([h, last], [w, gate], [torch.ones_like(h), torch.ones_like(last)])
        step = S.gated_step(gate.detach()[:3], h.detach()[:3], state, slots)
        return [h.detach(), last.detach(), dw, dg, step, state]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = work()
    for k in range(4):
        with torch.no_grad():
            gate.copy_(torch.randn(N, D, generator=g))
            ids.copy_(torch.randint(-1, 40, (N,), generator=g))
            off.copy_(torch.tensor([0, 5 * k, 700, 7000 + k, N]))
            state.fill_(float(k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        with torch.no_grad():
            state.fill_(float(k))
        want = work()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


# ------------------------------------------------------------------------------------------------------- used together

def test_gradients_are_not_differentiable_again():
    w = torch.randn(4, 8).cuda().requires_grad_(True)
    ids = torch.tensor([1, 2, 1], device="cuda")
    with pytest.raises(RuntimeError, match="differentiable again"):
        torch.autograd.grad(S.embed(w, ids).sum(), [w], create_graph=True)
    gate = torch.randn(1, 5, 8).cuda().requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiable again"):
        torch.autograd.grad(S.gated_scan(gate, gate.detach())[0].sum(), [gate], create_graph=True)


def test_the_graph_keeps_its_rules():
    """kept graphs, recomputed segments, hooks on saved tensors, freed graphs, inputs changed in place, gradients of some inputs only"""
    g = gen(41)
    N, D = 300, 24
    w = torch.randn(30, D, generator=g).cuda().requires_grad_(True)
    gate = torch.randn(N, D, generator=g).cuda().requires_grad_(True)
    h0 = torch.randn(3, D, generator=g).cuda().requires_grad_(True)
    ids, off = torch.randint(0, 30, (N,), generator=g).cuda(), torch.tensor([0, 7, 7, N]).cuda()
    up = torch.randn(N, D, generator=g).cuda()

    def work(w, gate, h0):
        return S.gated_scan(gate, S.embed(w, ids), off, h0)[0]

    h = work(w, gate, h0)
    first = torch.autograd.grad(h, [w, gate, h0], up, retain_graph=True)
    again = torch.autograd.grad(h, [w, gate, h0], up)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(h, [w], up)
    h = torch.utils.checkpoint.checkpoint(work, w, gate, h0, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(h, [w, gate, h0], up)))
    with torch.autograd.graph.save_on_cpu():
        h = work(w, gate, h0)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(h, [w, gate, h0], up)))
    for k, only in enumerate((w, gate, h0)):  # the others need none
        args = [t if t is only else t.detach() for t in (w, gate, h0)]
        assert torch.equal(first[k], torch.autograd.grad(work(*args), [only], up)[0])
        assert torch.equal(first[k], torch.autograd.grad(work(w, gate, h0), [only], up)[0])
    x = S.embed(w, ids).detach()
    h = S.gated_scan(gate, x, off)[0]
    x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, [gate], up)
    # h0 without offsets
    g3, x3, h3 = gate.detach().view(3, 100, D).requires_grad_(True), x.view(3, 100, D), h0.detach().requires_grad_(True)
    dg, dh = torch.autograd.grad(S.gated_scan(g3, x3, h0=h3)[0], [g3, h3], up.view(3, 100, D))
    even = torch.tensor([0, 100, 200, 300]).cuda()
    dg2, dh2 = torch.autograd.grad(S.gated_scan(gate, x, even, h0)[0], [gate, h0], up)
    assert torch.equal(dg.view(N, D), dg2) and torch.equal(dh, dh2)


def test_two_threads_at_once():
    import threading
    g = gen(42)
    jobs = [(torch.randn(40, 64, generator=g).cuda().requires_grad_(True), torch.randint(0, 40, (9000,), generator=g).cuda(),
             torch.randn(9000, 64, generator=g).cuda()) for _ in range(4)]

    def work(w, ids, up):
        return torch.autograd.grad(S.gated_scan(up.view(3, 3000, 64), S.embed(w, ids).view(3, 3000, 64))[0], [w], up.view(3, 3000, 64))[0]

    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    got = [None] * len(jobs)

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k] = work(*jobs[k])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(k,)) for k in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_operators_in_inference_mode():
    g = gen(40)
    w, ids = torch.randn(5, 8, generator=g).cuda(), torch.tensor([4, 0, 9], device="cuda")
    gate, x = torch.randn(3, 8, generator=g).cuda().requires_grad_(True), torch.randn(3, 8, generator=g).cuda()
    off = torch.tensor([0, 1, 3], device="cuda")
    with torch.no_grad():
        state = torch.zeros(3, 8, device="cuda")
        want = [S.embed(w, ids), S.gated_scan(gate, x, off)[0], S.gated_step(gate, x, state), dvae_amd.optim.orthogonalize(w, out=torch.empty_like(w))]
    with torch.inference_mode():
        mine = torch.zeros(3, 8, device="cuda")
        got = [S.embed(w, ids), S.gated_scan(gate, x, off)[0], S.gated_step(gate, x, mine), dvae_amd.optim.orthogonalize(w, out=torch.empty_like(w))]
        assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(state, mine)
    version = state._version
    with torch.no_grad():
        S.gated_step(gate, x, state)
    assert state._version > version  # autograd sees that the state was written


def test_refusals_on_the_device():
    w, ids = torch.randn(4, 8).cuda(), torch.tensor([1, 2], device="cuda")
    for bad in (lambda: S.embed(w, ids.float()), lambda: S.embed(w, ids.cpu()), lambda: S.embed(w.t(), ids), lambda: S.embed(w[:0], ids),
                lambda: S.embed(w[:, :0], ids), lambda: S.embed(w[:1].expand(4, 8), ids)):
        with pytest.raises(ValueError):
            bad()
    g, off = torch.randn(6, 8).cuda(), torch.tensor([0, 6], device="cuda")
    for bad in (lambda: S.gated_scan(g, g.half(), off), lambda: S.gated_scan(g, g[:5], off), lambda: S.gated_scan(g, g, off.float()),
                lambda: S.gated_scan(g, g, off[:0]), lambda: S.gated_scan(g, g, off[None]), lambda: S.gated_scan(g, g, off.cpu()),
                lambda: S.gated_scan(g, g, off, torch.zeros(2, 8).cuda()), lambda: S.gated_scan(g, g, off, torch.zeros(1, 8).cuda().half()),
                lambda: S.gated_scan(g[:, :0], g[:, :0], off), lambda: S.gated_scan(g, g)):
        with pytest.raises(ValueError):
            bad()
    st = torch.zeros(9, 8).cuda()
    for bad in (lambda: S.gated_step(g, g, st.half()), lambda: S.gated_step(g, g, st[:, :7]), lambda: S.gated_step(g, g, st[:5]),
                lambda: S.gated_step(g, g, st, off), lambda: S.gated_step(g, g, st.t().contiguous().t()), lambda: S.gated_step(g, g, st.cpu()),
                lambda: S.gated_step(g.clone().requires_grad_(True), g, st), lambda: S.gated_step(g, g, st[:1].expand(9, 8))):
        with pytest.raises(ValueError):
            bad()
    assert not st.any()


def test_a_training_step_of_a_sequence_encoder():
    """lookup -> projection -> recurrence -> readout -> loss, its gradients, and the orthogonalised update of the projection,
    against the same in 64 bits.  Five stages, each off by at most 200 u of its sums of absolute values, which exceed the
    sums themselves by less than 10 here: 10^4 u relative."""
    g = gen(20)
    V, E, D, lengths = 40, 24, 32, [5, 0, 70, 1, 33]
    off = offsets_of(lengths)
    N = off[-1]
    table, proj, out = torch.randn(V, E, generator=g), torch.randn(E, 2 * D, generator=g) / 5, torch.randn(D, 6, generator=g)
    ids = torch.randint(-1, V, (N,), generator=g)

    def loss_of(table, proj, out, lookup, scan):
        both = lookup(table) @ proj
        h, last = scan(both[:, :D], both[:, D:])
        logp = torch.log_softmax(last @ out, 1)
        return (h * h).mean() - logp[:, 2].sum()

    leaves = [t.cuda().requires_grad_(True) for t in (table, proj, out)]
    loss = loss_of(*leaves, lambda t: S.embed(t, ids.cuda(), E ** 0.5), lambda a, b: S.gated_scan(a, b, torch.tensor(off).cuda()))
    got = torch.autograd.grad(loss, leaves)
    update = dvae_amd.optim.orthogonalize(got[1])

    def lookup64(t):
        return t[ids.clamp(min=0)] * E ** 0.5 * (ids >= 0)[:, None]

    def scan64(gate, x):
        hs, lasts = [], []
        for s in range(len(lengths)):
            h = torch.zeros(D, dtype=torch.float64)
            for t in range(off[s], off[s + 1]):
                h = torch.sigmoid(gate[t]) * h + torch.sigmoid(-gate[t]) * x[t]
                hs.append(h)
            lasts.append(h)
        return torch.stack(hs), torch.stack(lasts)

    leaves64 = [t.double().requires_grad_(True) for t in (table, proj, out)]
    want = torch.autograd.grad(loss_of(*leaves64, lookup64, scan64), leaves64)
    for a, b in zip(got, want):
        assert float((a.double().cpu() - b).norm() / b.norm()) < 1e4 * U
    x = got[1].double().cpu()  # the update of the gradient that the device has
    x = x / x.norm()
    for _ in range(5):
        s = x @ x.t()
        x = 3.4445 * x + (-4.7750 * s + 2.0315 * (s @ s)) @ x
    assert float((update.double().cpu() - x).norm() / x.norm()) < 341 * 16 * 2.0 ** -22


def test_rows_and_sides_past_32_bits_are_refused():
    n = 2 ** 32 + 5  # would arrive as 5
    one = torch.zeros(1, 1, device="cuda")
    with pytest.raises(dvae_amd._lib.DvaeHipError, match="rows"):
        S.gated_step(one.expand(n, 1), one.expand(n, 1), torch.empty(n, 1, device="cuda"))  # 17 GB, not touched
    with pytest.raises(ValueError, match="32768"):
        dvae_amd.optim.orthogonalize(one.expand(n, 1))


def test_forward_mode_is_refused_not_dropped():
    import torch.autograd.forward_ad as fwd
    w, ids = torch.randn(4, 8).cuda(), torch.tensor([1, 2], device="cuda")
    gate, off = torch.randn(6, 8).cuda(), torch.tensor([0, 6], device="cuda")
    for call in (lambda t: S.embed(t[:4], ids), lambda t: S.gated_scan(t, gate, off)[0], lambda t: S.gated_scan(gate, t, off)[0],
                 lambda t: S.gated_step(t, gate, gate.clone()), lambda t: dvae_amd.optim.orthogonalize(t)):
        with fwd.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            call(fwd.make_dual(gate.clone(), gate))
        with fwd.dual_level():
            call(gate)  # no tangent: as ever
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(call, (gate,), (gate,))
    wl = w.clone().requires_grad_(True)
    out = S.embed(wl, ids)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):  # a tangent of the upstream gradient
        torch.autograd.grad(out, [wl], fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_views_of_negated_elements():
    """z.conj().imag holds -imag(z) as imag(z) and a mark"""
    g = gen(50)

    def negated(*shape):
        z = torch.complex(torch.randn(*shape, generator=g), torch.randn(*shape, generator=g)).cuda()
        assert z.conj().imag.is_neg()
        return z.conj().imag

    ids, off = torch.tensor([1, 0, 4, -1], device="cuda"), torch.tensor([0, 2, 5], device="cuda")
    for D in (1, 6):
        w, gate, x, h0, dh, dlast = negated(5, D), negated(5, D), negated(5, D), negated(2, D), negated(5, D), negated(2, D)
        plainly = [t.clone().resolve_neg() for t in (w, gate, x, h0, dh, dlast)]

        def work(w, gate, x, h0, dh, dlast):
            w, gate, x, h0 = (t.detach().requires_grad_(True) for t in (w, gate, x, h0))
            e = S.embed(w, ids)
            h, last = S.gated_scan(gate, x, off, h0)
            out = [e, *torch.autograd.grad(e, [w], dh[:4]), h, last, *torch.autograd.grad([h, last], [gate, x, h0], [dh, dlast])]
            state = torch.ones(5, D, device="cuda")
            with torch.no_grad():
                return out + [S.gated_step(gate, x, state), state, dvae_amd.optim.orthogonalize(x)]

        if D == 1:  # (rows whose elements do not lie side by side are refused in a table)
            assert all(torch.equal(a, b) for a, b in zip(work(w, gate, x, h0, dh, dlast), work(*plainly)))
        else:
            assert all(torch.equal(a, b) for a, b in zip(work(plainly[0], gate, x, h0, dh, dlast), work(*plainly)))
    state = negated(5, 1)
    with pytest.raises(ValueError, match="negated"):
        S.gated_step(torch.ones(5, 1, device="cuda"), torch.ones(5, 1, device="cuda"), state)
    with pytest.raises(ValueError, match="negated"):
        dvae_amd.optim.orthogonalize(torch.ones(5, 1, device="cuda"), out=state)


def test_gated_step_on_rows_of_the_pool_itself():
    g = gen(51)
    P, D = 20000, 96  # more rows than run at a time
    pool, gate = torch.randn(P, D, generator=g).cuda(), torch.randn(P, D, generator=g).cuda()
    slots = torch.arange(P).flip(0).cuda()
    want = pool.clone()
    h = S.gated_step(gate, pool, want, slots)
    got = pool.clone()
    assert torch.equal(S.gated_step(gate, got, got, slots), h) and torch.equal(got, want)
    want = pool.clone()
    h = S.gated_step(pool[:5000], gate[:5000], want, slots[:5000])
    got = pool.clone()
    assert torch.equal(S.gated_step(got[:5000], gate[:5000], got, slots[:5000]), h) and torch.equal(got, want)
    both = torch.cat([pool, gate], 1)  # states and gates side by side, in one range of addresses
    h = S.gated_step(gate, pool.clone(), pool, slots)
    assert torch.equal(S.gated_step(both[:, D:], both[:, :D], both[:, :D], slots), h) and torch.equal(both[:, :D], pool)
    assert torch.equal(both[:, D:], gate)
    parts = torch.cat([want, gate, gate], 1)  # states, gates and candidates beside each other, at an odd place, read where they lie
    wide = torch.zeros(P, 3 * D + 1, device="cuda")
    wide[:, 1:] = parts
    for flip in (False, True):
        st, ga, xx = want.clone(), gate.clone(), gate.clone()
        h = S.gated_step(ga, xx, st, slots)
        cols = [wide[:, 1:D + 1], wide[:, D + 1:2 * D + 1], wide[:, 2 * D + 1:]]
        wide[:, 1:] = parts
        if flip:
            cols = cols[::-1]
            cols[0].copy_(want), cols[1].copy_(gate), cols[2].copy_(gate)
        assert torch.equal(S.gated_step(cols[1], cols[2], cols[0], slots), h) and torch.equal(cols[0], st)
        assert torch.equal(cols[1], gate) and torch.equal(cols[2], gate)
