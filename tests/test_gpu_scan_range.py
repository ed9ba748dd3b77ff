"""The gated recurrence where states, gates and gradients span their range: masks of a type's lowest value, states that stay long.

Tolerances as in test_gpu_sequence: u = 2^-24; M bounds the values of x and h0 and so of every state; a step is off by at most
8 u M and passes older errors on times z <= zmax: 8 u M min(T, 1 / (1 - zmax)) + 32 u M in all, and alike with the gradients'
bound in the place of M on the way back."""
import pytest
import torch

from _dvae_pkg import dvae_amd
from test_gpu_sequence import DT, U, close, gen, plain_scan

S = dvae_amd.sequence
pytestmark = pytest.mark.gpu


def masked(dtype, D=70, N=300):
    """rows whose x is masked with the type's lowest value, each before a row whose gate is closed: nothing of them is left
    behind it.  The masked rows are the last of a wave's rows, of a tile's, and others."""
    dt, g = DT[dtype], gen(3)
    low = torch.finfo(dt).min
    gate = (torch.randn(N, D, generator=g) + 3).clamp(-5, 5).to(dt)
    x = torch.randn(N, D, generator=g).clamp(-3, 3).to(dt)
    rows = torch.tensor([15, 63, 127, 128, 191, 255, 280])
    x[rows], gate[rows] = low, 0
    gate[rows + 1] = low if dtype != "fp16" else -float("inf")  # (sigmoid(-65504) is 0 as well)
    gate[192] = -200.0  # not the lowest value, and closed all the same
    keep = torch.ones(N, dtype=torch.bool)
    keep[rows] = False
    return gate, x, keep, rows


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_masked_rows_leave_nothing_behind_a_closed_gate(dtype):
    gate, x, keep, rows = masked(dtype)
    off = [0, 300]
    ref, last = plain_scan(gate.double(), x.double(), off, None)
    h, mine = S.gated_scan(gate.cuda(), x.cuda(), torch.tensor(off).cuda())
    tol = (8 * 149 + 32) * U * 3.0
    close(h[keep.cuda()], ref[keep], tol, "h")
    close(mine, last, tol, "last")
    close(h[~keep.cuda()], ref[~keep], float(ref[rows].abs().max()) * 64 * U, "masked rows")
    one = S.gated_step(gate[16:17].cuda(), x[16:17].cuda(), h[15:16].float())
    close(one, ref[16:17], tol, "step")


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_gradients_of_masked_rows_are_finite(dtype):
    gate, x, keep, rows = masked(dtype)
    dt, g, off = DT[dtype], gen(4), [0, 300]
    dh = torch.randn(x.shape, generator=g).clamp(-2, 2).to(dt)  # nothing comes back through a closed gate: G = dh in a masked row
    dlast = torch.randn(1, x.shape[1], generator=g)
    ref = plain_scan(gate.double(), x.double(), off, None, dh.double(), dlast.double())
    leaves = [gate.cuda().requires_grad_(True), x.cuda().requires_grad_(True)]
    h, last = S.gated_scan(*leaves, torch.tensor(off).cuda())
    dg, dx = torch.autograd.grad([h, last], leaves, [dh.cuda(), dlast.cuda()])
    big = max(ref[5], 1.0)
    tol_G, tol_h = (8 * 149 + 32) * U * big, (8 * 149 + 32) * U * 3.0
    close(dx, ref[3], tol_G + 4 * U * big, "dx")
    closed = keep.clone()
    closed[:] = False
    closed[rows + 1] = True
    closed[192] = True
    plain = keep & ~closed
    close(dg[plain.cuda()], ref[2][plain], (tol_G * 6 + big * tol_h + 32 * U * big * 6) / 4, "dgate")
    assert not dg[closed.cuda()].any()  # z (1 - z) is 0 in 32 bits, whatever the state before
    # a masked row: G = dh exactly, (prev - x) z (1 - z) off by its roundings alone, a few u relative (and u |h| of prev)
    close(dg[rows.cuda()], ref[2][rows], ref[2][rows].abs() * 32 * U + 2 * tol_h, "dgate of masked rows")


# ------------------------------------------------------------------------------------ states that stay over many tiles of rows

LONG = [([3077], 0, 0), ([1500, 0, 3, 1574], 7, 5), ([2600, 477], 0, 0)]


def long_memory(k, dim, dtype):
    """every channel keeps its own retention between 0.3 and 0.9995; what comes first (h0, early x) and last (dlast) is large.
    More than 20 tiles of rows in either direction."""
    lengths, front, behind = LONG[k]
    dt, g = DT[dtype], gen(10 * k + dim)
    off = [front]
    for n in lengths:
        off.append(off[-1] + n)
    N, Sn = off[-1] + behind, len(lengths)
    z = torch.linspace(0.9995, 0.3, dim).double()
    gate = (torch.log(z / (1 - z)) + 0.1 * torch.randn(N, dim, generator=g)).to(dt)
    x = torch.randn(N, dim, generator=g).clamp(-3, 3)
    x[front:front + 100] = 3 * torch.sign(x[:1])
    h0 = 3 * torch.sign(torch.randn(Sn, dim, generator=g))
    dh, dlast = torch.randn(N, dim, generator=g).to(dt), 30 * torch.sign(torch.randn(Sn, dim, generator=g))
    return off, gate, x.to(dt), h0, dh, dlast


def long_bounds(off, gate, big):
    """what h and last, and G may be off by (the head of the file), channel by channel"""
    mem = (1 / (1 - torch.sigmoid(gate.double()).max(0).values)).clamp(max=max(b - a for a, b in zip(off, off[1:])))
    return (8 * mem + 32) * U * 3.0, (8 * mem + 32) * U * big


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [1, 66, 129])
@pytest.mark.parametrize("k", range(len(LONG)))
def test_states_and_gradients_that_stay_over_many_tiles(k, dim, dtype):
    off, gate, x, h0, dh, dlast = long_memory(k, dim, dtype)
    ref = plain_scan(gate.double(), x.double(), off, h0.double(), dh.double(), dlast.double())
    leaves = [gate.cuda().requires_grad_(True), x.cuda().requires_grad_(True), h0.cuda().requires_grad_(True)]
    h, last = S.gated_scan(leaves[0], leaves[1], torch.tensor(off).cuda(), leaves[2])
    dg, dx, dh0 = torch.autograd.grad([h, last], leaves, [dh.cuda(), dlast.cuda()])
    tol_h, tol_G = long_bounds(off, gate, ref[5])
    close(h, ref[0], tol_h, "h")
    close(last, ref[1], tol_h, "last")
    close(dx, ref[3], tol_G + 4 * U * ref[5], "dx")
    close(dg, ref[2], (tol_G * 6 + ref[5] * tol_h + 32 * U * ref[5] * 6) / 4, "dgate")
    close(dh0, ref[4], tol_G, "dh0")
    alone = S.gated_scan(gate.cuda(), x.cuda(), torch.tensor(off).cuda(), h0.cuda())  # without what the backward pass keeps
    assert torch.equal(alone[0], h) and torch.equal(alone[1], last)


def test_the_gradient_of_h0_comes_back_over_the_whole_sequence():
    g = gen(60)
    T, D = 700, 40
    gate = torch.full((2, T, D), 6.0) + 0.5 * torch.randn(2, T, D, generator=g)
    h0 = torch.zeros(2, D, device="cuda", requires_grad=True)
    h, last = S.gated_scan(gate.cuda(), torch.zeros(2, T, D, device="cuda"), h0=h0)
    dh0, = torch.autograd.grad(last.sum(), [h0])
    want = torch.sigmoid(gate.double()).prod(1)
    assert want.min() > 0.05
    close(dh0, want, (8 * T + 32) * U, "dh0")
