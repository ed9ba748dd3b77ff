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
