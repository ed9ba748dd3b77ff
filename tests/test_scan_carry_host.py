"""That the cases of test_gpu_scan_range see what a tile of rows hands to the next one: the walk over tiles as the kernels do it,
in float32 on the CPU, with and without mistakes in what is carried."""
import pytest
import torch

from test_gpu_scan_range import LONG, long_bounds, long_memory
from test_gpu_sequence import plain_scan


def tiled(gate, x, off, h0, dh, dlast, rows, mistake):
    """(h, G) by tiles of `rows` rows; every tile is a map s -> A s + B of what flows into it.
    mistake: "no A s", "one tile late" (the state before the previous tile) or None"""
    N = x.shape[0]
    z, omz = torch.sigmoid(gate), torch.sigmoid(-gate)
    start = {off[s]: s for s in range(len(off) - 1) if off[s] < off[s + 1]}
    end = {off[s + 1] - 1: s for s in range(len(off) - 1) if off[s] < off[s + 1]}
    inside = torch.zeros(N, dtype=torch.bool)
    for s in range(len(off) - 1):
        inside[off[s]:off[s + 1]] = True

    def over_tiles(order, step):
        """step(t, s): row t with s flowing in -> (what the row holds, what flows out); linear in s"""
        out, flows = torch.zeros_like(x), [torch.zeros_like(x[0])]
        tiles = [order[i:i + rows] for i in range(0, N, rows)]
        for n, tile in enumerate(tiles):
            held = flows[-2] if mistake == "one tile late" and n > 0 else flows[-1]
            if mistake == "no A s" and n > 0:  # the tile before hands on its B alone
                held = torch.zeros_like(x[0])
                for t in tiles[n - 1]:
                    held = step(t, held)[1]
            flow = held
            for t in tile:
                out[t], flow = step(t, flow)
            flows.append(flow)
        return out

    def forward(t, s):
        s = h0[start[t]] if t in start else s
        s = z[t] * s + omz[t] * x[t] if inside[t] else s
        return (s if inside[t] else torch.zeros_like(s)), s

    def backward(t, c):
        if not inside[t]:
            return torch.zeros_like(c), c
        G = dh[t] + (dlast[end[t]] if t in end else 0) + c
        return G, (torch.zeros_like(c) if t in start else z[t] * G)

    return over_tiles(list(range(N)), forward), over_tiles(list(range(N))[::-1], backward)


@pytest.mark.parametrize("dim", [1, 66])
@pytest.mark.parametrize("k", range(len(LONG)))
def test_the_long_cases_see_what_is_carried_from_tile_to_tile(k, dim):
    off, gate, x, h0, dh, dlast = long_memory(k, dim, "fp32")
    ref = plain_scan(gate.double(), x.double(), off, h0.double(), dh.double(), dlast.double())
    tol_h, tol_G = long_bounds(off, gate, ref[5])
    omz = torch.sigmoid(-gate.double())

    begin = [(s, off[s]) for s in range(len(off) - 1) if off[s] < off[s + 1]]

    def errors(rows, mistake):
        """largest errors of h, dx and dh0, in tolerances"""
        h, G = tiled(gate, x, off, h0, dh, dlast, rows, mistake)
        dh0 = max(float(((torch.sigmoid(gate[t]) * G[t]).double() - ref[4][s]).abs().div(tol_G).max()) for s, t in begin)
        return (float((h.double() - ref[0]).abs().div(tol_h).max()),
                float((omz * G.double() - ref[3]).abs().div(tol_G + 4 * 2.0 ** -24 * ref[5]).max()), dh0)

    assert max(errors(64, None)) <= 1
    for rows in (64, 128):
        for mistake in ("no A s", "one tile late"):
            wrong = errors(rows, mistake)
            assert wrong[0] > 3 and max(wrong[1:]) > 3, (rows, mistake, wrong)  # (dx of a channel that keeps all is small)
