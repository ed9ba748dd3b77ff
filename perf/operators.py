"""Cases that measure the sequence operators and the orthogonalised update of the framework.

Three groups of operators, each in a plain form (elementary torch operations in 32 bits, rounded once at the end) and as
the framework's own call:

  embed   rows of a table looked up by tokens, times a scale; its gradient sums the rows of equal tokens
          (dvae_amd.sequence.embed)
  scan    the gated linear recurrence h_t = z_t h_{t-1} + (1 - z_t) x_t, z = sigmoid(gate), along packed sequences, with
          its backward pass (dvae_amd.sequence.gated_scan), and its form for one token per sequence with the states
          kept in a pool (dvae_amd.sequence.gated_step)
  ortho   a set of matrices orthogonalised by Newton-Schulz products (dvae_amd.optim.orthogonalize)
"""
import math

import torch

own = False  # False: run() computes the plain forms; True: it calls the framework

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # the quintic p(s) = a s + b s^3 + c s^5 of every Newton-Schulz step
STEPS = 5


def listed():
    cfg2 = "1503x501 1503x501 1503x501 56x501 56x501 501x56 1002x501 2004x1002 501x509 501x509 501x509 501x509 501x1002"
    return [
        # the vertex types of one batch of 32 graphs of 8 vertices: latency counts
        {"name": "embed 256 of 8 fp32", "op": "embed", "train": False, "n": 256, "vocab": 8, "dim": 501, "dtype": "fp32", "skew": 0.5, "pad": 0.0},
        # the types of a batch of 1024 graphs of 8 vertices in training: few rows, each with a thousand tokens
        {"name": "embed train 8192 of 8 fp32", "op": "embed", "train": True, "n": 8192, "vocab": 8, "dim": 501, "dtype": "fp32", "skew": 0.5, "pad": 0.0},
        # a training batch of text-like tokens: a large table, a few hot rows, many that no token names, some padding
        {"name": "embed train 65521 of 50001 bf16", "op": "embed", "train": True, "n": 65521, "vocab": 50001, "dim": 1024, "dtype": "bf16", "skew": 1.0, "pad": 0.02},
        # the vertices of 32 small graphs as packed sequences of different lengths, in training: latency counts
        {"name": "scan train 32 short fp32", "op": "scan", "train": True, "seqs": 32, "rows": 331, "dim": 501, "dtype": "fp32", "h0": False},
        # a training batch of ragged sequences that go on from given states
        {"name": "scan train 24 ragged bf16", "op": "scan", "train": True, "seqs": 24, "rows": 40003, "dim": 1024, "dtype": "bf16", "h0": True},
        # two long sequences in training: nearly all of the parallel work has to come from the time axis
        {"name": "scan train 2 long bf16", "op": "scan", "train": True, "seqs": 2, "rows": 131072, "dim": 1024, "dtype": "bf16", "h0": False},
        # reading in one long prompt before answering: forward alone
        {"name": "scan prompt 32768 fp16", "op": "scan", "train": False, "seqs": 1, "rows": 32768, "dim": 1024, "dtype": "fp16", "h0": False},
        # the next token of 32 sequences: latency counts
        {"name": "step 32 fp32", "op": "step", "rows": 32, "pool": 32, "dim": 501, "dtype": "fp32"},
        # the next token of a large serving batch, its states scattered over a pool
        {"name": "step 2048 bf16", "op": "step", "rows": 2048, "pool": 4096, "dim": 1024, "dtype": "bf16"},
        # one hidden-to-hidden matrix: every product is small and the fifteen of them depend on each other
        {"name": "ortho 501x501 fp32", "op": "ortho", "shapes": "501x501", "dtype": "fp32"},
        # all the matrices of the ENAS model (hidden size 501, latent size 56), as an optimiser step has them
        {"name": "ortho cfg2 fp32", "op": "ortho", "shapes": cfg2, "dtype": "fp32"},
        # one large weight
        {"name": "ortho 4096x4096 bf16", "op": "ortho", "shapes": "4096x4096", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "scan", "step", "ortho"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "embed":
        return {"op": op, "train": rng.random() < 0.7, "n": _log(rng, 1, 65536), "vocab": _log(rng, 2, 50000),
                "dim": _log(rng, 8, 1024), "dtype": dtype, "skew": rng.choice([0.0, 0.5, 1.0]), "pad": rng.choice([0.0, 0.02, 0.5])}
    if op == "scan":
        rows = _log(rng, 1, 100000)
        return {"op": op, "train": rng.random() < 0.7, "seqs": min(_log(rng, 1, 128), rows), "rows": rows, "dim": _log(rng, 8, 1024),
                "dtype": dtype, "h0": rng.random() < 0.5}
    if op == "step":
        rows = _log(rng, 1, 2048)
        return {"op": op, "rows": rows, "pool": rows + _log(rng, 1, 4096), "dim": _log(rng, 8, 2048), "dtype": dtype}
    shapes = []
    for _ in range(_log(rng, 1, 16)):
        shapes.append("%dx%d" % (_log(rng, 8, 2048), _log(rng, 8, 2048)))
    return {"op": op, "shapes": " ".join(shapes), "dtype": dtype}


# ----------------------------------------------------------------------------------------------------------------- inputs

def _lengths(case, g, dev):
    """`seqs` lengths that sum to `rows`: spread by a factor of about ten; with more than eight sequences the second is empty"""
    S, N = case["seqs"], case["rows"]
    w = torch.rand(S, generator=g, device=dev, dtype=torch.float64) * 2.3
    w = w.exp()
    if S > 8:
        w[1] = 0
    edge = (w.cumsum(0) / w.sum() * N).round().long()
    edge[-1] = N
    return torch.cat([torch.zeros(1, dtype=torch.long, device=dev), edge])


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": dict(case)}
    if case["op"] == "embed":
        n, V, D = case["n"], case["vocab"], case["dim"]
        p = (torch.arange(V, device=dev, dtype=torch.float64) + 1) ** -case["skew"]
        p = p[torch.randperm(V, generator=g, device=dev)].cumsum(0)
        u = torch.rand(n, generator=g, device=dev, dtype=torch.float64) * p[-1]
        ids = torch.searchsorted(p, u).clamp_(max=V - 1)
        if case["pad"]:
            ids[torch.rand(n, generator=g, device=dev) < case["pad"]] = -1  # padding: a row of zeros, no gradient
        s.update(ids=ids.to(torch.int32), weight=(normal(V, D) / math.sqrt(D)).to(dt), scale=math.sqrt(D))
        if case["train"]:
            s.update(dout=normal(n, D).to(dt))
            s["weight"].requires_grad_(True)
    elif case["op"] in ("scan", "step"):
        rows, D = case["rows"], case["dim"]
        # how long a channel remembers differs from channel to channel: retention 0.3 to 0.998
        bias = torch.rand(D, generator=g, device=dev) * 7 - 1
        both = torch.empty(rows, 2 * D, device=dev, dtype=dt)  # one projection gives gates and candidates side by side
        both[:, :D] = (normal(rows, D) + bias).to(dt)
        both[:, D:] = torch.tanh(normal(rows, D)).to(dt)
        s.update(both=both, gate=both[:, :D], x=both[:, D:])
        if case["op"] == "step":
            s.update(state=normal(case["pool"], D).mul_(0.5), slots=torch.randperm(case["pool"], generator=g, device=dev)[:rows].to(torch.int32))
            return s
        s.update(offsets=_lengths(case, g, dev).to(torch.int32), h0=normal(case["seqs"], D).mul_(0.5) if case["h0"] else None)
        if case["train"]:
            s.update(dh=normal(rows, D).to(dt), dlast=normal(case["seqs"], D))
            s["gate"].requires_grad_(True)
            s["x"].requires_grad_(True)
            if s["h0"] is not None:
                s["h0"].requires_grad_(True)
    else:
        s["mats"] = []
        for m, n in _shapes(case):
            # an averaged gradient: noise, and a few directions that carry most of it
            r = min(4, m, n)
            s["mats"].append(((normal(m, n) + normal(m, r) @ normal(r, n) * 3) * 1e-3).to(dt))
    return s


# ------------------------------------------------------------------------------------------------------------- plain forms

def _plain_embed(weight, ids, scale):
    ok = (ids >= 0) & (ids < weight.shape[0])
    rows = weight[ids.long().clamp(0, weight.shape[0] - 1)].float()
    return (rows * scale * ok[:, None]).to(weight.dtype)


def _plain_embed_grad(weight, ids, scale, dout):
    ok = (ids >= 0) & (ids < weight.shape[0])
    dw = torch.zeros(weight.shape, device=weight.device, dtype=torch.float32)
    dw.index_add_(0, ids.long().clamp(0, weight.shape[0] - 1), dout.float() * ok[:, None])
    return (dw * scale).to(weight.dtype)


def _linear_scan(a, b):
    """y_t = a_t y_{t-1} + b_t by doubling, in place; where a sequence begins, a_t is 0"""
    step = 1
    while step < a.shape[0]:
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_scan(gate, x, offsets, h0):
    """h of every row in 32 bits, the last state of every sequence, and what the backward pass uses of them"""
    off = offsets.long()
    begin, length = off[:-1], off[1:] - off[:-1]
    some = (length > 0)[:, None]
    first = begin.clamp(max=gate.shape[0] - 1)
    z = torch.sigmoid(gate.float())
    b = (1 - z) * x.float()
    init = torch.zeros(begin.shape[0], gate.shape[1], device=gate.device) if h0 is None else h0.float()
    b.index_add_(0, first, z[first] * init * some)
    a = z.clone()
    seq = torch.searchsorted(off, torch.arange(gate.shape[0], device=gate.device), right=True) - 1
    starts = begin[seq] == torch.arange(gate.shape[0], device=gate.device)
    a *= ~starts[:, None]
    h = _linear_scan(a, b)
    last = torch.where(some, h[(off[1:] - 1).clamp(min=0)], init)
    return h, last, z, a, starts, seq, init, some


def _plain_scan_grad(x, offsets, dh, dlast, h, z, a, starts, seq, init, some):
    off = offsets.long()
    e = dh.float().index_add(0, (off[1:] - 1).clamp(min=0), dlast.float() * some)
    up = torch.cat([a[1:], torch.zeros_like(a[:1])]).flip(0)  # G_t = e_t + a_{t+1} G_{t+1}, walked from the end
    grad = _linear_scan(up, e.flip(0)).flip(0)
    prev = torch.where(starts[:, None], init[seq], torch.cat([h[:1], h[:-1]]))
    dx = (1 - z) * grad
    dgate = grad * (prev - x.float()) * z * (1 - z)
    first = off[:-1].clamp(max=h.shape[0] - 1)
    dh0 = torch.where(some, grad[first] * z[first], dlast.float())
    return dgate, dx, dh0


def _plain_ortho(g):
    a, b, c = COEFFICIENTS
    x = g.float()
    if x.shape[0] > x.shape[1]:
        x = x.t()
    x = x / x.double().square().sum().sqrt().float()
    for _ in range(STEPS):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    if g.shape[0] > g.shape[1]:
        x = x.t()
    return x.to(g.dtype).contiguous()


# --------------------------------------------------------------------------------------------------------------------- run

def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        from _dvae_pkg import dvae_amd
        if op == "embed":
            if not case["train"]:
                return dvae_amd.sequence.embed(state["weight"], state["ids"], state["scale"])
            out = dvae_amd.sequence.embed(state["weight"], state["ids"], state["scale"])
            return [out.detach()] + list(torch.autograd.grad(out, [state["weight"]], state["dout"]))
        if op == "scan":
            h, last = dvae_amd.sequence.gated_scan(state["gate"], state["x"], state["offsets"], state["h0"])
            if not case["train"]:
                return [h, last]
            wanted = [state["gate"], state["x"]] + ([state["h0"]] if case["h0"] else [])
            return [h.detach(), last.detach()] + list(torch.autograd.grad([h, last], wanted, [state["dh"], state["dlast"]]))
        if op == "step":
            return [dvae_amd.sequence.gated_step(state["gate"], state["x"], state["state"], state["slots"]), state["state"]]
        return dvae_amd.optim.orthogonalize(state["mats"], steps=STEPS, coefficients=COEFFICIENTS)
    with torch.no_grad():
        if op == "embed":
            out = _plain_embed(state["weight"], state["ids"], state["scale"])
            if not case["train"]:
                return out
            return [out, _plain_embed_grad(state["weight"], state["ids"], state["scale"], state["dout"])]
        if op == "scan":
            dt = state["x"].dtype
            h, last, *kept = _plain_scan(state["gate"], state["x"], state["offsets"], state["h0"])
            if not case["train"]:
                return [h.to(dt), last]
            dgate, dx, dh0 = _plain_scan_grad(state["x"], state["offsets"], state["dh"], state["dlast"], h, *kept)
            return [h.to(dt), last, dgate.to(dt), dx.to(dt)] + ([dh0] if case["h0"] else [])
        if op == "step":
            slots = state["slots"].long()
            z = torch.sigmoid(state["gate"].float())
            h = z * state["state"][slots] + (1 - z) * state["x"].float()
            state["state"][slots] = h
            return [h.to(state["x"].dtype), state["state"]]
        return [_plain_ortho(g) for g in state["mats"]]


# -------------------------------------------------------------------------------------------------------------------- work

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "embed":
        n, V, D = case["n"], case["vocab"], case["dim"]
        read = min(n, V) * D * e + 4 * n
        if not case["train"]:
            return {"bytes": read + n * D * e, "flops": n * D}
        return {"bytes": read + n * D * e + n * D * e + V * D * e, "flops": 2 * n * D}
    if case["op"] == "scan":
        n, D, S = case["rows"], case["dim"], case["seqs"]
        states = S * D * 4
        fwd = 3 * n * D * e + states * (2 if case["h0"] else 1) + 4 * (S + 1)
        if not case["train"]:
            return {"bytes": fwd, "flops": 8 * n * D}
        return {"bytes": fwd + 3 * n * D * e + states * (2 if case["h0"] else 1), "flops": 24 * n * D}
    if case["op"] == "step":
        n, D = case["rows"], case["dim"]
        return {"bytes": 3 * n * D * e + 8 * n * D + 4 * n, "flops": 8 * n * D}
    flops = size = 0
    for r, k in _shapes(case):
        m, n = min(r, k), max(r, k)
        # of the two symmetric products (X X^T and its square) one triangle each; the update product in full
        flops += STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)
        size += 2 * m * n * e
    return {"bytes": size, "flops": flops}


# ------------------------------------------------------------------------------------------------------------------- exact

def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        if case["op"] == "embed":
            w, ids = s["weight"].detach().double(), s["ids"].long()
            table = torch.cat([w, torch.zeros_like(w[:1])])  # the last row answers for tokens outside the table
            at = torch.where((ids < 0) | (ids >= w.shape[0]), w.shape[0], ids)
            out = table.index_select(0, at) * s["scale"]
            if not case["train"]:
                return out
            order = torch.argsort(at, stable=True)
            total = torch.cat([torch.zeros_like(w[:1]), (s["dout"].double()[order]).cumsum(0)])
            edge = torch.searchsorted(at[order], torch.arange(w.shape[0] + 1, device=at.device))
            return [out, (total[edge[1:]] - total[edge[:-1]]) * s["scale"]]
        if case["op"] == "step":
            z = 1 / (1 + torch.exp(-s["gate"].double()))
            at = s["slots"].long()
            pool = s["state"].double()
            h = s["x"].double() + z * (pool[at] - s["x"].double())
            return [h, pool.index_copy(0, at, h)]
        if case["op"] == "ortho":
            outs = []
            for g in s["mats"]:
                x = g.double() / g.double().norm()
                wide = x.shape[0] <= x.shape[1]
                for _ in range(STEPS):
                    gram = x @ x.mT if wide else x.mT @ x
                    eye = torch.eye(gram.shape[0], device=x.device, dtype=x.dtype)
                    poly = COEFFICIENTS[0] * eye + gram @ (COEFFICIENTS[1] * eye + COEFFICIENTS[2] * gram)
                    x = poly @ x if wide else x @ poly
                outs.append(x)
            return outs
        return _exact_scan(case, s)


def _chunked(a, b):
    """y_t = a_t y_{t-1} + b_t, y_{-1} = 0, in chunks whose rows are walked one by one, all chunks at once"""
    N, D = a.shape
    C = max(1, int(math.sqrt(N)))
    n = -(-N // C)
    pad = n * C - N
    if pad:
        a = torch.cat([a, torch.zeros(pad, D, device=a.device, dtype=a.dtype)])
        b = torch.cat([b, torch.zeros(pad, D, device=a.device, dtype=a.dtype)])
    a, b = a.view(n, C, D), b.view(n, C, D)
    y, p = torch.empty_like(b), torch.empty_like(a)
    y[:, 0], p[:, 0] = b[:, 0], a[:, 0]
    for t in range(1, C):
        y[:, t] = a[:, t] * y[:, t - 1] + b[:, t]
        p[:, t] = a[:, t] * p[:, t - 1]
    for k in range(1, n):
        y[k] += p[k] * y[k - 1, -1]
    return y.view(n * C, D)[:N]


def _exact_scan(case, s):
    off = s["offsets"].tolist()
    N, D = s["x"].shape
    gate, x = s["gate"].double(), s["x"].double()
    z = 1 / (1 + torch.exp(-gate))
    init = s["h0"].double() if s["h0"] is not None else torch.zeros(len(off) - 1, D, device=x.device, dtype=x.dtype)
    a, b = z.clone(), x - z * x
    prev = torch.empty_like(x)
    for q in range(len(off) - 1):
        if off[q + 1] > off[q]:
            a[off[q]] = 0
            b[off[q]] += z[off[q]] * init[q]
    h = _chunked(a, b)
    prev[1:] = h[:-1]
    last = init.clone()
    for q in range(len(off) - 1):
        if off[q + 1] > off[q]:
            prev[off[q]] = init[q]
            last[q] = h[off[q + 1] - 1]
    if not case["train"]:
        return [h, last]
    e, dh0 = s["dh"].double(), s["dlast"].double().clone()
    back = torch.zeros_like(a)
    back[:-1] = a[1:]
    for q in range(len(off) - 1):
        if off[q + 1] > off[q]:
            e[off[q + 1] - 1] += s["dlast"].double()[q]
    grad = _chunked(back.flip(0), e.flip(0)).flip(0)
    for q in range(len(off) - 1):
        if off[q + 1] > off[q]:
            dh0[q] = grad[off[q]] * z[off[q]]
    found = [h, last, grad * (prev - x) * z * (1 - z), grad - grad * z]
    return found + ([dh0] if case["h0"] else [])
