"""Sequence operators on the HIP library: a token table and a gated linear recurrence over packed sequences.

  embed        rows of a table looked up by tokens, times a scale; the gradient sums the rows of equal tokens
  gated_scan   h_t = z_t h_{t-1} + (1 - z_t) x_t, z = sigmoid(gate), along sequences of any lengths, differentiable
  gated_step   the same for one token of each sequence, the states kept in a pool and updated in place (serving)

The DAG model keeps its own paths (at most 32 vertex types as a table inside the GRU kernels, chains of at most 64
vertices); these are for encoders of long or many token sequences beside it -- the reference's sequence baselines
(models.py:18-338) run on one-hot inputs and nn.GRU.  Matrices are float32, bfloat16 or float16, the states of the
recurrence always float32.  Like the rest of the package there is no CPU or PyTorch fallback.
"""
import torch

from . import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # DVAE_F32, DVAE_BF16, DVAE_F16


def _need(cond, text):
    if not cond:
        raise ValueError(text)


def _matrix(t, name, dims):
    """a floating-point matrix (or batch of them) on a HIP device; returns the element type code of the C-ABI"""
    _need(torch.is_tensor(t) and t.dim() == dims, "%s must be a tensor with %d dimensions" % (name, dims))
    _need(t.dtype in DTYPES, "%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))
    if not t.is_cuda:
        raise _lib.DvaeHipError("%s is on %s; the operator only runs on a HIP device. There is no CPU fallback." % (name, t.device))
    return DTYPES[t.dtype]


def _index(t, name, device):
    _need(torch.is_tensor(t) and t.dtype in (torch.int32, torch.int64), "%s must be an int32 or int64 tensor" % name)
    _need(t.device == device, "%s is on %s, the matrices on %s" % (name, t.device, device))
    return t.contiguous()


def _rows(t):
    """(t, row stride) of a [N, D] matrix whose elements lie side by side in a row; other layouts are copied"""
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and 0 < t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _flat_rows(t):
    """[N, D] stays; [B, T, D] becomes its B T rows: a view where the rows have one stride, else a copy"""
    if t.dim() == 2:
        return _rows(t)
    B, T, D = t.shape
    if B == 1 or T == 0 or t.stride(0) == T * t.stride(1):
        return _rows(t.as_strided((B * T, D), (t.stride(1), t.stride(2))))
    if T == 1:
        return _rows(t[:, 0])
    return _rows(t.reshape(B * T, D))


class _On(object):
    """the device of the operands as the current one while the library enqueues on its current stream"""

    def __init__(self, device):
        self.index = device.index
        self.guard = None

    def __enter__(self):
        if self.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


def _workspace(n_bytes, device, what):
    if n_bytes < 0:
        _lib.check(-1, what)
    return torch.empty(n_bytes, dtype=torch.uint8, device=device)


# ------------------------------------------------------------------------------------------------------------------ embed

class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale):
        lib = _lib.load()
        V, D = weight.shape
        out = torch.empty(tuple(ids.shape) + (D,), dtype=weight.dtype, device=weight.device)
        with _On(weight.device) as stream:
            _lib.check(lib.dvae_embed_fwd(weight.data_ptr(), weight.stride(0) if V > 1 else D, ids.data_ptr(),
                                          int(ids.dtype == torch.int64), out.data_ptr(), ids.numel(), V, D, scale,
                                          DTYPES[weight.dtype], stream), "dvae_embed_fwd")
        ctx.save_for_backward(ids)
        ctx.table, ctx.scale = (V, D), scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        lib = _lib.load()
        ids, = ctx.saved_tensors
        V, D = ctx.table
        n = ids.numel()
        dout, ld = _rows(dout.reshape(n, D))
        dw = torch.empty(V, D, dtype=dout.dtype, device=dout.device)
        ws = _workspace(lib.dvae_embed_bwd_ws_bytes(n, V, D), dout.device, "dvae_embed_bwd_ws_bytes")
        with _On(dout.device) as stream:
            _lib.check(lib.dvae_embed_bwd(dout.data_ptr(), ld, ids.data_ptr(), int(ids.dtype == torch.int64), dw.data_ptr(),
                                          ws.data_ptr(), n, V, D, ctx.scale, DTYPES[dout.dtype], stream), "dvae_embed_bwd")
        return dw, None, None


def embed(weight, ids, scale=1.0):
    """scale * weight[ids]: `weight` [V, D] with its elements side by side in a row, `ids` int32 / int64 of any shape;
    returns [*ids.shape, D].  A token outside [0, V) (padding) gives a row of zeros and takes no part in the gradient.
    The gradient of `weight` is dense, summed in float32 in the order of the tokens' positions and rounded once; it does
    not vary from run to run."""
    _matrix(weight, "weight", 2)
    V, D = weight.shape
    _need(V > 0 and D > 0, "weight is empty")
    _need((D == 1 or weight.stride(1) == 1) and (V == 1 or weight.stride(0) >= D), "the elements of a row of weight must lie side by side")
    return _EmbedFn.apply(weight, _index(ids, "ids", weight.device), float(scale))


# ------------------------------------------------------------------------------------------------------------- recurrence

class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, offsets, h0, seqs):
        lib = _lib.load()
        g, ld_g = _flat_rows(gate)
        y, ld_y = _flat_rows(x)
        n, D = g.shape
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        last = torch.empty(seqs, D, dtype=torch.float32, device=x.device)
        states = None
        if any(ctx.needs_input_grad[i] for i in (0, 1, 3)):
            states = torch.empty(lib.dvae_scan_state_floats(n, D), dtype=torch.float32, device=x.device)
        ws = _workspace(lib.dvae_scan_ws_bytes(n, D), x.device, "dvae_scan_ws_bytes")
        with _On(x.device) as stream:
            _lib.check(lib.dvae_scan_fwd(g.data_ptr(), ld_g, y.data_ptr(), ld_y, _lib.ptr(offsets),
                                         int(offsets is not None and offsets.dtype == torch.int64), _lib.ptr(h0), h.data_ptr(),
                                         last.data_ptr(), _lib.ptr(states), ws.data_ptr(), n, seqs, D, DTYPES[x.dtype], stream),
                       "dvae_scan_fwd")
        ctx.save_for_backward(gate, x, offsets, h0)
        ctx.states, ctx.seqs = states, seqs
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        lib = _lib.load()
        gate, x, offsets, h0 = ctx.saved_tensors
        g, ld_g = _flat_rows(gate)
        y, ld_y = _flat_rows(x)
        n, D = g.shape
        ld_dh = 0
        if dh is not None:
            dh, ld_dh = _flat_rows(dh)
        if dlast is not None:
            dlast = dlast.contiguous()
        dgate = torch.empty(gate.shape, dtype=x.dtype, device=x.device)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dh0 = torch.empty(ctx.seqs, D, dtype=torch.float32, device=x.device) if ctx.needs_input_grad[3] else None
        ws = _workspace(lib.dvae_scan_ws_bytes(n, D), x.device, "dvae_scan_ws_bytes")
        with _On(x.device) as stream:
            _lib.check(lib.dvae_scan_bwd(g.data_ptr(), ld_g, y.data_ptr(), ld_y, _lib.ptr(offsets),
                                         int(offsets is not None and offsets.dtype == torch.int64), _lib.ptr(h0),
                                         ctx.states.data_ptr(), _lib.ptr(dh), ld_dh, _lib.ptr(dlast), dgate.data_ptr(),
                                         dx.data_ptr(), _lib.ptr(dh0), ws.data_ptr(), n, ctx.seqs, D, DTYPES[x.dtype], stream),
                       "dvae_scan_bwd")
        return dgate, dx, None, dh0, None


def gated_scan(gate, x, offsets=None, h0=None):
    """h_t = z_t h_{t-1} + (1 - z_t) x_t with z = sigmoid(gate), per channel, along every sequence -> (h, last).

    offsets [S + 1] (int32 / int64, on the device, not decreasing): gate and x are [N, D] and sequence s is the rows
    offsets[s] : offsets[s + 1]; empty sequences are allowed, rows of no sequence give zeros in h and in the gradients.
    Values outside [0, N] count as the nearer end.  Without offsets gate and x are [S, T, D].
    h0 [S, D] float32: the state before each sequence (default zeros).  last [S, D] float32: the state after it.

    gate and x may be the two halves of one projection's output: rows of any stride are read in place.  Differentiable in
    gate, x and h0; the states are float32 inside, h and the gradients of gate and x are rounded once to x's type."""
    dims = 2 if offsets is not None else 3
    _matrix(gate, "gate", dims)
    _matrix(x, "x", dims)
    _need(gate.dtype == x.dtype and gate.device == x.device, "gate and x differ in type or device")
    _need(gate.shape == x.shape, "gate has the shape %s, x %s" % (tuple(gate.shape), tuple(x.shape)))
    D = x.shape[-1]
    _need(D > 0, "gate and x have no channels")
    if offsets is not None:
        offsets = _index(offsets, "offsets", x.device)
        _need(offsets.dim() == 1 and offsets.numel() >= 1, "offsets must have one dimension and at least one value")
        seqs = offsets.numel() - 1
    else:
        seqs = x.shape[0]
    if h0 is not None:
        _need(torch.is_tensor(h0) and h0.dtype == torch.float32 and h0.device == x.device and tuple(h0.shape) == (seqs, D),
              "h0 must be a float32 tensor of shape (%d, %d) on %s" % (seqs, D, x.device))
        h0 = h0.contiguous()
    return _ScanFn.apply(gate, x, offsets, h0, seqs)


def gated_step(gate, x, state, slots=None):
    """One token of each of B sequences: gate, x [B, D]; returns h [B, D] in x's type and updates `state` [P, D] (float32)
    in place at the rows `slots` [B] (int32 / int64; default: row b has state b).  A slot outside [0, P) marks a padding
    row: its h is zero and no state changes.  Rows that name the same slot advance it one after the other, in their order.
    For serving: not differentiable, inputs that need gradients are refused outside torch.no_grad()."""
    code = _matrix(gate, "gate", 2)
    _matrix(x, "x", 2)
    _need(gate.dtype == x.dtype and gate.device == x.device and gate.shape == x.shape, "gate and x differ in type, device or shape")
    B, D = x.shape
    _need(D > 0, "gate and x have no channels")
    _need(torch.is_tensor(state) and state.dtype == torch.float32 and state.device == x.device and state.dim() == 2 and
          state.shape[1] == D, "state must be a float32 tensor of shape (P, %d) on %s" % (D, x.device))
    P = state.shape[0]
    _need((D == 1 or state.stride(1) == 1) and (P <= 1 or state.stride(0) >= D), "the elements of a row of state must lie side by side")
    if torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or state.requires_grad):
        raise ValueError("gated_step is not differentiable: call it under torch.no_grad(), or use gated_scan")
    if slots is not None:
        slots = _index(slots, "slots", x.device)
        _need(tuple(slots.shape) == (B,), "slots must have the shape (%d,)" % B)
    else:
        _need(B <= P, "%d rows, but %d states" % (B, P))
    g, ld_g = _rows(gate)
    y, ld_y = _rows(x)
    h = torch.empty(B, D, dtype=x.dtype, device=x.device)
    with _On(x.device) as stream:
        _lib.check(_lib.load().dvae_scan_step(g.data_ptr(), ld_g, y.data_ptr(), ld_y, state.data_ptr(),
                                              state.stride(0) if P > 1 else D, P, _lib.ptr(slots),
                                              int(slots is not None and slots.dtype == torch.int64), h.data_ptr(), B, D, code,
                                              stream), "dvae_scan_step")
    torch.autograd.graph.increment_version(state)
    return h
