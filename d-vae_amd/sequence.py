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


def _matrix(t, name, dims):
    """a floating-point matrix (or batch of them) on a HIP device; returns the element type code of the C-ABI"""
    if not torch.is_tensor(t) or t.dim() != dims:
        raise ValueError("%s must be a tensor with %d dimensions" % (name, dims))
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError("%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))
    if not t.is_cuda:
        raise _lib.DvaeHipError("%s is on %s; the operator only runs on a HIP device. There is no CPU fallback." % (name, t.device))
    return code


def _index(t, name, device):
    """an index tensor beside the matrices; (contiguous, is it int64)"""
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError("%s must be an int32 or int64 tensor" % name)
    if t.device != device:
        raise ValueError("%s is on %s, the matrices on %s" % (name, t.device, device))
    return t.contiguous()


def _wide(t):
    return 1 if t is not None and t.dtype == torch.int64 else 0


def _rows(t, most=1 << 23):
    """(t, row stride) of a [N, D] matrix whose elements lie side by side in a row; other layouts, and rows more than `most`
    elements apart (the recurrence addresses a few rows with 32-bit offsets), are copied"""
    n, d = t.shape
    s0, s1 = t.stride()
    if d > 1 and s1 != 1 or n > 1 and (0 < s0 < d or s0 > most):
        return t.contiguous(), d
    return t, s0 if n > 1 else d


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


def _enqueue(device, name, *args):
    """calls the library's function `name` with the current stream of `device`, that device being the current one"""
    fn = getattr(_lib.load(), name)
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        _lib.check(rc, name)


def _workspace(n_bytes, device, what):
    if n_bytes < 0:
        _lib.check(-1, what)
    return torch.empty(n_bytes, dtype=torch.uint8, device=device)


def _written(*tensors):
    """the library wrote into these: their autograd versions move as by an in-place operation"""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _once(name):
    if torch.is_grad_enabled():  # create_graph=True: the backward pass itself is not recorded
        raise RuntimeError("%s: the gradient is not differentiable again" % name)


# ------------------------------------------------------------------------------------------------------------------ embed

def _embed_forward(weight, ids, scale):
    V, D = weight.shape
    out = torch.empty(ids.shape + (D,), dtype=weight.dtype, device=weight.device)
    _enqueue(weight.device, "dvae_embed_fwd", weight.data_ptr(), weight.stride(0) if V > 1 else D, ids.data_ptr(), _wide(ids),
             out.data_ptr(), ids.numel(), V, D, scale, DTYPES[weight.dtype])
    return out


class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale):
        ctx.save_for_backward(ids)
        ctx.table, ctx.scale = tuple(weight.shape), scale
        return _embed_forward(weight, ids, scale)

    @staticmethod
    def backward(ctx, dout):
        _once("embed")
        ids, = ctx.saved_tensors
        V, D = ctx.table
        n = ids.numel()
        dout, ld = _rows(dout.reshape(n, D))
        dw = torch.empty(V, D, dtype=dout.dtype, device=dout.device)
        ws = _workspace(_lib.load().dvae_embed_bwd_ws_bytes(n, V, D), dout.device, "dvae_embed_bwd_ws_bytes")
        _enqueue(dout.device, "dvae_embed_bwd", dout.data_ptr(), ld, ids.data_ptr(), _wide(ids), dw.data_ptr(), ws.data_ptr(),
                 n, V, D, ctx.scale, DTYPES[dout.dtype])
        return dw, None, None


def embed(weight, ids, scale=1.0):
    """scale * weight[ids]: `weight` [V, D] with its elements side by side in a row, `ids` int32 / int64 of any shape;
    returns [*ids.shape, D].  A token outside [0, V) (padding) gives a row of zeros and takes no part in the gradient.
    The gradient of `weight` is dense, summed in float32 in the order of the tokens' positions and rounded once; it does
    not vary from run to run."""
    _matrix(weight, "weight", 2)
    V, D = weight.shape
    if V == 0 or D == 0:
        raise ValueError("weight is empty")
    if D > 1 and weight.stride(1) != 1 or V > 1 and weight.stride(0) < D:
        raise ValueError("the elements of a row of weight must lie side by side")
    ids = _index(ids, "ids", weight.device)
    if weight.requires_grad and torch.is_grad_enabled():
        return _EmbedFn.apply(weight, ids, float(scale))
    return _embed_forward(weight, ids, float(scale))


# ------------------------------------------------------------------------------------------------------------- recurrence

def _scan_forward(gate, x, offsets, h0, seqs, keep):
    """(h, last, the states that the backward pass reads if `keep`)"""
    lib = _lib.load()
    g, ld_g = _flat_rows(gate)
    y, ld_y = _flat_rows(x)
    n, D = g.shape
    dev = x.device
    h = torch.empty(x.shape, dtype=x.dtype, device=dev)
    last = torch.empty(seqs, D, dtype=torch.float32, device=dev)
    states = torch.empty(lib.dvae_scan_state_floats(n, D), dtype=torch.float32, device=dev) if keep else None
    ws = _workspace(lib.dvae_scan_ws_bytes(n, D), dev, "dvae_scan_ws_bytes")
    _enqueue(dev, "dvae_scan_fwd", g.data_ptr(), ld_g, y.data_ptr(), ld_y, _lib.ptr(offsets), _wide(offsets), _lib.ptr(h0),
             h.data_ptr(), last.data_ptr(), _lib.ptr(states), ws.data_ptr(), n, seqs, D, DTYPES[x.dtype])
    return h, last, states


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, offsets, h0, seqs):
        h, last, ctx.states = _scan_forward(gate, x, offsets, h0, seqs, True)
        ctx.save_for_backward(gate, x, offsets, h0)
        ctx.seqs = seqs
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        _once("gated_scan")
        gate, x, offsets, h0 = ctx.saved_tensors
        g, ld_g = _flat_rows(gate)
        y, ld_y = _flat_rows(x)
        n, D = g.shape
        dev = x.device
        ld_dh = 0
        if dh is not None:
            dh, ld_dh = _flat_rows(dh)
        if dlast is not None:
            dlast = dlast.contiguous()
        dgate = torch.empty(gate.shape, dtype=x.dtype, device=dev)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        dh0 = torch.empty(ctx.seqs, D, dtype=torch.float32, device=dev) if ctx.needs_input_grad[3] else None
        ws = _workspace(_lib.load().dvae_scan_ws_bytes(n, D), dev, "dvae_scan_ws_bytes")
        _enqueue(dev, "dvae_scan_bwd", g.data_ptr(), ld_g, y.data_ptr(), ld_y, _lib.ptr(offsets), _wide(offsets), _lib.ptr(h0),
                 ctx.states.data_ptr(), _lib.ptr(dh), ld_dh, _lib.ptr(dlast), dgate.data_ptr(), dx.data_ptr(), _lib.ptr(dh0),
                 ws.data_ptr(), n, ctx.seqs, D, DTYPES[x.dtype])
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
    if gate.dtype != x.dtype or gate.device != x.device:
        raise ValueError("gate and x differ in type or device")
    if gate.shape != x.shape:
        raise ValueError("gate has the shape %s, x %s" % (tuple(gate.shape), tuple(x.shape)))
    D = x.shape[-1]
    if D == 0:
        raise ValueError("gate and x have no channels")
    if offsets is not None:
        offsets = _index(offsets, "offsets", x.device)
        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must have one dimension and at least one value")
        seqs = offsets.numel() - 1
    else:
        seqs = x.shape[0]
    if h0 is not None:
        if not torch.is_tensor(h0) or h0.dtype != torch.float32 or h0.device != x.device or tuple(h0.shape) != (seqs, D):
            raise ValueError("h0 must be a float32 tensor of shape (%d, %d) on %s" % (seqs, D, x.device))
        h0 = h0.contiguous()
    if torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or (h0 is not None and h0.requires_grad)):
        return _ScanFn.apply(gate, x, offsets, h0, seqs)
    return _scan_forward(gate, x, offsets, h0, seqs, False)[:2]


def gated_step(gate, x, state, slots=None):
    """One token of each of B sequences: gate, x [B, D]; returns h [B, D] in x's type and updates `state` [P, D] (float32)
    in place at the rows `slots` [B] (int32 / int64, B at most 65536; default: row b has state b).  A slot outside [0, P)
    marks a padding row: its h is zero and no state changes.  Rows that name the same slot advance it one after the other,
    in their order.
    For serving: not differentiable, inputs that need gradients are refused outside torch.no_grad()."""
    code = _matrix(gate, "gate", 2)
    _matrix(x, "x", 2)
    dev = x.device
    if gate.dtype != x.dtype or gate.device != dev or gate.shape != x.shape:
        raise ValueError("gate and x differ in type, device or shape")
    B, D = x.shape
    if D == 0:
        raise ValueError("gate and x have no channels")
    if not torch.is_tensor(state) or state.dtype != torch.float32 or state.device != dev or state.dim() != 2 or state.shape[1] != D:
        raise ValueError("state must be a float32 tensor of shape (P, %d) on %s" % (D, dev))
    P = state.shape[0]
    if D > 1 and state.stride(1) != 1 or P > 1 and state.stride(0) < D:
        raise ValueError("the elements of a row of state must lie side by side")
    if (gate.requires_grad or x.requires_grad or state.requires_grad) and torch.is_grad_enabled():
        raise ValueError("gated_step is not differentiable: call it under torch.no_grad(), or use gated_scan")
    if slots is not None:
        slots = _index(slots, "slots", dev)
        if slots.dim() != 1 or slots.shape[0] != B:
            raise ValueError("slots must have the shape (%d,)" % B)
    elif B > P:
        raise ValueError("%d rows, but %d states" % (B, P))
    g, ld_g = _rows(gate)
    y, ld_y = _rows(x)
    h = torch.empty(B, D, dtype=x.dtype, device=dev)
    _enqueue(dev, "dvae_scan_step", g.data_ptr(), ld_g, y.data_ptr(), ld_y, state.data_ptr(), state.stride(0) if P > 1 else D, P,
             _lib.ptr(slots), _wide(slots), h.data_ptr(), B, D, code)
    _written(state)
    return h
