"""Sequence operators on the HIP library: a token table and a gated linear recurrence over packed sequences.

  embed        rows of a table looked up by tokens, times a scale; the gradient sums the rows of equal tokens
  gated_scan   h_t = z_t h_{t-1} + (1 - z_t) x_t, z = sigmoid(gate), along sequences of any lengths, differentiable
  gated_step   the same for one token of each sequence, the states kept in a pool and updated in place (serving)

The DAG model keeps its own paths (at most 32 vertex types as a table inside the GRU kernels, chains of at most 64
vertices); these are for encoders of long or many token sequences beside it -- the reference's sequence baselines
(models.py:18-338) run on one-hot inputs and nn.GRU.  Matrices are float32, bfloat16 or float16, the states of the
recurrence always float32.  Like the rest of the package there is no CPU or PyTorch fallback.  Gradients are those of the
backward pass alone: tensors that carry a tangent (forward-mode derivatives) are refused.
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
    """an index tensor beside the matrices, contiguous"""
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError("%s must be an int32 or int64 tensor" % name)
    if t.device != device:
        raise ValueError("%s is on %s, the matrices on %s" % (name, t.device, device))
    return t.resolve_neg().contiguous()


_ops = None


def _native():
    """the host side in C++ (csrc/sequence_ops.cpp): allocation, launch, autograd"""
    global _ops
    if _ops is None:
        _ops = _lib.load_sequence_ops()
    return _ops


# ------------------------------------------------------------------------------------------------------------------ embed

def embed(weight, ids, scale=1.0):
    """scale * weight[ids]: `weight` [V, D] with its elements side by side in a row, `ids` int32 / int64 of any shape;
    returns [*ids.shape, D].  A token outside [0, V) (padding) gives a row of zeros and takes no part in the gradient.
    The gradient of `weight` is dense (up to 2^28 - 32 tokens), summed in float32 in an order that depends on the tokens alone
    and rounded once; it does not vary from run to run."""
    out = (_ops or _native()).usual_embed(weight, ids, scale)
    if out is not None:
        return out
    _matrix(weight, "weight", 2)
    V, D = weight.shape
    if V == 0 or D == 0:
        raise ValueError("weight is empty")
    if D > 1 and weight.stride(1) != 1 or V > 1 and weight.stride(0) < D:
        raise ValueError("the elements of a row of weight must lie side by side")
    ids = _index(ids, "ids", weight.device)
    return _ops.embed(weight, ids, float(scale))


# ------------------------------------------------------------------------------------------------------------- recurrence

def gated_scan(gate, x, offsets=None, h0=None):
    """h_t = z_t h_{t-1} + (1 - z_t) x_t with z = sigmoid(gate), per channel, along every sequence -> (h, last).

    offsets [S + 1] (int32 / int64, on the device, not decreasing): gate and x are [N, D] and sequence s is the rows
    offsets[s] : offsets[s + 1]; empty sequences are allowed, rows of no sequence give zeros in h and in the gradients.
    Values outside [0, N] count as the nearer end.  Without offsets gate and x are [S, T, D].
    h0 [S, D] float32: the state before each sequence (default zeros).  last [S, D] float32: the state after it.

    gate and x may be the two halves of one projection's output: rows of any stride are read in place.  Differentiable in
    gate, x and h0; the states are float32 inside, h and the gradients of gate and x are rounded once to x's type."""
    out = (_ops or _native()).usual_scan(gate, x, offsets, h0)
    if out is not None:
        return out
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
    return _ops.scan(gate, x, offsets, h0, seqs)


def gated_step(gate, x, state, slots=None):
    """One token of each of B sequences: gate, x [B, D]; returns h [B, D] in x's type and updates `state` [P, D] (float32)
    in place at the rows `slots` [B] (int32 / int64, B at most 65536; default: row b has state b).  A slot outside [0, P)
    marks a padding row: its h is zero and no state changes.  Rows that name the same slot advance it one after the other,
    in their order.  gate and x may lie in the pool itself: they are read before it is written.
    For serving: not differentiable, inputs that need gradients are refused outside torch.no_grad()."""
    out = (_ops or _native()).usual_step(gate, x, state, slots)
    if out is not None:
        return out
    _matrix(gate, "gate", 2)
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
    if state.is_neg():
        raise ValueError("state is a view of negated elements and cannot be updated in place")
    if (gate.requires_grad or x.requires_grad or state.requires_grad) and torch.is_grad_enabled():
        raise ValueError("gated_step is not differentiable: call it under torch.no_grad(), or use gated_scan")
    if slots is not None:
        slots = _index(slots, "slots", dev)
        if slots.dim() != 1 or slots.shape[0] != B:
            raise ValueError("slots must have the shape (%d,)" % B)
    elif B > P:
        raise ValueError("%d rows, but %d states" % (B, P))
    return _ops.step(gate, x, state, slots)
