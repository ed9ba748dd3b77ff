"""Adam for the train step: one HIP launch over a flat parameter buffer.

Same update as `torch.optim.Adam(model.parameters(), lr=1e-4)` of the reference
(`/root/reference/train.py:174`): the parameters the step touches become views of one
flat fp32 buffer (their values, names and `state_dict` are unchanged), gradients are
the views of `dist.GradSumReducer`'s flat buffer, and `step()` is `dvae_adam_step_f32`.
Parameters the step never touches (grad None in the reference: `hv_unify`, the backward
encoder's when unidirectional) are left alone, exactly as torch's Adam skips them.
"""
import bisect
import ctypes as C
import itertools

import torch
from torch.autograd import forward_ad

from . import _lib
from .dist import GradSumReducer
from .sequence import _matrix


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


def _kept_apart(srcs, outs):
    """`srcs`, copied where they share memory with the output of another matrix: the library reads and writes the matrices in
    groups, and a group's outputs must not reach what a later one reads.  (Address ranges: rows between those of a matrix count.)"""
    def span(t):
        return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size()
    spans = sorted(span(o) + (k,) for k, o in enumerate(outs))
    begins = [b for b, _, _ in spans]
    reach = list(itertools.accumulate((e for _, e, _ in spans), max))
    apart = []
    for k, g in enumerate(srcs):
        begin, end = span(g)
        j = bisect.bisect_left(begins, end) - 1
        while j >= 0 and reach[j] > begin and not (spans[j][1] > begin and spans[j][2] != k):
            j -= 1
        apart.append(g.clone() if j >= 0 and reach[j] > begin else g)
    return apart


HALF_PRODUCTS = 16  # DVAE_HALF_PRODUCTS
QUINTIC = (3.4445, -4.7750, 2.0315)  # p(s) = a s + b s^3 + c s^5: five steps take singular values from 0.002 up to 0.7 .. 1.2


def _iteration(steps, coefficients):
    """(number of steps, their coefficients as the library takes them); refuses what the library would"""
    steps, coefficients = int(steps), list(coefficients)
    if not 1 <= steps <= 32:
        raise ValueError("steps must lie in 1 .. 32")
    if coefficients and not hasattr(coefficients[0], "__len__"):
        coefficients = [coefficients] * steps
    triples = [tuple(c) for c in coefficients]
    if len(triples) != steps or any(len(c) != 3 for c in triples):
        raise ValueError("coefficients must be (a, b, c) or one such triple for each of the %d steps" % steps)
    abc = (C.c_float * (3 * steps))(*[v for c in triples for v in c])
    _lib.check(_lib.load().dvae_orthogonalize((_lib.MatrixDesc * 1)(), 0, steps, abc, None, 0, None), "dvae_orthogonalize")  # of no matrix
    return steps, abc


def orthogonalize(updates, steps=5, coefficients=QUINTIC, out=None, products="full"):
    """The nearest (semi-)orthogonal matrix to each of `updates`, approximately: `steps` Newton-Schulz steps
    X <- a X + (b A + c A A) X with A = X X^T (on the smaller side) from X = G / |G|_F.

    updates: a matrix or a list of matrices (float32, bfloat16 or float16, one type, on one HIP device); a list goes through
    every product in one launch.  coefficients: (a, b, c), or one such triple for each step; a set that lets a singular value
    leave [-2, 2] is refused.  out: where to write (same shapes and type; matrices may be their own outputs, or each other's),
    default new tensors.  A zero matrix gives zeros, one with a NaN or an infinity NaN.  Not differentiable (it acts on updates):
    inputs and outputs that need gradients are refused outside torch.no_grad().

    Accuracy of float32, rounded once to the matrices' type.  products="half" (bfloat16 only): matrices with both sides of at
    least 512 multiply operands of 11 bits, for a third of the work; their error is then of the order of the result's own
    rounding and adds to it.  What other matrices a call has changes a result in the last bits of float32 alone."""
    one = torch.is_tensor(updates)
    mats = [updates] if one else list(updates)
    if out is not None:
        outs = [out] if one else list(out)
        if len(outs) != len(mats):
            raise ValueError("out has %d matrices, updates %d" % (len(outs), len(mats)))
    steps, abc = _iteration(steps, coefficients)
    if not mats:
        return []
    if torch.is_grad_enabled() and any(torch.is_tensor(g) and g.requires_grad for g in mats + (outs if out is not None else [])):
        raise ValueError("orthogonalize is not differentiable: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(torch.is_tensor(g) and forward_ad.unpack_dual(g).tangent is not None
                                              for g in mats + (outs if out is not None else [])):
        raise ValueError("orthogonalize has no forward-mode derivative")
    code = _matrix(mats[0], "updates", 2)
    if products not in ("full", "half"):
        raise ValueError("products must be 'full' or 'half'")
    if products == "half":
        if mats[0].dtype != torch.bfloat16:
            raise ValueError("products='half' is for bfloat16 matrices")
        code |= HALF_PRODUCTS
    dtype, device = mats[0].dtype, mats[0].device
    with torch.no_grad():
        srcs = []
        for g in mats:
            _matrix(g, "updates", 2)
            if g.dtype != dtype or g.device != device:
                raise ValueError("the matrices of one call must have one type and one device")
            if g.numel() == 0:
                raise ValueError("updates: an empty matrix")
            if max(g.shape) > 32768:  # (the descriptions below hold the sides in 32 bits)
                raise ValueError("updates: a matrix of %d x %d; sides of up to 32768 are supported" % tuple(g.shape))
            g = g.resolve_neg()  # (the library reads memory)
            srcs.append(g if (g.shape[1] == 1 or g.stride(1) == 1) and (g.shape[0] == 1 or g.stride(0) >= g.shape[1]) else g.contiguous())
        if out is None:
            outs = [torch.empty(g.shape, dtype=dtype, device=device) for g in mats]
        else:
            for o, g in zip(outs, mats):
                if o.shape != g.shape or o.dtype != dtype or o.device != device:
                    raise ValueError("out must have the shapes, type and device of updates")
                if o.is_neg():
                    raise ValueError("out is a view of negated elements")
                if (o.shape[1] > 1 and o.stride(1) != 1) or (o.shape[0] > 1 and o.stride(0) < o.shape[1]):
                    raise ValueError("out: the elements of a row must lie side by side")
            if len(mats) > 32 or products == "half":  # more than one group
                srcs = _kept_apart(srcs, outs)
        lib = _lib.load()
        descs = (_lib.MatrixDesc * len(mats))(*[
            _lib.MatrixDesc(g.data_ptr(), o.data_ptr(), g.stride(0) if g.shape[0] > 1 else g.shape[1],
                            o.stride(0) if o.shape[0] > 1 else o.shape[1], g.shape[0], g.shape[1]) for g, o in zip(srcs, outs)])
        ws = _workspace(lib.dvae_orthogonalize_ws_bytes(descs, len(mats), code), device, "dvae_orthogonalize_ws_bytes")
        _enqueue(device, "dvae_orthogonalize", descs, len(mats), steps, abc, ws.data_ptr(), code)
        if out is not None:
            _written(*outs)
    return outs[0] if one else outs


class FlatAdam(torch.optim.Optimizer):
    def __init__(self, model, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, reducer=None, extra_params=None, capturable=False):
        """extra_params: parameters outside the hot path (e.g. the optional `model.predictor` head of
        train.py:165-172); they are stepped by a torch.optim.Adam with the same hyper-parameters.
        capturable: the learning rate and the step count live in device memory (dvae_adam_step_dev_f32; the
        counterpart of torch.optim.Adam(capturable=True)), so that a captured train step can be replayed
        (harness.GraphedTrainStep); same arithmetic."""
        self.model = model
        extra = [p for p in (extra_params or [])]
        self.extra = torch.optim.Adam(extra, lr=lr, betas=betas, eps=eps) if extra else None
        self.reducer = reducer if reducer is not None else GradSumReducer(model)
        r = self.reducer
        r.add_extra(extra)  # their gradients join the exchange step (the head's loss is a sum over the rank's graphs too)
        if not r.flat.is_cuda:
            raise _lib.DvaeHipError("FlatAdam runs on a HIP device; move the model first (no CPU fallback)")
        super(FlatAdam, self).__init__(r.params, dict(lr=lr, betas=betas, eps=eps))
        self.flat_p = torch.zeros_like(r.flat)
        with torch.no_grad():
            for p, o in zip(r.params, r.offsets):
                view = self.flat_p[o:o + p.numel()].view_as(p)
                view.copy_(p)
                p.data = view
        self.exp_avg = torch.zeros_like(r.flat)
        self.exp_avg_sq = torch.zeros_like(r.flat)
        self.steps = 0
        self.capturable = bool(capturable)
        self._lr_dev = self._step_dev = None   # device copies of lr / steps (capturable)
        self._dev_mirror = (None, None)        # the (lr, steps) the device copies are known to hold
        model._pw = None  # parameter storage moved: pack afresh

    def zero_grad(self, set_to_none=False):
        self.reducer.zero()
        if self.extra is not None:
            self.extra.zero_grad()

    def _check_views(self):
        r = self.reducer
        base_p, base_g = self.flat_p.data_ptr(), r.flat.data_ptr()
        for p, o in zip(r.params, r.offsets):
            # .to() / .cuda() / .float() on the model re-allocate parameters: the views would be gone
            pg = p.grad
            if pg is None or p.data_ptr() != base_p + 4 * o or pg.data_ptr() != base_g + 4 * o:
                raise _lib.DvaeHipError("FlatAdam: a parameter (or its .grad) no longer lives in the flat buffers "
                                        "(was the model moved or its gradients set to None after the optimizer "
                                        "was built?); build the optimizer after the last .to()")

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        g = self.param_groups[0]
        r = self.reducer
        self._check_views()
        lib = _lib.load()
        # zero_grad: with the gradient sink attached every write to the flat gradient buffer goes through the model
        # (which clears `reducer.clean`), so the kernel can leave the buffer zeroed and the next zero_grad() is free
        zero = int(bool(getattr(self.model, "_grad_sink", False)) and getattr(self.model, "_reducer", None) is r)
        stream = C.c_void_p(torch._C._cuda_getCurrentRawStream(self.flat_p.device.index))
        if self.capturable:
            self.sync_device_state()
            _lib.check(lib.dvae_adam_step_dev_f32(self.flat_p.data_ptr(), r.flat.data_ptr(), self.exp_avg.data_ptr(),
                                                  self.exp_avg_sq.data_ptr(), self.flat_p.numel(), self._lr_dev.data_ptr(),
                                                  float(g["betas"][0]), float(g["betas"][1]), float(g["eps"]),
                                                  self._step_dev.data_ptr(), zero, stream), "dvae_adam_step_dev_f32")
            self.steps += 1
            self._dev_mirror = (self._dev_mirror[0], self.steps)  # the kernel pair advanced the device count
        else:
            self.steps += 1
            _lib.check(lib.dvae_adam_step_f32(self.flat_p.data_ptr(), r.flat.data_ptr(), self.exp_avg.data_ptr(),
                                              self.exp_avg_sq.data_ptr(), self.flat_p.numel(), float(g["lr"]),
                                              float(g["betas"][0]), float(g["betas"][1]), float(g["eps"]), self.steps, zero,
                                              stream), "dvae_adam_step_f32")
        # (set either way: with the sink detached autograd's own accumulation writes into the .grad views behind the
        # reducer's back, so the buffer is only known to be zero when THIS step's kernel zeroed it)
        r.clean = bool(zero)
        # the kernel wrote through raw pointers: tensor versions did not move, so the packed copy is stale
        self.model._pw_dirty = True
        if self.extra is not None:
            for eg in self.extra.param_groups:
                eg["lr"] = g["lr"]  # follows a scheduler attached to this optimizer
            self.extra.step()
        return loss

    def sync_device_state(self):
        """capturable: brings the device copies of (lr, steps) up to the host's values where they differ (a scheduler
        changed lr, a checkpoint was loaded).  Two tiny fills at most; nothing when they agree."""
        dev = self.flat_p.device
        if self._lr_dev is None:
            self._lr_dev = torch.zeros(1, dtype=torch.float32, device=dev)
            self._step_dev = torch.zeros(1, dtype=torch.int32, device=dev)
            self._dev_mirror = (None, None)
        lr = float(self.param_groups[0]["lr"])
        if self._dev_mirror[0] != lr:
            self._lr_dev.fill_(lr)
        if self._dev_mirror[1] != self.steps:
            self._step_dev.fill_(self.steps)
        self._dev_mirror = (lr, self.steps)

    def replayed(self):
        """a captured step() was replayed: the device count advanced by one, the host's follows"""
        self.steps += 1
        self._dev_mirror = (self._dev_mirror[0], self.steps)

    # ------------------------------------------------------------------ checkpoints
    # The layout written and read is torch.optim.Adam's own (what the reference saves as
    # optimizer_checkpoint<epoch>.pth, train.py:705-712, and loads back with --continue-from, train.py:185-192):
    #   {"state": {i: {"step", "exp_avg", "exp_avg_sq"}}, "param_groups": [{..., "params": [0 .. N-1]}]}
    # with i numbering `model.parameters()` in order (the reference builds optim.Adam(model.parameters())),
    # parameters that never received a gradient having no entry.  So a reference run resumes here and a run
    # of this package resumes under torch.optim.Adam.
    def _ordered_params(self):
        params = list(self.model.parameters())
        seen = {id(p) for p in params}
        if self.extra is not None:  # extra parameters that are not sub-modules of the model come last
            params += [p for g in self.extra.param_groups for p in g["params"] if id(p) not in seen]
        return params

    def state_dict(self):
        r = self.reducer
        slot = {id(p): (o, p.numel()) for p, o in zip(r.params, r.offsets)}
        state = {}
        extra_state = {id(k): v for k, v in self.extra.state.items()} if self.extra is not None else {}
        for i, p in enumerate(self._ordered_params()):
            if id(p) in slot:
                if self.steps > 0:
                    o, n = slot[id(p)]
                    state[i] = {"step": torch.tensor(float(self.steps)),
                                "exp_avg": self.exp_avg[o:o + n].view_as(p).clone(),
                                "exp_avg_sq": self.exp_avg_sq[o:o + n].view_as(p).clone()}
            elif id(p) in extra_state:
                state[i] = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in extra_state[id(p)].items()}
        probe = torch.zeros(1, requires_grad=True)
        group = dict(torch.optim.Adam([probe]).state_dict()["param_groups"][0])  # this torch version's keys and defaults
        mine = self.param_groups[0]
        group.update(lr=mine["lr"], betas=tuple(mine["betas"]), eps=mine["eps"])
        for k in ("initial_lr",):  # what a scheduler attached to this optimizer left in the group
            if k in mine:
                group[k] = mine[k]
        group["params"] = list(range(len(self._ordered_params())))
        return {"state": state, "param_groups": [group]}

    def load_state_dict(self, sd):
        if "names" in sd and "state" not in sd:
            return self._load_flat_state(sd)  # files written by the first version of this class
        if "state" not in sd or "param_groups" not in sd:
            raise ValueError("not an Adam state dict (expected the keys 'state' and 'param_groups')")
        params = self._ordered_params()
        ids = [i for g in sd["param_groups"] for i in g["params"]]
        if len(ids) != len(params):
            raise ValueError("optimizer state covers %d parameters, the model has %d" % (len(ids), len(params)))
        r = self.reducer
        slot = {id(p): (o, p.numel()) for p, o in zip(r.params, r.offsets)}
        self.exp_avg.zero_()
        self.exp_avg_sq.zero_()
        steps = 0
        extra_state = {}
        for i, p in zip(ids, params):
            st = sd["state"].get(i, sd["state"].get(str(i)))
            if st is None:
                continue
            if tuple(st["exp_avg"].shape) != tuple(p.shape):
                raise ValueError("optimizer state %d has shape %s, the parameter %s" % (i, tuple(st["exp_avg"].shape), tuple(p.shape)))
            if id(p) in slot:
                o, n = slot[id(p)]
                self.exp_avg[o:o + n].copy_(st["exp_avg"].reshape(-1))
                self.exp_avg_sq[o:o + n].copy_(st["exp_avg_sq"].reshape(-1))
                steps = max(steps, int(float(st["step"])))
            else:
                extra_state[id(p)] = st  # a parameter outside the hot path (predictor head), or one the step never touches
        self.steps = steps
        saved = sd["param_groups"][0]
        g = self.param_groups[0]
        g.update(lr=saved["lr"], betas=tuple(saved["betas"]), eps=saved["eps"])
        if "initial_lr" in saved:
            g["initial_lr"] = saved["initial_lr"]
        if self.extra is not None:
            own = self.extra.state_dict()
            eparams = [p for eg in self.extra.param_groups for p in eg["params"]]
            own["state"] = {j: extra_state[id(p)] for j, p in enumerate(eparams) if id(p) in extra_state}
            for eg in own["param_groups"]:
                eg.update(lr=saved["lr"], betas=tuple(saved["betas"]), eps=saved["eps"])
            self.extra.load_state_dict(own)

    def _load_flat_state(self, sd):
        if list(sd["names"]) != list(self.reducer.names):
            raise ValueError("optimizer state belongs to a different parameter set")
        self.steps = int(sd["steps"])
        self.exp_avg.copy_(sd["exp_avg"])
        self.exp_avg_sq.copy_(sd["exp_avg_sq"])
        for g, saved in zip(self.param_groups, sd["param_groups"]):
            g.update(saved)
        if self.extra is not None and sd.get("extra") is not None:
            self.extra.load_state_dict(sd["extra"])


def _of_matrices(key):
    """a value of FlatMuon's group of matrices as an attribute"""
    return property(lambda self: self.param_groups[0][key], lambda self, value: self.param_groups[0].update({key: value}))


class FlatMuon(FlatAdam):
    """Muon for the weight matrices, Adam for everything else, on FlatAdam's flat buffers: the momentum of a matrix is
    orthogonalised (`orthogonalize`, all matrices of the model together) before it is applied.  The arguments are those of
    torch.optim.Muon, whose counterpart this is:

      m += (1 - momentum) (g - m);  u = g + momentum (m - g) if nesterov else m
      p  = (1 - lr weight_decay) p - lr f orthogonalize(u),   f = sqrt(max(1, rows / columns))   ("original")
                                                               or 0.2 sqrt(max(rows, columns))    ("match_rms_adamw")

    matrices: names of the parameters that take this update; by default every weight matrix the train step touches except
    those that act on one-hot inputs (*.weight_ih, and the gates and mappers of DVAE_BN: rows of a table) and the last layers
    of the two predictors.  The rest, and `extra_params`, take Adam's with adam_lr, betas, eps.  param_groups[0] holds the
    matrices (lr, momentum, nesterov, weight_decay, ns_steps, ns_coefficients, adjust_lr_fn), param_groups[1] the rest;
    schedulers see both and checkpoints hold both."""

    def __init__(self, model, lr=2e-2, momentum=0.95, nesterov=True, weight_decay=0.0, adam_lr=1e-4, betas=(0.9, 0.999),
                 eps=1e-8, ns_steps=5, ns_coefficients=QUINTIC, adjust_lr_fn="original", matrices=None, reducer=None,
                 extra_params=None):
        self._check_adjust(adjust_lr_fn)
        _iteration(ns_steps, ns_coefficients)
        if not 0.0 <= momentum < 1.0 or lr < 0.0 or weight_decay < 0.0:
            raise ValueError("FlatMuon: momentum must lie in [0, 1), lr and weight_decay must not be negative")
        super(FlatMuon, self).__init__(model, lr=adam_lr, betas=betas, eps=eps, reducer=reducer, extra_params=extra_params)
        r = self.reducer
        if matrices is None:
            heads = ("add_vertex.2.weight", "add_edge.2.weight")
            tables = ("gate_forward.0.weight", "gate_backward.0.weight", "mapper_forward.0.weight", "mapper_backward.0.weight")
            matrices = [k for k, p in zip(r.names, r.params) if p.dim() == 2 and not k.endswith("weight_ih") and k not in heads
                        and not (model._is_bn and k in tables)]
        matrices = list(matrices)
        at = dict(zip(r.names, range(len(r.names))))
        for k in matrices:
            if k not in at or r.params[at[k]].dim() != 2:
                raise ValueError("FlatMuon: %s is not a weight matrix of the train step" % k)
        self.matrices = [k for k in r.names if k in set(matrices)]
        self.is_matrix = [k in set(matrices) for k in r.names]
        rest = self.param_groups[0]
        first = dict(rest, params=[p for p, mat in zip(r.params, self.is_matrix) if mat], lr=lr, momentum=momentum,
                     nesterov=bool(nesterov), weight_decay=weight_decay, ns_steps=int(ns_steps), ns_coefficients=ns_coefficients,
                     adjust_lr_fn=adjust_lr_fn)
        del first["betas"], first["eps"]
        rest["params"] = [p for p, mat in zip(r.params, self.is_matrix) if not mat]
        self.param_groups[:] = [first, rest]
        self._set_factor()
        self.flat_u = torch.zeros_like(self.flat_p)
        self.updates = [self.flat_u[o:o + p.numel()].view_as(p) for p, o, mat in zip(r.params, r.offsets, self.is_matrix) if mat]

    @staticmethod
    def _check_adjust(fn):
        if fn not in ("original", "match_rms_adamw"):
            raise ValueError("adjust_lr_fn must be 'original' or 'match_rms_adamw'")

    ns_steps, ns_coefficients = _of_matrices("ns_steps"), _of_matrices("ns_coefficients")

    def _set_factor(self):
        """the learning-rate factors of the matrices, for every 64 elements of the flat buffers; 0 elsewhere"""
        r, fn = self.reducer, self.param_groups[0]["adjust_lr_fn"]
        self._check_adjust(fn)
        factor = torch.zeros(r.numel // 64, dtype=torch.float32)
        for p, o, mat in zip(r.params, r.offsets, self.is_matrix):
            if mat:
                rows, cols = p.shape
                f = max(1.0, rows / cols) ** 0.5 if fn == "original" else 0.2 * max(rows, cols) ** 0.5
                factor[o // 64:(o + p.numel() + 63) // 64] = f
        self.factor, self._factor_fn = factor.to(self.flat_p.device), fn

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        mats, rest = self.param_groups
        r = self.reducer
        self._check_views()
        # what may be refused is, before anything has moved
        _iteration(mats["ns_steps"], mats["ns_coefficients"])
        if mats["adjust_lr_fn"] != self._factor_fn:
            self._set_factor()
        zero = int(bool(getattr(self.model, "_grad_sink", False)) and getattr(self.model, "_reducer", None) is r)
        n = self.flat_p.numel()
        self.steps += 1
        dev = self.flat_p.device
        _enqueue(dev, "dvae_muon_begin_f32", self.flat_p.data_ptr(), r.flat.data_ptr(), self.exp_avg.data_ptr(),
                 self.exp_avg_sq.data_ptr(), self.flat_u.data_ptr(), self.factor.data_ptr(), n, float(mats["momentum"]),
                 int(mats["nesterov"]), float(rest["lr"]), float(rest["betas"][0]), float(rest["betas"][1]), float(rest["eps"]),
                 self.steps, zero)
        if self.updates:
            orthogonalize(self.updates, mats["ns_steps"], mats["ns_coefficients"], out=self.updates)
            _enqueue(dev, "dvae_muon_apply_f32", self.flat_p.data_ptr(), self.flat_u.data_ptr(), self.factor.data_ptr(), n,
                     float(mats["lr"]), float(mats["weight_decay"]))
        r.clean = bool(zero)
        self.model._pw_dirty = True  # written through raw pointers, as by FlatAdam
        if self.extra is not None:
            for eg in self.extra.param_groups:
                eg["lr"] = rest["lr"]
            self.extra.step()
        return loss

    # Checkpoints: {"state": {i: {"momentum_buffer"} or {"step", "exp_avg", "exp_avg_sq"}}, "param_groups": [matrices, rest]},
    # i numbering model.parameters() as in FlatAdam's; the rest as torch.optim.Adam writes it, the matrices as torch.optim.Muon.
    def _adam_part(self, call, *args):
        """a FlatAdam method with the group of Adam's parameters as the only one"""
        mats, rest = self.param_groups
        self.param_groups[:] = [rest]
        try:
            return call(*args)
        finally:
            self.param_groups[:] = [mats, rest]

    def _matrix_numbers(self):
        number = {id(p): i for i, p in enumerate(self._ordered_params())}
        return sorted(number[id(p)] for p in self.param_groups[0]["params"])

    def state_dict(self):
        sd = self._adam_part(super(FlatMuon, self).state_dict)
        mats = self._matrix_numbers()
        for i in mats:
            if i in sd["state"]:
                sd["state"][i] = {"momentum_buffer": sd["state"][i]["exp_avg"]}
        adam = sd["param_groups"][0]
        adam["params"] = [i for i in adam["params"] if i not in mats]
        mine = {k: v for k, v in self.param_groups[0].items() if k != "params"}
        sd["param_groups"] = [dict(mine, params=mats), adam]
        sd["steps"] = self.steps
        return sd

    def load_state_dict(self, sd):
        if len(sd.get("param_groups", ())) != 2 or "steps" not in sd:
            raise ValueError("not a FlatMuon state dict (expected two parameter groups and the key 'steps')")
        params, mats = self._ordered_params(), self._matrix_numbers()
        if list(sd["param_groups"][0]["params"]) != mats:
            raise ValueError("the state belongs to another choice of matrices")
        first = dict(self.param_groups[0], **sd["param_groups"][0])
        self._check_adjust(first["adjust_lr_fn"])
        _iteration(first["ns_steps"], first["ns_coefficients"])
        state = {}
        for i, st in sd["state"].items():
            if int(i) in mats:
                m = st["momentum_buffer"]
                st = {"step": torch.tensor(float(sd["steps"])), "exp_avg": m, "exp_avg_sq": torch.zeros_like(m)}
            state[int(i)] = st
        adam = dict(sd["param_groups"][1], params=list(range(len(params))))
        self._adam_part(super(FlatMuon, self).load_state_dict, {"state": state, "param_groups": [adam]})
        self.param_groups[0].update({k: v for k, v in sd["param_groups"][0].items() if k != "params"})
        self.steps = int(sd["steps"])
