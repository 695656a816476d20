"""Orthogonalised updates of weight matrices: :func:`orthogonalize` and the optimizer made of it, :class:`ShardMuon`
(``include/jabas_muon.h``).

The update of a matrix is its momentum taken to the nearest matrix whose singular values all lie near one, by a few Newton-Schulz
products: with X of the shorter side first, X = G / max(|G|, eps), then X <- a X + (b A + c A A) X with A = X X^T. The
reference has no such optimizer; the surface is that of ``torch.optim.Muon`` with the conventions of the other ``Shard``
optimizers beside it (``step(gradients)``, replicas, state in the caller's hands).

Everything runs on the current stream of the tensors' device; there is no CPU path. Launches are queued without synchronisation. A list of
matrices that a step has not seen (gradients in other memory make it another) is laid out on the host first and copied to the
device, and the host waits for that copy: 96 matrices of 1024 x 1024 to 1024 x 4096 take 5 to 30 ms and 10 MB of tables. Gradients that keep their memory
(``zero_grad(set_to_none=False)``, a bucket's views, the engine's arenas) are laid out once.
"""
import ctypes as C
import math

import numpy as np
import torch
from torch.autograd import forward_ad

from .. import _lib as L
from ..loss import _direct
from ..sync import _stream_ptr
from .shard import ShardAdamW, _ShardOptimizer

COEFFICIENTS = (3.4445, -4.775, 2.0315)
_PRECISION = {torch.float32: L.F32, torch.bfloat16: L.BF16}
_ADJUST = {"original": lambda rows, cols: math.sqrt(max(1.0, rows / cols)),
           "match_rms_adamw": lambda rows, cols: 0.2 * math.sqrt(max(rows, cols))}


def _newton_schulz(steps, coefficients, eps, dtype):
    """The JabasNewtonSchulz of a call, with what can be said about it in words said here."""
    if dtype not in _PRECISION:
        raise TypeError(f"matrices are orthogonalised in float32 or bfloat16, not {dtype}")
    if len(coefficients) != 3:
        raise ValueError(f"three coefficients expected, got {len(coefficients)}")
    if not 1 <= int(steps) <= L.MUON_MAX_STEPS:
        raise ValueError(f"1..{L.MUON_MAX_STEPS} Newton-Schulz steps, got {steps}")
    a, b, c = (float(x) for x in coefficients)
    if not 1e-30 <= float(eps) < float("inf"):
        raise ValueError(f"eps must be positive (at least 1e-30) and finite, got {eps}")
    return L.JabasNewtonSchulz(a, b, c, float(eps), int(steps), _PRECISION[dtype])


_GROWN = "coefficients {} let singular values grow past 256"


def _grown(status, coefficients, where):
    if status == L.ERR_OPT:
        raise ValueError(_GROWN.format(tuple(coefficients)))
    L.check(status, where)


def _check_growth(ns):
    """Whether the library takes the polynomial, asked without a launch."""
    if not L.lib().jabas_orthogonalize_workspace_bytes(C.byref(L.JabasOrthogonalize(dtype=L.F32, ns=ns))):
        raise ValueError(_GROWN.format((ns.a, ns.b, ns.c)))


# ---------------------------------------------------------------------------------------------------------- orthogonalize
def _launch(x, out, steps, coefficients, eps):
    if x.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return _launch(x, out, steps, coefficients, eps)
    rows, cols = x.shape[-2:]
    if x.dim() != 3:
        x = x.reshape(-1, rows, cols) if x.numel() else x.new_empty((0, rows, cols))
    if (x.stride(2) != 1 and cols > 1) or (x.stride(1) < cols and rows > 1):
        x = x.contiguous()
    o = L.JabasOrthogonalize()
    setattr(o, "in", x.data_ptr())
    o.out, o.batch, o.rows, o.cols = out.data_ptr(), x.shape[0], rows, cols
    o.in_batch_stride = x.stride(0) if x.shape[0] > 1 else 0
    o.in_row_stride = x.stride(1) if rows > 1 else cols
    o.dtype = _PRECISION[x.dtype]
    o.ns = _newton_schulz(steps, coefficients, eps, x.dtype)
    n = L.lib().jabas_orthogonalize_workspace_bytes(C.byref(o))
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=x.device)
    _grown(L.lib().jabas_orthogonalize(C.byref(o), ws.data_ptr(), ws.numel(), _stream_ptr()), coefficients, "jabas_orthogonalize")
    return out


# For whoever watches operations (torch.compile, make_fx, modes): a launch through the C ABI is not seen by a recorder.
_LIBRARY = torch.library.Library("jabas", "FRAGMENT")
_LIBRARY.define("orthogonalize(Tensor x, int steps, float[] coefficients, float eps) -> Tensor")
_LIBRARY.impl("orthogonalize", lambda x, steps, coefficients, eps: _launch(
    x, torch.empty(x.shape, dtype=x.dtype, device=x.device), steps, coefficients, eps), "CUDA")


@torch.library.register_fake("jabas::orthogonalize", lib=_LIBRARY)
def _fake(x, steps, coefficients, eps):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _no_gradient(ctx, *upstream):
    raise RuntimeError("orthogonalize has no derivative")


torch.library.register_autograd("jabas::orthogonalize", _no_gradient, lib=_LIBRARY)


def orthogonalize(x, *, steps=5, coefficients=COEFFICIENTS, eps=1e-7, out=None):
    """The matrices ``x`` (..., rows, cols) with their singular values taken to the ones that ``steps`` Newton-Schulz products make of
    them, near 1 with the default coefficients; singular vectors stay. float32 or bfloat16, as is the result. A matrix whose
    length is under ``eps`` is divided by ``eps`` instead, so zeros stay zeros; one that holds an infinity or a NaN becomes NaN.

    float32: the products keep 22 bits of every factor. bfloat16: 11 bits of each in the products and 22 of the running matrix, one
    rounding to bfloat16 at the end.

    ``coefficients`` (a, b, c) may not let singular values grow past 256. ``out``: contiguous, of x's shape and type, not overlapping it.
    Leading sizes are a batch; sides up to 65536 x 4194304. There is no derivative: an ``x`` that requires grad is refused while
    gradients are recorded, and so is a tangent."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("x: expected a tensor")
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in (x, out)):
        raise RuntimeError("orthogonalize has no forward-mode derivative")
    if not x.is_cuda:
        raise ValueError(f"x: must live on the GPU, got {x.device}")
    if x.dtype not in _PRECISION:
        raise TypeError(f"x: must be float32 or bfloat16, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError(f"x: needs rows and columns, got shape {tuple(x.shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("orthogonalize has no derivative: call it under torch.no_grad() or on x.detach()")
    _newton_schulz(steps, coefficients, eps, x.dtype)
    rows, cols = x.shape[-2:]
    if min(rows, cols) > L.MUON_MAX_SIDE or max(rows, cols) > L.MUON_MAX_LENGTH:
        raise ValueError(f"x: sides up to {L.MUON_MAX_SIDE} and {L.MUON_MAX_LENGTH}, got {rows} x {cols}")
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
            raise ValueError("out: expected a tensor of x's shape, type and device")
        if not out.is_contiguous():
            raise ValueError("out: must be contiguous")
        if out.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("out: requires grad")
    if not _direct(x, out):
        made = torch.ops.jabas.orthogonalize(x, int(steps), [float(c) for c in coefficients], float(eps))
        return made if out is None else out.copy_(made)
    if out is None:
        return _launch(x, torch.empty(x.shape, dtype=x.dtype, device=x.device), steps, coefficients, eps)
    _launch(x, out, steps, coefficients, eps)
    torch.autograd.graph.increment_version(out)     # autograd does not see the launch: whoever saved out is told
    return out


def _recording(x):
    """Whether launches on x's device are being recorded in a graph."""
    return x.is_cuda and torch.cuda.is_current_stream_capturing()


# ------------------------------------------------------------------------------------------------------------------- plans
class MuonPlan:
    """A validated, device-resident list of matrices; ``run`` queues their step. ``items``: dicts of ``grad``, ``momentum``, ``param``
    (contiguous float32 of one device, any shape with as many elements), ``rows``, ``cols``, ``group``, ``lr_factor`` and ``fanout``
    (replicas that receive the new weights). The plan names their memory and keeps no tensor: a gradient that it held would never be
    freed."""

    def __init__(self, items, dtype=torch.float32):
        if not items:
            raise ValueError("a plan needs at least one matrix")
        if _recording(items[0]["grad"]):
            raise RuntimeError("a list of matrices is prepared before its step is recorded")
        self.precision = _PRECISION[dtype]
        self.device = items[0]["grad"].device
        table = (L.JabasMatrix * len(items))()
        for c, i in zip(table, items):
            n = i["rows"] * i["cols"]
            fanout = list(i.get("fanout", ()))
            for what, t in (("grad", i["grad"]), ("momentum", i["momentum"]), ("param", i["param"]), *(("fanout", f) for f in fanout)):
                if t.dtype != torch.float32 or t.device != self.device or t.numel() != n or not t.is_contiguous() or not t.is_cuda:
                    raise ValueError(f"{what}: expected {n} contiguous float32 elements on {self.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
            if len(fanout) > L.MAX_K - 1:
                raise ValueError(f"at most {L.MAX_K - 1} replicas")
            c.grad, c.momentum, c.param = i["grad"].data_ptr(), i["momentum"].data_ptr(), i["param"].data_ptr()
            c.rows, c.cols, c.lr_factor, c.group, c.n_fanout = i["rows"], i["cols"], float(i.get("lr_factor", 1.0)), int(i.get("group", 0)), len(fanout)
            for f, t in enumerate(fanout):
                c.fanout[f] = t.data_ptr()
        lib = L.lib()
        nbytes = lib.jabas_muon_plan_bytes(table, len(items), self.precision)
        self._host = torch.from_numpy(np.zeros(max(nbytes, 8) // 8, dtype=np.int64))
        L.check(lib.jabas_muon_plan_encode(table, len(items), self.precision, self._host.data_ptr(), nbytes), "jabas_muon_plan_encode")
        self.workspace_bytes = lib.jabas_muon_workspace_bytes(self._host.data_ptr())
        with torch.cuda.device(self.device):
            self._dev = self._host.to(self.device)
            self._made_on = _stream_ptr()

    def run(self, args, stream=None):
        """Queues the step. The workspace is the allocator's: steps on different streams, and recorded ones, have one each."""
        if self.device.index != torch._C._cuda_getDevice():
            with torch.cuda.device(self.device):
                return self.run(args, stream)
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.run(args)
        at = _stream_ptr()
        if at != self._made_on:
            self._dev.record_stream(torch.cuda.current_stream())
        ws = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=self.device)
        _grown(L.lib().jabas_muon_step(self._host.data_ptr(), self._dev.data_ptr(), C.byref(args), ws.data_ptr(), self.workspace_bytes, at),
               (args.ns.a, args.ns.b, args.ns.c), "jabas_muon_step")


def make_muon_args(groups, *, momentum, nesterov, steps=5, coefficients=COEFFICIENTS, eps=1e-7, dtype=torch.float32, lr_scale=1.0, grad_scale=None):
    """The JabasMuonArgs of one step; ``groups``: dicts with ``lr`` and ``weight_decay``."""
    if not 1 <= len(groups) <= L.MAX_GROUPS:
        raise ValueError(f"1..{L.MAX_GROUPS} parameter groups supported, got {len(groups)}")
    if not 0.0 <= momentum < 1.0:
        raise ValueError(f"momentum must be in [0, 1), got {momentum}")
    a = L.JabasMuonArgs()
    a.ns = _newton_schulz(steps, coefficients, eps, dtype)
    _check_growth(a.ns)
    a.momentum, a.nesterov, a.n_groups = float(momentum), int(bool(nesterov)), len(groups)
    for i, g in enumerate(groups):
        a.lr[i], a.weight_decay[i] = float(g["lr"]) * float(lr_scale), float(g.get("weight_decay", 0.0))
    if grad_scale is not None:
        if grad_scale.dtype != torch.float32 or not grad_scale.is_cuda:
            raise TypeError("grad_scale must be an fp32 scalar on the GPU")
        a.grad_scale = grad_scale.data_ptr()
        a._keep_grad_scale = grad_scale
    return a


def lr_factor(adjust_lr_fn, rows, cols):
    """What the learning rate of a rows x cols matrix is multiplied by: "original" (None) sqrt(max(1, rows / cols)), "match_rms_adamw"
    0.2 sqrt(max(rows, cols))."""
    name = "original" if adjust_lr_fn is None else adjust_lr_fn
    if name not in _ADJUST:
        raise ValueError(f"unknown adjust_lr_fn {adjust_lr_fn!r}: original or match_rms_adamw")
    return _ADJUST[name](rows, cols)


def matrix_shape(p):
    """Rows and columns that a parameter is taken as: its first size and all others together, as a convolution's weight is read."""
    if p.dim() < 2 or p.numel() == 0:
        raise ValueError(f"a parameter of shape {tuple(p.shape)} is no matrix: give its group use_muon=False")
    return p.shape[0], p.numel() // p.shape[0]


# --------------------------------------------------------------------------------------------------------------- optimizer
class ShardMuon(_ShardOptimizer):
    """Momentum, orthogonalised, as the update of weight matrices; AdamW for what is none.

    Arguments and state (``momentum_buffer``) of ``torch.optim.Muon``: checkpoints go both ways. Parameters of more than two sizes
    are taken as matrices of their first size by all others. Per step and matrix ``buf += (1 - momentum) (g - buf)``, ``u = g + momentum
    (buf - g)`` with nesterov (else buf), ``p = p (1 - lr weight_decay) - lr f orthogonalize(u)``, f by ``adjust_lr_fn``
    (:func:`lr_factor`). All matrices of a step go through the same launches.

    ``ns_dtype``: torch.float32 (22 bits of every factor in the products) or torch.bfloat16 (11 bits and a third of the products:
    the update is off by about 2e-3 of its length). A parameter group with ``use_muon=False`` is updated by AdamW with the group's ``betas`` and
    ``eps`` (``adam_eps`` unless the group names one): biases, norms, embeddings. ``step(gradients)``, ``attach_replicas``: as for the others.

    Parameters and gradients are float32 on one GPU, parameters contiguous. A step can be recorded in a graph from the third on with the same
    gradients' memory (the first makes the state, the second the list of matrices); learning rates and the like are then the recorded ones. One that
    updates anything by AdamW is refused while recording: its step count could not rise."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, ns_coefficients=COEFFICIENTS, eps=1e-7, ns_steps=5,
                 adjust_lr_fn=None, ns_dtype=torch.float32, betas=(0.9, 0.999), adam_eps=1e-8):
        if not 0.0 <= lr:
            raise ValueError("Invalid learning rate: {}".format(lr))
        if not 0.0 <= weight_decay:
            raise ValueError("Invalid weight_decay value: {}".format(weight_decay))
        self._adam_eps = adam_eps
        self._adam = None
        self._recorded = {}         # plans that a graph's launches read
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, ns_coefficients=tuple(ns_coefficients),
                                      eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn, ns_dtype=ns_dtype, use_muon=True, betas=betas,
                                      amsgrad=False))

    def add_param_group(self, param_group):
        if not param_group.get("use_muon", True):
            param_group.setdefault("eps", self._adam_eps)
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(group):
        if not group["use_muon"]:
            b1, b2 = group["betas"]
            if not 0.0 <= b1 < 1.0 or not 0.0 <= b2 < 1.0:
                raise ValueError("Invalid beta parameters: {}".format(group["betas"]))
            if not 0.0 <= group["eps"]:
                raise ValueError("Invalid epsilon value: {}".format(group["eps"]))
            return
        if not 0.0 <= group["momentum"] < 1.0:
            raise ValueError("Invalid momentum value: {}".format(group["momentum"]))
        _check_growth(_newton_schulz(group["ns_steps"], group["ns_coefficients"], group["eps"], group["ns_dtype"]))
        for p in group["params"]:
            lr_factor(group["adjust_lr_fn"], *matrix_shape(p))

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:             # a checkpoint of torch's optimizer names none of these
            for name, value in (("use_muon", True), ("ns_dtype", torch.float32), ("betas", (0.9, 0.999)), ("amsgrad", False)):
                group.setdefault(name, value)

    def attach_replicas(self, main_params=(), *replica_params):
        super().attach_replicas(main_params, *replica_params)
        self._adam = None
        return self

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        self._adam = None

    def _state_names(self):
        return ("momentum_buffer",)

    def _signature(self, counts, params, grads, where, states):
        return super()._signature(counts, params, grads, where, states) + tuple([p.shape for p in params]) + tuple([g.dtype for g in grads])

    def _others(self):
        """The AdamW that updates the groups without orthogonalisation, on this optimizer's groups and state."""
        groups = [g for g in self.param_groups if not g["use_muon"]]
        if not groups:
            return None
        if self._adam is None:
            self._adam = ShardAdamW([p for g in groups for p in g["params"]])
            self._adam._replicas = self._replicas
        self._adam.param_groups, self._adam.state = groups, self.state
        return self._adam

    def _matched(self, gradients):
        counts, params, grads, where = super()._matched(gradients)
        keep, at = [], 0
        for gi, n in enumerate(counts):
            if self.param_groups[gi]["use_muon"]:
                keep += range(at, at + n)
            else:
                counts[gi] = 0
            at += n
        if len(keep) == at:
            return counts, params, grads, where
        return counts, [params[i] for i in keep], [grads[i] for i in keep], [where[i] for i in keep] if where else where

    @staticmethod
    def _key(group):
        """What a launch takes one value of."""
        return (float(group["momentum"]), bool(group["nesterov"]), tuple(group["ns_coefficients"]), float(group["eps"]), int(group["ns_steps"]),
                group["ns_dtype"])

    @torch.no_grad()
    def step(self, gradients=None, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if gradients is not None:
            gradients = list(gradients)
        matched = self._matched(gradients)
        states = list(map(self.state.get, matched[1]))
        sig = self._signature(*matched, states)
        if matched[1] and sig not in self._recipes and _recording(matched[1][0]):
            raise RuntimeError("a step is prepared before it is recorded: take two with these gradients first")
        launches, held = self._remembered(sig), None        # held: copies of gradients that the launches are to read
        if matched[1] and launches is None:
            launches, held = self._prepare_launches(matched)
        others = self._others()
        if others is not None and torch.cuda.is_current_stream_capturing() and others._matched(gradients)[1]:
            raise RuntimeError("AdamW's bias corrections are by value: a step that updates anything by it cannot be recorded")
        # whatever is refused is refused here, before any weight moves
        runs = [(plan, self._args(key, places)) for plan, key, places, _ in launches or ()]
        if others is not None:
            others.step(gradients)
        for plan, args in runs:
            if torch.cuda.is_current_stream_capturing():
                self._recorded[id(plan)] = plan
            plan.run(args)
        if held is not None and not self._volatile:
            self._remember(sig, launches)
        return loss

    def _prepare_launches(self, matched):
        """[(plan, what its launch takes one value of, its groups, their adjust_lr_fn)] of a call, and what has to live until they are queued."""
        self._volatile, launches, self._late_copies = False, [], []
        batches = {}
        for gi, p, g in self._pairs(*matched):
            group = self.param_groups[gi]
            rows, cols = matrix_shape(p)
            if not p.is_contiguous():
                raise ValueError(f"a parameter of shape {tuple(p.shape)} is not contiguous: its columns have no order")
            g = self._prepare(p, g)
            st = self.state[p]
            if st.get("momentum_buffer") is None:
                st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                self._volatile = True             # state created in this call: remember the next one
            batches.setdefault(self._key(group), []).append((gi, dict(
                grad=g, momentum=st["momentum_buffer"], param=p.data, rows=rows, cols=cols, lr_factor=lr_factor(group["adjust_lr_fn"], rows, cols),
                fanout=[q.data for q in self._replicas.get(id(p), ())])))
        for key, items in batches.items():
            slots = {}
            for gi, item in items:
                item["group"] = slots.setdefault(gi, len(slots))
                if len(slots) > L.MAX_GROUPS:
                    raise RuntimeError(f"more than {L.MAX_GROUPS} parameter groups in one launch")
            plan = self._plan([item for _, item in items], key[-1], keep=not self._volatile)
            launches.append((plan, key, list(slots), [self.param_groups[gi]["adjust_lr_fn"] for gi in slots]))
        return launches, batches

    def _args(self, key, places):
        momentum, nesterov, coefficients, eps, steps, dtype = key
        return make_muon_args([self.param_groups[gi] for gi in places], momentum=momentum, nesterov=nesterov, steps=steps,
                              coefficients=coefficients, eps=eps, dtype=dtype)

    def _plan(self, items, dtype, keep):
        if not keep:                                  # names copies that are gone after this call
            return MuonPlan(items, dtype)
        key = (dtype, *((*[i[t].data_ptr() for t in ("grad", "momentum", "param")], i["rows"], i["cols"], i["group"], i["lr_factor"],
                         *[f.data_ptr() for f in i["fanout"]]) for i in items))
        plan = self._plans.get(key)
        if plan is None:
            if len(self._plans) >= self._max_cached_plans:
                self._plans.clear()
            plan = self._plans[key] = MuonPlan(items, dtype)
        return plan

    def _remembered(self, sig):
        """The launches of a remembered call, None when a value changed that they were split by or that their plans hold."""
        launches, _ = self._recipes.get(sig, (None, None))
        for _, key, places, adjust in launches or ():
            for gi, how in zip(places, adjust):
                group = self.param_groups[gi]
                if self._key(group) != key or group["adjust_lr_fn"] != how:
                    return None
        return launches
