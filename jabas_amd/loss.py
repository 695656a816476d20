"""Losses over a large vocabulary, forward and backward, as hand-written kernels (``include/jabas_loss.h``).

What ends a virtual stream worker's forward pass: cross entropy and distillation from a teacher's top logits, either over
logits in hand or straight from the hidden states and the classifier's weight. The latter never keep the logits: the
product is worked through in tiles whose maxima and sums are all that leaves the chip, and the backward pass computes them
again, a piece of the vocabulary at a time. K workers on one GPU hold K sets of activations, and [tokens, vocabulary] logits
are the largest of them (6400 tokens over 32317 in fp32: 0.83 GB per worker, once for the logits and once for their gradient).
Between the passes a call holds nothing of that size; while one runs, its workspace holds copies of the operands and a piece's
row gradients: over a vocabulary of 32317 and 1024 features, forward and backward, 169 and 672 MB for 6400 rows in fp32, 23 and
324 in bf16. Logits and their gradient would be 1655 and 827; up to about 1600 rows (142 and 396 MB in fp32, 414 of logits) they would be
the smaller, so few tokens gain what is not held between the passes, and nothing at the peak.

They stand in for the translation model's classifier (examples/gnmt/seq2seq/models/decoder.py) with its criterion and for
the vision examples' ``CrossEntropyLoss``; a trainer calls them as ``criterion(model(x), y)`` (jabas/train/trainer.py:82-86,
171-174), see :class:`LinearCrossEntropy` and :class:`LinearTopkDistillation`.

All of them are autograd functions on the current stream of the tensors' device, once differentiable; there is no CPU path, and a
forward-mode derivative or a function transform that differentiates is refused. What records or replaces operations (torch.jit.trace,
make_fx, torch.compile, a dispatch or function mode) sees them as the operators ``jabas::loss_forward`` and ``jabas::loss_backward``.
Every input keeps its place in memory: nothing is changed in place, nothing is kept between calls but what autograd saves (the
inputs, 16 bytes a row, 8 bytes an entry of the teacher). Results are the same from run to run: no sum depends on the order of
atomics.
"""
import ctypes as C
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .sync import _stream_ptr, _watched

REDUCTIONS = {"none": L.LOSS_NONE, "mean": L.LOSS_MEAN, "sum": L.LOSS_SUM}
MAX_ENTRIES = L.LOSS_MAX_ENTRIES


def _matrix(t, what, dtype=None):
    """Refuses what is no fp32 or bf16 tensor (``dtype``: none of that type) on the GPU."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor")
    if not t.is_cuda:
        raise ValueError(f"{what}: must live on the GPU, got {t.device}")
    if dtype is None:
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"{what}: must be float32 or bfloat16, got {t.dtype}")
    elif t.dtype != dtype:
        raise TypeError(f"{what}: expected {dtype}, got {t.dtype}")


def _rows_of(t):
    """``t`` as a matrix (its leading sizes as one) of contiguous rows: as it lies where it has that form, else a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_row_tensor(t, shape, dtype, device, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor")
    if t.dtype != dtype:
        raise TypeError(f"{what}: expected {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{what}: on {t.device}, expected {device}")
    if t.shape != shape:
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _flat(t):
    return t if t.dim() == 1 and t.is_contiguous() else t.reshape(-1).contiguous()


def _reduction(name):
    if name not in REDUCTIONS:
        raise ValueError(f"unknown reduction {name!r}: none, mean or sum")
    return REDUCTIONS[name]


# JabasLoss as one write: a foreign assignment per field costs more than the launches of a short call (10 us in a backward thread)
_LOSS = struct.Struct("4Q6q2iQqd3Qqd3Q")
assert _LOSS.size == C.sizeof(L.JabasLoss)


def _call(spec, hidden, weight, bias, logits, target, teacher_index, teacher_logits, teacher_lse, state):
    """The JabasLoss of a call. ``spec``: reduction, ignore_index, label_smoothing, temperature; ``state``: the rows' states, then the
    entries' probabilities, then their tokens."""
    if hidden is None:
        rows, vocab = logits.shape
        ptrs, strides, width, dtype = (0, 0, 0, logits.data_ptr()), (0, 0, _row_stride(logits)), 0, logits.dtype
    else:
        rows, width = hidden.shape
        vocab, dtype = weight.shape[0], hidden.dtype
        ptrs = hidden.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), 0
        strides = _row_stride(hidden), _row_stride(weight), 0
    at = state.data_ptr()
    if teacher_index is None:
        k, against, entries = 0, (0, 0, 0), (0, 0)
    else:
        k = teacher_index.shape[1]
        against = teacher_index.data_ptr(), teacher_logits.data_ptr(), 0 if teacher_lse is None else teacher_lse.data_ptr()
        p = at + 16 * rows + 16
        entries = p + 4 * rows * k, p
    c = L.JabasLoss()
    reduction, ignore_index, smoothing, temperature = spec
    _LOSS.pack_into(c, 0, *ptrs, *strides, rows, vocab, width, L.F32 if dtype == torch.float32 else L.BF16, reduction,
                    0 if target is None else target.data_ptr(), ignore_index, smoothing, *against, k, temperature, at, *entries)
    return c


def _sizes(rows, k, reduction):
    """Shapes of the loss and of the state."""
    return (rows,) if reduction == L.LOSS_NONE else (), 4 * rows + 4 + 2 * rows * k


def _workspace(c, backward, device):
    n = L.lib().jabas_loss_workspace_bytes(C.byref(c), backward)
    # 256 bytes are what the caching allocator aligns to at least
    return torch.empty(n, dtype=torch.uint8, device=device), n


def _forward(spec, tensors):
    """(loss, state) on the current stream of the tensors' device."""
    main = tensors[3] if tensors[0] is None else tensors[0]
    device, rows = main.device, main.shape[0]
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _forward(spec, tensors)
    k = 0 if tensors[5] is None else tensors[5].shape[1]
    shape, words = _sizes(rows, k, spec[0])
    state = torch.empty(words, dtype=torch.float32, device=device)
    out = torch.empty(shape, dtype=torch.float32, device=device)
    c = _call(spec, *tensors, state)
    ws, n = _workspace(c, 0, device)
    L.check(L.lib().jabas_loss_forward(C.byref(c), out.data_ptr(), ws.data_ptr(), n, _stream_ptr()), "jabas_loss_forward")
    return out, state


def _backward(spec, tensors, state, needs, upstream):
    device = upstream.device
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _backward(spec, tensors, state, needs, upstream)
    if upstream.dtype != torch.float32 or not upstream.is_contiguous():
        upstream = upstream.to(torch.float32).contiguous()
    grads = [torch.empty(t.shape, dtype=t.dtype, device=device) if t is not None and need else None for t, need in zip(tensors, needs)]
    c = _call(spec, *tensors, state)
    ws, n = _workspace(c, 1, device)
    L.check(L.lib().jabas_loss_backward(C.byref(c), upstream.data_ptr(), *[None if t is None else t.data_ptr() for t in grads],
                                        ws.data_ptr(), n, _stream_ptr()), "jabas_loss_backward")
    return grads


# The same two steps as operators, for whoever watches operations: a launch through the C ABI is not seen by a recorder, which would hold
# the results' memory and nothing that writes it. Their dispatch costs more than a small call's launches, so others go without.
_LIBRARY = torch.library.Library("jabas", "DEF")
_TENSORS = ("hidden", "weight", "bias", "logits", "target", "teacher_index", "teacher_logits", "teacher_lse")
_CALL = ", ".join(f"Tensor? {t}" for t in _TENSORS) + ", int reduction, int ignore_index, float label_smoothing, float temperature"
_LIBRARY.define(f"loss_forward({_CALL}) -> (Tensor, Tensor)")
_LIBRARY.define(f"loss_backward({_CALL}, Tensor state, Tensor upstream, bool[] needs) -> Tensor[]")


def _op_forward(*args):
    return _forward(args[8:12], args[:8])


def _op_backward(*args):
    *_, state, upstream, needs = args
    return [g for g in _backward(args[8:12], args[:8], state, needs, upstream) if g is not None]


_LIBRARY.impl("loss_forward", _op_forward, "CUDA")
_LIBRARY.impl("loss_backward", _op_backward, "CUDA")


@torch.library.register_fake("jabas::loss_forward", lib=_LIBRARY)
def _fake_forward(*args):
    main = args[3] if args[0] is None else args[0]
    shape, words = _sizes(main.shape[0], 0 if args[5] is None else args[5].shape[1], args[8])
    return main.new_empty(shape, dtype=torch.float32), main.new_empty(words, dtype=torch.float32)


@torch.library.register_fake("jabas::loss_backward", lib=_LIBRARY)
def _fake_backward(*args):
    return [t.new_empty(t.shape) for t, need in zip(args[:4], args[-1]) if t is not None and need]


def _op_setup(ctx, inputs, output):
    ctx.spec = inputs[8:]
    ctx.save_for_backward(*inputs[:8], output[1])


def _op_grads(spec, tensors, state, needs, upstream):
    """What ``_backward`` returns, through the operator."""
    needs = [t is not None and need for t, need in zip(tensors, needs)]
    grads = iter(torch.ops.jabas.loss_backward(*tensors, *spec, state, upstream, needs))
    return [next(grads) if need else None for need in needs]


def _op_gradient(ctx, upstream, _):
    *tensors, state = ctx.saved_tensors
    return (*_op_grads(ctx.spec, tensors, state, ctx.needs_input_grad[:4], upstream), *[None] * 8)


def _op_no_gradient(ctx, *upstream):
    raise RuntimeError("the losses can be differentiated once")


torch.library.register_autograd("jabas::loss_forward", _op_gradient, setup_context=_op_setup, lib=_LIBRARY)
torch.library.register_autograd("jabas::loss_backward", _op_no_gradient, lib=_LIBRARY)
_HELD = torch.Tensor, torch.nn.Parameter
_compiles, _traces, _transform = torch.compiler.is_dynamo_compiling, torch._C._is_tracing, torch._C._functorch.peek_interpreter_stack
_dispatch_modes, _function_modes = torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack


def _direct(*tensors):
    """Whether kernels may read the tensors, and write others, without anyone being told: nothing watches (``_watched``, in fewer steps: a
    small call's time is the host's), no function transform is under way, and memory holds what the tensors stand for (tensors
    without memory of their own have no address to ask for)."""
    if _compiles() or _traces() or _dispatch_modes() or _transform() is not None or (_function_modes() and _watched()):
        return False
    for t in tensors:
        if t is not None and (type(t) not in _HELD or t.is_neg() or t._is_zerotensor()):
            return False
    return True


class _Loss(torch.autograd.Function):
    """``spec``: what is no tensor. The tensors come one by one so that autograd sees them."""

    @staticmethod
    def forward(ctx, spec, *tensors):
        out, state = _forward(spec, tensors)
        ctx.spec = spec
        ctx.save_for_backward(*tensors, state)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        *tensors, state = ctx.saved_tensors
        run = _backward if _direct(upstream) else _op_grads         # the others are what the forward pass read
        return (None, *run(ctx.spec, tensors, state, ctx.needs_input_grad[1:5], upstream), None, None, None, None)


def _apply(spec, *tensors):
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors[:4]):
        raise RuntimeError("the losses have no forward-mode derivative")
    if not _direct(*tensors):
        return torch.ops.jabas.loss_forward(*tensors, *spec)[0]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors[:4]):
        return _Loss.apply(spec, *tensors)
    return _forward(spec, tensors)[0]


def _linear_inputs(hidden, weight, bias):
    _matrix(hidden, "hidden")
    _matrix(weight, "weight", hidden.dtype)
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)}: the last sizes must agree, weight has two")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("weight: needs at least one token and one feature")
    if weight.device != hidden.device:
        raise ValueError(f"weight: on {weight.device}, expected {hidden.device}")
    if bias is not None:
        _check_row_tensor(bias, weight.shape[:1], hidden.dtype, hidden.device, "bias")
        bias = bias.contiguous()
    return _rows_of(hidden), _rows_of(weight), bias


def _teacher_inputs(lead, device, dtype, teacher_index, teacher_logits, teacher_lse, temperature):
    if not isinstance(teacher_index, torch.Tensor) or teacher_index.dim() != len(lead) + 1:
        raise ValueError(f"teacher_index: expected a tensor of shape {tuple(lead)} and the entries")
    k = teacher_index.shape[-1]
    if not 1 <= k <= MAX_ENTRIES:
        raise ValueError(f"teacher_index: 1..{MAX_ENTRIES} entries per row, got {k}")
    _check_row_tensor(teacher_index, (*lead, k), torch.int64, device, "teacher_index")
    _check_row_tensor(teacher_logits, (*lead, k), dtype, device, "teacher_logits")
    if teacher_lse is not None:
        _check_row_tensor(teacher_lse, lead, torch.float32, device, "teacher_lse")
        teacher_lse = _flat(teacher_lse.detach())
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    return teacher_index.reshape(-1, k).contiguous(), teacher_logits.detach().reshape(-1, k).contiguous(), teacher_lse


def linear_cross_entropy(hidden, weight, target, bias=None, *, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """Cross entropy of the classifier ``hidden @ weight.T + bias`` against ``target``, without keeping the logits.

    hidden: (..., width) float32 or bfloat16; weight: (vocab, width) of the same type; bias: (vocab,) of the same type or
    None (-inf rules a token out); target: (...) int64. The loss of a row with logits z and label t is
    ``logsumexp(z) - (1 - e) z[t] - e mean(z)``, e = label_smoothing. Rows whose label is ``ignore_index`` do not count:
    loss and gradient are 0 whatever their hidden states hold; a row whose upstream gradient is 0 has gradient 0 too. Any
    other label outside the vocabulary gives NaN, one that is ruled out an infinite loss.

    reduction: "mean" over the rows that count (0 where none does), "sum" or "none" (the shape of target). The loss is
    float32, sums are kept in 32 bits; gradients have the inputs' type.

    Up to 64 rows (bfloat16 over a large weight: 32) the products are float32's, or with bfloat16 take the inputs as they are
    and the row gradients dz = dL/dz as two bfloat16 planes (16 bits at any size). More rows take dz as fp16: with bfloat16 one plane,
    an eighth of bfloat16's step down to 2^-29 of the row's upstream gradient and steps of 2^-39 of it below, so that the part of dW or of
    dX that comes from tokens less probable than 2^-40 is 0; with float32 two, 22 bits down to 2^-25 and steps of 2^-50. float32's
    other factors are two fp16 planes too, the products three: 22 bits of a hidden state down to 2^-16 of the largest of its row
    (for dW: of its feature), of a weight down to 2^-27 of the largest of its token (in the backward pass: of a piece of the vocabulary),
    and a fixed step below."""
    x, w, b = _linear_inputs(hidden, weight, bias)
    lead = hidden.shape[:-1]
    _check_row_tensor(target, lead, torch.int64, hidden.device, "target")
    if not 0.0 <= label_smoothing < 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1), got {label_smoothing}")
    spec = _reduction(reduction), int(ignore_index), float(label_smoothing), 1.0
    out = _apply(spec, x, w, b, None, _flat(target), None, None, None)
    return out.view(lead) if reduction == "none" else out


def topk_distillation(logits, teacher_index, teacher_logits, *, temperature=1.0, teacher_lse=None, reduction="mean"):
    """Distillation of ``logits`` (..., vocab) from a teacher's top logits, logits in hand.

    teacher_index: (..., k) int64, the tokens the teacher's logits belong to, k up to 255; teacher_logits: (..., k) of the
    logits' type. A place with a negative index or logit -inf holds no entry; a row without any does not count (loss and gradient
    0); places that name one token are one event with the sum of their probabilities. With q = softmax(logits / T) over the
    whole vocabulary the loss of a row is ``T^2 sum_j p_j (log p_j - log q_j)``:

    - ``teacher_lse`` None: p is the softmax of the entries' logits / T;
    - ``teacher_lse`` (...) float32, the teacher's logsumexp(logits / T) over its whole vocabulary: p are its true
      probabilities, and what they leave, r = max(0, 1 - sum p), is one more event that the student meets with all tokens
      that are no entry: ``+ T^2 r (log r - log sum_others q)``. Where all of those are ruled out (logits of -inf) a rest costs an
      infinite loss, as a label does that is ruled out: entries that are all there is to choose from take no ``teacher_lse``.

    reduction as in :func:`linear_cross_entropy`. No gradient flows to the teacher."""
    _matrix(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits: needs at least one token")
    lead = logits.shape[:-1]
    index, t, lse = _teacher_inputs(lead, logits.device, logits.dtype, teacher_index, teacher_logits, teacher_lse, temperature)
    out = _apply((_reduction(reduction), 0, 0.0, float(temperature)), None, None, None, _rows_of(logits), None, index, t, lse)
    return out.view(lead) if reduction == "none" else out


def linear_topk_distillation(hidden, weight, teacher_index, teacher_logits, bias=None, *, temperature=1.0, teacher_lse=None,
                             reduction="mean"):
    """:func:`topk_distillation` of the classifier ``hidden @ weight.T + bias`` without keeping its logits; hidden, weight
    and bias as in :func:`linear_cross_entropy`, teacher_logits of their type."""
    x, w, b = _linear_inputs(hidden, weight, bias)
    lead = hidden.shape[:-1]
    index, t, lse = _teacher_inputs(lead, hidden.device, hidden.dtype, teacher_index, teacher_logits, teacher_lse, temperature)
    out = _apply((_reduction(reduction), 0, 0.0, float(temperature)), x, w, b, None, None, index, t, lse)
    return out.view(lead) if reduction == "none" else out


class LinearCrossEntropy(torch.nn.Module):
    """:func:`linear_cross_entropy` as a trainer's criterion: ``criterion((hidden, weight, bias), target)`` for a model whose
    forward returns its last hidden states with its classifier's weight and bias (None where it has none)."""

    def __init__(self, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
        super().__init__()
        self.ignore_index, self.label_smoothing, self.reduction = ignore_index, label_smoothing, reduction

    def forward(self, output, target):
        hidden, weight, bias = output
        return linear_cross_entropy(hidden, weight, target, bias, ignore_index=self.ignore_index,
                                    label_smoothing=self.label_smoothing, reduction=self.reduction)


class LinearTopkDistillation(torch.nn.Module):
    """:func:`linear_topk_distillation` as a trainer's criterion: ``criterion((hidden, weight, bias), (teacher_index,
    teacher_logits))`` or ``(teacher_index, teacher_logits, teacher_lse)``."""

    def __init__(self, temperature=1.0, reduction="mean"):
        super().__init__()
        self.temperature, self.reduction = temperature, reduction

    def forward(self, output, teacher):
        hidden, weight, bias = output
        index, logits, lse = teacher if len(teacher) == 3 else (*teacher, None)
        return linear_topk_distillation(hidden, weight, index, logits, bias, temperature=self.temperature, teacher_lse=lse,
                                        reduction=self.reduction)
