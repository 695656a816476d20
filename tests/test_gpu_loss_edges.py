"""The losses (jabas_amd.loss) where their paths have to agree with the definition and with each other: rests that no token can meet, rows of any
size beside ordinary ones, weights of very different sizes, tokens ruled out that are named all the same, recorders, and means.

The bounds are those of ``Reference`` in test_gpu_loss.py, in whose terms a case says where it needs another.
"""
import math

import pytest
import torch

from jabas_amd import loss as losses
from tests.test_gpu_loss import F64, IGNORE, TYPES, Reference, _entries, _gen, _grads, _inputs

pytestmark = pytest.mark.gpu


def _cpu(t):
    return None if t is None else t.detach().cpu().to(F64)


class Given(Reference):
    """The bounds of ``Reference`` for row gradients that a test states itself: ``dz``, ``size`` (what their parts sum to without
    their signs) and the rows' losses, all without the upstream gradient ``up``."""

    def __init__(self, dz, size, row_losses, Z, up, hidden=None, weight=None, bias=None, T=1.0):
        x, w, b = _cpu(hidden), _cpu(weight), _cpu(bias)
        self.Z, self.T, self.counted = Z, T, torch.ones(len(dz), dtype=torch.bool)
        self.loss, self.loss_size = row_losses, row_losses.abs()
        dz, size = dz * up[:, None], size * up[:, None].abs()
        self.dz, self.size = dz, size
        if x is None:
            self.grads, self.sizes = [dz], [size]
        else:
            self.grads, self.sizes = [dz @ w, dz.t() @ x], [size @ w.abs(), size.t() @ x.abs()]
            if b is not None:
                self.grads.append(dz.sum(0))
                self.sizes.append(size.sum(0))


def _largest_logit(x, w, b=None):
    x, w, b = _cpu(x), _cpu(w), _cpu(b)
    return (x.abs() @ w.abs().t()).max().item() + (0.0 if b is None else b[torch.isfinite(b)].abs().max().item())


PATHS = {"whole": (200, 3000, 0), "parts": (6, 50000, 0), "few": (20, 600, 64), "tiles": (80, 600, 64), "large_tiles": (514, 17000, 64)}


# ------------------------------------------------------------------ what the entries leave
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
@pytest.mark.parametrize("path", list(PATHS))
def test_a_rest_that_no_token_can_meet(gpu, path, mask, dtype):
    """Every token but the entries is ruled out and the teacher leaves a rest: the loss is infinite (at the lowest finite value as large as
    that makes it), the entries' gradients are T (M q - p) with the rest in M, and the tokens at -inf have none. Without a rest (a teacher whose entries sum to
    more than 1) the loss is finite."""
    rows, vocab, width = PATHS[path]
    k, gen = 5, _gen(rows)
    low = -math.inf if mask == "-inf" else torch.finfo(TYPES[dtype]).min
    names = torch.randperm(vocab, generator=gen)[:k]
    index = torch.stack([names[torch.randperm(k, generator=gen)] for _ in range(rows)])
    teacher = torch.randn(rows, k, generator=gen).to(TYPES[dtype])
    lse = torch.logsumexp(teacher.float(), 1) + 0.5
    lse[::3] -= 1.5
    others = torch.ones(vocab, dtype=torch.bool)
    others[names] = False
    up = torch.rand(rows, generator=gen) + 0.5
    args = index.to(gpu), teacher.to(gpu)
    if width:
        (x, w, b), _ = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
        with torch.no_grad():
            b[others.to(gpu)] = low
        loss = losses.linear_topk_distillation(x, w, *args, b, teacher_lse=lse.to(gpu), reduction="none")
        grads = _grads(loss, (x, w, b), up.to(gpu))
        z = _cpu(x) @ _cpu(w)[names].t() + _cpu(b)[names]
        Z = _largest_logit(x, w, b.detach().clamp(min=-100.0))
    else:
        x = w = b = None
        logits = torch.randn(rows, vocab, generator=gen).to(TYPES[dtype])
        logits[:, others] = low
        logits = logits.to(gpu).requires_grad_(True)
        loss = losses.topk_distillation(logits, *args, teacher_lse=lse.to(gpu), reduction="none")
        grads = _grads(loss, (logits,), up.to(gpu))
        z = _cpu(logits)[:, names]
        Z = z.abs().max().item()
    at = torch.argsort(names)[torch.searchsorted(names.sort().values, index)]       # which of the names an entry is
    p = torch.zeros(rows, k, dtype=F64).scatter_(1, at, (teacher.to(F64) - lse.to(F64)[:, None]).exp())
    r = (1.0 - p.sum(1)).clamp(min=0.0)
    logq = torch.log_softmax(z, 1)
    M = p.sum(1) + r
    dz, size = torch.zeros(rows, vocab, dtype=F64), torch.zeros(rows, vocab, dtype=F64)
    dz[:, names], size[:, names] = M[:, None] * logq.exp() - p, M[:, None] * logq.exp() + p
    if mask == "lowest":        # equal logits share what the rest asks for
        dz[:, others] = -(r / int(others.sum()))[:, None]
        size[:, others] = -dz[:, others]
    finite = (p * (p.log() - logq)).sum(1)
    got = loss.detach().cpu().to(F64)
    left = r > 0
    assert bool(left.any()) and not bool(left.all())
    if mask == "-inf":
        assert bool((got[left] == math.inf).all())
    else:
        assert bool((got[left] >= 0.99 * r[left] * -low).all())
    ref = Given(dz, size, finite, Z, up.to(F64), x, w, b)
    ref.loss, ref.loss_size = finite[~left], finite[~left].abs()
    ref.check(loss[~left.to(gpu)], grads, dtype)
    if mask == "-inf":
        assert not bool((grads[1][others.to(gpu)] if width else grads[0][:, others.to(gpu)]).any())


@pytest.mark.parametrize("path", ["whole", "few", "tiles"])
def test_rows_whose_entries_are_all_there_is_count(gpu, path):
    """Every token is an entry of a teacher that gives all of them next to nothing: a loss of 0, in a mean over all the rows."""
    rows, _, width = PATHS[path]
    gen = _gen(2)
    index = torch.arange(3).expand(rows, 3).contiguous()
    teacher = torch.randn(rows, 3, generator=gen)
    lse = torch.logsumexp(teacher, 1) + 0.25
    lse[::2] = 300.0
    if width:
        (x, w, _), _ = _inputs(gpu, rows, 3, width, "fp32", seed=1)
        call = lambda reduction: losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), teacher_lse=lse.to(gpu), reduction=reduction)
    else:
        z = torch.randn(rows, 3, generator=gen).to(gpu)
        call = lambda reduction: losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), teacher_lse=lse.to(gpu), reduction=reduction)
    each = call("none").detach().cpu().to(F64)
    assert not bool(each[::2].any()) and bool(each[1::2].any())
    assert float(call("mean").detach()) == pytest.approx(float(each.sum()) / rows, rel=2.0 ** -22)


# ------------------------------------------------------------------ rows and weights of any size
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [20, 80, 300])
@pytest.mark.parametrize("how", ["2^42", "inf"])
def test_a_row_far_above_one_leaves_the_others_alone(gpu, rows, dtype, how):
    """One row's probabilities sum to 2^42, or to infinity: the losses and the hidden states' gradients of the other rows are what they are without it. The
    row's own p are off by the rounding of t - teacher_lse, 2^-24 (|t| + |lse| + |t - lse|) < 2^-17."""
    vocab, width, k, far = 2001, 64, 8, 7
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
    index, teacher = _entries(gen, rows, vocab, k, dtype)
    lse = torch.logsumexp(teacher.float(), 1) + 0.5
    lse[far] = lse[far] - 30.0 if how == "2^42" else -math.inf
    up = torch.rand(rows, generator=gen) + 0.5
    loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b, teacher_lse=lse.to(gpu), reduction="none")
    grads = _grads(loss, (x, w, b), up.to(gpu))
    keep = torch.arange(rows) != far
    ref = Reference(x[keep.to(gpu)], w, b, index=index[keep], teacher=teacher[keep], lse=lse[keep], reduction="none", upstream=up[keep])
    ref.check(loss[keep.to(gpu)], [grads[0][keep.to(gpu)]], dtype)
    if how == "inf":
        assert not bool(loss[far].isfinite())
        return
    ref = Reference(x, w, b, index=index, teacher=teacher, lse=lse, reduction="none", upstream=up)
    rel = 2.0 ** -20 * (ref.Z + 4.0) + 2.0 ** -17 + (2.0 ** -10 if dtype == "bf16" else 0.0)
    last = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -22
    for g, want, size in zip(grads, ref.grads, ref.sizes):
        assert bool(((_cpu(g) - want).abs() <= rel * size + last * want.abs()).all())


@pytest.mark.parametrize("rows", [20, 80, 300, 514])
@pytest.mark.parametrize("form", ["labels", "entries"])
@pytest.mark.parametrize("outlier", [1e5, 1e8])
def test_one_large_weight_does_not_blur_the_others(gpu, rows, form, outlier):
    """fp32, one weight far above the others in a feature that no hidden state uses: the logits of the backward pass are as good as the
    forward pass's, so dW and db are. dX sums over the tokens, and its planes of the weight have one scale for a piece: off by 2^-40 of the largest
    weight for each unit of a row's dz."""
    vocab, width = 17000 if rows == 514 else 2001, 64
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, "fp32", True, seed=rows)
    with torch.no_grad():
        x[:, 5] = 0.0
        w[77, 5] = outlier
    if form == "labels":
        target = torch.randint(0, vocab, (rows,), generator=gen)
        loss = losses.linear_cross_entropy(x, w, target.to(gpu), b)
        ref = Reference(x, w, b, target=target)
    else:
        index, teacher = _entries(gen, rows, vocab, 9, "fp32")
        loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b)
        ref = Reference(x, w, b, index=index, teacher=teacher)
    grads = _grads(loss, (x, w, b))
    gx, sx = ref.grads.pop(0), ref.sizes.pop(0)
    ref.check(loss, grads[1:], "fp32")
    each = ref.sizes[1].sum() / rows * 1.5                   # the sum of a row's |dz|, about the same for all of them
    unit = 2.0 ** -20 * (ref.Z + 4.0)
    assert bool(((_cpu(grads[0]) - gx).abs() <= (unit + 2.0 ** -20) * sx + 2.0 ** -40 * outlier * each + 2.0 ** -22 * gx.abs()).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [80, 514])
def test_improbable_tokens_to_the_absolute_step(gpu, rows, dtype):
    """Tokens whose every probability is about e^-25: with many rows their row gradients are held in steps of 2^-39 (bf16) and 2^-50 (fp32) of the
    upstream gradient, so their rows of dW are off by half a step for each hidden state beside what is relative."""
    vocab, width = 17000, 64
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
    with torch.no_grad():
        b[1000:1200] -= 25.0
        b[1200:1300] -= 15.0
    target = torch.randint(0, 1000, (rows,), generator=gen)
    loss = losses.linear_cross_entropy(x, w, target.to(gpu), b, reduction="sum")
    grads = _grads(loss, (x, w, b))
    ref = Reference(x, w, b, target=target, reduction="sum")
    half = 2.0 ** (-40 if dtype == "bf16" else -51)
    unit = 2.0 ** -20 * (ref.Z + 4.0) + (2.0 ** -10 if dtype == "bf16" else 2.0 ** -20)
    last = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -22
    off, rare = (_cpu(grads[1]) - ref.grads[1]).abs(), slice(1000, 1300)
    assert bool((off <= unit * ref.sizes[1] + half * _cpu(x).abs().sum(0) + last * ref.grads[1].abs())[rare].all())
    # db is summed in 32 bits in front of the rounding
    off = (_cpu(grads[2]) - ref.grads[2]).abs()
    assert bool((off <= (unit + last) * ref.sizes[2])[rare].all())


# ------------------------------------------------------------------ tokens ruled out, and named all the same
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [20, 80, 514])
@pytest.mark.parametrize("form", ["labels", "smoothed", "entries"])
def test_ruled_out_tokens_that_are_named(gpu, rows, dtype, form):
    """A bias of -inf at a token that is a row's label or entry: the loss is infinite, and the gradients are dz W and dz^T X all the same,
    with dz = -p there; under label smoothing every token is named. Tokens that are ruled out and not named have none, whatever their weight."""
    vocab, width = 17000 if rows == 514 else 700, 64
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
    out = torch.arange(3, vocab, 5)
    with torch.no_grad():
        b[out.to(gpu)] = -math.inf
        if form != "smoothed":
            w[out[4::7].to(gpu)] = 1e30
    e = 0.1 if form == "smoothed" else 0.0
    fine = torch.tensor([v for v in range(vocab) if v % 5 != 3])
    target = fine[torch.randint(0, len(fine), (rows,), generator=gen)]
    target[::4] = out[2]
    up = torch.rand(rows, generator=gen) + 0.5
    p = torch.zeros(rows, vocab, dtype=F64)
    if form == "entries":
        index = torch.stack([target, fine[torch.randint(0, len(fine), (rows,), generator=gen)]], 1)
        teacher = torch.randn(rows, 2, generator=gen).to(TYPES[dtype])
        loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b, reduction="none")
        p.scatter_add_(1, index, torch.softmax(teacher.to(F64), 1))
    else:
        loss = losses.linear_cross_entropy(x, w, target.to(gpu), b, label_smoothing=e, reduction="none")
        p.scatter_(1, target[:, None], 1.0 - e)
        p += e / vocab
    grads = _grads(loss, (x, w, b), up.to(gpu))
    wd = _cpu(w)
    if form != "smoothed":
        wd[out[4::7]] = 0.0
    z = _cpu(x) @ wd.t() + _cpu(b)
    q = torch.softmax(z, 1)
    infinite = torch.ones(rows, dtype=torch.bool) if e else target == int(out[2])
    assert bool((loss.detach().cpu()[infinite] == math.inf).all())
    row_losses = torch.where(p > 0, p * (p.clamp(min=1e-300).log() * (form == "entries") - torch.log_softmax(z, 1)), torch.zeros_like(p)).sum(1)
    ref = Given(q - p, q + p, row_losses[~infinite], _largest_logit(x, wd, b), up.to(F64), x, wd, b)
    if infinite.all():
        ref.loss = ref.loss_size = torch.zeros((), dtype=F64)
        ref.check(torch.zeros(()), grads, dtype)
    else:
        ref.check(loss[~infinite.to(gpu)], grads, dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("path", list(PATHS))
def test_rows_without_upstream_have_no_gradient(gpu, path, dtype):
    """Rows whose upstream gradient is 0 (a program that weighs the losses itself), over hidden states or logits that are NaN: as if they were not there."""
    rows, vocab, width = PATHS[path]
    gen = _gen(rows)
    up = torch.rand(rows, generator=gen) + 0.5
    up[::3] = 0.0
    keep = up != 0
    index, teacher = _entries(gen, rows, vocab, 4, dtype)
    if not width:
        z = torch.randn(rows, vocab, generator=gen).to(TYPES[dtype]).to(gpu)
        z[::3] = float("nan")
        z.requires_grad_(True)
        loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), reduction="none")
        grad = _grads(loss, (z,), up.to(gpu))[0]
        assert not bool(grad[::3].any())
        Reference(logits=z[keep.to(gpu)], index=index[keep], teacher=teacher[keep], reduction="none", upstream=up[keep]).check(
            loss[keep.to(gpu)], [grad[keep.to(gpu)]], dtype)
        return
    (x, w, b), _ = _inputs(gpu, rows, vocab, width, dtype, True, seed=1)
    with torch.no_grad():
        x[::3] = float("nan")
    target = torch.randint(0, vocab, (rows,), generator=gen)
    for call, held in ((lambda: losses.linear_cross_entropy(x, w, target.to(gpu), b, reduction="none"), dict(target=target[keep])),
                       (lambda: losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b, reduction="none"),
                        dict(index=index[keep], teacher=teacher[keep]))):
        loss = call()
        grads = _grads(loss, (x, w, b), up.to(gpu))
        assert not bool(grads[0][::3].any())
        Reference(x[keep.to(gpu)], w, b, reduction="none", upstream=up[keep], **held).check(
            loss[keep.to(gpu)], [grads[0][keep.to(gpu)], *grads[1:]], dtype)


# ------------------------------------------------------------------ means, and weights past 32 bits
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,width", [(20, 3001, 64), (64, 3001, 64), (130, 1003, 192), (514, 17000, 72), (2500, 2001, 70)])
def test_a_mean_is_as_good_as_its_rows(gpu, rows, vocab, width, dtype):
    """A mean of rows that are each off by 2^-19 (Z + 4) T^2 and 2^-20 of themselves is off by no more."""
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
    target = torch.randint(0, vocab, (rows,), generator=gen)
    target[::7] = IGNORE
    index = torch.randint(0, vocab // 8, (rows, 8), generator=gen) + torch.arange(8) * (vocab // 8)
    index[1::7] = -1
    teacher = torch.randn(rows, 8, generator=gen).to(TYPES[dtype])
    lse = torch.logsumexp(teacher.float(), 1) + 0.5
    z = (x.detach().float() @ w.detach().float().t()).to(TYPES[dtype])
    entries = index.to(gpu), teacher.to(gpu)
    for loss, ref in ((losses.linear_cross_entropy(x, w, target.to(gpu), b, label_smoothing=0.1), Reference(x, w, b, target=target, smoothing=0.1)),
                      (losses.linear_topk_distillation(x, w, *entries, b, teacher_lse=lse.to(gpu)), Reference(x, w, b, index=index, teacher=teacher, lse=lse)),
                      (losses.topk_distillation(z, *entries, teacher_lse=lse.to(gpu)), Reference(logits=z, index=index, teacher=teacher, lse=lse))):
        bound = 2.0 ** -19 * (ref.Z + 4.0) + 2.0 ** -20 * float(ref.loss_size)
        assert abs(float(loss.detach()) - float(ref.loss)) <= bound


def test_gradients_of_a_weight_past_32_bits_of_offset(gpu):
    """Two rows against 2.2e9 elements of weight: dX, summed over five pieces of the vocabulary, and dW at the pieces' borders and past element 2^31. dz is held
    in two bf16 planes (2^-16), the logits are off by 2^-20 Z, and a result by a unit of its own (2^-8)."""
    rows, vocab, width = 2, 540000, 4096
    w = torch.empty(vocab, width, dtype=torch.bfloat16, device=gpu)
    w.normal_(std=0.02, generator=torch.Generator(device=gpu).manual_seed(2))
    x = torch.randn(rows, width, generator=_gen(3)).bfloat16().to(gpu).requires_grad_(True)
    target = torch.tensor([vocab - 3, 1 << 17])
    w.requires_grad_(True)
    loss = losses.linear_cross_entropy(x, w, target.to(gpu), reduction="none")
    gx, gw = _grads(loss.sum(), (x, w))
    pieces = range(0, vocab, 30000)
    xd, wd = x.detach().to(F64), w.detach()
    z = torch.cat([xd @ wd[i:i + 30000].to(F64).t() for i in pieces], 1)
    Z = max(float((xd.abs() @ wd[i:i + 30000].to(F64).abs().t()).max()) for i in pieces)
    dz = torch.log_softmax(z, 1).exp_()
    size = dz.clone()
    for r in range(rows):
        dz[r, target[r]] -= 1.0
        size[r, target[r]] += 1.0
    rel = 2.0 ** -20 * (Z + 4.0) + 2.0 ** -15
    ref, sizes = torch.zeros(rows, width, dtype=F64, device=gpu), torch.zeros(rows, width, dtype=F64, device=gpu)
    for i in pieces:
        ref += dz[:, i:i + 30000] @ wd[i:i + 30000].to(F64)
        sizes += size[:, i:i + 30000] @ wd[i:i + 30000].to(F64).abs()
    assert bool(((gx.to(F64) - ref).abs() <= rel * sizes + 2.0 ** -8 * ref.abs()).all())
    for at in (0, 1 << 17, 1 << 18, 3 << 17, 1 << 19, vocab):        # 2^31 elements: token 2^19
        s = slice(max(0, at - 64), min(vocab, at + 64))
        ref, sizes = dz[:, s].t() @ xd, size[:, s].t() @ xd.abs()
        assert bool(((gw[s].to(F64) - ref).abs() <= rel * sizes + 2.0 ** -8 * ref.abs()).all())


# ------------------------------------------------------------------ recorders, derivatives, streams
def _scored(gpu, seed, rows=70):
    (x, w, b), gen = _inputs(gpu, rows, 300, 64, "fp32", True, seed=seed)
    target = torch.randint(0, 300, (rows,), generator=gen).to(gpu)
    index, teacher = (t.to(gpu) for t in _entries(gen, rows, 300, 5, "fp32"))
    return [t.detach() for t in (x, w, b)], target, index, teacher


def _score(x, w, b, target, index, teacher):
    return (losses.linear_cross_entropy(x, w, target, b, reduction="none"), losses.linear_topk_distillation(x, w, index, teacher, b),
            losses.topk_distillation(x, index % 64, teacher, temperature=2.0))


def _train(x, w, b, target, index, teacher):
    x, w, b = (t.detach().requires_grad_(True) for t in (x, w, b))
    a, c, d = _score(x, w, b, target, index, teacher)
    return a, c, d, *torch.autograd.grad(a.sum() + c + d, (x, w, b))


@pytest.mark.parametrize("rows", [20, 70])
@pytest.mark.parametrize("recorder,what", [(r, _score) for r in ("trace", "real", "fake", "symbolic", "aot_eager")] +
                         [(r, _train) for r in ("real", "fake", "symbolic")])        # the other two record no backward pass inside a program
def test_recorded_calls_answer_for_other_inputs(gpu, recorder, what, rows):
    """A recording of a call holds the loss, not the memory that it was written to."""
    from torch.fx.experimental.proxy_tensor import make_fx
    (leaves, *rest), (others, *others_rest) = _scored(gpu, 1, rows), _scored(gpu, 2, rows)
    args, other = (*leaves, *rest), (*others, *others_rest)
    if recorder == "trace":
        recorded = torch.jit.trace(what, args, check_trace=False)
    elif recorder == "aot_eager":
        recorded = torch.compile(what, backend="aot_eager")
        recorded(*args)
    else:
        recorded = make_fx(what, tracing_mode=recorder)(*args)
    want = what(*other)
    torch.empty(1 << 20, device=gpu).fill_(float("nan"))
    for got in (recorded(*other), recorded(*other)):
        assert len(got) == len(want)
        for p, q in zip(got, want):
            assert torch.equal(p, q)


def test_a_traced_module_trains(gpu):
    """The gradients of a recorded call are the eager ones."""
    (x, w, b), target, _, _ = _scored(gpu, 1)
    (y, v, c), t, _, _ = _scored(gpu, 2)
    call = lambda x, w, b, t: losses.linear_cross_entropy(x, w, t, b, label_smoothing=0.1)
    leaves = [t.requires_grad_(True) for t in (y, v, c)]
    want = torch.autograd.grad(call(*leaves, t), leaves)
    for recorded in (torch.jit.trace(call, (x.requires_grad_(True), w, b, target), check_trace=False), torch.compile(call, backend="aot_eager")):
        for _ in range(2):
            for p, q in zip(torch.autograd.grad(recorded(*leaves, t), leaves), want):
                assert torch.equal(p, q)


def test_calls_under_modes_are_the_same(gpu):
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Above(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    seen = []

    class Below(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    leaves, *rest = _scored(gpu, 3)
    want = _train(*leaves, *rest)
    for mode in (Above(), Below(), torch.device("cpu")):
        with mode:
            got = _train(*leaves, *rest)
        for p, q in zip(got, want):
            assert torch.equal(p, q)
    assert sum("jabas" in s for s in seen) == 6         # three losses and their gradients are seen
    x = leaves[0].clone().requires_grad_(True)
    with Below():
        grad = torch.autograd.grad(losses.linear_cross_entropy(x, *leaves[1:2], rest[0]), x, create_graph=True)[0]
        with pytest.raises(RuntimeError):
            grad.sum().backward()               # once differentiable


def test_values_that_memory_does_not_hold(gpu):
    """A lazy negation is taken as what it stands for; so are tensors inside a function transform."""
    (x, w, b), target, index, teacher = _scored(gpu, 4)
    got = losses.linear_cross_entropy(torch._neg_view(x), torch._neg_view(w), target, torch._neg_view(b), reduction="none")
    assert torch.equal(got, losses.linear_cross_entropy(-x, -w, target, -b, reduction="none"))
    got = losses.topk_distillation(torch._neg_view(x), index % 64, torch._neg_view(teacher), reduction="none")
    assert torch.equal(got, losses.topk_distillation(-x, index % 64, -teacher, reduction="none"))
    call = lambda x: losses.linear_cross_entropy(x, w, target, b)
    leaf = x.clone().requires_grad_(True)
    up = torch._neg_view(torch.rand(len(x), device=gpu))
    each = losses.linear_cross_entropy(leaf, w, target, b, reduction="none")
    assert torch.equal(torch.autograd.grad(each, leaf, up, retain_graph=True)[0], torch.autograd.grad(each, leaf, up.clone())[0])
    assert torch.equal(torch.func.vmap(call)(torch.stack([x, -x])), torch.stack([call(x), call(-x)]))
    with pytest.raises(RuntimeError):       # refused, not lost
        torch.func.grad(call)(x)


def test_forward_mode_is_refused(gpu):
    """There is no forward-mode derivative, and none is lost silently."""
    import torch.autograd.forward_ad as forward
    (x, w, b), target, index, teacher = _scored(gpu, 5)
    with forward.dual_level():
        dual = forward.make_dual(x, torch.ones_like(x))
        calls = [lambda: losses.linear_cross_entropy(dual, w, target, b), lambda: losses.linear_topk_distillation(dual, w, index, teacher, b),
                 lambda: losses.topk_distillation(dual, index % 64, teacher),
                 lambda: losses.linear_cross_entropy(x, w, target, forward.make_dual(b, b)),
                 lambda: losses.linear_cross_entropy(dual, w.clone().requires_grad_(True), target, b)]
        for call in calls:
            with pytest.raises(RuntimeError):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError):
                call()
        losses.linear_cross_entropy(x, w, target, b)
        losses.topk_distillation(x, index % 64, forward.make_dual(teacher, teacher))       # nothing flows to the teacher
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: losses.linear_cross_entropy(x, w, target, b), (x,), (x,))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_calls_of_several_streams_at_once(gpu, dtype):
    """Workers of different sizes on streams of their own, none waiting for another: each gets what it gets alone."""
    work = []
    for i, (rows, vocab, width) in enumerate([(300, 9000, 128), (20, 9000, 128), (514, 17000, 64), (90, 3000, 256)]):
        (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=i)
        target = torch.randint(0, vocab, (rows,), generator=gen).to(gpu)
        index, teacher = (t.to(gpu) for t in _entries(gen, rows, vocab, 20, dtype))
        work.append((x, w, b, target, index, teacher))

    def step(x, w, b, target, index, teacher):
        a = losses.linear_cross_entropy(x, w, target, b, label_smoothing=0.1)
        c = losses.linear_topk_distillation(x, w, index, teacher, b, temperature=2.0)
        return [a.detach(), c.detach(), *_grads(a, (x, w, b)), *_grads(c, (x, w, b))]

    alone = [step(*job) for job in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(3):
        got = []
        for stream, job in zip(streams, work):
            with torch.cuda.stream(stream):
                got.append(step(*job))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            for p, q in zip(a, b):
                assert torch.equal(p, q)


@pytest.mark.parametrize("rows", [80, 514])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e20])
def test_many_rows_of_any_size_keep_their_bits(gpu, rows, dtype, scale):
    """hidden * scale against weight / scale with many rows, whose operands are laid out by powers of two; the scale is one itself, so nothing is
    rounded on the way."""
    vocab, width = 17000 if rows == 514 else 700, 72
    (x, w, _), gen = _inputs(gpu, rows, vocab, width, dtype, seed=rows)
    scale = 2.0 ** round(math.log2(scale))
    target = torch.randint(0, vocab, (rows,), generator=gen)
    x, w = (x.detach() * scale).requires_grad_(True), (w.detach() / scale).requires_grad_(True)
    loss = losses.linear_cross_entropy(x, w, target.to(gpu))
    Reference(x, w, target=target).check(loss, _grads(loss, (x, w)), dtype)


@pytest.mark.parametrize("rows", [80, 514])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("name", ["first", "padding", 1 << 40, -7])
def test_names_outside_the_vocabulary_with_many_rows(gpu, rows, dtype, name):
    """A label or an entry past the vocabulary, inside the last tile's padding too: its row is NaN, the others' losses and gradients of hidden states are
    what they are without it."""
    vocab, width, bad = 17000 if rows == 514 else 700, 64, 5
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
    name = {"first": vocab, "padding": vocab + 60}.get(name, name)
    keep = torch.arange(rows) != bad
    on = keep.to(gpu)
    target = torch.randint(0, vocab, (rows,), generator=gen)
    target[bad] = name
    index, teacher = _entries(gen, rows, vocab, 4, dtype)
    index[bad, 2] = name
    calls = [(lambda: losses.linear_cross_entropy(x, w, target.to(gpu), b, reduction="none"), dict(target=target[keep]))]
    if name >= 0:       # a negative one is no entry
        calls.append((lambda: losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b, reduction="none"),
                      dict(index=index[keep], teacher=teacher[keep])))
    for call, held in calls:
        loss = call()
        grads = _grads(loss, (x, w, b), torch.ones(rows, device=gpu))
        assert bool(loss[bad].isnan()) and bool(grads[0][bad].isnan().all())
        Reference(x[on], w, b, reduction="none", **held).check(loss[on], [grads[0][on]], dtype)
