"""Losses over a large vocabulary (jabas_amd.loss) against the definition in 64 bits on the CPU.

Bounds, derived from the arithmetic. Z is the largest sum_h |x||w| + |b| (or |z|) of the case, over T. A logit's error is at most
2^-20 Z (fp32 sums of exact products, or of products of 22-bit factors), the exponential's and the sums' a few 2^-22 more; a
probability's relative error is the same. A row gradient dz = q - p is then off by 2^-20 (Z + 4) (q + p), and bf16 calls
round it to fp16 (2^-11). The gradients of hidden states and weight sum dz against the other factor, so they are off by that
times sum (q + p) |other factor|, plus the rounding of the result (bf16: half a unit, 2^-9; taken twice for a result that
falls on the other side).
"""
import math

import pytest
import torch

from jabas_amd import loss as losses

pytestmark = pytest.mark.gpu
F64 = torch.float64
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100


def _gen(seed):
    return torch.Generator().manual_seed(seed)


class Reference:
    """Loss and gradients in 64 bits on the CPU. ``p``, ``index`` (rows x k) and ``rest``: what a row is held against."""

    def __init__(self, hidden=None, weight=None, bias=None, logits=None, target=None, smoothing=0.0, index=None, teacher=None, lse=None,
                 T=1.0, reduction="mean", upstream=None, ignore=IGNORE):
        c = lambda t: None if t is None else t.detach().cpu().to(F64)
        x, w, b = c(hidden), c(weight), c(bias)
        z = c(logits) if x is None else x @ w.t() + (0.0 if b is None else b)
        n, vocab = z.shape
        self.losses = torch.zeros(n, dtype=F64)
        dz = torch.zeros(n, vocab, dtype=F64)
        size = torch.zeros(n, vocab, dtype=F64)          # q + p
        counted = torch.zeros(n, dtype=torch.bool)
        Z = 0.0
        for r in range(n):
            if target is not None:
                t = int(target[r])
                if t == ignore:
                    continue
                logq = torch.log_softmax(z[r], 0)
                p = torch.full((vocab,), smoothing / vocab, dtype=F64)
                p[t] += 1.0 - smoothing
                self.losses[r] = -(torch.where(p > 0, p * logq, torch.zeros_like(p))).sum()
                dz[r], size[r] = logq.exp() - p, logq.exp() + p
            else:
                s = z[r] / T
                logq = torch.log_softmax(s, 0)
                keep = [j for j in range(index.shape[1]) if int(index[r, j]) >= 0 and float(teacher[r, j]) != -math.inf]
                if not keep:
                    continue
                t = teacher[r, keep].detach().cpu().to(F64) / T
                logp = t - float(lse[r]) if lse is not None else torch.log_softmax(t, 0)
                p = torch.zeros(vocab, dtype=F64)
                p.index_add_(0, index[r, keep].cpu(), logp.exp())
                named = torch.zeros(vocab, dtype=torch.bool)
                named[index[r, keep].cpu()] = True
                mass, rest = float(p.sum()), 0.0
                row = torch.where(p > 0, p * (p.log() - logq), torch.zeros_like(p)).sum()
                grad = logq.exp() * mass - p
                if lse is not None and not bool(named.all()):
                    rest = max(0.0, 1.0 - mass)
                    others = logq[~named].logsumexp(0)
                    if rest > 0:
                        row = row + rest * (math.log(rest) - others)
                    grad = grad + rest * logq.exp()
                    grad[~named] -= rest * (logq[~named] - others).exp()
                self.losses[r] = T * T * row
                dz[r] = T * grad
                size[r] = T * (logq.exp() * (mass + rest) + p)
                if rest:
                    size[r][~named] += T * rest * (logq[~named] - others).exp()
            counted[r] = True
            if x is None:
                Z = max(Z, z[r][torch.isfinite(z[r])].abs().max().item() / T)
        if x is not None and bool(counted.any()):
            Z = ((x[counted].abs() @ w.abs().t()).max().item() + (0.0 if b is None else b[torch.isfinite(b)].abs().max().item())) / T
        self.Z, self.counted, self.T = Z, counted, T
        share = 1.0 / max(1, int(counted.sum())) if reduction == "mean" else 1.0
        g = (torch.ones(n, dtype=F64) if upstream is None else upstream.detach().cpu().to(F64).expand(n)) * share
        g = torch.where(counted, g, torch.zeros_like(g))
        dz, size = dz * g[:, None], size * g[:, None].abs()
        self.loss = self.losses if reduction == "none" else self.losses.sum() * share
        self.loss_size = (self.losses.abs() if reduction == "none" else self.losses.abs().sum() * share)
        if x is None:
            self.grads, self.sizes = [dz], [size]
        else:
            live = torch.where(counted[:, None], x, torch.zeros_like(x))
            wl = w if b is None else torch.where((b == -math.inf)[:, None], torch.zeros_like(w), w)
            self.grads, self.sizes = [dz @ wl, dz.t() @ live], [size @ wl.abs(), size.t() @ live.abs()]
            if b is not None:
                self.grads.append(dz.sum(0))
                self.sizes.append(size.sum(0))

    def check(self, loss, grads, dtype):
        unit = 2.0 ** -20 * (self.Z + 4.0)
        got = loss.detach().cpu().to(F64)
        if self.loss.dim():
            bound = self.T ** 2 * unit * 2 + 2.0 ** -20 * self.loss_size
        else:
            bound = self.T ** 2 * unit * 2 * (1 if self.loss_size.numel() else 0) * max(1.0, float(self.counted.sum())) + 2.0 ** -20 * self.loss_size
        assert bool(((got - self.loss).abs() <= bound).all()), f"loss off by {(got - self.loss).abs().max():.3g}"
        dz = unit + (2.0 ** -10 if dtype == "bf16" else 2.0 ** -20)
        last = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -22
        for i, (g, ref, size) in enumerate(zip(grads, self.grads, self.sizes)):
            off = (g.detach().cpu().to(F64) - ref).abs()
            over = off - (dz * size + last * ref.abs() + 1e-37)
            assert bool((over <= 0).all()), f"gradient {i}: {int((over > 0).sum())} of {off.numel()} out of bounds, worst {off.max():.3g}"


def _inputs(gpu, rows, vocab, width, dtype, bias=False, seed=0, std=1.5):
    gen = _gen(seed)
    hidden = torch.randn(rows, width, generator=gen).to(TYPES[dtype])
    weight = (torch.randn(vocab, width, generator=gen) * (std / math.sqrt(width))).to(TYPES[dtype])
    b = torch.randn(vocab, generator=gen).to(TYPES[dtype]) if bias else None
    out = [t if t is None else t.to(gpu).requires_grad_(True) for t in (hidden, weight, b)]
    return out, gen


def _entries(gen, rows, vocab, k, dtype):
    index = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(rows)])
    return index, (torch.randn(rows, k, generator=gen) * 2).to(TYPES[dtype])


def _grads(loss, wrt, upstream=None):
    wrt = [t for t in wrt if t is not None]
    return torch.autograd.grad(loss, wrt, grad_outputs=None if upstream is None else upstream)


SIZES = [(1, 1, 1), (1, 5, 3), (2, 1000, 64), (3, 129, 64), (64, 128, 64), (65, 257, 100), (17, 1000, 768), (130, 1003, 192), (257, 300, 65),
         (300, 2049, 128)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,width", SIZES)
@pytest.mark.parametrize("bias,smoothing,reduction", [(False, 0.0, "mean"), (True, 0.1, "sum"), (True, 0.0, "none")])
def test_linear_cross_entropy(gpu, rows, vocab, width, dtype, bias, smoothing, reduction):
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, bias, seed=rows + vocab)
    target = torch.randint(0, vocab, (rows,), generator=gen)
    target[rows // 2::5] = IGNORE
    target[0] = vocab - 1
    loss = losses.linear_cross_entropy(x, w, target.to(gpu), b, label_smoothing=smoothing, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == (() if reduction != "none" else (rows,))
    up = torch.randn(rows, generator=gen) if reduction == "none" else None
    grads = _grads(loss, (x, w, b), None if up is None else up.to(gpu))
    for g, t in zip(grads, [t for t in (x, w, b) if t is not None]):
        assert g.dtype == t.dtype and g.shape == t.shape
    Reference(x, w, b, target=target, smoothing=smoothing, reduction=reduction, upstream=up).check(loss, grads, dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,width,k", [(1, 3, 8, 1), (1, 300, 64, 255), (5, 1000, 64, 10), (65, 257, 100, 32), (130, 1003, 192, 64),
                                                (200, 128, 65, 128), (257, 515, 64, 7)])
@pytest.mark.parametrize("tail,T,reduction", [(False, 1.0, "mean"), (True, 2.0, "mean"), (True, 1.0, "none"), (False, 0.5, "sum")])
def test_linear_topk_distillation(gpu, rows, vocab, width, k, dtype, tail, T, reduction):
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, bias=k % 2 == 0, seed=rows + k)
    index, teacher = _entries(gen, rows, vocab, k, dtype)
    index[rows // 2::7] = -1
    index[0, 0] = vocab - 1 if not bool((index[0, 1:] == vocab - 1).any()) else index[0, 0]
    lse = torch.logsumexp(teacher.float() / T, 1) + torch.rand(rows, generator=gen) if tail else None
    loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b, temperature=T,
                                           teacher_lse=None if lse is None else lse.to(gpu), reduction=reduction)
    up = torch.randn(rows, generator=gen) if reduction == "none" else None
    grads = _grads(loss, (x, w, b), None if up is None else up.to(gpu))
    Reference(x, w, b, index=index, teacher=teacher, lse=lse, T=T, reduction=reduction, upstream=up).check(loss, grads, dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 7, 3), (3, 255, 255), (48, 1000, 10), (5, 8193, 100), (2, 70001, 64), (1, 131072, 128), (130, 515, 32)])
@pytest.mark.parametrize("tail,T,reduction", [(False, 1.0, "mean"), (True, 2.0, "sum"), (True, 1.0, "none")])
def test_topk_distillation(gpu, rows, vocab, k, dtype, tail, T, reduction):
    gen = _gen(rows + vocab + k)
    z = (torch.randn(rows, vocab, generator=gen) * 2).to(TYPES[dtype]).to(gpu).requires_grad_(True)
    index, teacher = _entries(gen, rows, vocab, k, dtype)
    if rows > 2:
        index[1] = -1
    lse = torch.logsumexp(teacher.float() / T, 1) + torch.rand(rows, generator=gen) if tail else None
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), temperature=T, teacher_lse=None if lse is None else lse.to(gpu), reduction=reduction)
    up = torch.randn(rows, generator=gen) if reduction == "none" else None
    grads = _grads(loss, (z,), None if up is None else up.to(gpu))
    Reference(logits=z, index=index, teacher=teacher, lse=lse, T=T, reduction=reduction, upstream=up).check(loss, grads, dtype)


# ------------------------------------------------------------------ layouts
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("form", ["rows_apart", "offset", "transposed", "one_row_for_all", "leading_sizes"])
def test_linear_inputs_of_any_layout(gpu, dtype, form):
    rows, vocab, width = 70, 333, 128
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=5)
    target = torch.randint(0, vocab, (rows,), generator=gen).to(gpu)
    x, w, b = (t.detach() for t in (x, w, b))
    if form == "rows_apart":
        big, bigw = torch.zeros(rows, width + 9, dtype=x.dtype, device=gpu), torch.zeros(vocab, 2 * width, dtype=x.dtype, device=gpu)
        big[:, 1:1 + width], bigw[:, width:] = x, w
        x, w = big[:, 1:1 + width], bigw[:, width:]
    elif form == "offset":
        flat, flatw = torch.zeros(rows * width + 3, dtype=x.dtype, device=gpu), torch.zeros(vocab * width + 1, dtype=x.dtype, device=gpu)
        flat[3:], flatw[1:] = x.reshape(-1), w.reshape(-1)
        x, w = flat[3:].view(rows, width), flatw[1:].view(vocab, width)
        flatb = torch.zeros(vocab + 1, dtype=b.dtype, device=gpu)
        flatb[1:] = b
        b = flatb[1:]
    elif form == "transposed":
        x, w = x.t().contiguous().t(), w.t().contiguous().t()
    elif form == "one_row_for_all":
        x = x[:1].expand(rows, width)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    if form == "leading_sizes":
        loss = losses.linear_cross_entropy(leaves[0].view(2, 5, 7, width), w, target.view(2, 5, 7), b, reduction="none")
        assert loss.shape == (2, 5, 7)
        loss = loss.reshape(-1)
    else:
        loss = losses.linear_cross_entropy(x, w, target, b, reduction="none")
    up = torch.rand(rows, generator=gen)
    grads = _grads(loss, leaves, up.to(gpu))
    Reference(x, w, b, target=target.cpu(), reduction="none", upstream=up).check(loss, grads, dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("form", ["rows_apart", "offset", "transposed", "one_row_for_all"])
def test_logits_of_any_layout(gpu, dtype, form):
    rows, vocab, k = 9, 2051, 20
    gen = _gen(8)
    z = torch.randn(rows, vocab, generator=gen).to(TYPES[dtype]).to(gpu)
    index, teacher = _entries(gen, rows, vocab, k, dtype)
    if form == "rows_apart":
        big = torch.full((rows, vocab + 30), float("nan"), dtype=z.dtype, device=gpu)
        big[:, 7:7 + vocab] = z
        z = big[:, 7:7 + vocab]
    elif form == "offset":
        flat = torch.full((rows * vocab + 5,), float("nan"), dtype=z.dtype, device=gpu)
        flat[5:] = z.reshape(-1)
        z = flat[5:].view(rows, vocab)
    elif form == "transposed":
        z = z.t().contiguous().t()
    else:
        z = z[:1].expand(rows, vocab)
    z = z.requires_grad_(True)
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu))
    Reference(logits=z, index=index, teacher=teacher).check(loss, _grads(loss, (z,)), dtype)


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_only_the_gradients_asked_for(gpu, need, dtype):
    (x, w, b), gen = _inputs(gpu, 100, 400, 64, dtype, True, seed=2)
    target = torch.randint(0, 400, (100,), generator=gen)
    leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, w, b), need)]
    loss = losses.linear_cross_entropy(leaves[0], leaves[1], target.to(gpu), leaves[2])
    loss.backward()
    ref = Reference(x, w, b, target=target)
    for i, (leaf, n) in enumerate(zip(leaves, need)):
        assert (leaf.grad is not None) == bool(n)
        if n:
            ref_one = Reference(x, w, b, target=target)
            ref_one.grads, ref_one.sizes = [ref.grads[i]], [ref.sizes[i]]
            ref_one.check(loss, [leaf.grad], dtype)


def test_several_pieces_of_the_vocabulary(gpu):
    """Enough rows that the backward pass takes the vocabulary in pieces, the last of them short and odd; the pieces' weights differ in size,
    so do the factors they are scaled by."""
    for dtype, rows, vocab, width, k in (("bf16", 2500, 50001, 70, 0), ("fp32", 1300, 40007, 64, 9)):
        (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=1)
        with torch.no_grad():
            w.mul_(torch.linspace(0.1, 1.6, vocab, device=gpu)[:, None])
        if k:
            steps = torch.randint(1, vocab // k, (rows, k), generator=gen)
            index, teacher = steps.cumsum(1) - 1, (torch.randn(rows, k, generator=gen) * 2).to(TYPES[dtype])
            loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b)
            ref = Reference(x, w, b, index=index, teacher=teacher)
        else:
            target = torch.randint(0, vocab, (rows,), generator=gen)
            loss = losses.linear_cross_entropy(x, w, target.to(gpu), b)
            ref = Reference(x, w, b, target=target)
        ref.check(loss, _grads(loss, (x, w, b)), dtype)


@pytest.mark.parametrize("dtype,rows,vocab,width", [("bf16", 64, 1000, 100), ("bf16", 40, 3300, 1000), ("bf16", 48, 13000, 1000), ("bf16", 64, 3300, 1000), ("fp32", 64, 3300, 1000),
                                                    ("fp32", 65, 3300, 128), ("bf16", 20, 140001, 64), ("fp32", 40, 140001, 64)])
def test_few_rows(gpu, dtype, rows, vocab, width):
    """Either side of the sizes up to which few rows have kernels of their own, and more tokens than those keep row gradients of."""
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
    target = torch.randint(0, vocab, (rows,), generator=gen)
    target[1::6] = IGNORE
    loss = losses.linear_cross_entropy(x, w, target.to(gpu), b, label_smoothing=0.1)
    Reference(x, w, b, target=target, smoothing=0.1).check(loss, _grads(loss, (x, w, b)), dtype)
    index = torch.randint(0, vocab // 30, (rows, 30), generator=gen) + torch.arange(30) * (vocab // 30)
    teacher = torch.randn(rows, 30, generator=gen).to(TYPES[dtype])
    lse = torch.logsumexp(teacher.float(), 1) + 0.5
    loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b, teacher_lse=lse.to(gpu))
    Reference(x, w, b, index=index, teacher=teacher, lse=lse).check(loss, _grads(loss, (x, w, b)), dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("form", ["labels", "entries"])
@pytest.mark.parametrize("rows,vocab,width", [(300, 22001, 128), (300, 22001, 1900), (514, 17000, 72)])
def test_large_tiles(gpu, dtype, form, rows, vocab, width):
    """Enough tiles for the large ones, of the logits and (1900 features) of the gradients, whose last row, token and feature tiles are odd."""
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, form == "labels", seed=width)
    if form == "labels":
        target = torch.randint(0, vocab, (rows,), generator=gen)
        target[torch.randperm(rows, generator=gen)[:rows // 9]] = IGNORE
        loss = losses.linear_cross_entropy(x, w, target.to(gpu), b, label_smoothing=0.1, reduction="sum")
        ref = Reference(x, w, b, target=target, smoothing=0.1, reduction="sum")
    else:
        index = torch.randint(0, vocab // 64, (rows, 64), generator=gen) + torch.arange(64) * (vocab // 64)
        index[torch.randperm(rows, generator=gen)[:rows // 9]] = -1
        teacher = (torch.randn(rows, 64, generator=gen) * 2).to(TYPES[dtype])
        lse = torch.logsumexp(teacher.float() / 2, 1) + torch.rand(rows, generator=gen)
        loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), temperature=2.0, teacher_lse=lse.to(gpu))
        ref = Reference(x, w, index=index, teacher=teacher, lse=lse, T=2.0)
    ref.check(loss, _grads(loss, (x, w) if b is None else (x, w, b)), dtype)


def test_forward_pieces_of_the_vocabulary(gpu):
    """A wide weight in 32 bits, whose planes are kept for a part of the vocabulary at a time in the forward pass too."""
    rows, vocab, width = 66, 50001, 4096
    (x, w, _), gen = _inputs(gpu, rows, vocab, width, "fp32", seed=3)
    target = torch.randint(0, vocab, (rows,), generator=gen)
    target[:2] = torch.tensor([vocab - 1, 0])
    loss = losses.linear_cross_entropy(x, w, target.to(gpu))
    Reference(x, w, target=target).check(loss, _grads(loss, (x, w)), "fp32")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [70, 300])
@pytest.mark.parametrize("counted", [0, 1])
def test_hardly_a_row_counts(gpu, dtype, rows, counted):
    vocab, width = 22001, 70
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
    target = torch.full((rows,), IGNORE)
    target[rows - 3:rows - 3 + counted] = 4242
    loss = losses.linear_cross_entropy(x, w, target.to(gpu), b)
    grads = _grads(loss, (x, w, b))
    if counted:
        Reference(x, w, b, target=target).check(loss, grads, dtype)
    else:
        assert float(loss.detach()) == 0.0 and not any(bool(g.any()) for g in grads)
    index = torch.full((rows, 3), -1)
    index[5:5 + counted] = torch.tensor([7, 22000, 9])
    teacher = torch.randn(rows, 3, generator=gen).to(TYPES[dtype])
    loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b)
    grads = _grads(loss, (x, w, b))
    if counted:
        Reference(x, w, b, index=index, teacher=teacher).check(loss, grads, dtype)
    else:
        assert float(loss.detach()) == 0.0 and not any(bool(g.any()) for g in grads)


@pytest.mark.parametrize("dtype,rows,vocab", [("fp32", 520, 131071), ("bf16", 1100, 131071), ("bf16", 192, 262147), ("fp32", 191, 49153), ("fp32", 20, 524289),
                                              ("bf16", 700, 9001)])
def test_many_and_long_rows_of_logits(gpu, dtype, rows, vocab):
    """Rows whole and in parts, through the caches and past them; some of the rows are checked, each by itself."""
    gen = _gen(rows)
    z = torch.empty(rows, vocab, dtype=TYPES[dtype], device=gpu).normal_(std=2.0, generator=torch.Generator(device=gpu).manual_seed(rows))
    index = torch.randint(0, vocab // 16, (rows, 16), generator=gen) + torch.arange(16) * (vocab // 16)
    index[:, 15] = vocab - 1
    teacher = (torch.randn(rows, 16, generator=gen) * 2).to(TYPES[dtype])
    lse = torch.logsumexp(teacher.float(), 1) + 0.5
    up = torch.randn(rows, generator=gen)
    z.requires_grad_(True)
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), teacher_lse=lse.to(gpu), reduction="none")
    grad = _grads(loss, (z,), up.to(gpu))[0]
    some = [0, 1, rows // 2, rows - 2, rows - 1]
    Reference(logits=z[some], index=index[some], teacher=teacher[some], lse=lse[some], reduction="none", upstream=up[some]).check(loss[some], [grad[some]], dtype)
    # a row's gradient sums to nothing: of the sizes' sum, bf16's results are off by 2^-9 each, fp32's by 2^-20 times a few
    mass = grad.float().sum(1).cpu()
    size = grad.float().abs().sum(1).cpu()
    assert bool((mass.abs() <= size * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -17)).all())


def test_criteria_are_the_functions(gpu):
    (x, w, b), gen = _inputs(gpu, 20, 300, 64, "fp32", True)
    target = torch.randint(0, 300, (4, 5), generator=gen).to(gpu)
    target[0, 2] = 0
    hidden = x.view(4, 5, 64)
    a = losses.LinearCrossEntropy(ignore_index=0, label_smoothing=0.1)((hidden, w, b), target)
    assert torch.equal(a, losses.linear_cross_entropy(hidden, w, target, b, ignore_index=0, label_smoothing=0.1))
    index, teacher = (t.view(4, 5, 6).to(gpu) for t in _entries(gen, 20, 300, 6, "fp32"))
    lse = torch.logsumexp(teacher, 2) + 0.1
    d = losses.LinearTopkDistillation(temperature=2.0, reduction="sum")
    assert torch.equal(d((hidden, w, None), (index, teacher)), losses.linear_topk_distillation(hidden, w, index, teacher, temperature=2.0, reduction="sum"))
    assert torch.equal(d((hidden, w, b), (index, teacher, lse)), losses.linear_topk_distillation(hidden, w, index, teacher, b, temperature=2.0, teacher_lse=lse, reduction="sum"))


# ------------------------------------------------------------------ masks and values
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("garbage", [float("nan"), float("inf"), 1e38, -1e38])
def test_rows_that_do_not_count_may_hold_anything(gpu, dtype, garbage):
    rows, vocab, width = 140, 500, 64
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=4)
    target = torch.randint(0, vocab, (rows,), generator=gen)
    target[::3] = 7
    bad = x.detach().clone()
    bad[::3] = garbage
    bad.requires_grad_(True)
    clean = x.detach().clone()
    clean[::3] = 0
    loss = losses.linear_cross_entropy(bad, w, target.to(gpu), b, ignore_index=7, label_smoothing=0.1)
    grads = _grads(loss, (bad, w, b))
    assert not bool(grads[0][::3].any())
    keep = target != 7
    Reference(clean, w, b, target=torch.where(keep, target, torch.tensor(IGNORE)), smoothing=0.1).check(loss, grads, dtype)
    index, teacher = _entries(gen, rows, vocab, 12, dtype)
    index[::3] = -1
    teacher[::6] = -math.inf
    loss = losses.linear_topk_distillation(bad, w, index.to(gpu), teacher.to(gpu), b)
    grads = _grads(loss, (bad, w, b))
    assert not bool(grads[0][::3].any())
    Reference(clean, w, b, index=index, teacher=teacher).check(loss, grads, dtype)
    z = torch.randn(rows, vocab, generator=gen).to(TYPES[dtype]).to(gpu)
    ref = Reference(logits=z, index=index, teacher=teacher)
    z[::3] = garbage
    z.requires_grad_(True)
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu))
    ref.check(loss, _grads(loss, (z,)), dtype)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_no_row_counts(gpu, dtype, reduction):
    (x, w, b), gen = _inputs(gpu, 20, 300, 64, dtype, True)
    loss = losses.linear_cross_entropy(x, w, torch.full((20,), IGNORE, device=gpu), b, reduction=reduction)
    grads = _grads(loss.sum(), (x, w, b))
    assert not bool(loss.any()) and not any(bool(g.any()) for g in grads)
    index, teacher = torch.full((20, 4), -1, device=gpu), torch.zeros(20, 4, dtype=TYPES[dtype], device=gpu)
    loss = losses.linear_topk_distillation(x, w, index, teacher, b, reduction=reduction)
    grads = _grads(loss.sum(), (x, w, b))
    assert not bool(loss.any()) and not any(bool(g.any()) for g in grads)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_no_rows(gpu, reduction):
    w = torch.randn(30, 64, device=gpu, requires_grad=True)
    b = torch.randn(30, device=gpu, requires_grad=True)
    x = torch.empty(0, 64, device=gpu, requires_grad=True)
    loss = losses.linear_cross_entropy(x, w, torch.empty(0, dtype=torch.int64, device=gpu), b, reduction=reduction)
    gx, gw, gb = torch.autograd.grad(loss.sum(), (x, w, b))
    assert loss.shape == ((0,) if reduction == "none" else ()) and float(loss.sum()) == 0.0
    assert gx.shape == (0, 64) and not bool(gw.any()) and not bool(gb.any())
    z = torch.empty(0, 30, device=gpu, requires_grad=True)
    loss = losses.topk_distillation(z, torch.empty(0, 3, dtype=torch.int64, device=gpu), torch.empty(0, 3, device=gpu), reduction=reduction)
    assert torch.autograd.grad(loss.sum(), z)[0].shape == (0, 30)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
def test_tokens_ruled_out_by_the_bias(gpu, dtype, mask):
    """A third of the vocabulary and a whole tile of it masked; the weight's rows of tokens at -inf may be any finite garbage."""
    rows, vocab, width = 70, 700, 64
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=6)
    value = -math.inf if mask == "-inf" else torch.finfo(TYPES[dtype]).min
    with torch.no_grad():
        b[::3] = value
        b[128:256] = value
        if mask == "-inf":
            w[128:256] = 1e30
    allowed = torch.tensor([v for v in range(vocab) if float(b[v]) > -1e30])
    target = allowed[torch.randint(0, len(allowed), (rows,), generator=gen)]
    loss = losses.linear_cross_entropy(x, w, target.to(gpu), b)
    grads = _grads(loss, (x, w, b))
    wr = w.detach().clone()
    if mask == "-inf":
        wr[128:256] = 0
    ref = Reference(x, wr, b, target=target)
    ref.check(loss, grads, dtype)
    assert not bool(grads[1][128:256].any())
    # a label that is ruled out: infinite loss, finite gradients
    t = torch.full((rows,), 3, device=gpu)
    with torch.no_grad():
        b[3] = -math.inf
    loss = losses.linear_cross_entropy(x, w, t, b, reduction="none")
    assert bool((loss == math.inf).all())
    assert all(bool(g.isfinite().all()) for g in _grads(loss.sum(), (x, w, b)))


def test_rows_of_the_lowest_value(gpu):
    """Every logit of a row at the type's lowest value is a uniform row, not NaN."""
    low = torch.finfo(torch.float32).min
    z = torch.full((3, 5000), low, device=gpu)
    z[1] = -math.inf
    z[1, 17] = 2.0
    z[2] = torch.randn(5000, generator=_gen(0)).to(gpu)
    z.requires_grad_(True)
    index = torch.tensor([[5, 9], [17, -1], [0, 4999]], device=gpu)
    teacher = torch.tensor([[low, low], [1.0, 1.0], [0.5, 0.25]], device=gpu)
    loss = losses.topk_distillation(z, index, teacher, reduction="none")
    grad = _grads(loss.sum(), (z,))[0]
    assert float(loss[0].detach()) == pytest.approx(math.log(2500.0), rel=1e-6)
    assert float(loss[1].detach()) == pytest.approx(0.0, abs=1e-6) and not bool(grad[1].any())
    assert grad[0, 5].item() == pytest.approx(1 / 5000 - 0.5, rel=1e-6) and grad[0, 6].item() == pytest.approx(1 / 5000, rel=1e-5)
    assert bool(grad.isfinite().all())


@pytest.mark.parametrize("label", [-1, 300, 1 << 40, -(1 << 62)])
def test_labels_outside_the_vocabulary_give_nan(gpu, label):
    (x, w, b), gen = _inputs(gpu, 10, 300, 64, "bf16", True)
    target = torch.randint(0, 300, (10,), generator=gen).to(gpu)
    target[4] = label
    loss = losses.linear_cross_entropy(x, w, target, b, reduction="none")
    nan = loss.isnan()
    assert bool(nan[4]) and int(nan.sum()) == 1
    gx = _grads(loss.sum(), (x, w, b))[0]
    assert bool(gx[4].isnan().all()) and not bool(gx[torch.arange(10, device=gpu) != 4].isnan().any())
    index = torch.tensor([[1, 2], [3, label if label > 0 else 300]], device=gpu)
    z = torch.randn(2, 300, device=gpu, requires_grad=True)
    loss = losses.topk_distillation(z, index, torch.zeros(2, 2, device=gpu), reduction="none")
    assert loss.isnan().tolist() == [False, True]
    g = _grads(loss.sum(), (z,))[0]
    assert bool(g[1].isnan().all()) and not bool(g[0].isnan().any())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(6, 50000), (200, 3000)])
def test_rows_of_logits_without_entries_or_outside(gpu, dtype, rows, vocab):
    """Rows in parts and whole: none of a row's places an entry, and one outside the vocabulary, beside rows that are neither."""
    gen = _gen(31)
    z = torch.randn(rows, vocab, generator=gen).to(TYPES[dtype])
    index, teacher = _entries(gen, rows, vocab, 5, dtype)
    index[1], teacher[2], index[4, 3] = -1, -math.inf, vocab
    clean, keep = z.clone(), [r for r in range(rows) if r != 4]
    z[1], z[2] = float("nan"), float("inf")
    z = z.to(gpu).requires_grad_(True)
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), reduction="none")
    grad = _grads(loss.sum(), (z,))[0]
    assert bool(loss[4].isnan()) and bool(grad[4].isnan().all())
    assert not bool(grad[1:3].any()) and float(loss[1].detach()) == float(loss[2].detach()) == 0.0
    Reference(logits=clean[keep], index=index[keep], teacher=teacher[keep], reduction="none").check(loss[keep], [grad[keep]], dtype)


@pytest.mark.parametrize("tail", [False, True])
def test_tokens_named_twice_are_one_event(gpu, tail):
    gen = _gen(3)
    z = torch.randn(4, 600, generator=gen).to(gpu).requires_grad_(True)
    index = torch.randint(0, 600, (4, 70), generator=gen) % 40           # many names twice and more
    teacher = torch.randn(4, 70, generator=gen)
    lse = torch.logsumexp(teacher, 1) + 0.3 if tail else None
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), teacher_lse=None if lse is None else lse.to(gpu))
    Reference(logits=z, index=index, teacher=teacher, lse=lse).check(loss, _grads(loss, (z,)), "fp32")


@pytest.mark.parametrize("rows", [20, 80, 300])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("why", ["low_lse", "one_token_often"])
def test_probabilities_that_sum_to_more_than_one(gpu, dtype, rows, why):
    """A teacher_lse below its entries' own, or one token named in many places: the formula holds, with the sum far above 1 in some rows."""
    vocab, width, k = 22001, 64, 40
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, dtype, True, seed=rows)
    index = torch.randint(0, vocab // k, (rows, k), generator=gen) + torch.arange(k) * (vocab // k)
    teacher = (torch.randn(rows, k, generator=gen) * 2).to(TYPES[dtype])
    lse = torch.logsumexp(teacher.float(), 1) + 0.5
    if why == "low_lse":
        lse[::5] -= 6.0
    else:
        index[3::7] = 11
        teacher[3::7] = 4.0
        lse[3::7] = 4.2
    index[1] = -1
    loss = losses.linear_topk_distillation(x, w, index.to(gpu), teacher.to(gpu), b, teacher_lse=lse.to(gpu))
    Reference(x, w, b, index=index, teacher=teacher, lse=lse).check(loss, _grads(loss, (x, w, b)), dtype)
    z = (x.detach().float() @ w.detach().float().t()).to(TYPES[dtype]).requires_grad_(True)
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), teacher_lse=lse.to(gpu))
    Reference(logits=z, index=index, teacher=teacher, lse=lse).check(loss, _grads(loss, (z,)), dtype)


def test_entries_far_above_the_rest(gpu):
    """The student's rest is e^-200 of its row: the slope of the other tokens is still finite and right."""
    z = torch.zeros(1, 1000)
    z[0, :3] = 200.0
    z = z.to(gpu).requires_grad_(True)
    index, teacher, lse = torch.tensor([[0, 1, 2]]), torch.zeros(1, 3), torch.tensor([math.log(3 / 0.9)])
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), teacher_lse=lse.to(gpu))
    Reference(logits=z, index=index, teacher=teacher, lse=lse).check(loss, _grads(loss, (z,)), "fp32")


def test_every_token_is_an_entry(gpu):
    gen = _gen(9)
    z = torch.randn(3, 100, generator=gen).to(gpu).requires_grad_(True)
    index, teacher = _entries(gen, 3, 100, 100, "fp32")
    lse = torch.logsumexp(teacher, 1) + 1e-3                             # no token is left for what the teacher's rest would be
    loss = losses.topk_distillation(z, index.to(gpu), teacher.to(gpu), teacher_lse=lse.to(gpu))
    Reference(logits=z, index=index, teacher=teacher, lse=lse).check(loss, _grads(loss, (z,)), "fp32")


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e20])
def test_inputs_of_any_size_keep_their_bits(gpu, scale):
    """hidden * scale against weight / scale: the planes of a 32-bit call are scaled, so the result stands."""
    (x, w, _), gen = _inputs(gpu, 40, 300, 100, "fp32")
    target = torch.randint(0, 300, (40,), generator=gen)
    x, w = (x.detach() * scale).requires_grad_(True), (w.detach() / scale).requires_grad_(True)
    loss = losses.linear_cross_entropy(x, w, target.to(gpu))
    Reference(x, w, target=target).check(loss, _grads(loss, (x, w)), "fp32")


# ------------------------------------------------------------------ gradients against differences
@pytest.mark.parametrize("op", ["ce", "topk", "linear"])
def test_gradients_against_differences(gpu, op):
    """(L(t + e d) - L(t - e d)) / 2e along random directions d of length 1, e = 2^-5: the loss is good to 2^-20 (Z + |L|) on either side,
    Z < 32, so the quotient to 2^-20 * 64 / 2e = 0.001; the third derivative of a log-sum-exp along d is at most the third power of the
    largest change of a logit, max |w| or |x| in length (4 here), times e^2 / 6: 0.011."""
    gen = _gen(11)
    (x, w, b), _ = _inputs(gpu, 6, 90, 16, "fp32", True, seed=12)
    z = torch.randn(6, 90, generator=gen).to(gpu).requires_grad_(True)
    target = torch.randint(0, 90, (6,), generator=gen).to(gpu)
    index, teacher = (t.to(gpu) for t in _entries(gen, 6, 90, 5, "fp32"))
    lse = torch.logsumexp(teacher, 1) + 0.2
    call, leaves = {
        "ce": (lambda x, w, b: losses.linear_cross_entropy(x, w, target, b, label_smoothing=0.1), (x, w, b)),
        "topk": (lambda z: losses.topk_distillation(z, index, teacher, teacher_lse=lse), (z,)),
        "linear": (lambda x, w, b: losses.linear_topk_distillation(x, w, index, teacher, b, teacher_lse=lse), (x, w, b)),
    }[op]
    grads = _grads(call(*leaves), leaves)
    e = 2.0 ** -5
    for i, (leaf, g) in enumerate(zip(leaves, grads)):
        for _ in range(3):
            d = torch.randn(leaf.shape, generator=gen).to(gpu)
            d /= d.norm()
            with torch.no_grad():
                up, down = (float(call(*[t + s * e * d if j == i else t for j, t in enumerate(leaves)])) for s in (1, -1))
            assert abs((up - down) / (2 * e) - float((g * d).sum())) <= 0.012


# ------------------------------------------------------------------ streams, graphs, repeats
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_the_same_bits_every_time_and_on_any_stream(gpu, dtype):
    (x, w, b), gen = _inputs(gpu, 300, 3000, 128, dtype, True)
    target = torch.randint(0, 3000, (300,), generator=gen).to(gpu)
    index, teacher = (t.to(gpu) for t in _entries(gen, 300, 3000, 20, dtype))

    def both():
        a = losses.linear_cross_entropy(x, w, target, b, label_smoothing=0.1)
        c = losses.linear_topk_distillation(x, w, index, teacher, b, temperature=2.0)
        return [a.detach(), c.detach(), *_grads(a, (x, w, b)), *_grads(c, (x, w, b))]

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both()
    torch.cuda.current_stream().wait_stream(side)
    third = both()
    torch.cuda.synchronize()
    for p, q, r in zip(first, second, third):
        assert torch.equal(p, q) and torch.equal(p, r)


def test_replays_of_a_recorded_step(gpu):
    """Forward and backward recorded in a HIP graph; every replay on new inputs gives what the eager call gives."""
    rows, vocab, width = 64, 1500, 128
    (x, w, b), gen = _inputs(gpu, rows, vocab, width, "bf16", True)
    target = torch.randint(0, vocab, (rows,), generator=gen).to(gpu)

    def step():
        loss = losses.linear_cross_entropy(x, w, target, b)
        return [loss.detach(), *_grads(loss, (x, w, b))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(rows, width, generator=gen).to(gpu))
            target.copy_(torch.randint(0, vocab, (rows,), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(recorded, step()):
            assert torch.equal(p, q)
        torch.cuda.synchronize()


@pytest.mark.parametrize("which", ["tiles_fp32", "tiles_bf16", "entries_bf16", "parts_of_rows", "whole_rows"])
def test_replays_of_other_recorded_steps(gpu, which):
    """The same for the calls of many rows and for logits in hand; the number of rows that count changes from replay to replay."""
    gen = _gen(21)
    dtype = "fp32" if which.endswith("fp32") or which == "parts_of_rows" else "bf16"
    rows, vocab, width = {"parts_of_rows": (7, 60001, 0), "whole_rows": (90, 5001, 0)}.get(which, (300, 9000, 72))
    index, teacher = (t.to(gpu) for t in _entries(gen, rows, vocab, 9, dtype))
    target = torch.randint(0, vocab, (rows,), generator=gen).to(gpu)
    if width:
        leaves, _ = _inputs(gpu, rows, vocab, width, dtype, True, seed=4)
        x, w, b = leaves
        call = (lambda: losses.linear_topk_distillation(x, w, index, teacher, b, temperature=2.0)) if which.startswith("entries") else \
               (lambda: losses.linear_cross_entropy(x, w, target, b, label_smoothing=0.1))
    else:
        z = torch.randn(rows, vocab, generator=gen).to(TYPES[dtype]).to(gpu).requires_grad_(True)
        leaves = [z]
        call = lambda: losses.topk_distillation(z, index, teacher)

    def step():
        loss = call()
        return [loss.detach(), *_grads(loss, leaves)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(leaves[0].shape, generator=gen).to(gpu))
            target.copy_(torch.randint(0, vocab, (rows,), generator=gen))
            target[: i * rows // 4] = IGNORE
            index.copy_(_entries(gen, rows, vocab, 9, dtype)[0])
            index[: i * rows // 4] = -1
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(recorded, step()):
            assert torch.equal(p, q)
        torch.cuda.synchronize()


# ------------------------------------------------------------------ offsets past 32 bits
def test_logits_past_32_bits_of_offset(gpu):
    rows, vocab = 17000, 131072          # 2.2e9 elements
    z = torch.empty(rows, vocab, dtype=torch.bfloat16, device=gpu)
    z.normal_(generator=torch.Generator(device=gpu).manual_seed(0))
    gen = _gen(0)
    index = torch.randint(0, vocab // 8, (rows, 8), generator=gen).add_(torch.arange(8) * (vocab // 8)).to(gpu)
    teacher = torch.randn(rows, 8, generator=gen).bfloat16().to(gpu)
    z.requires_grad_(True)
    loss = losses.topk_distillation(z, index, teacher, reduction="none")
    grad = _grads(loss.sum(), (z,))[0]
    last = z.detach()[-3:].clone().requires_grad_(True)
    again = losses.topk_distillation(last, index[-3:], teacher[-3:], reduction="none")
    Reference(logits=last, index=index[-3:].cpu(), teacher=teacher[-3:].cpu(), reduction="none").check(loss[-3:], [grad[-3:]], "bf16")
    Reference(logits=last, index=index[-3:].cpu(), teacher=teacher[-3:].cpu(), reduction="none").check(again, _grads(again.sum(), (last,)), "bf16")


def test_weight_past_32_bits_of_offset(gpu):
    rows, vocab, width = 2, 540000, 4096          # 2.2e9 elements
    w = torch.empty(vocab, width, dtype=torch.bfloat16, device=gpu)
    w.normal_(std=0.02, generator=torch.Generator(device=gpu).manual_seed(0))
    x = torch.randn(rows, width, generator=_gen(1)).bfloat16().to(gpu).requires_grad_(True)
    target = torch.tensor([vocab - 1, 11])
    w.requires_grad_(True)
    loss = losses.linear_cross_entropy(x, w, target.to(gpu), reduction="none")
    gx, gw = _grads(loss.sum(), (x, w))
    xd, wd = x.detach().float(), w.detach()
    z = torch.cat([(xd @ wd[i:i + 60000].float().t()) for i in range(0, vocab, 60000)], 1).cpu().to(F64)
    logq = torch.log_softmax(z, 1)
    ref = -logq[torch.arange(rows), target]
    assert torch.allclose(loss.detach().cpu().to(F64), ref, rtol=1e-5, atol=1e-5)
    dz = logq.exp()
    dz[torch.arange(rows), target] -= 1.0
    tail = dz[:, -500:].t() @ x.detach().cpu().to(F64)
    assert torch.allclose(gw[-500:].cpu().to(F64), tail, rtol=2.0 ** -7, atol=2.0 ** -10 * float(tail.abs().max()))
    assert bool(gx.isfinite().all()) and bool(gx.any())


# ------------------------------------------------------------------ refusals
def test_refusals(gpu):
    x, w, t = torch.randn(4, 64, device=gpu), torch.randn(30, 64, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    ce, kd, lin = losses.linear_cross_entropy, losses.topk_distillation, losses.linear_topk_distillation
    i, tl = torch.zeros(4, 3, dtype=torch.int64, device=gpu), torch.zeros(4, 3, device=gpu)
    for error, call in [
            (TypeError, lambda: ce([1.0], w, t)), (TypeError, lambda: ce(x.half(), w.half(), t)), (TypeError, lambda: ce(x, w.bfloat16(), t)),
            (ValueError, lambda: ce(x[:, :32], w, t)), (ValueError, lambda: ce(x, w[0], t)), (ValueError, lambda: ce(x, w[:0], t)),
            (TypeError, lambda: ce(x, w, t.int())), (ValueError, lambda: ce(x, w, t[:3])), (ValueError, lambda: ce(x, w, t.cpu())),
            (ValueError, lambda: ce(x, w, t, torch.zeros(29, device=gpu))), (TypeError, lambda: ce(x, w, t, torch.zeros(30, device=gpu).bfloat16())),
            (ValueError, lambda: ce(x, w, t, label_smoothing=1.0)), (ValueError, lambda: ce(x, w, t, label_smoothing=float("nan"))),
            (ValueError, lambda: ce(x, w, t, reduction="batchmean")), (ValueError, lambda: ce(x.cpu(), w, t)), (ValueError, lambda: ce(x, w.cpu(), t)),
            (ValueError, lambda: kd(x, i[:, :0], tl[:, :0])), (ValueError, lambda: kd(x, i.expand(4, 3)[:, :1].expand(4, 256), tl[:, :1].expand(4, 256))),
            (ValueError, lambda: kd(x, i, tl, temperature=0.0)), (ValueError, lambda: kd(x, i, tl, temperature=float("inf"))),
            (TypeError, lambda: kd(x, i.int(), tl)), (TypeError, lambda: kd(x, i, tl.bfloat16())), (ValueError, lambda: kd(x, i, tl[:3])),
            (TypeError, lambda: kd(x, i, tl, teacher_lse=torch.zeros(4, device=gpu).double())), (ValueError, lambda: kd(x, i, tl, teacher_lse=torch.zeros(3, device=gpu))),
            (ValueError, lambda: kd(x, i[0], tl[0])), (ValueError, lambda: lin(x, w[:, :9], i, tl)), (TypeError, lambda: lin(x, w, i, tl.bfloat16()))]:
        with pytest.raises(error):
            call()
    loss = ce(x.requires_grad_(True), w, t)
    g = torch.autograd.grad(loss, x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()              # once differentiable
