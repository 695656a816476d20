"""Performance cases of the losses at the end of a worker's forward pass: cross entropy and distillation over a large vocabulary.

  ce      ``loss.linear_cross_entropy``: hidden states and the classifier's weight in, the loss and their gradients out, no logits kept
  topk    ``loss.topk_distillation``: logits in hand against a teacher's top logits
  linear  ``loss.linear_topk_distillation``: the same from hidden states and the classifier's weight

``listed()`` holds the fixed cases, ``draw(rng)`` makes another one of the same ranges, ``prepare`` builds what the training program
holds before the call, ``run`` is one pass: in elementary torch operations in 32 bits, or with ``own`` through the framework's
operators; ``work`` the bytes and operations that one pass cannot do without and ``exact`` the same pass from the definition in 64 bits.
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
IGNORE = -100
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _case(op, **kw):
    """width: features of a hidden state (0: logits in hand); padding: share of rows that do not count; k: entries of the teacher;
    tail: the teacher's log-sum-exp is given, so what its entries leave is one event more; train: gradients too."""
    case = dict(op=op, rows=1, vocab=1000, width=0, dtype="bf16", bias=False, smoothing=0.0, padding=0.0, k=0,
                temperature=1.0, tail=False, reduction="mean", train=True)
    unknown = set(kw) - set(case) - {"name"}
    if unknown:
        raise KeyError(f"unknown case fields {sorted(unknown)}")
    case.update(kw)
    return case


def listed():
    return [
        # The smallest local batch of the ViT-B/16 configuration at its 1000-class head: a call whose launches weigh more than its bytes.
        _case("ce", name="ce_classes_16", rows=16, vocab=1000, width=768, bias=True),
        # One token scored against the translation vocabulary, as beam search and perplexity do: the weight is read once.
        _case("ce", name="ce_one_row_scored", rows=1, vocab=32317, width=1024, bias=True, reduction="none", train=False),
        # A translation worker in fp32, 64 sentences of about 25 tokens, label smoothing, a fifth of the rows padding.
        _case("ce", name="ce_translation_fp32", rows=1600, vocab=32317, width=1024, dtype="fp32", bias=True, smoothing=0.1, padding=0.2),
        # The same in bf16 with 128 sentences of 50 tokens.
        _case("ce", name="ce_translation_bf16", rows=6400, vocab=32317, width=1024, bias=True, smoothing=0.1, padding=0.2),
        # Evaluation of a held-out set: losses per token, no gradients, sizes that end inside every tile.
        _case("ce", name="ce_evaluation", rows=4099, vocab=50001, width=768, reduction="none", train=False),
        # A large vocabulary over wide states: the products alone.
        _case("ce", name="ce_large", rows=4096, vocab=131072, width=4096),
        # Classes distilled from a larger network's ten best, a batch of 48 images, logits in hand.
        _case("topk", name="topk_classes_48", rows=48, vocab=1000, dtype="fp32", k=10, temperature=4.0),
        # Few rows over a large vocabulary, losses only: rows must be shared between workgroups.
        _case("topk", name="topk_few_long_rows", rows=5, vocab=131072, dtype="fp32", k=100, tail=True, reduction="none", train=False),
        # Translation logits in hand; the odd vocabulary puts every row at another alignment.
        _case("topk", name="topk_translation", rows=3200, vocab=32317, k=32, temperature=2.0, padding=0.2),
        # A stored teacher's 64 best of a large vocabulary with its normaliser.
        _case("topk", name="topk_large", rows=4096, vocab=131072, k=64, tail=True),
        # A translation worker distilled without keeping its logits, fp32.
        _case("linear", name="linear_translation_fp32", rows=800, vocab=32317, width=1024, dtype="fp32", bias=True, k=32, temperature=2.0, padding=0.2),
        # The same operator at an ordinary language model's size in bf16, the rest of the vocabulary as one event.
        _case("linear", name="linear_large", rows=4096, vocab=50001, width=2048, k=64, tail=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ce", "ce", "topk", "linear"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    vocab = _log_uniform(rng, 1000, 131072)
    rows = _log_uniform(rng, 1, 8192)
    width = 0 if op == "topk" else _log_uniform(rng, 256, 4096)
    if width and rng.random() < 0.75:      # most models' widths are multiples of 64; the others are taken as drawn
        width = max(256, width // 64 * 64)
    limit = 4096 * 131072 if op == "topk" else 4096 * 131072 * 4096 // (4 if dtype == "fp32" else 1)
    rows = max(1, min(rows, limit // (vocab * max(1, width))))
    kd = op != "ce"
    return _case(op, rows=rows, vocab=vocab, width=width, dtype=dtype, bias=width > 0 and rng.random() < 0.5,
                 smoothing=0.0 if kd else rng.choice((0.0, 0.1)), padding=rng.choice((0.0, 0.0, 0.2)) if rows >= 8 else 0.0,
                 k=_log_uniform(rng, 4, 128) if kd else 0, temperature=rng.choice((1.0, 2.0, 4.0)) if kd else 1.0,
                 tail=kd and rng.random() < 0.4, reduction=rng.choice(("mean", "mean", "none")), train=rng.random() < 0.75)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, rows, vocab, k = TYPES[case["dtype"]], case["rows"], case["vocab"], case["k"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    state = dict(case)
    padded = torch.rand(rows, generator=gen, device=DEVICE) < case["padding"]
    padded[0] = False
    if k:   # distinct entries: steps of random length through the vocabulary, in an order of their own per row
        steps = torch.randint(1, max(2, vocab // k), (rows, k), generator=gen, device=DEVICE)
        index = (steps.cumsum(1) - 1).gather(1, torch.rand(rows, k, generator=gen, device=DEVICE).argsort(1))
        teacher = randn(rows, k).mul(2.0).sort(1, descending=True).values + 6.0
        favourite = index[:, 0]
        if case["tail"]:    # the entries hold most of the teacher's mass, not all of it
            share = 0.5 + 0.45 * torch.rand(rows, generator=gen, device=DEVICE)
            state["teacher_lse"] = torch.logsumexp(teacher.to(dtype).float() / case["temperature"], 1) - share.log()
        index = torch.where(padded[:, None], torch.full_like(index, -1), index)
        state["teacher_index"], state["teacher_logits"] = index, teacher.to(dtype)
    else:
        favourite = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE)
        state["target"] = torch.where(padded, torch.full_like(favourite, IGNORE), favourite)
    if case["width"]:
        weight = randn(vocab, case["width"]).mul_(2.0 / math.sqrt(case["width"])).to(dtype)
        # a model in the middle of training: the right answer's logit stands out, by more in some rows than in others
        lift = randn(rows, 1).add_(2.0)
        hidden = (randn(rows, case["width"]) + lift * weight[favourite].float()).to(dtype)
        state["hidden"], state["weight"] = hidden, weight
        state["bias"] = randn(vocab).mul_(0.5).to(dtype) if case["bias"] else None
        state["wrt"] = [t for t in (hidden, weight, state["bias"]) if t is not None]
    else:
        logits = randn(rows, vocab).mul_(2.0)
        logits.scatter_add_(1, favourite[:, None], randn(rows, 1).add_(2.0).mul_(4.0))
        state["logits"] = logits.to(dtype)
        state["wrt"] = [state["logits"]]
    if case["reduction"] == "none":       # a weight per row, as a program has that sums the losses itself
        state["upstream"] = torch.rand(rows, generator=gen, device=DEVICE) / rows
    else:
        state["upstream"] = torch.ones((), device=DEVICE)
    if case["train"]:
        for t in state["wrt"]:
            t.requires_grad_(True)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from jabas_amd import loss as losses
    if s["op"] == "ce":
        loss = losses.linear_cross_entropy(s["hidden"], s["weight"], s["target"], s["bias"], ignore_index=IGNORE,
                                           label_smoothing=s["smoothing"], reduction=s["reduction"])
    elif s["op"] == "topk":
        loss = losses.topk_distillation(s["logits"], s["teacher_index"], s["teacher_logits"], temperature=s["temperature"],
                                        teacher_lse=s.get("teacher_lse"), reduction=s["reduction"])
    else:
        loss = losses.linear_topk_distillation(s["hidden"], s["weight"], s["teacher_index"], s["teacher_logits"], s["bias"],
                                               temperature=s["temperature"], teacher_lse=s.get("teacher_lse"), reduction=s["reduction"])
    if not s["train"]:
        return [loss.detach()]
    return [loss.detach(), *torch.autograd.grad(loss, s["wrt"], grad_outputs=s["upstream"])]


@torch.no_grad()
def _run_plain(s):
    """The formulas as they stand, logits and all, in 32 bits."""
    if s["op"] == "topk":
        z = s["logits"].float()
    else:
        x, w = s["hidden"].float(), s["weight"].float()
        z = x @ w.t()
        if s["bias"] is not None:
            z += s["bias"].float()
    rows, dz = _entropy_plain(s, z) if s["op"] == "ce" else _distillation_plain(s, z)
    counted = (s["target"] != IGNORE) if s["op"] == "ce" else (s["teacher_index"] >= 0).any(1)
    scale = 1.0 / counted.sum().clamp(min=1).float() if s["reduction"] == "mean" else torch.ones((), device=z.device)
    rows = torch.where(counted, rows, torch.zeros_like(rows))
    loss = rows if s["reduction"] == "none" else rows.sum() * scale
    if not s["train"]:
        return [loss]
    dz *= torch.where(counted, s["upstream"] * scale, torch.zeros_like(rows))[:, None]
    if s["op"] == "topk":
        return [loss, dz.to(s["logits"].dtype)]
    grads = [(dz @ w).to(s["hidden"].dtype), (dz.t() @ x).to(s["weight"].dtype)]
    if s["bias"] is not None:
        grads.append(dz.sum(0).to(s["bias"].dtype))
    return [loss, *grads]


def _entropy_plain(s, z):
    e, vocab = s["smoothing"], z.shape[1]
    t = s["target"].clamp(min=0)[:, None]
    top = z.amax(1, keepdim=True)
    q = torch.exp(z - top)
    total = q.sum(1, keepdim=True)
    lse = top + torch.log(total)
    rows = (lse - (1.0 - e) * z.gather(1, t)).squeeze(1)
    if e:
        rows -= e * z.mean(1)
    if s["train"]:
        q /= total
        if e:
            q -= e / vocab
        q.scatter_add_(1, t, torch.full_like(lse, e - 1.0))
    return rows, q


def _distillation_plain(s, z):
    T = s["temperature"]
    z = z / T
    there = s["teacher_index"] >= 0
    index = s["teacher_index"].clamp(min=0)
    t = torch.where(there, s["teacher_logits"].float() / T, torch.full((), -math.inf, device=z.device))
    if s["tail"]:
        norm = s["teacher_lse"][:, None]
    else:
        peak = t.amax(1, keepdim=True).clamp(min=-3e38)
        norm = peak + torch.log(torch.exp(t - peak).sum(1, keepdim=True))
    p = torch.where(there, torch.exp(t - norm), torch.zeros_like(t))
    top = z.amax(1, keepdim=True)
    q = torch.exp(z - top)
    total = q.sum(1, keepdim=True)
    lse = top + torch.log(total)
    rows = torch.where(p > 0, p * ((t - norm) - (z.gather(1, index) - lse)), torch.zeros_like(p)).sum(1)
    q /= total
    mass, factor = p.sum(1, keepdim=True), 0.0
    if s["tail"]:
        rest = (1.0 - mass).clamp(min=0.0)
        held = q.gather(1, index)
        left = q.scatter(1, index, 0.0).sum(1, keepdim=True)
        rows += torch.where(rest > 0, rest * (torch.log(rest) - torch.log(left)), torch.zeros_like(rest)).squeeze(1)
        mass = mass + rest
        factor = rest / left
    if s["train"]:
        q *= (mass - factor)
        if s["tail"]:
            q.scatter_(1, index, held * mass)
        q.scatter_add_(1, index, -p)
        q *= T
    return rows * (T * T), q


def exact(case, seed):
    """Loss and gradients from the definition in 64 bits, some rows at a time: the classifier's product, the distribution that the row
    is held against, and the derivative of their divergence."""
    with torch.no_grad():
        return _exact(prepare(case, seed))


def _exact(s):
    f64 = torch.float64
    n, vocab, T = s["rows"], s["vocab"], s["temperature"]
    w = b = None
    if s["op"] != "topk":
        w = s["weight"].detach().to(f64)
        b = s["bias"].detach().to(f64) if s["bias"] is not None else None
    counted = (s["target"] != IGNORE) if s["op"] == "ce" else (s["teacher_index"] >= 0).any(1)
    share = s["upstream"].to(f64).expand(n).clone()
    if s["reduction"] == "mean":
        share /= max(1, int(counted.sum()))
    share[~counted] = 0.0
    losses = torch.zeros(n, dtype=f64, device=DEVICE)
    out = [torch.zeros(t.shape, dtype=f64, device=DEVICE) for t in s["wrt"]] if s["train"] else []
    step = max(1, (1 << 28) // vocab)
    for at in range(0, n, step):
        r = torch.arange(at, min(n, at + step), device=DEVICE)
        r = r[counted[r]]
        if not len(r):
            continue
        x = None if s["op"] == "topk" else s["hidden"].detach()[r].to(f64)
        z = s["logits"].detach()[r].to(f64) if x is None else x @ w.t() + (0.0 if b is None else b)
        logq = torch.log_softmax(z / T, 1)
        del z
        if s["op"] == "ce":
            e = s["smoothing"]
            hard = s["target"][r][:, None]
            losses[r] = -(1.0 - e) * logq.gather(1, hard).squeeze(1)
            if e:
                losses[r] -= e * logq.mean(1)
            if s["train"]:
                dz = logq.exp_().sub_(e / vocab)
                dz[torch.arange(len(r), device=DEVICE), hard.squeeze(1)] -= 1.0 - e
        else:
            index, t = s["teacher_index"][r], s["teacher_logits"].detach()[r].to(f64) / T
            logp = t - s["teacher_lse"][r].to(f64)[:, None] if s["tail"] else torch.log_softmax(t, 1)
            p, logh = logp.exp(), logq.gather(1, index)
            row = (p * (logp - logh)).sum(1)
            mass = p.sum(1, keepdim=True)
            slope = mass.clone()
            if s["tail"]:
                rest = (1.0 - mass).clamp(min=0.0)
                left = logq.scatter(1, index, -math.inf).logsumexp(1, keepdim=True)
                row += (rest * (rest.log() - left)).squeeze(1)
                mass = mass + rest
                slope = mass - rest / left.exp()
            losses[r] = row * T * T
            if s["train"]:
                dz = logq.exp_().mul_(slope)
                dz.scatter_(1, index, logh.exp() * mass - p)
                dz *= T
        if s["train"]:
            dz *= share[r][:, None]
            if x is None:
                out[0][r] = dz
            else:
                out[0][r] = dz @ w
                out[1].addmm_(dz.t(), x)
                if b is not None:
                    out[2] += dz.sum(0)
    loss = losses if s["reduction"] == "none" else losses.sum() / (max(1, int(counted.sum())) if s["reduction"] == "mean" else 1)
    return [loss, *out]


def work(case):
    """Every input read once and every output written once; products of the loss and, in training, of both gradients. What a program
    computes again because it keeps no logits is not counted."""
    n, v, h, k = case["rows"], case["vocab"], case["width"], case["k"]
    s = 4 if case["dtype"] == "fp32" else 2
    moved = s * (n * h + v * h + (v if case["bias"] else 0)) if h else s * n * v
    asked = n * k * (8 + s) + (4 * n if case["tail"] else 0) if k else 8 * n
    lost = 4 * n if case["reduction"] == "none" else 4
    ops = (2.0 * n * v * h if h else 0.0) + 4.0 * n * v
    if case["train"]:
        return {"bytes": 2 * moved + asked + lost, "flops": ops + (4.0 * n * v * h if h else 0.0) + 3.0 * n * v}
    return {"bytes": moved + asked + lost, "flops": ops}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
