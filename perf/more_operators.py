"""Performance cases of the orthogonalised update: Newton-Schulz products of a gradient matrix, and the optimizer steps made of them.

  ortho  ``optim.orthogonalize``: a matrix, or a batch of one shape, to the nearest matrix with singular values around one
  step   ``optim.ShardMuon.step``: momentum, orthogonalised update, decay and weights of a list of matrices, AdamW for what is no matrix
  sync   ``engine.VSWFlatSync.step`` with ``kind="muon"``: the gradients of K workers joined by their batch sizes, then the same step

``listed()`` holds the fixed cases, ``draw(rng)`` makes another one of the same ranges, ``prepare`` builds what the training program
holds before the call, ``run`` is one pass: in elementary torch operations in 32 bits, or with ``own`` through the framework's
operators; ``work`` the bytes and operations that one pass cannot do without and ``exact`` the same pass from the definition in 64 bits.
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
COEFFICIENTS, STEPS, EPS = (3.4445, -4.775, 2.0315), 5, 1e-7
MU, BETAS, ADAM_EPS, ADAM_STEP = 0.95, (0.9, 0.999), 1e-8, 7


def _case(op, **kw):
    """shapes: "rowsxcols*count" of the matrices, by commas (ortho: one, the count is the batch); vectors: lengths of parameters that
    are no matrices, as "length*count"; workers: gradients that are joined first; adjust: how the learning rate goes by the shape."""
    case = dict(op=op, shapes="64x64", vectors="", dtype="fp32", workers=1, nesterov=True, decay=0.0, lr=0.02, adjust="original")
    unknown = set(kw) - set(case) - {"name"}
    if unknown:
        raise KeyError(f"unknown case fields {sorted(unknown)}")
    case.update(kw)
    return case


def listed():
    return [
        # A 1 x 1 convolution of a residual network's first stage: a call whose launches weigh more than its products.
        _case("ortho", name="ortho_small", shapes="64x64*1", dtype="bf16"),
        # The attention outputs of a ViT-B/16, stacked.
        _case("ortho", name="ortho_attention_fp32", shapes="768x768*12"),
        # The classifier of ResNet-50, one matrix with a ragged edge.
        _case("ortho", name="ortho_classifier_bf16", shapes="1000x2048*1", dtype="bf16"),
        # Many small odd matrices, as heads or experts have them.
        _case("ortho", name="ortho_many_odd", shapes="129x257*64"),
        # The feed-forward weight of a wide layer: the products alone.
        _case("ortho", name="ortho_large_bf16", shapes="4096x16384*1", dtype="bf16"),
        # One recurrent gate matrix of the translation model in a bucket of its own.
        _case("step", name="step_one_matrix", shapes="4096x1024*1"),
        # The convolutions of one stage of ResNet-50 as matrices, of many shapes, and its norms' vectors.
        _case("step", name="step_convolutions", shapes="64x64*1,64x576*3,256x64*4,64x256*2,128x1152*4,512x128*4,128x512*3", vectors="256*4", decay=0.01),
        # The gate matrices of the translation model's encoder.
        _case("step", name="step_translation", shapes="4096x1024*8,4096x2048*2", vectors="4096*4", lr=1e-3, decay=0.1, adjust="match_rms_adamw"),
        # Four blocks of a ViT-L/16's square and wide matrices.
        _case("step", name="step_transformer", shapes="1024x1024*4,4096x1024*4,1024x4096*4", nesterov=False, decay=0.05),
        # Two workers' gradients of a small network's matrices.
        _case("sync", name="sync_small", shapes="384x384*4,1000x384*1", vectors="384*4", workers=2, lr=0.01),
        # Four workers of a ViT-B/16: attention outputs and their biases.
        _case("sync", name="sync_attention", shapes="768x768*12", vectors="768*12", workers=4, decay=0.05, lr=1e-3, adjust="match_rms_adamw"),
        # Eight workers with bfloat16 buckets, blocks of a ViT-L/16.
        _case("sync", name="sync_transformer_bf16", shapes="1024x1024*4,1024x4096*4", vectors="1024*8", dtype="bf16", workers=8, decay=0.05),
    ]


def _parse(text):
    return [tuple(int(n) for n in part.split("*")[0].split("x")) for part in text.split(",") if part for _ in range(int(part.split("*")[1]))]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _flops(rows, cols):
    """Of one matrix: X X^T and its square are symmetric, half of either is enough."""
    m, n = float(min(rows, cols)), float(max(rows, cols))
    return STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)


def draw(rng):
    op = rng.choice(("ortho", "ortho", "step", "step", "sync"))
    limit = _flops(4096, 16384) / 2

    def shape():
        rows, cols = _log_uniform(rng, 16, 4096), _log_uniform(rng, 16, 4096)
        if rng.random() < 0.6:              # most models' widths are multiples of 64; the others are taken as drawn
            rows, cols = max(64, rows // 64 * 64), max(64, cols // 64 * 64)
        return rows, cols

    parts, left, some = [], limit, 0
    for _ in range(1 if op == "ortho" else rng.randint(1, 4)):
        rows, cols = shape()
        count = min(_log_uniform(rng, 1, 64 if op == "ortho" else 6), max(1, int(left / _flops(rows, cols))), max(1, (1 << 26) // (rows * cols)))
        if _flops(rows, cols) * count > left:
            continue
        left -= _flops(rows, cols) * count
        some += count
        parts.append(f"{rows}x{cols}*{count}")
    adjust = rng.choice(("original", "match_rms_adamw"))
    vectors = f"{_log_uniform(rng, 16, 4096)}*{rng.randint(1, 4)}" if op != "ortho" and rng.random() < 0.5 else ""
    return _case(op, shapes=",".join(parts), vectors=vectors, dtype="fp32" if op == "step" else rng.choice(("fp32", "bf16")),
                 workers=rng.choice((2, 3, 4, 8)) if op == "sync" else 1, nesterov=rng.random() < 0.75, decay=rng.choice((0.0, 0.01, 0.1)),
                 lr=0.02 if adjust == "original" else 1e-3, adjust=adjust)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    shapes, dtype, K = _parse(case["shapes"]), TYPES[case["dtype"]], case["workers"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    def gradient(*shape):
        """Some directions far stronger than the rest, as a layer's gradient has them."""
        if len(shape) == 1:
            return randn(*shape).mul_(1e-3)
        *lead, rows, cols = shape
        rank = max(1, min(rows, cols) // 16)
        strong = randn(*lead, rows, rank).mul_(torch.logspace(0.0, -1.0, rank, device=DEVICE)) @ randn(*lead, rank, cols)
        return strong.mul_(4.0 / math.sqrt(rank)).add_(randn(*shape)).mul_(1e-3)

    state = dict(case)
    if case["op"] == "ortho":
        batch = () if len(shapes) == 1 else (len(shapes),)
        state["x"] = gradient(*batch, *shapes[0]).to(dtype)
        return state
    shapes = shapes + _parse(case["vectors"])
    state["params"] = [randn(*s).mul_(0.02) for s in shapes]
    state["grads"] = [[gradient(*s).to(dtype) for s in shapes] for _ in range(K)]
    state["momentum"] = [gradient(*s).mul_(0.3) if len(s) == 2 else None for s in shapes]
    state["first"] = [randn(*s).mul_(3e-4) if len(s) == 1 else None for s in shapes]
    state["second"] = [randn(*s).mul_(1e-3).square_() if len(s) == 1 else None for s in shapes]
    state["step"] = ADAM_STEP
    state["batches"] = [32 - 4 * (k % 3) for k in range(K)]
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from jabas_amd import optim
    if s["op"] == "ortho":
        return [optim.orthogonalize(s["x"])]
    if s["op"] == "step":
        return _step_own(s)
    return _sync_own(s)


def _groups(s):
    """The parameters of the two kinds, as an optimizer takes them."""
    lists = [[i for i, p in enumerate(s["params"]) if (p.dim() == 2) == matrices] for matrices in (True, False)]
    return [(matrices, places) for matrices, places in zip((True, False), lists) if places]


def _step_own(s):
    from jabas_amd import optim
    if "optimizer" not in s:        # made once, as a program does before its first step; the state is what a checkpoint brings
        for p, g in zip(s["params"], s["grads"][0]):
            p.grad = g
        groups = [dict(params=[s["params"][i] for i in places], use_muon=matrices) for matrices, places in _groups(s)]
        opt = s["optimizer"] = optim.ShardMuon(groups, lr=s["lr"], weight_decay=s["decay"], momentum=MU, nesterov=s["nesterov"],
                                               adjust_lr_fn=s["adjust"], betas=BETAS, adam_eps=ADAM_EPS)
        for p, buf, m, v in zip(s["params"], s["momentum"], s["first"], s["second"]):
            opt.state[p] = dict(momentum_buffer=buf) if buf is not None else dict(step=s["step"], exp_avg=m, exp_avg_sq=v)
    s["optimizer"].step()
    return _held(s["params"], s["momentum"], s["first"], s["second"])


def _sync_own(s):
    from jabas_amd.engine import VSWFlatSync
    from jabas_amd.workloads import ParamSpec
    if "engine" not in s:           # the arenas that a program's models and buckets are views of, filled once
        groups, group_of = [], {}
        for matrices, places in _groups(s):
            group_of.update({i: len(groups) for i in places})
            groups.append(dict(lr=s["lr"], weight_decay=s["decay"], use_muon=matrices))
        opt = dict(kind="muon", momentum=MU, nesterov=s["nesterov"], adjust_lr_fn=s["adjust"], betas=BETAS, eps=ADAM_EPS, groups=groups)
        specs = [ParamSpec(f"p{i}", p.numel(), group_of[i]) for i, p in enumerate(s["params"])]
        eng = s["engine"] = VSWFlatSync(specs, s["batches"], grad_dtype=TYPES[s["dtype"]], opt=opt, in_place=False,
                                        shapes=[tuple(p.shape) for p in s["params"]])
        eng.step_count = s["step"]
        for i, p in enumerate(s["params"]):
            eng.param_view(i).copy_(p.view(-1))
            for k in range(s["workers"]):
                eng.grad_view(k, i).copy_(s["grads"][k][i].view(-1))
            for j, state in enumerate((s["momentum"][i] if p.dim() == 2 else s["first"][i], s["second"][i])):
                if state is not None:
                    eng.state_view(j, i).copy_(state.view(-1))
        views = lambda of, dims: [of(i).view(p.shape) if p.dim() in dims else None for i, p in enumerate(s["params"])]
        s["views"] = (views(eng.param_view, (1, 2)), views(lambda i: eng.state_view(0, i), (2,)),
                      views(lambda i: eng.state_view(0, i), (1,)), views(lambda i: eng.state_view(1, i), (1,)))
    s["engine"].step()
    return _held(*s["views"])


def _held(params, momentum, first, second):
    """Weights, momenta of the matrices, both moments of the others."""
    return [list(params), *[[t for t in ts if t is not None] for ts in (momentum, first, second)]]


@torch.no_grad()
def _run_plain(s):
    """The formulas as they stand, in 32 bits; the length of a whole matrix in 64."""
    if s["op"] == "ortho":
        return [_orthogonal(s["x"].float()).to(s["x"].dtype)]
    s["step"] += 1
    total = float(sum(s["batches"]))
    for i, p in enumerate(s["params"]):
        g = s["grads"][0][i].float()
        if s["op"] == "sync":
            g = sum(s["grads"][k][i].float() * (s["batches"][k] / total) for k in range(s["workers"]))
        p.mul_(1.0 - s["lr"] * s["decay"])
        if p.dim() == 2:
            buf = s["momentum"][i]
            buf.mul_(MU).add_(g, alpha=1.0 - MU)
            u = g * (1.0 - MU) + buf * MU if s["nesterov"] else buf
            p.sub_(_orthogonal(u), alpha=_adjusted(s["lr"], p.shape, s["adjust"]))
        else:
            m, v = s["first"][i], s["second"][i]
            m.mul_(BETAS[0]).add_(g, alpha=1.0 - BETAS[0])
            v.mul_(BETAS[1]).add_(g * g, alpha=1.0 - BETAS[1])
            down = (v / (1.0 - BETAS[1] ** s["step"])).sqrt() + ADAM_EPS
            p.sub_(m / down, alpha=s["lr"] / (1.0 - BETAS[0] ** s["step"]))
    return _held(s["params"], s["momentum"], s["first"], s["second"])


def _adjusted(lr, shape, how):
    rows, cols = shape
    return lr * math.sqrt(max(1.0, rows / cols)) if how == "original" else lr * 0.2 * math.sqrt(max(rows, cols))


def _orthogonal(x):
    a, b, c = COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2).contiguous()
    length = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = x / length.clamp(min=EPS).float()
    for _ in range(STEPS):
        A = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.transpose(-1, -2).contiguous() if tall else x


def exact(case, seed):
    """Weights and state from the definition in 64 bits."""
    with torch.no_grad():
        s = prepare(case, seed)
        if case["op"] == "ortho":
            x = s["x"]
            return [_polynomial(x.double()) if x.dim() == 2 else torch.stack([_polynomial(one.double()) for one in x])]
        return _exact_step(s)


def _polynomial(g):
    """sum of odd powers, applied to the shorter side: X <- X + ((a - 1) I + b S + c S S) X with S = X X^T."""
    if g.shape[0] > g.shape[1]:
        return _polynomial(g.t()).t()
    a, b, c = COEFFICIENTS
    x = g / torch.linalg.vector_norm(g).clamp(min=EPS)
    for _ in range(STEPS):
        s = torch.mm(x, x.t())
        q = torch.addmm(b * s, s, s, alpha=c)
        q.diagonal().add_(a)
        x = torch.mm(q, x)
    return x


def _exact_step(s):
    share = torch.tensor(s["batches"], dtype=torch.float64) / sum(s["batches"])
    t = s["step"] + 1
    params, momentum, first, second = [], [], [], []
    for i, p in enumerate(s["params"]):
        g = s["grads"][0][i].double() if s["op"] == "step" else sum(float(w) * s["grads"][k][i].double() for k, w in enumerate(share))
        w = p.double() * (1.0 - s["lr"] * s["decay"])
        if p.dim() == 2:
            buf = s["momentum"][i].double()
            buf = buf + (1.0 - MU) * (g - buf)
            o = _polynomial(g + MU * (buf - g) if s["nesterov"] else buf)
            rows, cols = p.shape
            scale = max(1.0, rows / cols) ** 0.5 if s["adjust"] == "original" else 0.2 * max(rows, cols) ** 0.5
            params.append(w - s["lr"] * scale * o)
            momentum.append(buf)
        else:
            m = BETAS[0] * s["first"][i].double() + (1.0 - BETAS[0]) * g
            v = BETAS[1] * s["second"][i].double() + (1.0 - BETAS[1]) * g * g
            params.append(w - s["lr"] * (m / (1.0 - BETAS[0] ** t)) / ((v / (1.0 - BETAS[1] ** t)).sqrt() + ADAM_EPS))
            first.append(m)
            second.append(v)
    return [params, momentum, first, second]


def work(case):
    """Every input read once, every output written once; the products with symmetry's half left out."""
    shapes, vectors, size = _parse(case["shapes"]), _parse(case["vectors"]), 4 if case["dtype"] == "fp32" else 2
    flops = sum(_flops(*s) for s in shapes)
    elements, others = sum(r * c for r, c in shapes), sum(n for n, in vectors)
    if case["op"] == "ortho":
        return {"bytes": 2 * size * elements, "flops": flops}
    return {"bytes": (case["workers"] * size + 16) * elements + (case["workers"] * size + 24) * others, "flops": flops}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
