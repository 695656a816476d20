"""Orthogonalised updates (optim.orthogonalize, optim.ShardMuon, the engine's and the trainer's step with kind "muon") against the definition in
64 bits on the CPU.

Bounds (oracle.muon.allowed): the documented precision is so many bits of every factor of a product; the definition is computed
in 64 bits with factors off by evenly random amounts of that size, and a result may be 8 times as far off as that carries, plus
the rounding of the result itself. The factor covers that the sums are fp32 too and that one random draw is no bound. Lengths of differences are
compared (2-norm): a rounding of X turns singular vectors, so single elements have no bound of their own.
"""
import copy

import pytest
import torch

from jabas_amd import optim
from oracle import muon as M

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _matrices(*shape, kind="even", seed=0):
    gen = _gen(seed)
    x = torch.randn(*shape, generator=gen)
    if kind == "steep":                 # few strong directions over a floor
        *lead, rows, cols = shape
        rank = max(1, min(rows, cols) // 8)
        x = torch.randn(*lead, rows, rank, generator=gen) @ (torch.logspace(0, -2, rank)[:, None] * torch.randn(*lead, rank, cols, generator=gen)) + 1e-2 * x
    return x


def _close(got, x, **kw):
    far, e = M.allowed(x, x.dtype == torch.bfloat16, **kw)
    off = M.off_by(got, e)
    assert off <= far, (off, far)


# ------------------------------------------------------------------------------------------------------- orthogonalize
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["even", "steep"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (7, 1), (5, 3), (64, 64), (63, 65), (65, 128), (64, 577), (129, 127), (200, 64), (256, 256), (257, 300),
                                   (40, 1000), (1000, 384), (513, 514)])
def test_matrices_of_any_size(gpu, dtype, kind, shape):
    x = _matrices(*shape, kind=kind).to(TYPES[dtype])
    _close(optim.orthogonalize(x.to(gpu)), x)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 100, 130), (2, 3, 70, 33), (40, 17, 19), (5, 1, 300, 100), (3, 640, 640)])
def test_batches(gpu, dtype, shape):
    x = _matrices(*shape).to(TYPES[dtype]) * torch.logspace(-3, 3, shape[0]).view(-1, *[1] * (len(shape) - 1)).to(TYPES[dtype])
    got = optim.orthogonalize(x.to(gpu)).cpu()
    assert got.shape == x.shape and got.is_contiguous()
    for one, o in zip(x.view(-1, *shape[-2:]), got.view(-1, *shape[-2:])):
        _close(o, one)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1100, 1030), (300, 2100), (2050, 70)])
def test_tiles_of_every_size_that_end_inside(gpu, dtype, rows, cols):
    """Large enough, or often enough, for the larger tiles; the sides end inside all of them."""
    x = _matrices(4, rows, cols, kind="steep").to(TYPES[dtype])
    got = optim.orthogonalize(x.to(gpu))
    _close(got[0], x[0])
    _close(got[3], x[3])
    many = x[:1].to(gpu).expand(24, rows, cols)
    for o in optim.orthogonalize(many)[::23]:
        _close(o, x[0])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(250, 4000), (3, 64, 9001), (2, 3001, 130), (448, 4100), (1, 20, 20000), (800, 2100), (2600, 1000)])
def test_long_matrices_whose_tiles_are_shared(gpu, dtype, shape):
    """Few tiles over a long axis: workgroups share them. The last to finish adds up, in a fixed order, and the tickets are good for the next call."""
    x = _matrices(*shape, kind="steep").to(TYPES[dtype])
    held = x.to(gpu)
    first = optim.orthogonalize(held)
    for one, o in zip(x.view(-1, *shape[-2:]), first.view(-1, *shape[-2:])):
        _close(o, one)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams * 4:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(optim.orthogonalize(held))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(4096, 4096), (2500, 5000), (6, 1030, 2050)])
def test_large_matrices(gpu, dtype, shape):
    x = _matrices(*shape, kind="steep").to(TYPES[dtype]).to(gpu)
    got = optim.orthogonalize(x)
    far, e = M.allowed(x, dtype == "bf16", device=gpu)
    for o, y in zip(got.view(-1, *shape[-2:]), e.view(-1, *shape[-2:])):
        assert M.off_by(o, y) <= far


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_very_many_small_matrices(gpu, dtype):
    x = _matrices(70001, 5, 3).to(TYPES[dtype])
    got = optim.orthogonalize(x.to(gpu))
    _close(got, x)
    for i in (0, 1, 65535, 65536, 70000):
        _close(got[i], x[i])


def test_calls_that_overlap(gpu):
    """Two streams at once, other shapes and inputs on either."""
    a, b = [_matrices(200, 300, seed=s).to(gpu) for s in range(6)], [_matrices(4, 64, 3000, seed=s).to(gpu) for s in range(6)]
    alone = [optim.orthogonalize(x) for x in a], [optim.orthogonalize(x) for x in b]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [], []
    for x, y in zip(a, b):
        for z, s, out in zip((x, y), streams, outs):
            with torch.cuda.stream(s):
                out.append(optim.orthogonalize(z))
    torch.cuda.synchronize()
    for one, two in zip(alone, outs):
        assert all(torch.equal(o, t) for o, t in zip(one, two))


def test_a_batch_that_goes_through_the_workspace_some_at_a_time(gpu):
    x = torch.randn(40, 512, 1024, generator=torch.Generator(gpu).manual_seed(0), device=gpu)
    got = optim.orthogonalize(x)
    for i in (0, 17, 39):
        assert torch.equal(got[i], optim.orthogonalize(x[i:i + 1])[0]) or M.off_by(got[i], M.newton_schulz(x[i])) < 1e-5
        _close(got[i], x[i].cpu())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_views(gpu, dtype):
    base = _matrices(4, 90, 150).to(TYPES[dtype]).to(gpu)
    for view in (base[:, 1:80, 3:140], base.mT, base[::2], base[:, ::2], base[..., ::3], base[0][:, 5:70].mT, base[:1].expand(3, 90, 150),
                 base[0, :1].expand(30, 150), base.flip(0), base.permute(1, 0, 2)):
        assert torch.equal(optim.orthogonalize(view), optim.orthogonalize(view.contiguous()))
    negative = torch._neg_view(base)
    assert torch.equal(optim.orthogonalize(negative), optim.orthogonalize(-base))
    before = base.clone()
    optim.orthogonalize(base)
    assert torch.equal(before, base)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_offsets_past_32_bits(gpu, dtype):
    """Matrices 2^32 elements apart, and rows 2^26 apart."""
    store = torch.empty((1 << 32) + (1 << 16), dtype=TYPES[dtype], device=gpu)
    x = _matrices(2, 60, 70).to(TYPES[dtype])
    far = store.as_strided((2, 60, 70), (1 << 32, 70, 1))
    far.copy_(x)
    assert torch.equal(optim.orthogonalize(far), optim.orthogonalize(x.to(gpu)))
    far = store.as_strided((60, 70), (1 << 26, 1))
    far.copy_(x[0])
    assert torch.equal(optim.orthogonalize(far), optim.orthogonalize(x[0].to(gpu)))
    del store, far


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_empty_zero_and_nothing_finite(gpu, dtype):
    t = TYPES[dtype]
    for shape in ((0, 5), (5, 0), (0, 4, 4), (3, 0, 0)):
        assert optim.orthogonalize(torch.empty(shape, dtype=t, device=gpu)).shape == shape
    x = _matrices(5, 70, 90).to(t)
    x[0] = 0.0
    x[1, 69, 89] = float("nan")
    x[2, 3, 4] = float("-inf")
    x[3, :, 1:] = 0.0                  # one direction
    got = optim.orthogonalize(x.to(gpu)).cpu()
    assert (got[0] == 0).all() and got[1].isnan().all() and got[2].isnan().all()
    _close(got[3], x[3])
    _close(got[4], x[4])


@pytest.mark.parametrize("scale", [1e-18, 1e-5, 1e15, 1e37])
def test_lengths_far_from_one(gpu, scale):
    """Squares of these entries leave fp32's range at both ends."""
    x = _matrices(30, 50) * scale / 4.0
    _close(optim.orthogonalize(x.to(gpu), eps=1e-30), x, eps=1e-30)


def test_a_length_under_eps(gpu):
    x = _matrices(40, 40)
    x *= 1e-9 / x.norm()
    _close(optim.orthogonalize(x.to(gpu)), x)
    assert M.off_by(optim.orthogonalize(x.to(gpu)), M.newton_schulz(x, eps=1e-30)) > 0.5


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kw", [dict(steps=1), dict(steps=2), dict(steps=8), dict(coefficients=(1.5, -0.5, 0.0), steps=12), dict(coefficients=(3.0, -3.2, 1.2), steps=6),
                                dict(coefficients=(2.0, -1.5, 0.5)), dict(coefficients=(1.0, 0.0, 0.0)), dict(coefficients=(8.0, -22.0, 16.0), steps=1)])
def test_steps_and_coefficients(gpu, dtype, kw):
    x = _matrices(100, 140).to(TYPES[dtype])
    _close(optim.orthogonalize(x.to(gpu), **kw), x, **kw)


def test_one_huge_entry(gpu):
    """A matrix that is one entry is its own direction; the rest are kept beside it down to the documented steps."""
    x = torch.zeros(80, 100)
    x[17, 31] = -3.0
    got = optim.orthogonalize(x.to(gpu)).cpu()
    _close(got, x)
    x += 1e-3 * _matrices(80, 100)
    _close(optim.orthogonalize(x.to(gpu)), x)


def test_results_are_the_same_every_time_and_on_any_stream(gpu):
    x = _matrices(300, 700).to(gpu)
    first = optim.orthogonalize(x)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s in streams * 3:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(optim.orthogonalize(x))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_out(gpu):
    x = _matrices(3, 30, 40).to(gpu)
    store = torch.full((3 * 1200 + 2,), 7.0, device=gpu)
    out = store[1:-1].view(3, 30, 40)                       # off the 16-byte lines
    assert optim.orthogonalize(x, out=out) is out
    assert torch.equal(out, optim.orthogonalize(x)) and store[0] == 7.0 and store[-1] == 7.0
    from jabas_amd._lib import JabasSyncError
    with pytest.raises(JabasSyncError):
        optim.orthogonalize(x, out=x)
    for bad in (out[:2], out.bfloat16(), out.cpu(), out.mT):
        with pytest.raises(ValueError):
            optim.orthogonalize(x, out=bad)


def test_what_was_saved_of_out_is_known_to_have_changed(gpu):
    x, out = _matrices(30, 40).to(gpu), _matrices(30, 40, seed=1).to(gpu)
    w = torch.ones(30, 40, device=gpu, requires_grad=True)
    y = (w * out).sum()                                     # keeps out for its backward pass
    before = out._version
    optim.orthogonalize(x, out=out)
    assert out._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(gpu):
    x = _matrices(30, 40).to(gpu)
    with pytest.raises(RuntimeError, match="no derivative"):
        optim.orthogonalize(x.clone().requires_grad_())
    with torch.no_grad():
        assert torch.equal(optim.orthogonalize(x.clone().requires_grad_()), optim.orthogonalize(x))
    for bad, error in ((x.half(), TypeError), (x.double(), TypeError), (x[0], ValueError), (x.cpu(), ValueError)):
        with pytest.raises(error):
            optim.orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=33), dict(eps=0.0), dict(eps=float("inf")), dict(coefficients=(1.0, 2.0)), dict(coefficients=(30.0, 40.0, 5.0)),
               dict(coefficients=(8.0, -22.0, 16.0), steps=2)):         # 1 -> 2 -> 352
        with pytest.raises(ValueError):
            optim.orthogonalize(x, **kw)
    with pytest.raises(ValueError, match="sides"):
        optim.orthogonalize(torch.empty(1, (1 << 22) + 1, device=gpu))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_recorded_calls_answer_for_other_inputs(gpu, dtype):
    """A HIP graph, and a graph of operations."""
    x = _matrices(3, 130, 70).to(TYPES[dtype]).to(gpu)
    optim.orthogonalize(x)
    held, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = optim.orthogonalize(held)
    for seed in range(4):
        y = _matrices(3, 130, 70, seed=seed).to(TYPES[dtype]).to(gpu)
        expected = optim.orthogonalize(y)
        held.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expected)
    from torch.fx.experimental.proxy_tensor import make_fx
    traced = make_fx(lambda t: optim.orthogonalize(t) * 2)(x)
    assert torch.equal(traced(y), expected * 2)


def test_a_tangent_is_refused_and_not_lost(gpu):
    import torch.autograd.forward_ad as fwd
    x, out = torch.randn(30, 20, device=gpu), torch.empty(30, 20, device=gpu)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            optim.orthogonalize(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            optim.orthogonalize(dual)
        with pytest.raises(RuntimeError, match="forward-mode"):
            optim.orthogonalize(x, out=fwd.make_dual(out, torch.ones_like(x)))
        assert torch.equal(optim.orthogonalize(fwd.unpack_dual(dual).primal), optim.orthogonalize(x))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(optim.orthogonalize, (x,), (torch.ones_like(x),))


# ----------------------------------------------------------------------------------------------------------- ShardMuon
SHAPES = [(64, 64), (33, 70), (100, 30), (20, 6, 3, 3), (1, 50), (300, 129), (7,), (129,)]


def _parameters(gpu, shapes=SHAPES, seed=1):
    gen = _gen(seed)
    params = [torch.nn.Parameter((torch.randn(*s, generator=gen) * 0.05).to(gpu)) for s in shapes]
    for i, p in enumerate(params):
        p.index = i
    return params


def _gradients(shapes=SHAPES, seed=2):
    gen = _gen(seed)
    return [torch.randn(*s, generator=gen) * 1e-3 for s in shapes]


def _split(params):
    return [dict(params=[p for p in params if p.dim() > 1]), dict(params=[p for p in params if p.dim() == 1], use_muon=False, lr=3e-3, weight_decay=0.2)]


class Expected:
    """The optimizer's arithmetic on the CPU, carried from the kernels' own state so that a step is judged by itself."""

    def __init__(self, opt, **kw):
        self.opt, self.kw = opt, kw

    def before(self):
        self.held = {}
        for group in self.opt.param_groups:
            for p in group["params"]:
                st = self.opt.state.get(p, {})
                self.held[p] = p.detach().clone(), {k: (v.clone() if torch.is_tensor(v) else v) for k, v in st.items()}

    def check(self, p, g):
        group = next(gr for gr in self.opt.param_groups if any(q is p for q in gr["params"]))
        old, st = self.held[p]
        zero = torch.zeros_like(old)
        if group["use_muon"]:
            new, buf, far = M.muon_step(old, g, st.get("momentum_buffer", zero), group["lr"], group["weight_decay"], group["momentum"], group["nesterov"],
                                        group["adjust_lr_fn"], **self.kw)
            assert float((p.detach().cpu().double() - new).norm()) <= far
            got = self.opt.state[p]["momentum_buffer"].cpu().double()
            assert float((got - buf).norm()) <= 2.0 ** -22 * (float(buf.norm()) + float(g.norm()))
        else:
            new, m, v = M.adamw_step(old, g, st.get("exp_avg", zero), st.get("exp_avg_sq", zero), st.get("step", 0) + 1, group["lr"], group["weight_decay"],
                                     group["betas"], group["eps"])
            assert torch.allclose(p.detach().cpu().double(), new, rtol=1e-6, atol=1e-8)
            assert torch.allclose(self.opt.state[p]["exp_avg"].cpu().double(), m, rtol=1e-6, atol=1e-9)

    def unchanged(self, p):
        old, st = self.held[p]
        assert torch.equal(p.detach(), old)
        if "momentum_buffer" in st:
            assert torch.equal(self.opt.state[p]["momentum_buffer"], st["momentum_buffer"])


@pytest.mark.parametrize("kw", [dict(), dict(nesterov=False, momentum=0.5), dict(momentum=0.0, weight_decay=0.0), dict(adjust_lr_fn="match_rms_adamw", lr=1e-3),
                                dict(ns_dtype=torch.bfloat16), dict(ns_steps=2, eps=1e-3)])
def test_steps_of_a_list(gpu, kw):
    params = _parameters(gpu)
    opt = optim.ShardMuon(_split(params), **{**dict(lr=0.02, weight_decay=0.1), **kw})
    exp = Expected(opt, bf16=kw.get("ns_dtype") is torch.bfloat16, steps=kw.get("ns_steps", 5), eps=kw.get("eps", 1e-7))
    for step in range(3):
        grads = _gradients(seed=10 + step)
        for p, g in zip(params, grads):
            p.grad = g.to(gpu)
        opt.param_groups[0]["lr"] *= 0.9
        exp.before()
        opt.step()
        for p, g in zip(params, grads):
            exp.check(p, g)


def test_gradients_in_place_are_remembered_and_follow_every_change(gpu):
    params = _parameters(gpu)
    opt = optim.ShardMuon(_split(params), lr=0.02)
    exp = Expected(opt)
    for p in params:
        p.grad = torch.zeros_like(p)
    for step in range(6):
        grads = _gradients(seed=20 + step)
        for p, g in zip(params, grads):
            p.grad.copy_(g)
        group = opt.param_groups[0]
        if step == 2:
            group["momentum"] = 0.8
        if step == 3:
            group["adjust_lr_fn"] = "match_rms_adamw"
        if step == 4:
            group["nesterov"], group["weight_decay"] = False, 0.3
        if step == 5:
            opt.state[params[0]]["momentum_buffer"] = torch.ones_like(params[0])
        exp.before()
        opt.step()
        assert opt._recipes or step == 0
        for p, g in zip(params, grads):
            exp.check(p, g)


def test_a_buckets_gradients_update_only_their_parameters(gpu):
    params = _parameters(gpu)
    opt = optim.ShardMuon(_split(params), lr=0.02)
    exp = Expected(opt)
    for step, chosen in enumerate(([0, 2, 6], [1, 3, 4], [5, 7], [0, 5, 6, 7], [6])):
        grads = _gradients(seed=30 + step)
        bucket = []
        for i in chosen:
            g = grads[i].to(gpu)
            g.index = i
            bucket.append(g)
        exp.before()
        opt.step(iter(bucket))
        for i, p in enumerate(params):
            exp.check(p, grads[i]) if i in chosen else exp.unchanged(p)
    with pytest.raises(ValueError, match="index"):
        opt.step([torch.zeros(64, 64, device=gpu)])


def test_weights_and_gradients_anywhere_in_memory(gpu):
    """Views at every position of a 16-byte line, gradients that are transposed, what lies beside left as it was."""
    shapes = [(40, 52), (52, 40), (31, 33)]
    stores, params = [], []
    gen = _gen(3)
    for i, s in enumerate(shapes * 4):
        n = s[0] * s[1]
        stores.append(torch.full((n + 8,), 5.0, device=gpu))
        view = stores[-1][1 + i // 3:1 + i // 3 + n].view(s)
        view.copy_(torch.randn(*s, generator=gen) * 0.05)
        params.append(torch.nn.Parameter(view))
    assert all(p.data_ptr() - st.data_ptr() == 4 * (1 + i // 3) for i, (p, st) in enumerate(zip(params, stores)))
    opt = optim.ShardMuon(params, lr=0.02)
    exp = Expected(opt)
    for step in range(2):
        grads = _gradients([tuple(p.shape) for p in params], seed=40 + step)
        for i, (p, g) in enumerate(zip(params, grads)):
            wide = torch.zeros(g.numel() + 3, device=gpu)
            p.grad = wide[i % 4:i % 4 + g.numel()].view(g.shape).copy_(g) if i % 2 else g.t().contiguous().to(gpu).t()
        exp.before()
        opt.step()
        for i, (p, g, st) in enumerate(zip(params, grads, stores)):
            exp.check(p, g)
            at = 1 + i // 3
            assert (st[:at] == 5.0).all() and (st[at + p.numel():] == 5.0).all()


def test_replicas_receive_the_weights(gpu):
    params, a, b = _parameters(gpu), _parameters(gpu, seed=5), _parameters(gpu, seed=6)
    store = torch.zeros(64 * 64 + 1, device=gpu)
    b[0] = torch.nn.Parameter(store[1:].view(64, 64))
    opt = optim.ShardMuon(_split(params), lr=0.02).attach_replicas(params, a, b)
    exp = Expected(opt)
    for step in range(3):
        if step == 2:
            opt.attach_replicas()
        grads = _gradients(seed=50 + step)
        for p, g in zip(params, grads):
            p.grad = g.to(gpu)
        held = [q.detach().clone() for q in a]
        exp.before()
        opt.step()
        for p, g, q, r, old in zip(params, grads, a, b, held):
            exp.check(p, g)
            if step < 2:
                assert torch.equal(p, q) and torch.equal(p, r)
            else:
                assert torch.equal(q, old)


@pytest.mark.parametrize("shapes", [[(16, 16), (64, 40), (33, 64), (1, 9), (50, 3)], [(128, 100), (97, 128), (20, 6, 3, 3)], [(30, 1000), (700, 17)], [(60, 500)], [(300, 90), (5, 5)]])
def test_lists_of_small_matrices(gpu, shapes):
    """What a workgroup's LDS holds is stepped in one launch: weights off the 16-byte lines, replicas, decay, state that is kept."""
    gen = _gen(9)
    params, twins, stores = [], [], []
    for i, s in enumerate(shapes):
        n = torch.Size(s).numel()
        stores.append(torch.full((n + 8,), 5.0, device=gpu))
        params.append(torch.nn.Parameter(stores[-1][i % 4 + 1:i % 4 + 1 + n].view(s)))
        twins.append(torch.nn.Parameter(torch.zeros(s, device=gpu)))
        with torch.no_grad():
            params[-1].copy_(torch.randn(s, generator=gen) * 0.05)
    opt = optim.ShardMuon(params, lr=0.02, weight_decay=0.2).attach_replicas(params, twins)
    exp = Expected(opt)
    for step in range(3):
        grads = _gradients(shapes, seed=100 + step)
        for p, g in zip(params, grads):
            p.grad = g.to(gpu)
        opt.param_groups[0]["nesterov"] = step != 1
        exp.before()
        opt.step()
        for i, (p, g, q, st) in enumerate(zip(params, grads, twins, stores)):
            exp.check(p, g)
            assert torch.equal(p, q)
            assert (st[:i % 4 + 1] == 5.0).all() and (st[i % 4 + 1 + p.numel():] == 5.0).all()


def test_a_list_with_long_matrices(gpu):
    shapes = [(64, 4000), (3000, 200), (40, 50), (130, 1500)]
    params = _parameters(gpu, shapes)
    opt = optim.ShardMuon(params, lr=0.02)
    exp = Expected(opt)
    for step in range(3):
        grads = _gradients(shapes, seed=110 + step)
        for p, g in zip(params, grads):
            p.grad = g.to(gpu)
        exp.before()
        opt.step()
        for p, g in zip(params, grads):
            exp.check(p, g)


def test_lists_that_go_through_the_workspace_some_at_a_time(gpu):
    shapes = [(1024, 1500)] * 9 + [(1500, 900)] * 3 + [(30, 40)] * 40
    params = _parameters(gpu, shapes)
    opt = optim.ShardMuon(params, lr=0.02)
    exp = Expected(opt)
    grads = _gradients(shapes)
    for p, g in zip(params, grads):
        p.grad = g.to(gpu)
    exp.before()
    opt.step()
    alone = _parameters(gpu, shapes)
    one = optim.ShardMuon([alone[8]], lr=0.02)
    alone[8].grad = grads[8].to(gpu)
    one.step()
    assert M.off_by(params[8], alone[8]) < 1e-6
    for i in (0, 8, 11, 12, 51):
        exp.check(params[i], grads[i])


@pytest.mark.parametrize("ns_dtype", [torch.float32, torch.bfloat16])
def test_lists_with_matrices_too_large_to_share_the_workspace(gpu, ns_dtype):
    """Feed-forward weights, each of which is alone in its part, among small ones; the second step, whose momentum is the first one's."""
    shapes = [(300, 129), (4096, 16384), (64, 64), (14336, 4096)]
    gen = torch.Generator(gpu).manual_seed(3)
    params = [torch.nn.Parameter(torch.randn(*s, generator=gen, device=gpu) * 0.05) for s in shapes]
    opt = optim.ShardMuon(params, lr=0.02, weight_decay=0.1, ns_dtype=ns_dtype)
    for step in range(2):
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen, device=gpu) * 1e-3
        held = [(p.detach().double(), opt.state[p]["momentum_buffer"].double() if step else 0.0) for p in params]
        opt.step()
    for p, (old, buf) in zip(params, held):
        g = p.grad.double()
        buf = buf + (1.0 - 0.95) * (g - buf)
        assert float((opt.state[p]["momentum_buffer"].double() - buf).norm()) <= 2.0 ** -22 * float(buf.norm() + g.norm())
        far, o = M.allowed(g + 0.95 * (buf - g), ns_dtype is torch.bfloat16, device=gpu)
        rate = 0.02 * M.lr_factor(None, *p.shape)
        new = old * (1.0 - 0.02 * 0.1) - rate * o
        assert float((p.detach().double() - new).norm()) <= rate * far * float(o.norm()) + 2.0 ** -22 * float(old.norm())


def test_checkpoints_go_to_torch_and_back(gpu):
    shapes = [(40, 30), (30, 64)]
    params, theirs = _parameters(gpu, shapes), _parameters(gpu, shapes)
    opt = optim.ShardMuon(params, lr=0.02, weight_decay=0.05)
    torchs = torch.optim.Muon(theirs, lr=0.02, weight_decay=0.05)
    for step in range(2):
        grads = _gradients(shapes, seed=60 + step)
        for p, q, g in zip(params, theirs, grads):
            p.grad, q.grad = g.to(gpu), g.to(gpu)
        opt.step()
        torchs.step()
        for p, q in zip(params, theirs):        # torch's products are bfloat16's: 8 bits, some of them lost five times over
            assert float((p - q).detach().norm()) <= 2 * 0.02 * (step + 1) * 0.1 * q.shape[0] ** 0.5
            assert torch.allclose(opt.state[p]["momentum_buffer"], torchs.state[q]["momentum_buffer"], rtol=1e-5, atol=1e-8)
    fresh = _parameters(gpu, shapes, seed=1)
    back = optim.ShardMuon(fresh, lr=1.0)
    with torch.no_grad():
        for p, q in zip(fresh, theirs):
            p.copy_(q)
    back.load_state_dict(copy.deepcopy(torchs.state_dict()))
    assert back.param_groups[0]["lr"] == 0.02 and back.param_groups[0]["use_muon"]
    exp = Expected(back)
    grads = _gradients(shapes, seed=63)
    for p, g in zip(fresh, grads):
        p.grad = g.to(gpu)
    exp.before()
    back.step()
    for p, g in zip(fresh, grads):
        exp.check(p, g)
    torchs.load_state_dict(back.state_dict())
    assert torch.equal(torchs.state[theirs[0]]["momentum_buffer"], back.state[fresh[0]]["momentum_buffer"])


def test_what_the_optimizer_refuses(gpu):
    p = torch.nn.Parameter(torch.randn(30, 40, device=gpu).t())
    p.grad = torch.zeros(40, 30, device=gpu)
    with pytest.raises(ValueError, match="contiguous"):
        optim.ShardMuon([p]).step()
    p = torch.nn.Parameter(torch.randn(30, 40, device=gpu).bfloat16())
    p.grad = torch.zeros_like(p)
    with pytest.raises(TypeError):
        optim.ShardMuon([p]).step()
    p = torch.nn.Parameter(torch.randn(30, 40, device=gpu))
    p.grad = torch.zeros(30, 40, device=gpu).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        optim.ShardMuon([p]).step()
    many = [dict(params=[torch.nn.Parameter(torch.randn(3, 4, device=gpu))]) for _ in range(17)]
    for g in many:
        g["params"][0].grad = torch.ones(3, 4, device=gpu)
    with pytest.raises(RuntimeError, match="groups"):
        optim.ShardMuon(many).step()


def test_a_step_recorded_in_a_graph(gpu):
    params = _parameters(gpu)
    opt = optim.ShardMuon([p for p in params if p.dim() > 1], lr=0.02)
    exp = Expected(opt)
    for p in params:
        p.grad = torch.zeros_like(p)
    for seed in (70, 71):               # makes the state, then the plan
        for p, g in zip(params, _gradients(seed=seed)):
            p.grad.copy_(g)
        opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for seed in (72, 73, 74):
        grads = _gradients(seed=seed)
        for p, g in zip(params, grads):
            p.grad.copy_(g)
        exp.before()
        graph.replay()
        torch.cuda.synchronize()
        for p, g in zip(params, grads):
            if p.dim() > 1:
                exp.check(p, g)
        optim.orthogonalize(params[0].detach())


def test_a_recorded_step_outlives_the_optimizers_other_lists(gpu):
    params = [torch.nn.Parameter(torch.randn(s, generator=torch.Generator(gpu).manual_seed(5), device=gpu)) for s in ((40, 200), (300, 70))]
    opt = optim.ShardMuon(params, lr=0.02)
    opt._max_cached_plans = 2
    exp = Expected(opt)
    mine = [torch.zeros_like(p) for p in params]

    def steps(grads, n=1):
        for p, g in zip(params, grads):
            p.grad = g
        for _ in range(n):
            opt.step()

    def some(seed):
        return [torch.randn(p.shape, generator=torch.Generator(gpu).manual_seed(seed), device=gpu) for p in params]

    first = some(0)
    with pytest.raises(RuntimeError, match="recorded"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            steps(first)
    assert not any(opt.state.values())          # memory of a graph that never ran is no state
    steps(some(1), 2)
    steps(mine, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    others = [some(seed) for seed in range(2, 8)]
    for seed in range(3):
        for other in others:            # more lists than are kept
            steps(other, 2)
        grads = some(10 + seed)
        for g, new in zip(mine, grads):
            g.copy_(new)
        exp.before()
        graph.replay()
        torch.cuda.synchronize()
        for p, g in zip(params, grads):
            exp.check(p, g)


def test_a_parameter_that_changes_its_shape_in_place(gpu):
    p = torch.nn.Parameter(torch.randn(30, 80, device=gpu))
    p.grad = torch.randn(30, 80, device=gpu)
    opt = optim.ShardMuon([p], lr=0.02)
    opt.step()
    opt.step()
    grad = p.grad
    p.grad = None
    p.data, p.grad = p.data.view(80, 30), None
    p.grad = grad.view(80, 30)
    opt.state[p]["momentum_buffer"] = opt.state[p]["momentum_buffer"].view(80, 30)
    exp = Expected(opt)
    exp.before()
    opt.step()
    exp.check(p, p.grad)


def _held(opt, params):
    return [p.detach().clone() for p in params] + [v.clone() for p in params for v in opt.state.get(p, {}).values() if torch.is_tensor(v)]


def test_a_call_that_is_refused_moves_nothing(gpu):
    """Matrices are looked over before AdamW updates the others: whoever mends the call and takes it again updates them once."""
    params = _parameters(gpu)
    opt = optim.ShardMuon(_split(params), lr=0.02)
    grads = [g.to(gpu) for g in _gradients()]
    for p, g in zip(params, grads):
        p.grad = g
    opt.step()
    opt.step()
    vector, matrix, group = params[-1], params[0], opt.param_groups[0]
    good = dict(group)

    def refused(error, gradients=None, **kw):
        held, count = _held(opt, params), opt.state[vector]["step"]
        group.update(kw)
        with pytest.raises(error):
            opt.step(gradients)
        group.update(good)
        assert opt.state[vector]["step"] == count
        assert all(torch.equal(a, b) for a, b in zip(held, _held(opt, params)))

    for kw in (dict(momentum=1.0), dict(ns_steps=0), dict(eps=0.0), dict(ns_coefficients=(30.0, 40.0, 5.0)), dict(adjust_lr_fn="none")):
        refused(ValueError, **kw)
    halves = [g.bfloat16() for g in grads]
    for i, h in enumerate(halves):
        h.index = i
    refused(TypeError, gradients=halves)
    held = matrix.data
    matrix.data = held.t().contiguous().t()
    refused(ValueError)
    matrix.data = held
    buf = opt.state[matrix]["momentum_buffer"]
    opt.state[matrix]["momentum_buffer"] = buf.bfloat16()
    refused(ValueError)
    opt.state[matrix]["momentum_buffer"] = buf
    exp = Expected(opt)
    exp.before()
    opt.step()
    for p, g in zip(params, grads):
        exp.check(p, g.cpu())


def test_too_many_groups_move_nothing(gpu):
    params = [torch.nn.Parameter(torch.randn(3, 4, device=gpu)) for _ in range(17)] + [torch.nn.Parameter(torch.randn(5, device=gpu))]
    for p in params:
        p.grad = torch.ones_like(p)
    opt = optim.ShardMuon([dict(params=[p]) for p in params[:-1]] + [dict(params=params[-1:], use_muon=False)])
    held = [p.detach().clone() for p in params]
    with pytest.raises(RuntimeError, match="groups"):
        opt.step()
    assert all(torch.equal(p, h) for p, h in zip(params, held)) and not opt.state.get(params[-1])


def test_a_gradient_of_another_type_at_the_same_address(gpu):
    p = torch.nn.Parameter(torch.randn(64, 64, device=gpu))
    opt = optim.ShardMuon([p], lr=0.02)
    p.index = 0
    g = torch.randn(64, 64, device=gpu)
    half = g.view(torch.bfloat16).view(-1)[:4096].view(64, 64)
    g.index = half.index = 0
    for _ in range(3):
        opt.step([g])
    held = p.detach().clone()
    with pytest.raises(TypeError):
        opt.step([half])
    assert torch.equal(p, held)


def test_a_step_that_updates_others_by_adamw_is_not_recorded(gpu):
    """Its bias corrections are by value: a replay would repeat the recorded ones, and no count would rise."""
    params = _parameters(gpu)
    opt = optim.ShardMuon(_split(params), lr=0.02)
    grads = _gradients()
    for some in (params, params[-1:]):
        for p, g in zip(params, grads):
            p.grad = g.to(gpu) if any(q is p for q in some) else None
        for _ in range(3):
            opt.step()
        torch.cuda.synchronize()
        held, count = _held(opt, params), opt.state[params[-1]]["step"]
        with pytest.raises(RuntimeError, match="recorded"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                opt.step()
        torch.cuda.synchronize()
        assert opt.state[params[-1]]["step"] == count and all(torch.equal(a, b) for a, b in zip(held, _held(opt, params)))
    exp = Expected(opt)                     # and eager steps go on from there
    exp.before()
    opt.step()
    exp.check(params[-1], grads[-1])


# ------------------------------------------------------------------------------------------------ the engine's and the trainer's step
def _engine(gpu, batches, dtype, shapes, n_fanout=0, caps=None, **kw):
    from jabas_amd.engine import VSWFlatSync
    from jabas_amd.workloads import ParamSpec
    specs = [ParamSpec(f"p{i}", torch.Size(s).numel(), 0 if len(s) > 1 else 1) for i, s in enumerate(shapes)]
    opt = dict(kind="muon", momentum=0.9, nesterov=True, betas=(0.8, 0.95), eps=1e-8, groups=[dict(lr=0.02, weight_decay=0.1), dict(lr=1e-3, weight_decay=0.0, use_muon=False)])
    return VSWFlatSync(specs, batches, grad_dtype=dtype, opt=opt, device=gpu, n_fanout=n_fanout, shapes=shapes, caps=caps, **kw)


@pytest.mark.parametrize("dtype,batches,clip,keep", [("fp32", (8,), None, True), ("fp32", (8, 4, 4), None, True), ("bf16", (8, 4, 4, 2, 2, 2, 2, 2), None, True),
                                                     ("fp32", (4, 4), 0.02, True), ("bf16", (4, 4), 0.02, False), ("fp32", (4, 4), 1e9, False)])
def test_engine_steps(gpu, dtype, batches, clip, keep):
    """Many small buckets, so that matrices and vectors alternate inside them and stretches begin anywhere."""
    shapes = [(64, 64), (7,), (33, 70), (129,), (5,), (100, 30), (20, 6, 3, 3), (3,), (40, 41)]
    K = len(batches)
    eng = _engine(gpu, batches, TYPES[dtype], shapes, n_fanout=K - 1, caps=(8192, 20000), keep_clipped_grads=keep)
    gen = _gen(7)
    for i, s in enumerate(shapes):
        eng.param_view(i).copy_(torch.randn(eng.layout.specs[i].numel, generator=gen) * 0.05)
    for step in range(1, 4):
        grads = [[(torch.randn(s, generator=gen) * 1e-2).to(TYPES[dtype]) for s in shapes] for _ in range(K)]
        for k in range(K):
            for i in range(len(shapes)):
                eng.grad_view(k, i).copy_(grads[k][i].reshape(-1))
        total = float(sum(batches))
        mean = [sum(grads[k][i].double() * (batches[k] / total) for k in range(K)) for i in range(len(shapes))]
        norm = float(torch.cat([g.reshape(-1) for g in mean]).norm())
        coef = min(1.0, clip / (norm + 1e-6)) if clip else 1.0
        old = [(eng.param_view(i).cpu(), eng.state_view(0, i).cpu(), eng.state_view(1, i).cpu()) for i in range(len(shapes))]
        rows = eng.step(stats="similarity" if step == 2 else False, lr_scale=0.5 * step, clip_norm=clip)
        assert (rows is not None) == (step == 2)
        if rows is not None:
            assert abs(float(rows[:, 3].sum()) ** 0.5 - norm) <= 1e-5 * norm
        for i, s in enumerate(shapes):
            g, (p, m, v) = mean[i] * coef, old[i]
            if len(s) > 1:
                new, buf, far = M.muon_step(p.view(s), g, m.view(s), 0.02 * 0.5 * step, 0.1, 0.9, True)
                assert float((eng.param_view(i).cpu().double().view(s) - new).norm()) <= far
                assert float((eng.state_view(0, i).cpu().double().view(s) - buf).norm()) <= 1e-6 * (float(buf.norm()) + float(g.norm()))
            else:
                new, m1, v1 = M.adamw_step(p, g, m, v, step, 1e-3 * 0.5 * step, 0.0, (0.8, 0.95))
                assert torch.allclose(eng.param_view(i).cpu().double(), new, rtol=1e-5, atol=1e-7)
                assert torch.allclose(eng.state_view(1, i).cpu().double(), v1, rtol=1e-5, atol=1e-12)
            assert torch.allclose(eng.agg_view(i).cpu().double(), (g if keep else mean[i]).reshape(-1), rtol=1e-5, atol=1e-9)
            for f in eng.fanout:
                assert torch.equal(eng._view(f, i), eng.param_view(i))
    eng.reconfigure((4,) * (K + 1))
    for a in eng.grads:
        a.zero_()
    before = eng.state_view(0, 0).clone()
    eng.step()
    assert torch.allclose(eng.state_view(0, 0), before * 0.9, rtol=1e-6, atol=0)
    with pytest.raises(ValueError, match="cannot be replayed"):
        eng.capture()


def test_engine_refusals(gpu):
    from jabas_amd.engine import VSWFlatSync
    from jabas_amd.workloads import ParamSpec
    opt = dict(kind="muon", groups=[dict(lr=0.02)])
    specs = [ParamSpec("a", 12, 0)]
    for shapes, match in ((None, "shape of every parameter"), ([], "shape of every parameter"), ([(3, 5)], "cannot have shape"), ([(12,)], "no matrix")):
        with pytest.raises(ValueError, match=match):
            VSWFlatSync(specs, (1,), opt=opt, device=gpu, shapes=shapes)


class _Net(torch.nn.Module):
    def __init__(self, seed, bias=True):
        super().__init__()
        torch.manual_seed(seed)
        self.a, self.b = torch.nn.Linear(37, 64, bias=bias), torch.nn.Linear(64, 10, bias=bias)

    def forward(self, x):
        return self.b(torch.relu(self.a(x)))


def _data(gpu, batches, seed):
    gen = _gen(seed)
    return [(torch.randn(b, 37, generator=gen).to(gpu), torch.randn(b, 10, generator=gen).to(gpu)) for b in batches]


def _own(model):
    return optim.ShardMuon([dict(params=[p for p in model.parameters() if p.dim() > 1]), dict(params=[p for p in model.parameters() if p.dim() == 1], use_muon=False, lr=1e-3)],
                           lr=0.02, weight_decay=0.01)


@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("clip", [None, 0.05])
def test_trainer_steps_as_the_optimizer_does(gpu, share, clip):
    """Two workers through the trainer, and one worker on both batches with the optimizer's own step."""
    from jabas_amd.train import VSWSyncTrainer
    batches, crit = (6, 6), torch.nn.MSELoss()
    t = VSWSyncTrainer(gpu, batches, interval=2, share_weights=share, clip_norm=clip, keep_grads=True)
    t.prepare_stream_parallel(_Net(3), crit)
    t.prepare_weight_sync_method(_own(t.main_model))
    plain = _Net(3).to(gpu)
    opt = _own(plain)
    for step in range(4):
        data = _data(gpu, batches, 80 + step)
        t.compute(data)
        t.step()
        for p in plain.parameters():
            p.grad = None
        (sum(crit(plain(x), y) for x, y in data) / 2).backward()
        if clip:
            torch.nn.utils.clip_grad_norm_(plain.parameters(), clip)
        opt.step()
        for p, q, r in zip(t.main_model.parameters(), plain.parameters(), t.local_models[1].parameters()):
            assert torch.allclose(p.grad, q.grad, rtol=1e-4, atol=1e-7)
            assert M.off_by(p, q) < 1e-4 and torch.equal(p, r)
    for p, q in zip(t.main_model.parameters(), plain.parameters()):
        mine, theirs = t.main_optimizer.state[p], opt.state[q]
        assert set(mine) == set(theirs)
        assert all(M.off_by(mine[k], theirs[k]) < 1e-4 for k in mine if torch.is_tensor(theirs[k]))


def test_trainer_resumes_from_its_checkpoint(gpu, tmp_path):
    from jabas_amd.train import VSWSyncTrainer
    crit = torch.nn.MSELoss()

    def make(seed):
        t = VSWSyncTrainer(gpu, (4, 4), interval=2)
        t.prepare_stream_parallel(_Net(seed), crit)
        t.prepare_weight_sync_method(_own(t.main_model))
        return t

    def run(t, first, last):
        for step in range(first, last):
            t.compute(_data(gpu, (4, 4), 90 + step))
            t.step()
        torch.cuda.synchronize()

    a = make(1)
    run(a, 0, 3)
    torch.save(a.state_dict(), tmp_path / "t.pth")
    run(a, 3, 6)
    b = make(2)
    b.load_state_dict(torch.load(tmp_path / "t.pth", map_location=gpu, weights_only=True))
    run(b, 3, 6)
    for p, q in zip(a.main_model.parameters(), b.main_model.parameters()):
        assert torch.equal(p, q)


def test_trainer_takes_torchs_own_and_follows_its_groups(gpu):
    from jabas_amd.train import VSWSyncTrainer
    t = VSWSyncTrainer(gpu, (4, 4))
    t.prepare_stream_parallel(_Net(5, bias=False), torch.nn.MSELoss())
    opt = torch.optim.Muon(t.main_model.parameters(), lr=0.02, weight_decay=0.0)
    t.prepare_weight_sync_method(opt)
    held = [p.detach().clone() for p in t.main_model.parameters()]
    t.compute(_data(gpu, (4, 4), 1))
    t.step()
    for p, old in zip(t.main_model.parameters(), held):
        # the first step's update is along its gradient, and so is the momentum
        far, e = M.allowed(opt.state[p]["momentum_buffer"].cpu(), False)
        rate = 0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        assert float((p.detach().cpu().double() - (old.cpu().double() - rate * e)).norm()) <= rate * far * float(e.norm()) + 2.0 ** -22 * float(old.norm())
    opt.param_groups[0]["lr"] = 0.0
    held = [p.detach().clone() for p in t.main_model.parameters()]
    t.compute(_data(gpu, (4, 4), 2))
    t.step()
    assert all(torch.equal(p, old) for p, old in zip(t.main_model.parameters(), held))
    opt.param_groups[0]["adjust_lr_fn"] = "match_rms_adamw"
    t.compute(_data(gpu, (4, 4), 3))
    with pytest.raises(ValueError, match="part of the launches' plan"):
        t.step()


def test_trainer_leaves_parameters_outside_the_groups_alone(gpu):
    """A frozen bias needs no group, a frozen matrix is not decayed, and checkpoints hold neither."""
    from jabas_amd.train import VSWSyncTrainer
    for share in (True, False):
        t = VSWSyncTrainer(gpu, (4, 4), interval=2, share_weights=share, clip_norm=0.05)
        net = _Net(6)
        for p in (net.a.weight, net.b.bias):
            p.requires_grad_(False)
        t.prepare_stream_parallel(net, torch.nn.MSELoss())
        mine = t.main_model
        t.prepare_weight_sync_method(optim.ShardMuon([dict(params=[mine.b.weight]), dict(params=[mine.a.bias], use_muon=False, lr=1e-2)], lr=0.02, weight_decay=0.3))
        held = [p.detach().clone() for p in mine.parameters()]
        for step in range(3):
            t.compute(_data(gpu, (4, 4), 50 + step))
            t.step()
        for p, q, old in zip(mine.parameters(), t.local_models[1].parameters(), held):
            assert torch.equal(p, q) and torch.equal(p, old) == (not p.requires_grad)
        state = t.state_dict()
        assert len(state["optimizer"]["state"]) == 2
        t.load_state_dict(state)
        t.compute(_data(gpu, (4, 4), 60))
        t.step()
        for p, old in zip(mine.parameters(), held):
            assert torch.equal(p, old) == (not p.requires_grad)


@pytest.mark.parametrize("change,error", [(dict(momentum=1.0), ValueError), (dict(ns_steps=0), ValueError), (dict(ns_eps=0.0), ValueError),
                                          (dict(ns_coefficients=(30.0, 40.0, 5.0)), ValueError)])
def test_an_engines_step_that_is_refused_moves_nothing(gpu, change, error):
    shapes = [(64, 64), (7,), (300, 129)]
    eng = _engine(gpu, (4, 4), torch.float32, shapes, in_place=False)
    for a in (eng.param, *eng.grads):
        a.copy_(torch.randn(a.numel(), generator=_gen(8)) * 0.05)
    eng.step()
    held = [t.clone() for t in (eng.param, eng.state1, eng.state2)]
    eng.opt.update(change)
    for clip in (None, 0.1):
        with pytest.raises(error):
            eng.step(clip_norm=clip)
    assert eng.step_count == 1 and all(torch.equal(a, b) for a, b in zip(held, (eng.param, eng.state1, eng.state2)))


def test_trainer_goes_on_refusing_what_its_plans_cannot_follow(gpu):
    from jabas_amd.train import VSWSyncTrainer
    t = VSWSyncTrainer(gpu, (4, 4))
    t.prepare_stream_parallel(_Net(5, bias=False), torch.nn.MSELoss())
    opt = optim.ShardMuon(t.main_model.parameters(), lr=0.02)
    t.prepare_weight_sync_method(opt)
    held = [p.detach().clone() for p in t.main_model.parameters()]
    for key, value in (("adjust_lr_fn", "match_rms_adamw"), ("ns_dtype", torch.bfloat16)):
        before = opt.param_groups[0][key]
        opt.param_groups[0][key] = value
        for seed in range(3):
            t.compute(_data(gpu, (4, 4), seed))
            with pytest.raises(ValueError, match="part of the launches' plan"):
                t.step()
        opt.param_groups[0][key] = before
    assert all(torch.equal(p, old) for p, old in zip(t.main_model.parameters(), held))
    t.step()
    assert not any(torch.equal(p, old) for p, old in zip(t.main_model.parameters(), held))


@pytest.mark.parametrize("change", [dict(ns_dtype=torch.bfloat16), dict(adjust_lr_fn="match_rms_adamw"),
                                    dict(groups=[dict(lr=0.02, use_muon=False), dict(lr=1e-3, use_muon=False)])])
def test_an_engines_step_that_its_plans_cannot_follow_moves_nothing(gpu, change):
    eng = _engine(gpu, (4, 4), torch.float32, [(64, 64), (7,), (300, 129)], in_place=False)
    for a in (eng.param, *eng.grads):
        a.copy_(torch.randn(a.numel(), generator=_gen(8)) * 0.05)
    held, before = [t.clone() for t in (eng.param, eng.state1, eng.state2, eng.agg)], dict(eng.opt)
    eng.opt.update(change)
    with pytest.raises(ValueError, match="part of the launches' plan"):
        eng.step()
    assert eng.step_count == 0 and all(torch.equal(a, b) for a, b in zip(held, (eng.param, eng.state1, eng.state2, eng.agg)))
    eng.opt.clear()
    eng.opt.update(before)
    eng.step()
    assert not torch.equal(held[0], eng.param)


def test_engine_leaves_parameters_without_a_shape_alone(gpu):
    """Between matrices and between vectors, in one bucket with them; they count for the aggregate and its norm."""
    from jabas_amd.engine import VSWFlatSync
    from jabas_amd.workloads import ParamSpec
    shapes = [(7,), (64, 40), (9,), (11,), (33, 70), (5,), (3,)]
    alone = {1, 3, 6}
    specs = [ParamSpec(f"p{i}", torch.Size(s).numel(), 0 if len(s) > 1 else 1) for i, s in enumerate(shapes)]
    opt = dict(kind="muon", groups=[dict(lr=0.02, weight_decay=0.5), dict(lr=1e-2, weight_decay=0.5, use_muon=False)])
    eng = VSWFlatSync(specs, (4, 4), opt=opt, device=gpu, in_place=False, n_fanout=1, shapes=[None if i in alone else s for i, s in enumerate(shapes)])
    for a in (eng.param, *eng.grads):
        a.copy_(torch.randn(a.numel(), generator=_gen(8)))
    eng.fanout[0].copy_(eng.param)
    held = [eng.param_view(i).clone() for i in range(len(shapes))]
    for _ in range(2):
        eng.step(clip_norm=1e6)
        eng.reconfigure((4, 4))
    for i, old in enumerate(held):
        assert torch.equal(eng.param_view(i), old) == (i in alone)
        assert torch.equal(eng._view(eng.fanout[0], i), eng.param_view(i))
        assert torch.allclose(eng.agg_view(i), eng.grad_view(0, i) / 2 + eng.grad_view(1, i) / 2)
        assert bool(eng.state_view(0, i).any()) == (i not in alone)


@pytest.mark.parametrize("dtype,clip,keep,ns_dtype", [("fp32", None, True, torch.float32), ("fp32", 0.02, False, torch.float32), ("bf16", 0.02, False, torch.bfloat16),
                                                      ("bf16", 0.02, True, torch.float32)])
def test_engine_steps_of_larger_matrices(gpu, dtype, clip, keep, ns_dtype):
    """Matrices that no workgroup holds alone: the clipping coefficient is read by both passes over the aggregate, which have to agree on it."""
    shapes, batches = [(300, 129), (129,), (200, 700), (5,), (64, 64)], (4, 2, 2)
    eng = _engine(gpu, batches, TYPES[dtype], shapes, n_fanout=2, caps=(200000,), keep_clipped_grads=keep)
    eng.opt["ns_dtype"] = ns_dtype
    eng.reconfigure(batches)
    gen, bf16 = _gen(17), ns_dtype is torch.bfloat16
    for i in range(len(shapes)):
        eng.param_view(i).copy_(torch.randn(eng.layout.specs[i].numel, generator=gen) * 0.05)
    for step in range(1, 4):
        grads = [[(torch.randn(s, generator=gen) * 1e-2).to(TYPES[dtype]) for s in shapes] for _ in batches]
        for k, mine in enumerate(grads):
            for i, g in enumerate(mine):
                eng.grad_view(k, i).copy_(g.reshape(-1))
        mean = [sum(mine[i].double() * (b / sum(batches)) for mine, b in zip(grads, batches)) for i in range(len(shapes))]
        coef = min(1.0, clip / (float(torch.cat([g.reshape(-1) for g in mean]).norm()) + 1e-6)) if clip else 1.0
        assert not clip or coef < 0.1
        old = [(eng.param_view(i).cpu(), eng.state_view(0, i).cpu(), eng.state_view(1, i).cpu()) for i in range(len(shapes))]
        eng.step(clip_norm=clip)
        for i, s in enumerate(shapes):
            g, (p, m, v), got = mean[i] * coef, old[i], eng.param_view(i).cpu().double()
            if len(s) > 1:
                new, buf, far = M.muon_step(p.view(s), g, m.view(s), 0.02, 0.1, 0.9, True, bf16=bf16)
                assert float((got.view(s) - new).norm()) <= far
                assert float((eng.state_view(0, i).cpu().double().view(s) - buf).norm()) <= 1e-6 * (float(buf.norm()) + float(g.norm()))
            else:
                new, _, _ = M.adamw_step(p, g, m, v, step, 1e-3, 0.0, (0.8, 0.95))
                assert torch.allclose(got, new, rtol=1e-5, atol=1e-7)
            for f in eng.fanout:
                assert torch.equal(eng._view(f, i), eng.param_view(i))


@pytest.mark.parametrize("kind", ["muon", "adamw"])
@pytest.mark.parametrize("keep", [True, False])
def test_a_first_clipped_step_on_another_stream(gpu, kind, keep):
    """What such a step makes for itself is filled on the current stream, which has work of its own to do first."""
    from jabas_amd.engine import VSWFlatSync
    from jabas_amd.workloads import ParamSpec
    shapes = [(64, 64), (7,), (300, 129)]
    specs = [ParamSpec(f"p{i}", torch.Size(s).numel(), 0 if len(s) > 1 else 1) for i, s in enumerate(shapes)]
    opt = dict(kind=kind, momentum=0.9, nesterov=True, betas=(0.8, 0.95), eps=1e-8, groups=[dict(lr=0.02, weight_decay=0.1), dict(lr=1e-3, weight_decay=0.0, use_muon=False)])

    def engine():
        eng = VSWFlatSync(specs, (4, 4), opt=opt, device=gpu, in_place=False, shapes=shapes, keep_clipped_grads=keep, write_aggregate=False)
        for a in (eng.param, *eng.grads):
            a.copy_(torch.randn(a.numel(), generator=_gen(8)) * 0.05)
        return eng

    here, there, side = engine(), engine(), torch.cuda.Stream()
    here.step(clip_norm=0.5)
    busy = torch.randn(4096, 4096, device=gpu)
    busy @ busy
    torch.cuda.synchronize()
    for _ in range(40):
        busy = busy @ busy
    there.step(clip_norm=0.5, stream=side)
    torch.cuda.synchronize()
    for a, b in ((here._coef, there._coef), (here.param, there.param), (here.agg, there.agg)):
        assert torch.equal(a, b)
    assert float(here._coef) < 0.2
