"""CPU-only checks of the orthogonalised update's C ABI (include/jabas_muon.h) and of the refusals above it. Nothing is launched."""
import ctypes as C
import os
import re
import subprocess
import sys

import pytest
import torch

from jabas_amd import _lib as L
from jabas_amd import optim

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "jabas_muon.h")
ADDRESS = 0x7f0000000000
STRUCTS = ("JabasNewtonSchulz", "JabasOrthogonalize", "JabasMatrix", "JabasMuonArgs")


def _ns(**kw):
    return L.JabasNewtonSchulz(**{**dict(a=3.4445, b=-4.775, c=2.0315, eps=1e-7, steps=5, precision=L.F32), **kw})


def _batch(ns=None, **kw):
    o = L.JabasOrthogonalize(out=2 * ADDRESS, batch=3, rows=100, cols=70, in_batch_stride=7000, in_row_stride=70, dtype=L.F32, ns=ns or _ns())
    setattr(o, "in", ADDRESS)
    for k, v in kw.items():
        setattr(o, k, v)
    return o


def _matrix(i=0, **kw):
    m = L.JabasMatrix(grad=ADDRESS + (3 * i << 30), momentum=ADDRESS + (3 * i + 1 << 30), param=ADDRESS + (3 * i + 2 << 30), rows=100, cols=70, lr_factor=1.0)
    for k, v in kw.items():
        setattr(m, k, v)
    return m


def _list(*matrices):
    return (L.JabasMatrix * len(matrices))(*matrices), len(matrices)


def _encode(*matrices, precision=L.F32):
    table, n = _list(*matrices)
    size = L.lib().jabas_muon_plan_bytes(table, n, precision)
    blob = torch.zeros(max(size, 8) // 8, dtype=torch.int64)
    return L.lib().jabas_muon_plan_encode(table, n, precision, blob.data_ptr(), size), blob, size


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(jabas_[a-z_]+)\s*\(", text))
    assert names == set(L.MUON_SIGNATURES)
    for n in names:
        assert hasattr(L.lib(), n)


def test_structs_and_constants_match_the_header(tmp_path):
    prints, expected = "", []
    for name in STRUCTS:
        kind = getattr(L, name)
        for f, _ in kind._fields_:
            prints += f'printf("%zu ", offsetof({name}, {f}));'
            expected.append(getattr(kind, f).offset)
        prints += f'printf("%zu ", sizeof({name}));'
        expected.append(C.sizeof(kind))
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include "jabas_muon.h"\nint main(void) {{ {prints} '
                   'printf("%d %lld %lld", JABAS_MUON_MAX_STEPS, JABAS_MUON_MAX_SIDE, JABAS_MUON_MAX_LENGTH); return 0; }')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    seen = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert seen == expected + [L.MUON_MAX_STEPS, L.MUON_MAX_SIDE, L.MUON_MAX_LENGTH]


def _orthogonalize(o, workspace=ADDRESS << 1, size=None):
    n = L.lib().jabas_orthogonalize_workspace_bytes(C.byref(o))
    return L.lib().jabas_orthogonalize(C.byref(o), workspace, n if size is None else size, None), n


@pytest.mark.parametrize("change,status", [
    (dict(dtype=7), L.ERR_DTYPE), (dict(batch=-1), L.ERR_SIZE), (dict(rows=-1), L.ERR_SIZE), (dict(rows=1 << 17, cols=1 << 17, in_row_stride=1 << 17), L.ERR_SIZE),
    (dict(cols=(1 << 22) + 1, in_row_stride=1 << 23), L.ERR_SIZE), (dict(in_row_stride=69), L.ERR_SIZE), (dict(in_batch_stride=-1), L.ERR_SIZE),
    (dict(out=None), L.ERR_NULL), (dict(out=ADDRESS), L.ERR_ALIAS), (dict(out=ADDRESS + 4 * 20999), L.ERR_ALIAS), (dict(out=ADDRESS - 4), L.ERR_ALIAS),
    (dict(out=2 * ADDRESS + 2), L.ERR_ALIGN), (dict(ns=_ns(steps=0)), L.ERR_OPT), (dict(ns=_ns(steps=33)), L.ERR_OPT), (dict(ns=_ns(eps=0.0)), L.ERR_OPT),
    (dict(ns=_ns(eps=float("nan"))), L.ERR_OPT), (dict(ns=_ns(a=float("inf"))), L.ERR_OPT), (dict(ns=_ns(a=30.0, b=40.0, c=5.0)), L.ERR_OPT),
    (dict(ns=_ns(precision=2)), L.ERR_DTYPE)])
def test_batches_that_are_refused(change, status):
    got, size = _orthogonalize(_batch(**change))
    assert got == status and size == 0


def test_what_lies_right_beside_is_no_overlap_and_little_workspace_is_refused():
    for o in (_batch(out=ADDRESS + 4 * 21000), _batch()):
        n = L.lib().jabas_orthogonalize_workspace_bytes(C.byref(o))
        assert n >= 256 and n % 256 == 0
        assert _orthogonalize(o, size=n - 256)[0] == L.ERR_WORKSPACE
        assert _orthogonalize(o, workspace=None)[0] == L.ERR_WORKSPACE
        assert _orthogonalize(o, workspace=ADDRESS + 128)[0] == L.ERR_WORKSPACE


@pytest.mark.parametrize("empty", [dict(batch=0), dict(rows=0), dict(cols=0, in_row_stride=0)])
def test_nothing_to_do_launches_nothing(empty):
    assert _orthogonalize(_batch(**empty), workspace=None, size=0) == (L.OK, 256)


def test_the_workspace_does_not_grow_with_the_batch():
    sizes = [L.lib().jabas_orthogonalize_workspace_bytes(C.byref(_batch(batch=n, rows=1024, cols=1024, in_row_stride=1024, in_batch_stride=1 << 20,
                                                                        out=1 << 45))) for n in (1, 4, 100, 1000)]
    assert sizes[0] < sizes[1] < sizes[2] == sizes[3] < 520 << 20


@pytest.mark.parametrize("change,status", [
    (dict(grad=None), L.ERR_NULL), (dict(momentum=None), L.ERR_NULL), (dict(param=None), L.ERR_NULL), (dict(rows=0), L.ERR_SIZE), (dict(cols=0), L.ERR_SIZE),
    (dict(rows=1 << 17, cols=1 << 17), L.ERR_SIZE), (dict(group=16), L.ERR_GROUP), (dict(n_fanout=16), L.ERR_K), (dict(n_fanout=1), L.ERR_NULL),
    (dict(lr_factor=float("nan")), L.ERR_OPT), (dict(grad=ADDRESS + 2), L.ERR_ALIGN), (dict(param=ADDRESS + 4 * 6999), L.ERR_ALIAS),
    (dict(momentum=ADDRESS), L.ERR_ALIAS)])
def test_matrices_that_are_refused(change, status):
    got, _, size = _encode(_matrix(), _matrix(1), _matrix(**change))
    assert got == status and size == 0


def test_replicas_may_not_lie_in_what_is_read():
    m = _matrix(n_fanout=2)
    m.fanout[0], m.fanout[1] = ADDRESS + (5 << 30), ADDRESS + (6 << 30)
    assert _encode(m)[0] == L.OK
    m.fanout[1] = m.fanout[0] + 4
    assert _encode(m)[0] == L.ERR_ALIAS
    m.fanout[1] = m.grad
    assert _encode(m)[0] == L.ERR_ALIAS


def test_plans_and_their_workspace():
    lib = L.lib()
    assert lib.jabas_muon_plan_bytes(None, 1, L.F32) == 0 and lib.jabas_muon_plan_bytes(_list(_matrix())[0], 0, L.F32) == 0
    status, blob, size = _encode(*[_matrix(i, rows=1024, cols=4096) for i in range(40)], _matrix(40, rows=3, cols=5, group=2))
    assert status == L.OK
    ws = lib.jabas_muon_workspace_bytes(blob.data_ptr())
    assert 0 < ws < 520 << 20 and ws % 256 == 0                # 40 matrices of 80 MB go through it some at a time
    again = _encode(*[_matrix(i, rows=1024, cols=4096) for i in range(40)], _matrix(40, rows=3, cols=5, group=2))[1]
    assert torch.equal(blob, again)
    table, n = _list(_matrix())
    assert lib.jabas_muon_plan_encode(table, n, L.F32, blob.data_ptr(), 64) == L.ERR_PLAN
    assert lib.jabas_muon_plan_encode(table, n, L.F32, None, size) == L.ERR_NULL
    assert lib.jabas_muon_workspace_bytes(None) == 0 and lib.jabas_muon_workspace_bytes(torch.zeros(64, dtype=torch.int64).data_ptr()) == 0


LARGE = {"feed_forward": [(4096, 16384)], "tall": [(14336, 4096)], "vocabulary": [(50257, 1600)], "three": [(32000, 4096)] * 3, "square": [(6144, 6144)] * 2,
         "mixed": [(32000, 4096), (1024, 1024), (32000, 4096)], "among_small": [(64, 64), (4096, 16384), (100, 70), (1000, 2048)]}


@pytest.mark.parametrize("precision", [L.F32, L.BF16])
@pytest.mark.parametrize("shapes", LARGE.values(), ids=LARGE)
def test_matrices_too_large_to_share_the_workspace(shapes, precision):
    """One that needs more than the 500 MiB that several may share goes through alone. In a process of its own: a crash of the encoder is a failure here."""
    code = ("import sys; sys.path.insert(0, 'tests'); import test_muon_cabi_host as t\n"
            f"print(*t._workspaces({shapes!r}, {precision}))")
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, env={**os.environ, "PYTHONPATH": ROOT})
    assert run.returncode == 0, (run.returncode, run.stderr)
    status, whole, *alone = [int(x) for x in run.stdout.split()]
    assert status == L.OK
    assert max(max(alone), 400 << 20) <= whole <= max(max(alone), 520 << 20)


def _workspaces(shapes, precision):
    lib, table = L.lib(), [_matrix(i, rows=r, cols=c) for i, (r, c) in enumerate(shapes)]
    status, blob, _ = _encode(*table, precision=precision)
    return [status] + [lib.jabas_muon_workspace_bytes(b.data_ptr()) for b in (blob, *[_encode(m, precision=precision)[1] for m in table])]


def test_steps_that_are_refused():
    lib = L.lib()
    status, blob, size = _encode(_matrix(), _matrix(1, group=2))
    assert status == L.OK
    ws = lib.jabas_muon_workspace_bytes(blob.data_ptr())

    def step(plan=blob.data_ptr(), dev=ADDRESS, workspace=ADDRESS, size=ws, **kw):
        a = L.JabasMuonArgs(**{**dict(ns=_ns(), momentum=0.9, n_groups=3), **kw})
        return lib.jabas_muon_step(plan, dev, C.byref(a), workspace, size, None)

    assert step(n_groups=2) == L.ERR_GROUP and step(n_groups=17) == L.ERR_GROUP
    assert step(momentum=1.0) == L.ERR_OPT and step(momentum=float("nan")) == L.ERR_OPT and step(momentum=-0.1) == L.ERR_OPT
    assert step(ns=_ns(precision=L.BF16)) == L.ERR_PLAN
    assert step(ns=_ns(steps=0)) == L.ERR_OPT
    assert step(plan=None) == L.ERR_NULL and step(dev=None) == L.ERR_NULL and step(dev=ADDRESS + 8) == L.ERR_PLAN
    assert step(plan=torch.zeros(64, dtype=torch.int64).data_ptr()) == L.ERR_PLAN
    assert step(size=ws - 1) == L.ERR_WORKSPACE and step(workspace=None) == L.ERR_WORKSPACE and step(workspace=ADDRESS + 16) == L.ERR_WORKSPACE


def test_tensors_that_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        optim.orthogonalize(torch.zeros(3, 3))
    with pytest.raises(TypeError):
        optim.orthogonalize([[1.0]])


def test_a_tangent_is_refused_and_not_lost():
    import torch.autograd.forward_ad as fwd
    x = torch.randn(3, 4)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones(3, 4))
        for call in (lambda: optim.orthogonalize(dual), lambda: optim.orthogonalize(x, out=dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="GPU"):
            optim.orthogonalize(x)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(optim.orthogonalize, (x,), (torch.ones(3, 4),))


def test_optimizers_that_are_refused():
    p = lambda *s: torch.nn.Parameter(torch.zeros(*s))
    with pytest.raises(ValueError, match="no matrix"):
        optim.ShardMuon([p(3, 4), p(5)])
    with pytest.raises(ValueError, match="no matrix"):
        optim.ShardMuon([p(0, 4)])
    for bad in (dict(lr=-1.0), dict(weight_decay=-1.0), dict(momentum=1.0), dict(momentum=-0.5), dict(ns_steps=0), dict(ns_steps=33), dict(eps=0.0),
                dict(ns_coefficients=(1.0, 2.0)), dict(ns_coefficients=(30.0, 40.0, 5.0)), dict(adjust_lr_fn="none")):
        with pytest.raises(ValueError):
            optim.ShardMuon([p(3, 4)], **bad)
    with pytest.raises(TypeError):
        optim.ShardMuon([p(3, 4)], ns_dtype=torch.float16)
    with pytest.raises(ValueError):
        optim.ShardMuon([dict(params=[p(3)], use_muon=False, betas=(1.0, 0.9))])
    opt = optim.ShardMuon([p(3, 4)])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[p(7)]))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[p(7)], use_muon=False))
    assert opt.param_groups[1]["eps"] == 1e-8 and opt.param_groups[0]["eps"] == 1e-7
    opt.param_groups[0]["params"][0].grad = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt.step()


def test_the_bucket_launches_refuse_it():
    from jabas_amd.local_sync import LocalBucketSync
    from jabas_amd.train.trainer import opt_from_torch_optimizer
    groups = [dict(params=[torch.nn.Parameter(torch.zeros(3, 4))], weight_decay=0.1), dict(params=[torch.nn.Parameter(torch.zeros(3))], use_muon=False, lr=0.3)]
    opt = optim.ShardMuon(groups, lr=0.02, betas=(0.8, 0.9), momentum=0.7)
    got = opt_from_torch_optimizer(opt)
    assert got["kind"] == "muon" and got["betas"] == (0.8, 0.9) and got["momentum"] == 0.7 and got["eps"] == 1e-8 and got["ns_eps"] == 1e-7
    assert [(g["lr"], g["weight_decay"], g["use_muon"]) for g in got["groups"]] == [(0.02, 0.1, True), (0.3, 0.1, False)]
    local = LocalBucketSync((2, 2))
    with pytest.raises(TypeError, match="no part of a bucket's launch"):
        local.bind_optimizer(opt)
    assert local.optimizer is None


def test_amsgrad_is_refused_where_the_sync_step_would_drop_it():
    from jabas_amd.engine import VSWFlatSync
    from jabas_amd.train.trainer import opt_from_torch_optimizer, refresh_opt_from_torch_optimizer
    from jabas_amd.workloads import ParamSpec
    groups = [dict(params=[torch.nn.Parameter(torch.zeros(3, 4))]), dict(params=[torch.nn.Parameter(torch.zeros(3))], use_muon=False, amsgrad=True)]
    opt = optim.ShardMuon(groups)
    with pytest.raises(ValueError, match="amsgrad"):
        opt_from_torch_optimizer(opt)
    opt.param_groups[1]["amsgrad"] = False
    got = opt_from_torch_optimizer(opt)
    opt.param_groups[1]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        refresh_opt_from_torch_optimizer(got, opt)
    opt.param_groups[1]["amsgrad"], opt.param_groups[0]["amsgrad"] = False, True        # of the matrices: means nothing
    opt_from_torch_optimizer(opt)
    specs = [ParamSpec("a", 12, 0), ParamSpec("b", 3, 1)]
    for where in (dict(amsgrad=True), dict(groups=[dict(lr=0.1), dict(lr=0.1, use_muon=False, amsgrad=True)])):
        with pytest.raises(ValueError, match="amsgrad"):
            VSWFlatSync(specs, (1,), opt={**dict(kind="muon", groups=[dict(lr=0.1), dict(lr=0.1, use_muon=False)]), **where}, device="cpu", shapes=[(3, 4), (3,)])


def test_a_refused_change_of_the_groups_is_refused_again():
    from jabas_amd.train.trainer import opt_from_torch_optimizer, refresh_opt_from_torch_optimizer
    opt = optim.ShardMuon([torch.nn.Parameter(torch.zeros(3, 4))])
    got = opt_from_torch_optimizer(opt)
    for key, value in (("adjust_lr_fn", "match_rms_adamw"), ("ns_dtype", torch.bfloat16)):
        before = opt.param_groups[0][key]
        opt.param_groups[0][key] = value
        for _ in range(2):
            with pytest.raises(ValueError, match="part of the launches' plan"):
                refresh_opt_from_torch_optimizer(got, opt)
        opt.param_groups[0][key] = before
    opt.param_groups[0]["momentum"] = 0.5
    refresh_opt_from_torch_optimizer(got, opt)
    assert got == opt_from_torch_optimizer(opt)
