"""CPU-only checks of the losses' C ABI (include/jabas_loss.h): exported symbols, struct layout, sizes, refusals. Nothing is launched."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from jabas_amd import _lib as L
from jabas_amd import loss as losses

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "jabas_loss.h")
ADDRESS = 0x7f0000000000


def _linear(**kw):
    c = L.JabasLoss()
    c.hidden, c.weight, c.target, c.row_state = ADDRESS, 2 * ADDRESS, 3 * ADDRESS, 4 * ADDRESS
    c.rows, c.vocab, c.width, c.hidden_stride, c.weight_stride = 100, 1000, 64, 64, 64
    c.dtype, c.reduction, c.ignore_index, c.temperature = L.BF16, L.LOSS_MEAN, -100, 1.0
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _teacher(**kw):
    c = _linear(target=None, teacher_index=5 * ADDRESS, teacher_logits=6 * ADDRESS, entry_index=7 * ADDRESS, entry_p=8 * ADDRESS,
                entries=8, temperature=2.0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _topk(**kw):
    return _teacher(**{**dict(hidden=None, weight=None, logits=ADDRESS, logits_stride=1000), **kw})


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(jabas_[a-z_]+)\s*\(", text))
    assert names == set(L.LOSS_SIGNATURES)
    for n in names:
        assert hasattr(L.lib(), n)


def test_struct_and_constants_match_the_header(tmp_path):
    fields = [name for name, _ in L.JabasLoss._fields_]
    prints = "".join(f'printf("%zu ", offsetof(JabasLoss, {f}));' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include "jabas_loss.h"\nint main(void) {{ {prints} '
                   'printf("%zu %d %d %d %d", sizeof(JabasLoss), JABAS_LOSS_MAX_ENTRIES, JABAS_LOSS_NONE, JABAS_LOSS_MEAN, JABAS_LOSS_SUM); return 0; }')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    seen = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert seen == [getattr(L.JabasLoss, f).offset for f in fields] + [C.sizeof(L.JabasLoss), L.LOSS_MAX_ENTRIES, L.LOSS_NONE, L.LOSS_MEAN, L.LOSS_SUM]


@pytest.mark.parametrize("make", [_linear, _teacher, _topk])
@pytest.mark.parametrize("dtype", [L.F32, L.BF16])
def test_workspace_is_sized_and_asked_for(make, dtype):
    lib = L.lib()
    for rows in (0, 1, 63, 64, 65, 5000):
        c = make(rows=rows, dtype=dtype)
        sizes = [lib.jabas_loss_workspace_bytes(C.byref(c), b) for b in (0, 1)]
        assert min(sizes) >= 256 and all(n % 256 == 0 for n in sizes)
        # too little, none, or misaligned: refused before any launch
        args = [C.byref(c), ADDRESS]
        assert lib.jabas_loss_forward(*args, None, sizes[0], None) == L.ERR_WORKSPACE
        assert lib.jabas_loss_forward(*args, ADDRESS + 8, sizes[0], None) == L.ERR_WORKSPACE
        if rows:
            assert lib.jabas_loss_forward(*args, ADDRESS, sizes[0] - 256, None) == L.ERR_WORKSPACE
            outs = (None, None, None, ADDRESS) if make is _topk else (ADDRESS, 2 * ADDRESS, None, None)
            assert lib.jabas_loss_backward(*args, *outs, ADDRESS, sizes[1] - 256, None) == L.ERR_WORKSPACE


@pytest.mark.parametrize("dtype", [L.F32, L.BF16])
@pytest.mark.parametrize("rows", [1, 100, 6400, 100000])
def test_backward_workspace_does_not_grow_with_the_vocabulary(dtype, rows):
    def size(vocab):
        c = _linear(rows=rows, vocab=vocab, width=1024, hidden_stride=1024, weight_stride=1024, dtype=dtype)
        return L.lib().jabas_loss_workspace_bytes(C.byref(c), 1)
    logits = rows * (1 << 20) * 4
    assert size(1 << 20) < max(size(1 << 18) * 1.5, logits / 8)
    assert size(1 << 20) < (1 << 30) + 40 * rows * 1024


@pytest.mark.parametrize("make,change,status", [
    (_linear, dict(dtype=2), L.ERR_DTYPE), (_linear, dict(reduction=3), L.ERR_SIZE), (_linear, dict(rows=-1), L.ERR_SIZE),
    (_linear, dict(vocab=0), L.ERR_SIZE), (_linear, dict(width=0), L.ERR_SIZE), (_linear, dict(vocab=1 << 31), L.ERR_SIZE),
    (_linear, dict(rows=1 << 30, vocab=1 << 30), L.ERR_SIZE), (_linear, dict(weight_stride=-1), L.ERR_SIZE),
    (_linear, dict(vocab=(1 << 28) + 1), L.ERR_SIZE), (_linear, dict(rows=(1 << 22) + 1), L.ERR_SIZE), (_linear, dict(rows=1 << 22, vocab=1 << 18), L.ERR_SIZE),
    (_topk, dict(rows=1 << 24, vocab=8), L.ERR_SIZE), (_linear, dict(width=(1 << 20) + 1), L.ERR_SIZE),
    (_linear, dict(weight=None), L.ERR_NULL), (_linear, dict(hidden=None), L.ERR_NULL), (_linear, dict(target=None), L.ERR_NULL),
    (_linear, dict(row_state=None), L.ERR_NULL), (_linear, dict(logits=ADDRESS), L.ERR_NULL),
    (_linear, dict(label_smoothing=1.0), L.ERR_SIZE), (_linear, dict(label_smoothing=-0.1), L.ERR_SIZE),
    (_linear, dict(label_smoothing=float("nan")), L.ERR_SIZE), (_linear, dict(temperature=2.0), L.ERR_SIZE),
    (_linear, dict(teacher_lse=ADDRESS), L.ERR_SIZE), (_linear, dict(hidden=ADDRESS + 1), L.ERR_ALIGN),
    (_linear, dict(row_state=ADDRESS + 4), L.ERR_ALIGN), (_linear, dict(target=ADDRESS + 4), L.ERR_ALIGN),
    (_linear, dict(dtype=L.F32, weight=ADDRESS + 2), L.ERR_ALIGN),
    (_teacher, dict(target=ADDRESS), L.ERR_NULL), (_teacher, dict(teacher_logits=None), L.ERR_NULL), (_teacher, dict(entry_p=None), L.ERR_NULL),
    (_teacher, dict(entries=0), L.ERR_SIZE), (_teacher, dict(entries=256), L.ERR_SIZE), (_teacher, dict(temperature=0.0), L.ERR_SIZE),
    (_teacher, dict(temperature=float("nan")), L.ERR_SIZE), (_teacher, dict(temperature=float("inf")), L.ERR_SIZE),
    (_teacher, dict(label_smoothing=0.1), L.ERR_SIZE), (_teacher, dict(teacher_lse=ADDRESS + 2), L.ERR_ALIGN),
    (_topk, dict(logits=None), L.ERR_NULL), (_topk, dict(bias=ADDRESS), L.ERR_NULL), (_topk, dict(logits_stride=-1), L.ERR_SIZE),
    (_topk, dict(rows=1 << 30, vocab=1 << 20), L.ERR_SIZE), (_topk, dict(teacher_index=None, teacher_logits=None, entries=0, target=ADDRESS, temperature=1.0), L.ERR_NULL)])
def test_malformed_losses_are_refused(make, change, status):
    lib, c = L.lib(), make(**change)
    assert lib.jabas_loss_workspace_bytes(C.byref(c), 0) == 0
    assert lib.jabas_loss_forward(C.byref(c), ADDRESS, ADDRESS, 1 << 40, None) == status
    assert lib.jabas_loss_backward(C.byref(c), ADDRESS, None, None, None, None, ADDRESS, 1 << 40, None) == status


def test_missing_results_are_refused():
    lib = L.lib()
    assert lib.jabas_loss_forward(None, ADDRESS, ADDRESS, 1 << 40, None) == L.ERR_NULL
    assert lib.jabas_loss_forward(C.byref(_linear()), None, ADDRESS, 1 << 40, None) == L.ERR_NULL
    big = (ADDRESS, 1 << 40, None)
    assert lib.jabas_loss_backward(C.byref(_linear()), None, ADDRESS, None, None, None, *big) == L.ERR_NULL
    assert lib.jabas_loss_backward(C.byref(_linear()), ADDRESS, None, None, None, ADDRESS, *big) == L.ERR_NULL      # no logits
    assert lib.jabas_loss_backward(C.byref(_linear()), ADDRESS, None, None, ADDRESS, None, *big) == L.ERR_NULL      # no bias
    assert lib.jabas_loss_backward(C.byref(_topk()), ADDRESS, ADDRESS, None, None, None, *big) == L.ERR_NULL
    assert lib.jabas_loss_backward(C.byref(_linear()), ADDRESS, ADDRESS + 1, None, None, None, *big) == L.ERR_ALIGN


def test_there_is_no_cpu_path():
    x, w, t = torch.randn(4, 8), torch.randn(16, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        losses.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="GPU"):
        losses.topk_distillation(torch.randn(4, 16), t[:, None], torch.zeros(4, 1))
    with pytest.raises(ValueError, match="GPU"):
        losses.linear_topk_distillation(x, w, t[:, None], torch.zeros(4, 1))
