"""examples/train_and_distil.py: the losses as trainer's criteria on K virtual stream workers, and their gradients against plain ones'."""
import importlib.util
import os

import pytest
import torch

from jabas_amd import loss as losses

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("train_and_distil", os.path.join(ROOT, "examples", "train_and_distil.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_teacher_and_student_learn(gpu, dtype):
    r = _example().main(["--vocab", "503", "--length", "9", "--steps", "40", "--workers", "12", "8", "--entries", "8", "--dtype", dtype])
    assert r["teacher"][1] < 0.6 * r["teacher"][0] and r["student"][1] < 0.6 * r["student"][0]
    assert r["teacher score"] < 0.5 * torch.tensor(503.0).log()
    # logits in hand are rounded to their type: 2^-8 of the largest for bfloat16, T^2 = 4 times over
    assert r["in hand"] == pytest.approx(r["linear"], rel=0.05 if dtype == "bf16" else 1e-4, abs=1e-3)


def test_workers_train_as_with_the_plain_loss(gpu):
    """The same two workers, three steps, with the criterion here and with torch's cross entropy over kept logits in 32 bits."""
    ex = _example()
    mapping = torch.randperm(300, generator=torch.Generator().manual_seed(2))
    mapping[mapping == 0], mapping[0] = mapping[0].clone(), 0
    work = ex.batches((6, 4), 11, mapping, gpu, torch.Generator().manual_seed(3))

    def plain(output, target):
        hidden, weight, bias = output
        return torch.nn.functional.cross_entropy((hidden @ weight.t() + bias).flatten(0, 1), target.flatten(), ignore_index=0, label_smoothing=0.1)

    ends = []
    for criterion in (losses.LinearCrossEntropy(ignore_index=0, label_smoothing=0.1), plain):
        torch.manual_seed(5)
        model = ex.Translator(300, 64, torch.float32)
        first, last, model = ex.train(model, criterion, 3, (6, 4), lambda step: work, gpu, 1e-3)
        ends.append((first, last, [p.detach().clone() for p in model.parameters()]))
    (a0, a1, pa), (b0, b1, pb) = ends
    assert a0 == pytest.approx(b0, rel=1e-5) and a1 == pytest.approx(b1, rel=1e-3)
    # Adam divides a gradient by its own size: where it is rounding noise a weight may move the other way, by 2 lr a step at most
    for p, q in zip(pa, pb):
        off = (p - q).abs()
        assert float(off.max()) <= 6.1e-3 and float((off > 1e-5).float().mean()) < 0.02
