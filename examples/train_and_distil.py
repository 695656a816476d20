"""Training with the losses over a large vocabulary, end to end on one GPU:

1. a teacher learns a toy translation by cross entropy with label smoothing and padding, on K virtual stream workers
   (``VSWSyncTrainer``, criterion ``LinearCrossEntropy``);
2. its top logits and their true normaliser are recorded for every target token;
3. a narrower student learns from them alone (criterion ``LinearTopkDistillation``);
4. both are scored token by token without gradients (``linear_cross_entropy(..., reduction="none")``), and the student's
   divergence from the teacher is taken once more from logits in hand (``topk_distillation``).

A model's forward returns its last hidden states with its classifier's weight and bias, and the criterion does the rest: no
pass keeps [tokens, vocabulary] logits. Data is synthetic: a fixed relabelling of random source sentences.

    python examples/train_and_distil.py [--vocab 32317] [--steps 60]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from jabas_amd import loss as losses                  # noqa: E402
from jabas_amd.train import VSWSyncTrainer            # noqa: E402

PAD = 0


class Translator(torch.nn.Module):
    """Source tokens to hidden states, token by token; ``dtype``: what the classifier's product and loss run in."""

    def __init__(self, vocab, width, dtype):
        super().__init__()
        self.dtype = dtype
        self.embed = torch.nn.Embedding(vocab, width, padding_idx=PAD)
        self.body = torch.nn.Sequential(torch.nn.Linear(width, 2 * width), torch.nn.GELU(), torch.nn.Linear(2 * width, width))
        self.norm = torch.nn.LayerNorm(width)
        self.classifier = torch.nn.Linear(width, vocab)
        torch.nn.init.normal_(self.classifier.weight, std=0.1 * width ** -0.5)

    def forward(self, source):
        x = self.embed(source)
        hidden = self.norm(x + self.body(x))
        return tuple(t.to(self.dtype) for t in (hidden, self.classifier.weight, self.classifier.bias))


def batches(sizes, length, mapping, device, gen):
    """A (source, target) pair per worker: sentences of different lengths, padded."""
    out = []
    for size in sizes:
        source = torch.randint(1, len(mapping), (size, length), generator=gen)
        ends = torch.randint(length // 2, length + 1, (size, 1), generator=gen)
        source[torch.arange(length) >= ends] = PAD
        out.append((source.to(device), mapping[source].to(device)))
    return out


@torch.no_grad()
def top_logits(model, source, k, temperature):
    """The teacher's k top logits per token and its logsumexp(logits / T); padding holds no entry."""
    hidden, weight, bias = model(source)
    logits = hidden @ weight.t() + bias
    top, index = logits.topk(k, dim=-1)
    index[source == PAD] = -1
    return index, top, torch.logsumexp(logits.float() / temperature, -1)


def train(model, criterion, steps, sizes, data, device, lr):
    """Adam over K workers; ``data(step)`` gives a pair per worker. Returns the first and the last step's mean loss."""
    opt = dict(kind="adam", betas=(0.9, 0.999), eps=1e-8, groups=[dict(lr=lr, weight_decay=0.0)])
    trainer = VSWSyncTrainer(device, sizes, opt)
    trainer.prepare_stream_parallel(model, criterion)
    first = last = None
    for step in range(steps):
        last = trainer.compute(data(step))
        trainer.step()
        first = first or [float(x) for x in last]
    mean = lambda v: sum(float(x) for x in v) / len(v)
    return mean(first), mean(last), trainer.main_model


def main(argv=None):
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--vocab", type=int, default=4001)
    a.add_argument("--length", type=int, default=25)
    a.add_argument("--steps", type=int, default=60)
    a.add_argument("--entries", type=int, default=16)
    a.add_argument("--temperature", type=float, default=2.0)
    a.add_argument("--workers", type=int, nargs="+", default=[48, 32, 16], help="sentences of each virtual stream worker")
    a.add_argument("--dtype", choices=["fp32", "bf16"], default="bf16")
    a = a.parse_args(argv)
    device, dtype = torch.device("cuda:0"), {"fp32": torch.float32, "bf16": torch.bfloat16}[a.dtype]
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(1)
    mapping = torch.cat([torch.zeros(1, dtype=torch.int64), torch.randperm(a.vocab - 1, generator=gen) + 1])
    corpus = [batches(a.workers, a.length, mapping, device, gen) for _ in range(8)]     # seen again and again
    tasks = lambda step: corpus[step % len(corpus)]
    results = {}

    criterion = losses.LinearCrossEntropy(ignore_index=PAD, label_smoothing=0.1)
    first, last, teacher = train(Translator(a.vocab, 256, dtype), criterion, a.steps, a.workers, tasks, device, 2e-3)
    results["teacher"] = first, last
    print(f"teacher: loss {first:.3f} -> {last:.3f}", flush=True)

    recorded = [[(x, top_logits(teacher, x, a.entries, a.temperature)) for x, _ in work] for work in corpus]
    criterion = losses.LinearTopkDistillation(temperature=a.temperature)
    first, last, student = train(Translator(a.vocab, 128, dtype), criterion, a.steps, a.workers, lambda step: recorded[step % len(corpus)], device, 2e-3)
    results["student"] = first, last
    print(f"student: divergence from the teacher {first:.3f} -> {last:.3f}", flush=True)

    with torch.no_grad():
        (source, target), (_, (index, top, lse)) = corpus[0][0], recorded[0][0]
        for name, model in (("teacher", teacher), ("student", student)):
            hidden, weight, bias = model(source)
            scores = losses.linear_cross_entropy(hidden, weight, target, bias, ignore_index=PAD, reduction="none")
            results[f"{name} score"] = float(scores.sum() / (target != PAD).sum())
            print(f"{name}: {results[f'{name} score']:.3f} nats per token; best sentence {int(scores.sum(1).argmin())}", flush=True)
        logits = hidden @ weight.t() + bias
        in_hand = losses.topk_distillation(logits, index, top, temperature=a.temperature, teacher_lse=lse)
        linear = losses.linear_topk_distillation(hidden, weight, index, top, bias, temperature=a.temperature, teacher_lse=lse)
        results["in hand"], results["linear"] = float(in_hand), float(linear)
        print(f"student against teacher: {float(linear):.4f} from hidden states, {float(in_hand):.4f} from logits in hand", flush=True)
    return results


if __name__ == "__main__":
    main()
