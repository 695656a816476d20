"""The orthogonalised update in 64 bits (on the CPU, large ones elsewhere), from its definition, and how far roundings of its factors carry."""
import math

import torch

COEFFICIENTS = (3.4445, -4.775, 2.0315)


def _rounded(x, bits, gen):
    """x off by up to half a step of `bits` bits, evenly: what a factor of so many bits is."""
    if bits is None:
        return x
    return x * (1.0 + (2.0 * torch.rand(x.shape, generator=gen, dtype=x.dtype, device=x.device) - 1.0) * 2.0 ** -bits)


def newton_schulz(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7, factor_bits=None, own_bits=None, seed=0, device="cpu"):
    """g (..., rows, cols). ``factor_bits``: of the products' factors; ``own_bits``: of the running matrix itself."""
    if g.shape[-2] > g.shape[-1]:
        return newton_schulz(g.transpose(-1, -2), steps, coefficients, eps, factor_bits, own_bits, seed, device).transpose(-1, -2)
    gen = torch.Generator(device).manual_seed(seed)
    a, b, c = coefficients
    x = g.detach().to(device).double()
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    for _ in range(steps):
        x = _rounded(x, own_bits, gen)
        f = _rounded(x, factor_bits, gen)
        A = _rounded(f @ f.transpose(-1, -2), factor_bits, gen)
        B = _rounded(b * A + c * (A @ A), factor_bits, gen)
        x = a * x + B @ f
    return x


def off_by(x, y):
    """Length of the difference over the length of y."""
    x, y = x.detach().to(y.device).double(), y.detach().double()
    length = float(y.norm())
    return float((x - y).norm()) / length if length else float((x - y).norm())


def allowed(g, bf16, **kw):
    """How far a kernel may be off: 8 times what evenly random roundings to the documented bits carry (float32: 22 bits, bfloat16: 11 of
    the factors, 22 of the running matrix; two random draws, the larger), and half a step of bfloat16 or two of float32 for the result."""
    e = newton_schulz(g, **kw)
    bits = dict(factor_bits=11 if bf16 else 21, own_bits=21)
    far = max(off_by(newton_schulz(g, seed=s, **bits, **kw), e) for s in (1, 2))
    return 8.0 * far + (2.0 ** -8 if bf16 else 2.0 ** -23), e


def lr_factor(how, rows, cols):
    return math.sqrt(max(1.0, rows / cols)) if how in (None, "original") else 0.2 * math.sqrt(max(rows, cols))


def muon_step(p, g, buf, lr, weight_decay, momentum=0.95, nesterov=True, adjust=None, **kw):
    """New weights and momentum of one matrix, and how far off the weights may be (elementwise, in units of their own)."""
    p, g, buf = (t.detach().cpu().double() for t in (p, g, buf))
    shape = p.shape
    rows, cols = shape[0], p.numel() // shape[0]
    bf16 = kw.pop("bf16", False)
    buf = buf + (1.0 - momentum) * (g - buf)
    u = (g + momentum * (buf - g) if nesterov else buf).reshape(rows, cols)
    far, o = allowed(u, bf16, **kw)
    rate = lr * lr_factor(adjust, rows, cols)
    new = p * (1.0 - lr * weight_decay) - rate * o.reshape(shape)
    return new, buf, rate * far * float(o.norm()) + 2.0 ** -22 * float(p.norm())


def adamw_step(p, g, m, v, step, lr, weight_decay, betas=(0.9, 0.999), eps=1e-8):
    p, g, m, v = (t.detach().cpu().double() for t in (p, g, m, v))
    m = betas[0] * m + (1.0 - betas[0]) * g
    v = betas[1] * v + (1.0 - betas[1]) * g * g
    new = p * (1.0 - lr * weight_decay) - lr * (m / (1.0 - betas[0] ** step)) / ((v / (1.0 - betas[1] ** step)).sqrt() + eps)
    return new, m, v
