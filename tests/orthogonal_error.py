"""How far an orthogonalised update may be off: its iteration in 64 bits beside the same with the kernels' roundings
as noise.

Iterates are pairs of halves: a value errs by up to 2^-22 of itself and half the halves' smallest spacing, 2^-25, in
units of its plane's scale.  A product of pairs leaves out lo lo, 2^-22 of a term, and adds 3 depth / 32 times in float:
sums of terms of either sign, whose errors grow with the root of their number.  Noise of these sizes (uniform up to
them, drawn anew for every entry) goes through the iteration; an entry's error is a sum of very many, so the norm of the
difference hardly varies, and eight times the largest of four draws is allowed.  Values of 11 bits in the place of 22
err 2^11 times as much."""

from __future__ import annotations

import math

import torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
PAIR = 2.0 ** -22


def scale_of(m: int, n: int) -> float:
    return 2.0 ** min(round(0.5 * math.log2(m * n)), 13)


def _iterate(x, steps, coefficients, scale, noise):
    """``noise(value, size)``: the value with an error of up to ``size``."""

    a, b, c = coefficients

    def held(value, unit):
        return noise(value, PAIR * value.abs() + 2.0 ** -25 / unit)

    def product(p, q):
        exact = p @ q
        walk = (p.square() @ q.square()).sqrt()
        return noise(exact, PAIR * walk + 2.0 ** -24 * math.sqrt(3 * p.size(1) / 32 + 1) * (walk + exact.abs()))

    x = held(x, scale)
    for _ in range(steps):
        turned = x.t().contiguous()
        gram = held(product(x, turned), 4096.0)
        poly = held(b * gram + c * product(gram, gram), 4096.0)
        x = held(a * x + product(poly, x), scale)
    return x


def orthogonalised(update, steps: int = 5, coefficients=COEFFICIENTS, eps: float = EPS):
    """The result in 64 bits and the norm of the error that the kernels may leave on it."""

    x = update.double()
    tall = x.size(0) > x.size(1)
    x = x.t().contiguous() if tall else x
    scale = scale_of(*x.shape)
    x = x / (x.norm() + eps)
    want = _iterate(x, steps, coefficients, scale, lambda value, size: value)
    g = torch.Generator(device=x.device)
    g.manual_seed(0)
    worst = 0.0
    for _ in range(4):
        noisy = _iterate(x, steps, coefficients, scale, lambda value, size: value + size * (
            2 * torch.rand(value.shape, generator=g, device=value.device, dtype=torch.float64) - 1))
        worst = max(worst, float((noisy - want).norm()))
    return (want.t() if tall else want), 8 * worst + PAIR * float(want.norm())
