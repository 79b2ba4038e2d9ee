"""The orthogonalised update's tolerance tells pairs of halves from single ones (simulated on the CPU)."""

from __future__ import annotations

import pytest
import torch

from .orthogonal_error import COEFFICIENTS, EPS, orthogonalised, scale_of


def _simulated(update, halves: int, steps: int = 5):
    """The iteration with every iterate held as one half or a pair, at the kernels' scales, products in 64 bits."""

    def held(x, scale):
        hi = (x * scale).half().double()
        lo = (x * scale - hi).half().double() if halves == 2 else torch.zeros_like(hi)
        return hi / scale, lo / scale

    def product(p, q):
        return p[0] @ q[0] + p[0] @ q[1] + p[1] @ q[0]

    a, b, c = COEFFICIENTS
    x = update.double()
    x = x / (x.norm() + EPS)
    scale = scale_of(*x.shape)
    x = held(x, scale)
    for _ in range(steps):
        gram = held(product(x, (x[0].t(), x[1].t())), 4096.0)
        poly = held(b * (gram[0] + gram[1]) + c * product(gram, gram), 4096.0)
        x = held(a * (x[0] + x[1]) + product(poly, x), scale)
    return x[0] + x[1]


@pytest.mark.parametrize("shape", [(32, 32), (96, 96), (31, 300), (129, 129), (260, 398)])
def test_one_half_in_the_place_of_two_is_outside(shape) -> None:
    update = torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))) * 1e-2
    want, allowed = orthogonalised(update)
    pair = float((_simulated(update, 2) - want).norm())
    single = float((_simulated(update, 1) - want).norm())
    assert pair <= 0.25 * allowed and single >= 4 * allowed, (pair, single, allowed)


@pytest.mark.parametrize("shape", [(96, 96), (260, 398)])
def test_a_missing_tile_is_outside(shape) -> None:
    """Entries of any tile are far past the error allowed to all of them together."""

    update = torch.randn(*shape, generator=torch.Generator().manual_seed(1))
    want, allowed = orthogonalised(update)
    assert float(want[:16, :16].abs().max()) > 4 * allowed
    assert allowed < 0.01 * float(want.abs().max())
