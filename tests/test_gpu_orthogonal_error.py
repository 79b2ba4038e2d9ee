"""``mp.orthogonalise`` on the GPU within the error of pairs of halves: in norm, and of every entry, so that no part of a
matrix is left out."""

from __future__ import annotations

import pytest
import torch

from .orthogonal_error import orthogonalised
from .test_gpu_orthogonal import DEV, DTYPES, SHAPES, UNIT, _gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def _check(got, update, **kw) -> None:
    want, allowed = orthogonalised(update, **kw)
    off, unit = (got.double() - want).abs(), UNIT[got.dtype]
    assert float((off - unit * want.abs()).clamp_min(0).norm()) <= allowed
    assert bool((off <= unit * want.abs() + allowed).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_within_the_error_of_pairs(shape, dtype) -> None:
    from relmo_amd import mp

    update = torch.randn(*shape, device=DEV, generator=_gen(sum(shape) + 1)).mul_(3e-3).to(dtype)
    _check(mp.orthogonalise(update), update)


@pytest.mark.parametrize("shape", [(48, 80), (300, 200)])
def test_within_the_error_of_pairs_far_apart_and_with_other_rules(shape) -> None:
    from relmo_amd import mp

    g = _gen(14)
    side = min(shape)
    u, v = (torch.linalg.qr(torch.randn(n, side, device=DEV, generator=g, dtype=torch.float64))[0] for n in shape)
    for values in (torch.logspace(0, -3, side, device=DEV, dtype=torch.float64), (torch.arange(side, device=DEV) < 3).double()):
        update = (u * values @ v.t()).float()
        _check(mp.orthogonalise(update), update)
        for steps, coefficients in ((1, (3.4445, -4.7750, 2.0315)), (9, (3.4445, -4.7750, 2.0315)), (6, (1.5, -0.5, 0.0))):
            _check(mp.orthogonalise(update, steps=steps, coefficients=coefficients), update, steps=steps, coefficients=coefficients)


def test_lists_within_the_error_of_pairs() -> None:
    from relmo_amd import mp

    g = _gen(15)
    updates = [torch.randn(*s, device=DEV, generator=g) for s in SHAPES[:-1]]
    for got, update in zip(mp.orthogonalise(updates), updates):
        _check(got, update)
