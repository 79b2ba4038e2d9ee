"""GPU tests of ``mp.orthogonalise`` against its definition in 64 bits.

Tolerance.  The iterates are held to 2^-22 of an entry (or 2^-25 of the matrix's scale) and a product of depth n adds
up to 6 sqrt(n) 2^-24 of its terms' magnitudes; a step multiplies what is wrong with a direction whose singular value is
small by at most a + |b| + |c| <= 10.3, and by its slope (at most a = 3.45 in magnitude over [0, 1.25]) otherwise, so
over `steps` steps an error of the norm |X|_F grows to at most sum of 3.45^k.  The sums are taken relative to the norm
of the result, whose singular values are about 1 but for those that start below 3.45^-steps; the 64-bit result's norm
is at least that of its largest value, 0.6."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]

# one value, vectors, sides off 16 and 32, the widest in one workgroup and the first past it, both tile sizes
SHAPES = [(1, 1), (1, 300), (7, 5), (16, 16), (31, 33), (32, 32), (96, 96), (64, 192), (128, 100), (128, 128), (97, 300),
          (33, 1000), (129, 129), (140, 20), (398, 11), (398, 387), (384, 398), (700, 65), (257, 1030), (64, 4000), (2000, 1500)]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _definition(update, steps=5, coefficients=COEFFICIENTS, eps=EPS):
    a, b, c = coefficients
    x = update.double()
    x = x / (x.square().sum().sqrt() + eps)
    left = x.size(0) <= x.size(1)
    for _ in range(steps):
        gram = x @ x.t().contiguous() if left else x.t().contiguous() @ x
        poly = b * gram + c * gram @ gram
        x = a * x + (poly @ x if left else x @ poly)
    return x


def _allowed(shape, steps=5) -> float:
    """Error of the result in units of its norm, before its own rounding."""

    grown = sum(3.45 ** k for k in range(steps + 1))
    return grown * (2.0 ** -22 + 6 * max(shape) ** 0.5 * 2.0 ** -24)


def _check(got, update, **kw) -> None:
    want = _definition(update, **kw)
    assert got.shape == update.shape and got.dtype == update.dtype
    norm = float(want.norm())
    err = float((got.double() - want).norm()) / norm
    assert err <= UNIT[got.dtype] + _allowed(update.shape, kw.get("steps", 5)), err
    # entry by entry: no part of the matrix is left out (a norm would hide a tile)
    worst = float((got.double() - want).abs().max())
    assert worst <= (UNIT[got.dtype] + _allowed(update.shape, kw.get("steps", 5))) * max(norm, 1.0), worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(shape, dtype) -> None:
    from relmo_amd import mp

    update = torch.randn(*shape, device=DEV, generator=_gen(sum(shape))).mul_(1e-2).to(dtype)
    got = mp.orthogonalise(update)
    _check(got, update)
    assert torch.equal(got, mp.orthogonalise(update))
    _check(mp.orthogonalise(update.t()), update.t())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(48, 80), (300, 200)])
def test_singular_values_far_apart_and_low_rank(shape, dtype) -> None:
    from relmo_amd import mp

    g = _gen(4)
    side = min(shape)
    u, v = (torch.linalg.qr(torch.randn(n, side, device=DEV, generator=g, dtype=torch.float64))[0] for n in shape)
    for values in (torch.logspace(0, -3, side, device=DEV, dtype=torch.float64),
                   (torch.arange(side, device=DEV) < 3).double()):
        _check(mp.orthogonalise((u * values @ v.t()).to(dtype)), (u * values @ v.t()).to(dtype))


@pytest.mark.parametrize("shape", [(40, 60), (200, 300)])
def test_result_is_nearly_orthogonal(shape) -> None:
    from relmo_amd import mp

    update = torch.randn(*shape, device=DEV, generator=_gen(2))
    values = torch.linalg.svdvals(mp.orthogonalise(update, steps=8).double())
    assert 0.6 < float(values.min()) and float(values.max()) < 1.3


def test_lists_of_many_shapes_equal_single_calls() -> None:
    from relmo_amd import mp

    g = _gen(7)
    shapes = SHAPES[:-1] + [(n, 2 * n) for n in range(1, 45)] + [(130 + n, 140) for n in range(35)]
    updates = [torch.randn(*s, device=DEV, generator=g) for s in shapes]
    for got, u in zip(mp.orthogonalise(updates), updates):
        # tiles go by the launch's matrices: equal up to the sums' order
        alone = mp.orthogonalise(u)
        assert float((got - alone).norm()) <= 2 * _allowed(u.shape) * float(alone.norm())


def test_small_matrices_beside_a_large_one() -> None:
    """They go through the tiles of the large one's launches, stay apart from it, and come out as alone up to the
    sums' order."""
    from relmo_amd import mp

    g = _gen(11)
    shapes = [(398, 387), (398, 11), (1, 1), (5, 300), (128, 128), (31, 33), (96, 96)]
    updates = [torch.randn(*s, device=DEV, generator=g) for s in shapes]
    for got, u in zip(mp.orthogonalise(updates), updates):
        _check(got, u)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e15, 3e30])
def test_any_magnitude(scale: float) -> None:
    """The norm is added in double: squares neither vanish nor overflow.  eps is 1e-7: tiny updates stay small."""
    from relmo_amd import mp

    for shape in ((50, 70), (300, 200)):
        update = torch.randn(*shape, device=DEV, generator=_gen(1)) * scale
        got, want = mp.orthogonalise(update), _definition(update)
        assert bool(got.isfinite().all())
        # below the pairs' range (2^-25 of the scale of about 2^5 to 2^8) an entry is lost, five steps grow what is left
        lost = 3.45 ** 5 * 2.0 ** -25 * max(shape) ** 0.5
        assert float((got.double() - want).norm()) <= _allowed(shape) * float(want.norm()) + lost


def test_zero_nan_and_infinite_updates_stay_apart() -> None:
    from relmo_amd import mp

    for shape in ((40, 64), (200, 140)):
        clean = torch.randn(*shape, device=DEV, generator=_gen(3))
        spoilt = clean.clone()
        spoilt[3, 7] = float("nan")
        inf = clean.clone()
        inf[0, 0] = float("inf")
        got = mp.orthogonalise([clean, torch.zeros_like(clean), spoilt, inf, clean])
        assert torch.equal(got[0], got[4]) and torch.equal(got[0], mp.orthogonalise([clean] * 5)[0])
        assert float(got[1].abs().sum()) == 0
        assert bool(got[2].isnan().all()) and bool(got[3].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_stacks_and_empty(dtype) -> None:
    from relmo_amd import mp

    base = torch.randn(6, 100, 150, device=DEV, generator=_gen(5)).to(dtype)
    stack = mp.orthogonalise(base[:, :90, 10:])
    for i in range(6):
        assert torch.equal(stack[i], mp.orthogonalise(base[i, :90, 10:].contiguous()))
        assert torch.equal(stack[i], mp.orthogonalise(base[i, :90, 10:]))       # rows apart
    every = base[0, ::2, ::3]
    assert torch.equal(mp.orthogonalise(every), mp.orthogonalise(every.contiguous()))
    assert mp.orthogonalise([]) == []
    assert mp.orthogonalise(base[:0]).shape == (0, 100, 150) and mp.orthogonalise(base[0, :0]).shape == (0, 150)


@pytest.mark.parametrize("shape", [(48, 48), (260, 150)])
def test_steps_and_other_coefficients(shape) -> None:
    from relmo_amd import mp

    update = torch.randn(*shape, device=DEV, generator=_gen(6))
    for steps in (1, 2, 3, 9):
        _check(mp.orthogonalise(update, steps=steps), update, steps=steps)
    cubic = (1.5, -0.5, 0.0)
    _check(mp.orthogonalise(update, steps=6, coefficients=cubic), update, steps=6, coefficients=cubic)


def test_runs_on_the_current_stream() -> None:
    from relmo_amd import mp

    update = torch.randn(400, 500, device=DEV, generator=_gen(8))
    want = mp.orthogonalise([update, update[:64, :64]])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        moved = (update * 4).mul_(0.25)
        got = mp.orthogonalise([moved, moved[:64, :64]])
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_refusals() -> None:
    from relmo_amd import capi, mp

    x = torch.ones(4, 8, device=DEV)
    with pytest.raises(ValueError, match="matrices"):
        mp.orthogonalise(x[0])
    with pytest.raises(ValueError, match="one dtype"):
        mp.orthogonalise([x, x.bfloat16()])
    with pytest.raises(ValueError, match="three"):
        mp.orthogonalise(x, coefficients=(1.5, -0.5))
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        mp.orthogonalise(x.double())
    for steps in (0, -1, 65, 1 << 40):
        with pytest.raises(RuntimeError, match="steps"):
            mp.orthogonalise(x, steps=steps)
    for eps in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="eps"):
            mp.orthogonalise(x, eps=eps)
    for coefficients in ((4.0, 0.0, 0.0), (float("nan"), 0.0, 0.0), (1.0, float("inf"), 0.0)):
        with pytest.raises(RuntimeError, match="past 2"):
            mp.orthogonalise(x, coefficients=coefficients)
    u = (capi.Update * 1)(capi.Update(x.data_ptr(), x.data_ptr(), 200, 300, 300))
    rc = capi.lib().relm_mp_orthogonalise(capi.F32, u, 1, 5, 1.5, -0.5, 0.0, 1e-7, None, 0, capi._stream(x))
    assert rc == capi.ERR_WORKSPACE
    u[0].row_stride = 299
    rc = capi.lib().relm_mp_orthogonalise(capi.F32, u, 1, 5, 1.5, -0.5, 0.0, 1e-7, None, 0, capi._stream(x))
    assert rc == capi.ERR_INVALID_ARGUMENT and "overlap" in capi.last_error()
