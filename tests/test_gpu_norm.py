"""GPU tests of the residual norm (``mp.add_rms_norm``, ``mp.rms_norm``, ``mp.add_rms_norm_fp8``) against its
definition in 64 bits.

Tolerances.  u is the unit roundoff: 2^-24 in float32, 2^-8 and 2^-11 where a result is stored in bfloat16 and
float16.  A pass adds at most max(32, width / 256) squares in a lane one after the other and the lanes' sums in a
tree, whose relative error the root halves; with the other roundings of y that is CHAIN(width) units of 2^-24,
relative.  The backward's sums have terms of both signs: their error counts in units of the sum of magnitudes.
A 16-bit h is rounded before the backward reads it, which moves n by one unit of its type."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = 1e-6
U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # spacing of subnormals
DTYPES = [torch.float32, torch.bfloat16, torch.float16]

# every number of lanes and units of a row, rows that are no whole units, rows of odd 16-bit widths (one value at
# a time), rows that are walked; one row and more rows than one round of workgroups holds
SIZES = [(1, 1), (3, 7), (200, 128), (65, 33), (5, 398), (1025, 32), (9000, 24), (70, 256), (3, 511), (7, 1030), (2, 2050),
         (4, 4097), (3, 8192), (2, 9001), (70, 20000), (300_000, 8)]


def chain(width: int) -> float:
    return 16 + max(32, width / 256) / 2 + 6


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def _inputs(rows: int, width: int, dtype, seed: int = 0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed + rows * 31 + width)
    make = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    return [t.to(dtype) for t in (make(rows, width), 2 * make(rows, width), 1 + 0.2 * make(width), make(rows, width),
                                  make(rows, width))]


def _definition(x, r, w):
    h = x.double() if r is None else x.double() + r.double()
    rstd = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return h * rstd * w.double(), h, rstd


def _close(got, want, tol) -> None:
    assert got.shape == want.shape
    over = (got.double() - want).abs() - tol
    assert bool((over <= 0).all()), float(over.max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", SIZES)
def test_forward_and_backward_against_64_bits(rows: int, width: int, dtype) -> None:
    from relmo_amd import mp

    x, r, w, gy, gh = _inputs(rows, width, dtype)
    u, tiny = UNIT[dtype], TINY[dtype]
    x.requires_grad_(True), r.requires_grad_(True), w.requires_grad_(True)
    y, h = mp.add_rms_norm(x, r, w, eps=EPS)
    gx, gr, gw = torch.autograd.grad((y, h), (x, r, w), (gy, gh))
    with torch.no_grad():
        y2, h2 = mp.add_rms_norm(x, r, w, eps=EPS)  # the same kernel without the backward's rstd
        assert torch.equal(y, y2) and torch.equal(h, h2)
        want, h64, rstd = _definition(x, r, w)
        _close(h, h64, (u + U32) * h64.abs() + tiny)
        _close(y, want, (u + chain(width) * U32) * want.abs() + tiny)
        n = h64 * rstd
        dn = gy.double() * w.double()
        mean_abs = (dn * n).abs().mean(-1, keepdim=True)
        dx = rstd * (dn - n * (dn * n).mean(-1, keepdim=True)) + gh.double()
        spread = rstd * (dn.abs() + n.abs() * mean_abs) + gh.double().abs()
        moved = (0 if dtype == torch.float32 else u) * rstd * n.abs() * 2 * mean_abs
        _close(gx, dx, u * dx.abs() + 2 * chain(width) * U32 * spread + moved + tiny)
        assert torch.equal(gx, gr)
        terms = gy.double() * n
        # a lane's rows one after the other (its share of at least 1024 workgroups' rows), the groups, the blocks
        rows_chain = rows / 1024 + 64 + 32 + 64 + 16 + chain(width)
        scale = terms.abs().sum(0)
        _close(gw, terms.sum(0), u * terms.sum(0).abs() + (rows_chain * U32 + (0 if dtype == torch.float32 else u)) * scale + tiny)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_residual_and_with_one_gradient(dtype) -> None:
    from relmo_amd import mp

    x, r, w, gy, gh = _inputs(37, 100, dtype)
    u = UNIT[dtype]
    y = mp.rms_norm(x, w, eps=EPS)
    want, h64, rstd = _definition(x, None, w)
    _close(y, want, (u + chain(100) * U32) * want.abs())
    y2, h2 = mp.add_rms_norm(x, None, w, eps=EPS)
    assert torch.equal(y, y2) and h2 is x
    x.requires_grad_(True)
    n = h64 * rstd
    dn = gy.double() * w.double()
    dx = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    spread = rstd * (dn.abs() + n.abs() * (dn * n).abs().mean(-1, keepdim=True))
    (gx,) = torch.autograd.grad(mp.rms_norm(x, w, eps=EPS), x, gy)
    _close(gx, dx, u * dx.abs() + 2 * chain(100) * U32 * spread)
    # the gradient of one output only
    r.requires_grad_(True)
    y, h = mp.add_rms_norm(x, r, w, eps=EPS)
    only_h = torch.autograd.grad(h, (x, r), gh, retain_graph=True)
    assert torch.equal(only_h[0], gh) and torch.equal(only_h[1], gh)
    only_y = torch.autograd.grad(y, (x, r), gy, retain_graph=True)
    both = torch.autograd.grad((y, h), (x, r), (gy, torch.zeros_like(gh)))
    assert torch.equal(only_y[0], both[0]) and torch.equal(only_y[1], both[1])


def test_gradient_against_differences() -> None:
    """The gradient's inner product with a direction, against the central difference of the 64-bit loss along it:
    the difference's own error is step^2 (1e-8) times third derivatives of order 1, the gradient's float32."""
    from relmo_amd import mp

    x, r, w, gy, gh = _inputs(19, 77, torch.float32)
    for t in (x, r, w):
        t.requires_grad_(True)
    grads = torch.autograd.grad(mp.add_rms_norm(x, r, w, eps=EPS), (x, r, w), (gy, gh))
    with torch.no_grad():
        g = torch.Generator(device=DEV)
        g.manual_seed(5)
        for i, (t, gt) in enumerate(zip((x, r, w), grads)):
            d = torch.randn(t.shape, device=DEV, generator=g, dtype=torch.float64)

            def loss(s):
                args = [a.double() for a in (x, r, w)]
                args[i] = args[i] + s * d
                y, h, _ = _definition(*args)
                return (y * gy.double()).sum() + (h * gh.double()).sum()

            want = (loss(1e-4) - loss(-1e-4)) / 2e-4
            got = (gt.double() * d).sum()
            assert abs(float(got - want)) <= 1e-6 * float((gt.double() * d).abs().sum()), i


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", SIZES)
def test_fp8_output(rows: int, width: int, dtype) -> None:
    from relmo_amd import mp

    x, r, w, _, _ = _inputs(rows, width, dtype)
    if rows > 1:
        x[1] = 0
        r[1] = 0
    q, scale, h = mp.add_rms_norm_fp8(x, r, w, eps=EPS)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == x.shape[:1]
    want, h64, _ = _definition(x, r, w)
    _close(h, h64, (UNIT[dtype] + U32) * h64.abs() + TINY[dtype])
    most = want.abs().amax(1)
    want_scale = torch.where(most == 0, 1.0, most / 448)
    _close(scale, want_scale, (chain(width) + 2) * U32 * want_scale)
    value = q.double() * scale.double().unsqueeze(1)
    # e4m3 keeps 4 significant bits (half a unit: 2^-4 relative), its subnormals are 2^-9 apart
    _close(value, want, (2.0 ** -4 + 2 * chain(width) * U32) * want.abs() + 2.0 ** -10 * want_scale.unsqueeze(1))
    at = q.double().abs().amax(1)
    assert bool(((at == 448) | (most == 0)).all())


def test_fp8_rows_too_small_for_a_scale() -> None:
    from relmo_amd import mp

    # y = x / sqrt(eps) * w: about 1e-44, whose 448th is no float; and subnormal scales
    x = torch.full((2, 16), 1e-30, device=DEV)
    w = torch.ones(16, device=DEV) * 1e-17
    x[1] *= 1e3
    q, scale, _ = mp.add_rms_norm_fp8(x, None, w, eps=1e-6)
    y = mp.rms_norm(x, w, eps=1e-6)
    assert float(scale[0]) == 1.0 and float(q[0].float().abs().sum()) == 0
    assert bool(q.float().isfinite().all())
    assert abs(float(scale[1]) * 448 - float(y[1].double().max())) <= 0.5 * 2.0 ** -149 * 448  # 16 units of 2^-149
    # a subnormal scale of a few units is off by up to half of one
    assert float(((q[1].double() * scale[1].double()) - y[1].double()).abs().max()) <= 0.5 * 2.0 ** -149 * 448 + 2.0 ** -4 * 1e-41


def test_fp8_rows_with_infinite_and_nan_values_stay_apart() -> None:
    from relmo_amd import mp

    x, r, w, _, _ = _inputs(6, 48, torch.float32)
    clean_q, clean_scale, _ = mp.add_rms_norm_fp8(x, r, w)
    clean_y, _ = mp.add_rms_norm(x, r, w)
    x[2, 5], x[4, 47] = float("nan"), float("inf")
    q, scale, _ = mp.add_rms_norm_fp8(x, r, w)
    y, h = mp.add_rms_norm(x, r, w)
    fine = [0, 1, 3, 5]
    assert torch.equal(q[fine].float(), clean_q[fine].float()) and torch.equal(scale[fine], clean_scale[fine])
    assert torch.equal(y[fine], clean_y[fine])
    assert bool(scale[2].isnan()) and bool(y[2].isnan().all()) and bool(q[2].float().isnan().all())
    assert bool(y[4, 47].isnan()) and bool(scale[4].isnan()) and bool(h[4, 47].isinf())  # inf * (1 / inf)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_offsets_and_leading_shapes(dtype) -> None:
    from relmo_amd import mp

    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    base = torch.randn(4, 6, 130, device=DEV, generator=g).to(dtype)
    other = torch.randn(6, 4, 65, device=DEV, generator=g).to(dtype)
    w = torch.rand(65, device=DEV, generator=g).to(dtype)
    x, r = base[..., ::2], other.transpose(0, 1)
    y, h = mp.add_rms_norm(x, r, w)
    y2, h2 = mp.add_rms_norm(x.contiguous(), r.contiguous(), w)
    assert torch.equal(y, y2) and torch.equal(h, h2) and y.shape == x.shape
    # contiguous, but starting off a dword or 16 bytes
    flat = torch.randn(1 + 40 * 64, device=DEV, generator=g).to(dtype)
    off = flat[1:].view(40, 64)
    w = w[1:]
    y, h = mp.add_rms_norm(off, off, w)
    y2, h2 = mp.add_rms_norm(off.clone(), off.clone(), w.clone())
    # the same sums in another order of lanes: equal to the tolerance of two results
    assert torch.equal(h, h2)
    _close(y, y2.double(), 2 * (UNIT[dtype] + chain(64) * U32) * y2.double().abs() + TINY[dtype])
    q, scale, _ = mp.add_rms_norm_fp8(off, off, w)
    _close(scale, (y2.double().abs().amax(1) / 448), (2 * UNIT[dtype] + 2 * chain(64) * U32) * scale.double())


def test_empty_inputs() -> None:
    from relmo_amd import mp

    w = torch.ones(16, device=DEV, requires_grad=True)
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    y, h = mp.add_rms_norm(x, x, w)
    gx, gw = torch.autograd.grad((y, h), (x, w), (y, h))
    assert y.shape == (0, 16) and gx.shape == (0, 16) and torch.equal(gw, torch.zeros(16, device=DEV))
    z = torch.zeros(3, 0, device=DEV)
    q, scale, _ = mp.add_rms_norm_fp8(z, z, torch.zeros(0, device=DEV))
    assert q.shape == (3, 0) and torch.equal(scale, torch.ones(3, device=DEV))


def test_runs_on_the_current_stream() -> None:
    from relmo_amd import mp

    x, r, w, gy, gh = _inputs(50_000, 128, torch.float32)
    want = mp.add_rms_norm(x, r, w)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        x2 = x * 2
        x2.mul_(0.5)
        got = mp.add_rms_norm(x2, r, w)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals() -> None:
    from relmo_amd import capi, mp

    x = torch.ones(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    with pytest.raises(ValueError, match="weight"):
        mp.add_rms_norm(x, x, torch.ones(7, device=DEV))
    with pytest.raises(ValueError, match="residual"):
        mp.add_rms_norm(x, x[:2], w)
    with pytest.raises(ValueError, match="dtype"):
        mp.add_rms_norm(x, x.bfloat16(), w)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        mp.add_rms_norm(x.double(), x.double(), w.double())
    with pytest.raises(RuntimeError, match="eps"):
        mp.add_rms_norm(x, x, w, eps=-1.0)
    with pytest.raises(RuntimeError, match="eps"):
        mp.add_rms_norm(x, x, w, eps=float("nan"))
    with pytest.raises(RuntimeError, match="no gradient"):
        mp.add_rms_norm_fp8(x.requires_grad_(True), x, w)
    x = x.detach()
    y = torch.empty_like(x)
    rc = capi.lib().relm_mp_add_rms_norm(capi.F64, x.data_ptr(), None, w.data_ptr(), 4, 8, 1e-6, y.data_ptr(), None, None,
                                         capi._stream(x))
    assert rc == capi.ERR_INVALID_ARGUMENT and "dtype" in capi.last_error()
    rc = capi.lib().relm_mp_add_rms_norm_backward(capi.F32, x.data_ptr(), None, x.data_ptr(), w.data_ptr(), w.data_ptr(), 4, 8,
                                                  y.data_ptr(), y.data_ptr(), None, 0, capi._stream(x))
    assert rc == capi.ERR_WORKSPACE
