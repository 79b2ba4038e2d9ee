"""GPU tests of ``mp.cross_attention`` where its numbers run out: probabilities that a 16-bit type cannot hold,
scores of any size, softmaxes of one key, infinities in keys and gradients.

Scores are made exact here (one value of a query, a power of two, meets one value of a key), so a probability errs by
its own roundings only: at most 16 units of 2^-24 and one for each unit of the score's distance from the row's maximum,
and by its type's unit where a product reads it rounded.  u is the unit roundoff of the values' type."""

from __future__ import annotations

import pytest
import torch

from .test_gpu_attention import DEV, DTYPES, U, UNIT, _check, _definition, _gen, _make, _offsets, _run, _walk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


# queries of a graph (16, 32, 64 and 128 rows to an item) and head sizes
ROWS = [(1, 64), (9, 32), (30, 64), (31, 128), (60, 32), (64, 128), (200, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,dim", ROWS)
@pytest.mark.parametrize("keys", [200, 4096, 30_001])
def test_values_far_below_the_dominant_key(queries, dim, keys, dtype) -> None:
    """One key of value 0 whose score lies 14 to 18 above all others': what the others add is the whole output."""
    from relmo_amd import mp

    g = _gen(queries + keys)
    plan = mp.attention_plan(_offsets([queries]), _offsets([keys]), 1)
    q = torch.zeros(queries, 1, dim, device=DEV)
    q[:, 0, 1] = 1.0
    v = (8.0 * torch.rand(keys, 1, dim, device=DEV, generator=g) + 1.0).to(dtype)
    for gap in (14.0, 16.0, 17.0, 18.0):
        for at in (0, keys // 2, keys - 1):
            k = torch.zeros(keys, 1, dim, device=DEV)
            k[at, 0, 1] = gap
            values = v.clone()
            values[at] = 0
            with torch.no_grad():
                out = mp.cross_attention(q.to(dtype), k.to(dtype), values, plan, scale=1.0)
            p = torch.softmax(torch.tensor([gap] + [0.0] * (keys - 1), dtype=torch.float64, device=DEV), 0)[1]
            want = p * values.double().sum(0, keepdim=True)
            # terms of one sign: the walk's error in units of the sum; the output's own rounding (its subnormals' spacing)
            tol = want * (2 * UNIT[dtype] + (16 + gap) * U + _walk(keys)) + (2.0 ** -24 if dtype == torch.float16 else 0)
            over = (out.double() - want).abs() - tol
            assert bool((over <= 0).all()), (gap, at, float((out.double() / want - 1).abs().max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,dim", [([0, 3], 64), ([9, 0], 33), ([0, 60], 128), ([0, 0], 5)])
def test_keys_of_graphs_without_queries_get_zeros(queries, dim, dtype) -> None:
    from relmo_amd import mp

    keys = [70_001, 5_000]
    g = _gen(dim)
    q, grad = (torch.randn(sum(queries), 2, dim, device=DEV, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(sum(keys), 1, dim, device=DEV, generator=g).to(dtype) for _ in range(2))
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), 2, 1)
    for _ in range(3):  # memory that the results will take
        torch.full_like(k, float("nan"))
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    _dq, dk, dv = torch.autograd.grad(mp.cross_attention(q, k, v, plan), (q, k, v), grad)
    edge = keys[0]
    for b, rows in enumerate((slice(0, edge), slice(edge, None))):
        for t in (dk, dv):
            assert bool(t[rows].isfinite().all()) and (queries[b] > 0) == bool(t[rows].abs().sum() > 0)


def _ladder(queries, keys, dim, dtype, size, scale=1.0, step=1):
    """q, k, v, grad whose scores are size * scale less 0 .. 5 steps, exactly."""

    g = _gen(keys)
    root = 2.0 ** round(0.5 * torch.tensor(float(size)).log2().item())
    level = torch.randint(0, 6, (keys,), device=DEV, generator=g)
    level[keys // 3] = 0
    q = torch.zeros(queries, 1, dim, device=DEV, dtype=torch.float64)
    k = torch.zeros(keys, 1, dim, device=DEV, dtype=torch.float64)
    q[:, 0, 0] = root
    k[:, 0, 0] = size / root - level.double() * step / root
    v, grad = torch.randn(keys, 1, dim, device=DEV, generator=g), torch.randn(queries, 1, dim, device=DEV, generator=g)
    return q.to(dtype), k.to(dtype), v.to(dtype), grad.to(dtype), -level.double() * step * scale


@pytest.mark.parametrize("queries,dim", ROWS)
@pytest.mark.parametrize("size", [2.0 ** 4, 2.0 ** 8, 2.0 ** 12, 2.0 ** 16])
def test_probabilities_of_large_scores_add_up_to_one(queries, dim, size) -> None:
    """Scores of a row a few units apart around a large one: the backward's probabilities are the forward's."""
    from relmo_amd import mp

    keys = 700
    q, k, v, grad, s = _ladder(queries, keys, dim, torch.float32, size)
    plan = mp.attention_plan(_offsets([queries]), _offsets([keys]), 1)
    out, dq, dk, dv = _run(q, k, v, grad, plan, None, scale=1.0)
    p = torch.softmax(s, 0)
    ep = (16 + 5) * U
    V, G = v[:, 0].double(), grad[:, 0].double()
    want = (p[:, None] * V).sum(0)
    assert float(((out[:, 0].double() - want).abs() - (ep + _walk(keys)) * (p[:, None] * V.abs()).sum(0)).max()) <= 0
    want = p[:, None] * G.sum(0)
    assert float(((dv[:, 0].double() - want).abs() - (ep + _walk(queries) + U) * p[:, None] * G.abs().sum(0)).max()) <= 0
    # ds adds up to nothing over a row's keys, up to its terms' errors
    ds = dk[:, 0, 0].double() / float(q[0, 0, 0])
    dp_err = 3 * _walk(dim) * (G.abs().sum(0) * V.abs().amax(0)).sum() + _walk(keys) * (G.abs().sum(0) * V.abs().amax(0)).sum()
    assert abs(float(ds.sum())) <= float(dp_err + 2 * ep * ds.abs().sum() + _walk(keys) * ds.abs().sum())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,keys,dim", [([3, 0, 9], [70, 5, 0], 32), ([60, 33], [70, 300], 64), ([1], [6_000], 40)])
def test_c_entries_from_the_logarithm_of_the_total(queries, keys, dim, dtype) -> None:
    """``relm_mp_cross_attention`` with its lse and the backward from it, without the torch binding."""
    import ctypes

    from relmo_amd import capi

    lib, code = capi.lib(), {torch.float32: capi.F32, torch.bfloat16: capi.BF16, torch.float16: capi.F16}[dtype]
    q, k, v, grad, mask = _make(queries, keys, 2, 1, dim, dtype, seed=dim, mask="random")
    offsets = [_offsets(n).cpu() for n in (queries, keys)]
    plan = capi.AttentionPlan()
    args = (offsets[0].data_ptr(), offsets[1].data_ptr(), len(queries), sum(queries), sum(keys), 2, 1)
    capi.check(lib.relm_mp_attention_plan_build(*args, None, 0, ctypes.byref(plan)))
    table = torch.empty(plan.table_bytes, dtype=torch.uint8)
    capi.check(lib.relm_mp_attention_plan_build(*args, table.data_ptr(), plan.table_bytes, ctypes.byref(plan)))
    table = table.to(DEV)
    plan.table = table.data_ptr()
    rows = [ctypes.byref(capi.HeadRows(t.data_ptr(), t.stride(0), t.stride(1))) for t in (q, k, v, grad)]
    scale, stream = dim ** -0.5, capi._stream(q)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    ws = torch.empty(max(lib.relm_mp_cross_attention_workspace_size(plan, dim),
                         lib.relm_mp_cross_attention_backward_workspace_size(plan, dim)), dtype=torch.uint8, device=DEV)
    capi.check(lib.relm_mp_cross_attention(code, plan, *rows[:3], dim, mask.data_ptr(), scale, out.data_ptr(), lse.data_ptr(),
                                           ws.data_ptr(), ws.numel(), stream))
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    capi.check(lib.relm_mp_cross_attention_backward(code, plan, rows[3], *rows[:3], dim, mask.data_ptr(), scale, out.data_ptr(),
                                                    lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(),
                                                    ws.numel(), stream))
    val, tol = _definition(q, k, v, grad, mask, queries, keys, scale)
    _check((out, dq, dk, dv), val, tol, 2.0 ** -24 if dtype == torch.float16 else 1e-30)
    q0 = k0 = 0
    for nq, nk in zip(queries, keys):
        kept = k[k0:k0 + nk, 0][mask[k0:k0 + nk]].double()
        s = torch.einsum("nhd,kd->nhk", q[q0:q0 + nq].double(), kept) * scale
        want = torch.logsumexp(s, 2) if kept.size(0) else torch.full(s.shape[:2], -torch.inf, device=DEV, dtype=torch.float64)
        got = lse[q0:q0 + nq].double()
        err = _walk(dim) * scale * q[q0:q0 + nq].double().norm(dim=2) * (kept.norm(dim=1).max() if kept.size(0) else 0)
        assert torch.equal(got.isinf(), want.isinf())
        fine = ~want.isinf()
        assert bool(((got - want).abs()[fine] <= (err + 16 * U * (1 + want.abs()))[fine]).all())
        q0, k0 = q0 + nq, k0 + nk
    null = lib.relm_mp_cross_attention_keep(code, plan, *rows[:3], dim, None, scale, out.data_ptr(), None, ws.data_ptr(), ws.numel(), stream)
    assert null == capi.ERR_INVALID_ARGUMENT and "NULL" in capi.last_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,dim", ROWS)
@pytest.mark.parametrize("keys", [100, 6_000])
def test_scores_past_the_floats_units(queries, dim, keys, dtype) -> None:
    """Scores whose neighbours in float lie hundreds apart: the largest takes all, two equal ones take half each."""
    from relmo_amd import mp

    g = _gen(3)
    plan = mp.attention_plan(_offsets([queries]), _offsets([keys]), 1)
    for scale in (1.0, 1.3):
        for ties in (1, 2):
            q = torch.zeros(queries, 1, dim, device=DEV)
            k = torch.zeros(keys, 1, dim, device=DEV)
            q[:, 0, 2] = 2.0 ** 14
            k[:, 0, 2] = -(2.0 ** 13)
            top = [7, keys - 9][:ties]
            k[top, 0, 2] = 57344.0  # 7 * 2^13
            v, grad = torch.randn(keys, 1, dim, device=DEV, generator=g), torch.randn(queries, 1, dim, device=DEV, generator=g)
            v, grad = v.to(dtype), grad.to(dtype)
            out, _dq, dk, dv = _run(q.to(dtype), k.to(dtype), v, grad, plan, None, scale=scale * 2.0 ** 12)
            u = max(UNIT[dtype], U)
            want = v[top].double().mean(0)
            assert bool(((out.double() - want).abs() <= 2 * u * want.abs() + 16 * U).all())
            G = grad.double().sum(0)
            tol = (2 * u + _walk(queries)) * grad.double().abs().sum(0) / ties
            assert bool(((dv[top].double() - G / ties).abs() <= tol).all())
            rest = torch.ones(keys, dtype=torch.bool, device=DEV)
            rest[top] = False
            assert float(dv[rest].abs().sum()) == 0 and float(dk[rest].abs().sum()) == 0


ONE_KEY = [([2, 1], 7), ([20, 3], 33), ([60, 33], 64), ([200, 130], 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,dim", ONE_KEY)
@pytest.mark.parametrize("keys", [1, 100, 129, 200, 5_000, 20_011])
def test_one_kept_key_among_any_number(queries, dim, keys, dtype) -> None:
    """A softmax over one kept key is 1 and its gradient nothing, however many keys are left out around it."""
    from relmo_amd import mp

    lengths = [keys, 3]
    q, k, v, grad, _ = _make(queries, lengths, 2, 1, dim, dtype, seed=dim + keys)
    mask = torch.zeros(sum(lengths), dtype=torch.bool, device=DEV)
    mask[keys // 2] = mask[keys + 1] = True
    plan = mp.attention_plan(_offsets(queries), _offsets(lengths), 2, 1)
    out, dq, dk, dv = _run(q, k, v, grad, plan, mask)
    assert torch.equal(out[:queries[0]], v[keys // 2].expand(queries[0], 2, dim))
    assert float(dq.abs().sum()) == 0 and float(dk.abs().sum()) == 0
    val, tol = _definition(q, k, v, grad, mask, queries, lengths, dim ** -0.5)
    _check((out, dq, dk, dv), val, tol, 2.0 ** -24 if dtype == torch.float16 else 1e-30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,dim", ONE_KEY)
@pytest.mark.parametrize("keys", [1, 100, 5_000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradients_that_are_no_numbers_show_through_one_kept_key(queries, dim, keys, dtype, bad) -> None:
    from relmo_amd import mp

    lengths = [keys, 3]
    q, k, v, grad, _ = _make(queries, lengths, 2, 1, dim, dtype, seed=dim + keys)
    mask = torch.zeros(sum(lengths), dtype=torch.bool, device=DEV)
    mask[keys // 2] = mask[keys + 1] = True
    grad[1, 1, dim // 2] = bad
    plan = mp.attention_plan(_offsets(queries), _offsets(lengths), 2, 1)
    _out, dq, dk, dv = _run(q, k, v, grad, plan, mask)
    assert bool(dq[1, 1].isnan().all()) and bool(dk[keys // 2].isnan().all())
    assert not bool(dv[keys // 2, 0, dim // 2].isfinite())
    dq[1, 1] = 0
    assert float(dq.abs().sum()) == 0 and float(dk[~mask].abs().sum()) == 0 and float(dv[~mask].abs().sum()) == 0
    assert float(dk[keys + 1].abs().sum()) == 0 and bool(dv[keys + 1].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,dim", ROWS)
@pytest.mark.parametrize("size", [2.0 ** 5, 2.0 ** 11, 2.0 ** 20, 2.0 ** 34])
def test_a_dominant_key_leaves_no_gradient_of_the_scores(queries, dim, size, dtype) -> None:
    """All but one key lie far below: their probabilities are 0 in float, as if they were left out."""
    from relmo_amd import mp

    keys = 300
    g = _gen(7)
    plan = mp.attention_plan(_offsets([queries]), _offsets([keys]), 1)
    q, k = torch.zeros(queries, 1, dim, device=DEV), torch.zeros(keys, 1, dim, device=DEV)
    q[:, 0, 0], k[:, 0, 0], k[211, 0, 0] = 8.0, -64.0, size / 8 if size < 2.0 ** 16 else 2.0 ** 13
    v, grad = torch.randn(keys, 1, dim, device=DEV, generator=g), torch.randn(queries, 1, dim, device=DEV, generator=g)
    scale = 1.3 if size < 2.0 ** 16 else 1.3 * size / 2.0 ** 16
    out, dq, dk, dv = _run(q.to(dtype), k.to(dtype), v.to(dtype), grad.to(dtype), plan, None, scale=scale)
    assert torch.equal(out, v[211:212].to(dtype).expand_as(out))
    assert float(dq.abs().sum()) == 0 and float(dk.abs().sum()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [[1, 2], [9, 1], [17, 30], [40, 33], [65, 1], [130, 250]])
@pytest.mark.parametrize("dim", [20, 64, 128])
def test_infinite_keys_that_no_query_attends_to(queries, dim, dtype) -> None:
    """A kept key whose scores are all -inf has the probability 0: dk and dv of it are 0, whatever fills a tile's
    rows past the graph's, and the other keys go on as if it were left out.  (dq is 0 times infinity, as by the formula.)"""
    from relmo_amd import mp

    keys = [70, 150]
    q, k, v, grad, _ = _make(queries, keys, 1, 1, dim, dtype, seed=dim)
    q[:, 0, 3] = q[:, 0, 3].abs() + 0.5
    spoilt = torch.zeros(sum(keys), dtype=torch.bool, device=DEV)
    spoilt[[11, 70, 219]] = True
    val, tol = _definition(q, k, v, grad, ~spoilt, queries, keys, dim ** -0.5)
    k[spoilt, 0, 3] = float("-inf")
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), 1)
    out, dq, dk, dv = _run(q, k, v, grad, plan, None)
    assert float(dk[spoilt].abs().sum()) == 0 and float(dv[spoilt].abs().sum()) == 0
    assert bool(dq[:, 0, 3].isnan().all())
    dq[:, 0, 3], val[1][:, 0, 3] = 0, 0
    _check((out, dq, dk, dv), val, tol, 2.0 ** -24 if dtype == torch.float16 else 1e-30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [[1, 2], [17, 30], [40, 33], [130, 250]])
def test_infinite_values_leave_their_own_gradient_alone(queries, dtype) -> None:
    """dv of a key is its probabilities' sum over the gradients, whatever the key's value is."""
    from relmo_amd import mp

    keys = [70, 150]
    q, k, v, grad, _ = _make(queries, keys, 1, 1, 32, dtype, seed=5)
    val, tol = _definition(q, k, v, grad, None, queries, keys, 32 ** -0.5)
    v = v.clone()
    v[11, 0, 3] = float("inf")
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), 1)
    _out, dq, dk, dv = _run(q, k, v, grad, plan, None)
    for at, g in ((1, dq), (2, dk)):  # the other graph's are as they were
        rows = queries[0] if at == 1 else keys[0]
        over = (g[rows:].double() - val[at][rows:]).abs() - tol[at][rows:] - 2.0 ** -24
        assert bool((over <= 0).all())
    assert bool(((dv.double() - val[3]).abs() <= tol[3] + 2.0 ** -24).all())


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("graphs,queries,dim", [(300, 16, 64), (150, 30, 32), (80, 60, 64), (30, 200, 128)])
@pytest.mark.parametrize("keys", [2, 3, 9])
def test_few_keys_lose_no_more_than_two_roundings(graphs, queries, dim, keys, dtype) -> None:
    """With few keys ds is the small difference of <grad, v> and delta.  dq and dk then err by two roundings to 16 bits of
    the same size, ds and the result: 1.42 times one of them, and not by the output's on top (1.6 times with 4 keys, 2.2
    with 2)."""
    from relmo_amd import mp

    lengths = [queries] * graphs, [keys] * graphs
    q, k, v, grad, _ = _make(*lengths, 1, 1, dim, dtype, seed=keys)
    plan = mp.attention_plan(_offsets(lengths[0]), _offsets(lengths[1]), 1)
    got = _run(q, k, v, grad, plan, None)
    val, _tol = _definition(q, k, v, grad, None, *lengths, dim ** -0.5)
    for name, g, w in (("dq", got[1], val[1]), ("dk", got[2], val[2])):
        once = float((w.to(dtype).double() - w).norm())
        assert float((g.double() - w).norm()) <= 1.55 * once, (name, float((g.double() - w).norm()) / once)
