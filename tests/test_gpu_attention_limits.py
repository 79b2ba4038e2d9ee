"""GPU tests of ``mp.cross_attention`` where its numbers run out: probabilities that a 16-bit type cannot hold.

Scores are made exact here (one value of a query, a power of two, meets one value of a key), so a probability errs by
its own roundings only: at most 16 units of 2^-24 and one for each unit of the score's distance from the row's maximum,
and by its type's unit where a product reads it rounded.  u is the unit roundoff of the values' type."""

from __future__ import annotations

import pytest
import torch

from .test_gpu_attention import DEV, DTYPES, U, UNIT, _gen, _offsets, _walk

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
