"""GPU tests of ``mp.cross_attention`` against its definition in 64 bits, graph by graph.

Tolerances follow the path of a value.  u is the unit roundoff (2^-24; 2^-8 and 2^-11 where a value is held in
bfloat16 and float16); sums of n float32 terms of either sign err by up to 6 sqrt(n) u times their magnitudes (a
random walk's six deviations).  A score errs by es = 6 sqrt(dim) u scale sum|q||k| + 4 u |s| (its scaling and the
total's logarithm enter the exponent at their size), a probability by ep = 2 max es + 16 u relatively, and by its type's
unit where a product reads it rounded.  The output adds the probabilities' errors over |v|; ds adds those of <grad, v>
and of delta, which is taken from the rounded output; dq, dk and dv add up over |k|, |q| and |grad|."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _offsets(counts):
    return torch.tensor([0] + list(counts), device=DEV).cumsum(0)


def _make(queries, keys, heads, kv_heads, dim, dtype, seed=0, mask=None):
    g = _gen(seed)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g).to(dtype)  # noqa: E731
    nq, nk = sum(queries), sum(keys)
    key_mask = None
    if mask == "random":
        key_mask = torch.rand(nk, device=DEV, generator=g) > 0.3
    elif mask == "first graph":
        key_mask = torch.rand(nk, device=DEV, generator=g) > 0.3
        key_mask[: keys[0]] = False
    elif mask == "last key":
        key_mask = torch.zeros(nk, dtype=torch.bool, device=DEV)
        key_mask[-1] = True
    return (rand(nq, heads, dim), rand(nk, kv_heads, dim), rand(nk, kv_heads, dim), rand(nq, heads, dim), key_mask)


def _walk(n) -> float:
    return 6 * math.sqrt(max(n, 1)) * U


def _definition(q, k, v, grad, key_mask, queries, keys, scale):
    """Results in 64 bits and how far each entry of ours may be off: out, dq, dk, dv."""

    ut = UNIT[q.dtype]
    heads, kv_heads, dim = q.size(1), k.size(1), q.size(2)
    group = heads // kv_heads
    shapes = [q, q, k, k]
    val = [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in shapes]
    tol = [torch.zeros_like(t) for t in val]
    q0 = k0 = 0
    for nq, nk in zip(queries, keys):
        seen = torch.arange(k0, k0 + nk, device=DEV)
        if key_mask is not None:
            seen = seen[key_mask[k0:k0 + nk]]
        if nq and seen.numel():
            rows = lambda t: t[q0:q0 + nq].double().view(nq, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, -1, dim)  # noqa: E731,B023
            back = lambda t: t.view(kv_heads, group, nq, dim).permute(2, 0, 1, 3).reshape(nq, heads, dim)  # noqa: E731,B023
            Q, G = rows(q), rows(grad)
            K, V = (t[seen].double().transpose(0, 1).contiguous() for t in (k, v))
            mm = lambda a, b: a @ b.contiguous()  # noqa: E731
            T = lambda t: t.transpose(1, 2).contiguous()  # noqa: E731
            s = mm(Q, T(K)) * scale
            p = torch.softmax(s, 2)
            es = _walk(dim) * scale * mm(Q.abs(), T(K.abs())) + 4 * U * s.abs() + 4 * U * math.log(seen.numel() + 1)
            ep = (2 * es.amax(2, keepdim=True) + 16 * U)
            nk_walk, nq_walk = _walk(seen.numel()), _walk(Q.size(1))
            o = mm(p, V)
            o_err = mm(p, V.abs()) * (ut + ep + nk_walk) + ut * o.abs()
            dp = mm(G, T(V))
            delta = (G * o).sum(2, keepdim=True)
            dp_err = _walk(dim) * mm(G.abs(), T(V.abs())) + (G.abs() * o_err).sum(2, keepdim=True) + \
                _walk(dim) * (G * o).abs().sum(2, keepdim=True)
            ds = p * (dp - delta)
            ds_err = p * (ep * (dp - delta).abs() + dp_err) + ut * ds.abs()
            dq = mm(ds, K) * scale
            dq_err = scale * (mm(ds_err, K.abs()) + nk_walk * mm(ds.abs(), K.abs())) + (ut + U) * dq.abs()
            dk = mm(T(ds), Q) * scale
            dk_err = scale * (mm(T(ds_err), Q.abs()) + nq_walk * mm(T(ds.abs()), Q.abs())) + (ut + U) * dk.abs()
            dv = mm(T(p), G)
            dv_err = mm(T(p * (ep + ut)), G.abs()) + nq_walk * mm(T(p), G.abs()) + (ut + U) * dv.abs()
            val[0][q0:q0 + nq], tol[0][q0:q0 + nq] = back(o), back(o_err)
            val[1][q0:q0 + nq], tol[1][q0:q0 + nq] = back(dq), back(dq_err)
            val[2][seen], tol[2][seen] = dk.transpose(0, 1), dk_err.transpose(0, 1)
            val[3][seen], tol[3][seen] = dv.transpose(0, 1), dv_err.transpose(0, 1)
        q0, k0 = q0 + nq, k0 + nk
    return val, tol


def _check(got, val, tol, tiny) -> None:
    for name, g, w, t in zip(("out", "dq", "dk", "dv"), got, val, tol):
        assert g.shape == w.shape and bool(g.isfinite().all()), name
        over = (g.double() - w).abs() - t - tiny
        assert bool((over <= 0).all()), (name, float(over.max()), float(w.abs().max()))


def _run(q, k, v, grad, plan, key_mask, scale=None):
    from relmo_amd import mp

    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = mp.cross_attention(q, k, v, plan, key_mask=key_mask, scale=scale)
    return (out, *torch.autograd.grad(out, (q, k, v), grad))


# (queries per graph, keys per graph, heads, key heads, head size)
RAGGED = [
    ([1], [1], 1, 1, 1),
    ([1], [200], 4, 4, 32),
    ([1, 0, 1, 1], [7, 5, 0, 64], 2, 1, 20),
    ([3, 16, 1], [63, 65, 129], 3, 3, 16),              # 16 rows
    ([8, 5], [200, 127], 2, 2, 33),
    ([4, 2, 0], [1, 128, 300], 8, 1, 64),               # 32 rows through the shared key head
    ([32, 31, 17], [100, 64, 513], 2, 2, 128),          # 32 rows
    ([40, 64, 33], [64, 1, 500], 4, 2, 48),             # 64 rows and more
    ([7, 50], [31, 33], 8, 2, 72),
    ([130, 1, 250], [190, 700, 66], 2, 2, 64),          # 128 rows
    ([300, 128], [257, 128], 6, 3, 100),
    ([257], [2000], 2, 1, 128),
    ([1], [20_011], 2, 1, 64),                          # one query: parts over the keys
    ([9, 1], [7_000, 3], 1, 1, 128),
    ([70], [9_000], 1, 1, 32),
    ([5_003, 2], [40, 1], 1, 1, 24),                    # few keys: parts over the rows
    ([600], [70], 8, 1, 128),
    ([20, 3], [50, 130], 2, 1, 7),                      # rows shorter than a unit, and cut ones
    ([5, 33], [90, 64], 2, 2, 9),
    ([33, 90], [200, 70], 2, 1, 65),
    ([12], [300], 1, 1, 127),
    ([2] * 700, [3, 11] * 350, 2, 2, 8),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,keys,heads,kv_heads,dim", RAGGED)
@pytest.mark.parametrize("mask", [None, "random"])
def test_forward_and_backward_against_64_bits(queries, keys, heads, kv_heads, dim, dtype, mask) -> None:
    from relmo_amd import mp

    q, k, v, grad, key_mask = _make(queries, keys, heads, kv_heads, dim, dtype, seed=len(queries) + dim, mask=mask)
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), heads, kv_heads)
    got = _run(q, k, v, grad, plan, key_mask)
    val, tol = _definition(q, k, v, grad, key_mask, queries, keys, dim ** -0.5)
    _check(got, val, tol, 2.0 ** -24 if dtype == torch.float16 else 1e-30)
    with torch.no_grad():  # without the backward's statistics, and again: the same bits
        assert torch.equal(mp.cross_attention(q, k, v, plan, key_mask=key_mask), got[0])
    again = _run(q, k, v, grad, plan, key_mask)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", ["first graph", "last key"])
@pytest.mark.parametrize("queries,keys,heads,kv_heads,dim", [
    ([2, 9, 4], [130, 64, 77], 2, 1, 32), ([60, 33], [70, 129], 2, 2, 64), ([140, 90], [200, 64], 2, 2, 128),
    ([1, 1], [6_000, 5_000], 2, 2, 64), ([30, 30, 30], [20, 700, 128], 1, 1, 64)])
def test_left_out_keys_never_enter(queries, keys, heads, kv_heads, dim, dtype, mask) -> None:
    """Whole graphs without a key, and NaN, infinities and the type's lowest value in what is left out."""
    from relmo_amd import mp

    q, k, v, grad, key_mask = _make(queries, keys, heads, kv_heads, dim, dtype, seed=3, mask=mask)
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), heads, kv_heads)
    val, tol = _definition(q, k, v, grad, key_mask, queries, keys, dim ** -0.5)
    junk = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min, torch.finfo(dtype).max],
                        device=DEV).to(dtype)
    out_of = ~key_mask
    fill = junk[torch.randint(0, 5, (int(out_of.sum()), kv_heads, dim), device=DEV, generator=_gen(1))]
    k, v = k.clone(), v.clone()
    k[out_of], v[out_of] = fill, fill.flip(0)
    got = _run(q, k, v, grad, plan, key_mask)
    _check(got, val, tol, 2.0 ** -24 if dtype == torch.float16 else 1e-30)
    assert float(got[2][out_of].abs().sum()) == 0 and float(got[3][out_of].abs().sum()) == 0
    first = _offsets(queries).tolist()[1]
    if mask == "first graph":
        assert float(got[0][:first].abs().sum()) == 0 and float(got[1][:first].abs().sum()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_scores_and_scales(dtype) -> None:
    """Scores far apart (a maximum that keeps rising, probabilities that underflow) and another scale."""
    from relmo_amd import mp

    queries, keys = [40, 3], [500, 1300]
    q, k, v, grad, _ = _make(queries, keys, 2, 2, 64, dtype, seed=9)
    ramp = torch.linspace(0.1, 6.0, sum(keys), device=DEV).view(-1, 1, 1)
    k = (k.float() * ramp).to(dtype)
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), 2, 2)
    for scale in (0.7, 0.01):
        got = _run(q, k, v, grad, plan, None, scale=scale)
        val, tol = _definition(q, k, v, grad, None, queries, keys, scale)
        _check(got, val, tol, 2.0 ** -24 if dtype == torch.float16 else 1e-30)


def test_infinite_scores_spoil_their_row_only() -> None:
    from relmo_amd import mp

    q, k, v, _, _ = _make([3, 2], [70, 40], 1, 1, 32, torch.float32, seed=4)
    plan = mp.attention_plan(_offsets([3, 2]), _offsets([70, 40]), 1, 1)
    clean = mp.cross_attention(q, k, v, plan)
    q = q.clone()
    q[1, 0, 5] = float("inf")
    out = mp.cross_attention(q, k, v, plan)
    rows = [0, 2, 3, 4]
    assert torch.equal(out[rows], clean[rows]) and bool(out[1].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [[2, 9, 4], [60, 33, 1], [200, 130, 9]])
def test_one_key_leaves_no_gradient_of_the_scores(queries, dtype) -> None:
    """A softmax over one key is 1: dq and dk are 0, not a rounding's rest, with one key and with one kept key."""
    from relmo_amd import mp

    for keys, mask in (([1, 1, 1], None), ([1, 0, 100], "one")):
        q, k, v, grad, _ = _make(queries, keys, 2, 1, 33, dtype, seed=15)
        key_mask = None
        if mask:
            key_mask = torch.zeros(sum(keys), dtype=torch.bool, device=DEV)
            key_mask[0] = key_mask[-7] = True
        plan = mp.attention_plan(_offsets(queries), _offsets(keys), 2, 1)
        out, dq, dk, dv = _run(q, k, v, grad, plan, key_mask)
        assert float(dq.abs().sum()) == 0 and float(dk.abs().sum()) == 0
        val, tol = _definition(q, k, v, grad, key_mask, queries, keys, 33 ** -0.5)
        _check((out, dq, dk, dv), val, tol, 2.0 ** -24 if dtype == torch.float16 else 1e-15)


@pytest.mark.parametrize("queries", [[2, 9], [60, 33], [200, 130]])
def test_infinite_queries_and_left_out_keys(queries) -> None:
    """An infinite query spoils neither the gradients of left-out keys nor the zeros of a graph without a key."""
    from relmo_amd import mp

    keys = [150, 90]
    q, k, v, grad, mask = _make(queries, keys, 1, 1, 32, torch.float32, seed=14, mask="first graph")
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), 1)
    clean = _run(q, k, v, grad, plan, mask)
    q = q.clone()
    q[0, 0, 3] = float("inf")  # in the graph without a key
    out, dq, dk, dv = _run(q, k, v, grad, plan, mask)
    assert torch.equal(out, clean[0]) and torch.equal(dk, clean[2]) and torch.equal(dv, clean[3])
    assert torch.equal(dq[queries[0]:], clean[1][queries[0]:]) and float(dq[:queries[0]].abs().sum()) == 0
    q[-1, 0, 3] = float("inf")
    out, dq, dk, dv = _run(q, k, v, grad, plan, mask)
    assert torch.equal(out[:-1], clean[0][:-1])
    assert float(dk[~mask].abs().sum()) == 0 and float(dv[~mask].abs().sum()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_offsets_and_alignment(dtype) -> None:
    from relmo_amd import mp

    g = _gen(6)
    queries, keys, heads, dim = [17, 40], [150, 90], 3, 40
    nq, nk = sum(queries), sum(keys)
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), heads)
    both = torch.randn(nk, 2, heads, dim, device=DEV, generator=g).to(dtype)      # a fused projection
    k, v = both[:, 0], both[:, 1]
    q = torch.randn(heads, nq, dim, device=DEV, generator=g).to(dtype).transpose(0, 1)  # heads first
    grad = torch.randn(nq, heads, dim, device=DEV, generator=g).to(dtype)
    want = _run(q.contiguous(), k.contiguous(), v.contiguous(), grad, plan, None)
    got = _run(q, k, v, grad, plan, None)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    # rows that start off a dword; values that are not side by side; an expanded gradient
    def shifted(t):
        flat = torch.empty(t.numel() + 1, device=DEV, dtype=dtype)
        return flat[1:].view(t.shape).copy_(t)
    got = _run(shifted(q), shifted(k.contiguous()), shifted(v.contiguous()), shifted(grad), plan, None)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    wide = torch.zeros(nk, heads, 2 * dim, device=DEV, dtype=dtype)
    wide[..., ::2] = k
    got = _run(q, wide[..., ::2], v, grad, plan, None)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    one = torch.ones((), device=DEV, dtype=dtype).expand(nq, heads, dim)
    got, want = _run(q, k, v, one, plan, None), _run(q, k, v, one.contiguous(), plan, None)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_keys_broadcast_over_heads_share_their_gradient() -> None:
    """One key head against query heads that read it through an expanded tensor: the sum of the heads' gradients."""
    from relmo_amd import mp

    queries, keys, heads, dim = [5, 20], [90, 33], 4, 32
    q, k, v, grad, _ = _make(queries, keys, heads, 1, dim, torch.float32, seed=8)
    qo, ko = _offsets(queries), _offsets(keys)
    shared = _run(q, k, v, grad, mp.attention_plan(qo, ko, heads, 1), None)
    k2, v2 = k.detach().requires_grad_(True), v.detach().requires_grad_(True)
    out = mp.cross_attention(q, k2.expand(-1, heads, -1), v2.expand(-1, heads, -1), mp.attention_plan(qo, ko, heads))
    gk, gv = torch.autograd.grad(out, (k2, v2), grad)
    val, tol = _definition(q, k, v, grad, None, queries, keys, dim ** -0.5)
    _check((out, shared[1], gk, gv), val, tol, 1e-30)
    _check(shared, val, tol, 1e-30)


def test_gradient_against_differences() -> None:
    from relmo_amd import mp

    queries, keys = [6, 11], [40, 75]
    q, k, v, grad, mask = _make(queries, keys, 4, 2, 24, torch.float32, seed=2, mask="random")
    plan = mp.attention_plan(_offsets(queries), _offsets(keys), 4, 2)
    grads = _run(q, k, v, grad, plan, mask)[1:]
    g = _gen(12)
    for i, gt in enumerate(grads):
        d = torch.randn(gt.shape, device=DEV, generator=g, dtype=torch.float64)

        def loss(step):
            args = [t.double() for t in (q, k, v)]
            args[i] = args[i] + step * d
            out = _definition(*args, grad.double(), mask, queries, keys, 24 ** -0.5)[0][0]
            return (out * grad.double()).sum()

        UNIT.setdefault(torch.float64, 0.0)
        want = (loss(1e-4) - loss(-1e-4)) / 2e-4  # its own error: step^2 times third derivatives of order 1
        assert abs(float((gt.double() * d).sum() - want)) <= 2e-6 * float((gt.double() * d).abs().sum()), i


def test_offsets_past_32_bits() -> None:
    """Rows far into a tensor whose last values lie past 2^31 values and 2^32 bytes from its start."""
    from relmo_amd import mp

    rows, heads, dim = 300, 1, 64
    stride = (1 << 31) // 290
    big = torch.empty((rows - 1) * stride + 2 * dim, device=DEV, dtype=torch.bfloat16)
    k = big.as_strided((rows, heads, dim), (stride, dim, 1))
    v = big.as_strided((rows, heads, dim), (stride, dim, 1), dim)
    g = _gen(5)
    kc, vc = (torch.randn(rows, heads, dim, device=DEV, generator=g).bfloat16() for _ in range(2))
    k.copy_(kc), v.copy_(vc)
    q, grad = (torch.randn(20, heads, dim, device=DEV, generator=g).bfloat16() for _ in range(2))
    plan = mp.attention_plan(_offsets([20]), _offsets([rows]), heads)
    got, want = _run(q, k, v, grad, plan, None), _run(q, kc, vc, grad, plan, None)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_plan_keeps_its_own_lengths_and_serves_other_streams() -> None:
    from relmo_amd import mp

    queries, keys = [8] * 300, [200] * 300
    q, k, v, grad, _ = _make(queries, keys, 2, 2, 32, torch.float32)
    qo, ko = _offsets(queries), _offsets(keys)
    plan = mp.attention_plan(qo, ko, 2)
    want = _run(q, k, v, grad, plan, None)
    qo.zero_(), ko.zero_()
    got = _run(q, k, v, grad, plan, None)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        q2 = (q * 2).mul_(0.5)
        got = _run(q2, k, v, grad, plan, None)
        del plan, q2
        torch.empty(1 << 20, device=DEV).fill_(1.0)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_the_plan_lives_as_long_as_its_graph_and_second_derivatives_raise() -> None:
    from relmo_amd import mp

    q, k, v, grad, _ = _make([3], [40], 1, 1, 16, torch.float32)
    plan = mp.attention_plan(_offsets([3]), _offsets([40]), 1)
    want = _run(q, k, v, grad, plan, None)
    x = q.detach().requires_grad_(True)
    out = mp.cross_attention(x, k, v, plan)
    del plan
    (gx,) = torch.autograd.grad(out, x, grad, create_graph=True)
    assert torch.equal(gx, want[1])
    with pytest.raises(RuntimeError, match="twice"):
        gx.sum().backward()


def test_empty_batches() -> None:
    from relmo_amd import mp

    for queries, keys in (([], []), ([0, 0], [0, 0]), ([3, 0], [0, 0]), ([0, 0], [5, 2])):
        q, k, v, grad, _ = _make(queries, keys, 2, 2, 16, torch.float32)
        got = _run(q, k, v, grad, mp.attention_plan(_offsets(queries), _offsets(keys), 2), None)
        assert [t.shape for t in got] == [q.shape, q.shape, k.shape, v.shape]
        assert all(float(t.abs().sum()) == 0 for t in got)


def test_refusals() -> None:
    from relmo_amd import capi, mp

    o = _offsets([4, 4])
    for bad in ([1, 2, 3], [0, 5, 3]):
        with pytest.raises(RuntimeError, match="q_offsets must"):
            mp.attention_plan(torch.tensor(bad, device=DEV), o, 2)
    with pytest.raises(ValueError, match="int64"):
        mp.attention_plan(o.int(), o, 2)
    with pytest.raises(ValueError, match="multiple"):
        mp.attention_plan(o, o, 4, 3)
    plan = mp.attention_plan(o, o, 2)
    x = torch.ones(8, 2, 16, device=DEV)
    with pytest.raises(ValueError, match="q must be"):
        mp.cross_attention(x[:7], x, x, plan)
    with pytest.raises(ValueError, match="k and v must be"):
        mp.cross_attention(x, x[:7], x[:7], plan)
    with pytest.raises(ValueError, match="dtype"):
        mp.cross_attention(x, x.bfloat16(), x, plan)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        mp.cross_attention(x.double(), x.double(), x.double(), plan)
    with pytest.raises(ValueError, match="key_mask"):
        mp.cross_attention(x, x, x, plan, key_mask=torch.ones(8, device=DEV))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            mp.cross_attention(x, x, x, plan, scale=scale)
    big = torch.ones(8, 2, 129, device=DEV)
    with pytest.raises(ValueError, match="head_dim"):
        mp.cross_attention(big, big, big, plan)
    with pytest.raises(ValueError, match="GPU"):
        mp.cross_attention(x, x, x, mp.attention_plan(o.cpu(), o.cpu(), 2))
    number = plan.number
    del plan
    with pytest.raises(ValueError, match="no longer exists"):
        torch.ops.relm_mp.cross_attention(x, x, x, number, None, 1.0)
    rc = capi.lib().relm_mp_cross_attention(capi.F32, None, None, None, None, 16, None, 1.0, None, None, None, 0, None)
    assert rc == capi.ERR_INVALID_ARGUMENT and "plan" in capi.last_error()
