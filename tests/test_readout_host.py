"""The readout ops without a GPU: the facade's ATen formulations against their definitions in 64 bits, their
gradients against differences, argument checks, and the host-side plan of the attention's work."""

from __future__ import annotations

import ctypes

import pytest
import torch

from relmo_amd import mp


def _gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def _randn(*shape, seed: int = 0, dtype=torch.float64):
    return torch.randn(*shape, generator=_gen(seed), dtype=dtype)


# ---- ATen formulations ----------------------------------------------------------------------


def test_norm_formulation_and_gradient() -> None:
    x, r, w = (_randn(5, 9, seed=1).requires_grad_(), _randn(5, 9, seed=2).requires_grad_(), _randn(9, seed=3).requires_grad_())
    y, h = mp.add_rms_norm(x, r, w, eps=1e-3)
    assert torch.equal(h, x + r)
    torch.testing.assert_close(y, (x + r) / ((x + r).square().mean(-1, keepdim=True) + 1e-3).sqrt() * w)
    assert torch.autograd.gradcheck(lambda *a: mp.add_rms_norm(*a, eps=1e-3), (x, r, w))
    torch.testing.assert_close(mp.rms_norm(x, w), mp.add_rms_norm(x, torch.zeros_like(x), w)[0])
    with torch.no_grad():
        q, scale, h2 = mp.add_rms_norm_fp8(x, r, w, eps=1e-3)
    assert q.dtype == torch.float8_e4m3fn and torch.equal(h2, h)
    # half a unit of 4 significant bits
    assert bool(((q.double() * scale.double().unsqueeze(1) - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * scale.unsqueeze(1)).all())


def test_norm_rounds_once_in_16_bits() -> None:
    x, r, w = (_randn(4, 33, seed=s).bfloat16() for s in (1, 2, 3))
    y, h = mp.add_rms_norm(x, r, w[0])
    exact = x.double() + r.double()
    assert torch.equal(h, exact.bfloat16())
    want = exact * (exact.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w[0].double()
    assert float(((y.double() - want).abs() / want.abs()).max()) <= 2.0 ** -8 * 1.001


@pytest.mark.parametrize("mask", [False, True])
def test_attention_formulation_and_gradient(mask) -> None:
    qo, ko = torch.tensor([0, 2, 2, 5, 6]), torch.tensor([0, 3, 7, 7, 12])
    q, k, v = (_randn(6, 4, 5, seed=1).requires_grad_(), _randn(12, 2, 5, seed=2).requires_grad_(),
               _randn(12, 2, 5, seed=3).requires_grad_())
    kept = torch.ones(12, dtype=torch.bool)
    if mask:
        kept[[0, 1, 2, 9]] = False
    plan = mp.attention_plan(qo, ko, 4, 2)
    out = mp.cross_attention(q, k, v, plan, key_mask=kept if mask else None, scale=0.7)
    for b in range(4):
        for i in range(int(qo[b]), int(qo[b + 1])):
            keys = [j for j in range(int(ko[b]), int(ko[b + 1])) if kept[j]]
            for h in range(4):
                if not keys:
                    assert float(out[i, h].abs().sum()) == 0
                    continue
                s = torch.stack([0.7 * q[i, h] @ k[j, h // 2] for j in keys])
                p = s.exp() / s.exp().sum()
                torch.testing.assert_close(out[i, h], sum(p[n] * v[j, h // 2] for n, j in enumerate(keys)))
    assert torch.autograd.gradcheck(
        lambda *a: mp.cross_attention(*a, plan, key_mask=kept if mask else None, scale=0.7), (q, k, v))


def test_plan_keeps_its_own_lengths() -> None:
    """Later writes to the offsets neither move a plan's graphs nor undo the check that was made of them."""

    qo, ko = torch.tensor([0, 2, 5]), torch.tensor([0, 3, 9])
    q, k, v = (_randn(n, 2, 4, seed=n) for n in (5, 9, 9))
    plan = mp.attention_plan(qo, ko, 2)
    want = mp.cross_attention(q, k, v, plan)
    ko[1], qo[1] = 5, 1
    assert torch.equal(mp.cross_attention(q, k, v, plan), want)
    ko[1] = 100
    assert torch.equal(mp.cross_attention(q, k, v, plan), want)
    assert plan.k_offsets.tolist() == [0, 3, 9] and plan.q_offsets.tolist() == [0, 2, 5]


def test_orthogonalise_formulation() -> None:
    tall = _randn(9, 4, seed=5)
    got = mp.orthogonalise(tall, steps=8, coefficients=(1.5, -0.5, 0.0))
    u, _s, vt = torch.linalg.svd(tall, full_matrices=False)
    x = _s / _s.norm()
    for _ in range(8):
        x = 1.5 * x - 0.5 * x ** 3
    torch.testing.assert_close(got, u * x @ vt, atol=1e-6, rtol=1e-6)
    stack = _randn(3, 4, 9, seed=6)
    outs = mp.orthogonalise([stack, tall])
    torch.testing.assert_close(outs[0][1], mp.orthogonalise(stack[1]))
    assert outs[1].shape == tall.shape and mp.orthogonalise([]) == []


def test_argument_checks() -> None:
    x, o = torch.ones(4, 2, 8), torch.tensor([0, 1, 4])
    plan = mp.attention_plan(o, o, 2)
    with pytest.raises(ValueError, match="weight"):
        mp.rms_norm(x, torch.ones(7))
    with pytest.raises(RuntimeError, match="no gradient"):
        mp.add_rms_norm_fp8(x.clone().requires_grad_(), x, torch.ones(8))
    with pytest.raises(ValueError, match="multiple"):
        mp.attention_plan(o, o, 3, 2)
    with pytest.raises(ValueError, match="int64"):
        mp.attention_plan(o, o.int(), 2)
    with pytest.raises(ValueError, match="int64"):
        mp.attention_plan(o, o[:2], 2)
    with pytest.raises(RuntimeError, match="k_offsets must ascend"):
        mp.attention_plan(o, torch.tensor([0, 3, 2]), 2)
    with pytest.raises(ValueError, match="numbers of queries"):
        mp.cross_attention(x[:3], x, x, plan)
    with pytest.raises(ValueError, match="heads and kv_heads"):
        mp.cross_attention(x[:, :1], x, x, plan)
    with pytest.raises(ValueError, match="scale"):
        mp.cross_attention(x, x, x, plan, scale=0.0)
    with pytest.raises(ValueError, match="key_mask"):
        mp.cross_attention(x, x, x, plan, key_mask=torch.ones(4))
    with pytest.raises(ValueError, match="three"):
        mp.orthogonalise(x[0], coefficients=(1.0,))
    with pytest.raises(ValueError, match="one dtype"):
        mp.orthogonalise([x[0], x[0].double()])


def test_cpu_tensors_are_refused_what_gpu_tensors_are() -> None:
    x, w = torch.ones(4, 8), torch.ones(8)
    for eps in (-1.0, float("nan"), float("inf")):
        for call in (lambda: mp.rms_norm(x, w, eps=eps), lambda: mp.add_rms_norm(x, x, w, eps=eps),
                     lambda: mp.add_rms_norm_fp8(x, x, w, eps=eps), lambda: mp.orthogonalise(x, eps=eps)):
            with pytest.raises(RuntimeError, match="eps"):
                call()
    for steps in (0, -1, 65, 1 << 40, 5 - (1 << 32)):
        with pytest.raises(RuntimeError, match="steps"):
            mp.orthogonalise(x, steps=steps)
    for coefficients in ((4.0, 0.0, 0.0), (float("nan"), 0.0, 0.0), (1.0, float("inf"), 0.0)):
        with pytest.raises(RuntimeError, match="past 2"):
            mp.orthogonalise(x, coefficients=coefficients)
    assert mp.orthogonalise([], steps=0) == []


# ---- the attention's plan ---------------------------------------------------------------------


@pytest.fixture(scope="module")
def capi():
    from relmo_amd import capi as c

    if not c.LIB_PATH.exists():
        pytest.skip("librelm_mp_hip.so is not built (run __graft_entry__.build())")
    return c


def _i64(values):
    return (ctypes.c_int64 * len(values))(*values)


def _offsets(counts):
    total, out = 0, [0]
    for c in counts:
        total += c
        out.append(total)
    return out


def _build(capi, queries, keys, heads, kv_heads):
    qo, ko = _offsets(queries), _offsets(keys)
    plan = capi.AttentionPlan()
    args = (_i64(qo), _i64(ko), len(queries), qo[-1], ko[-1], heads, kv_heads)
    capi.check(capi.lib().relm_mp_attention_plan_build(*args, None, 0, ctypes.byref(plan)))
    table = (ctypes.c_int32 * max(plan.table_bytes // 4, 1))()
    capi.check(capi.lib().relm_mp_attention_plan_build(*args, table, plan.table_bytes, ctypes.byref(plan)))
    records = [tuple(table[i:i + 8]) for i in range(0, plan.table_bytes // 4, 8)]
    cut = [plan.num_items, plan.num_idle_items, plan.num_joins, plan.num_key_items, plan.num_key_joins]
    parts, at = [], 0
    for n in cut:
        parts.append(records[at:at + n])
        at += n
    assert at == len(records)
    return plan, parts


@pytest.mark.parametrize("queries,keys,heads,kv_heads", [
    ([1], [200], 4, 4), ([1], [262_147], 8, 2), ([3, 0, 40], [0, 9, 64], 2, 1), ([8] * 512, [200] * 512, 2, 2),
    ([2048] * 4, [4096] * 4, 16, 4), ([100_003, 1], [5, 70_001], 1, 1), ([0, 0], [7, 0], 1, 1), ([], [], 1, 1),
    ([700, 3, 0, 12], [1, 90_000, 128, 129], 6, 3)])
def test_plan_covers_every_pair_once(capi, queries, keys, heads, kv_heads) -> None:
    """Every (row, key) of every graph lies in exactly one row item and one key item, parts are numbered once and
    joined completely, and nothing reaches past its graph."""

    plan, (items, idle, joins, key_items, key_joins) = _build(capi, queries, keys, heads, kv_heads)
    group = heads // kv_heads
    qo, ko = _offsets(queries), _offsets(keys)
    graph_of = {}
    for b, n in enumerate(queries):
        if n:
            graph_of[qo[b]] = b
    want = sum(n * group * max(k, 0) for n, k in zip(queries, keys))

    def check(records, tile_rows, tile_keys):
        pairs, seen, parts = 0, set(), []
        for q_first, row0, rows, key_first, n, part, *_ in records:
            assert 0 <= rows <= tile_rows and 0 <= n <= tile_keys
            if rows:
                b = graph_of[q_first]
                assert row0 + rows <= queries[b] * group and ko[b] <= key_first and key_first + n <= ko[b + 1]
                pairs += rows * n
            assert (q_first, row0, key_first, rows, n) not in seen
            seen.add((q_first, row0, key_first, rows, n))
            if part >= 0:
                parts.append(part)
        assert pairs == want and sorted(parts) == list(range(len(parts)))
        return len(parts)

    big = 1 << 30
    assert check(items, plan.row_tile, big) == plan.num_parts == sum(j[6] for j in joins)
    assert check(key_items, big, plan.key_tile) == plan.num_key_parts == sum(j[6] for j in key_joins)
    # every row is written and every key; keys that no query reads are listed apart
    assert {(r[3], r[4]) for r in idle} == {(ko[b], k) for b, k in enumerate(keys) if k and not queries[b]}
    assert all(r[2] == 0 and r[5] < 0 for r in idle)
    rows_whole = sum(r[2] for r in items if r[5] < 0) + sum(j[2] for j in joins)
    assert rows_whole == sum(queries) * group
    keys_whole = sum(r[4] for r in key_items if r[5] < 0) + sum(j[4] for j in key_joins)
    assert keys_whole == sum(keys)
    for j in joins:
        parts = [r for r in items if j[5] <= r[5] < j[5] + j[6]]
        assert len(parts) == j[6] and {(r[0], r[1], r[2]) for r in parts} == {j[:3]}
    for j in key_joins:
        parts = [r for r in key_items if j[5] <= r[5] < j[5] + j[6]]
        assert len(parts) == j[6] and {(r[3], r[4]) for r in parts} == {(j[3], j[4])}


@pytest.mark.parametrize("queries,keys", [([0], [1 << 27]), ([3, 0, 0, 2], [50, 1_000_001, 4, 0]), ([0, 0], [1024, 1025])])
def test_keys_without_queries_are_cut_into_short_ranges(capi, queries, keys) -> None:
    """A graph's keys that no query reads are listed once each, in order, in ranges short enough that a workgroup's
    share of them (keys times quarters of 128 values) counts in 32 bits and that many workgroups share a long graph."""

    plan, (_items, idle, *_rest) = _build(capi, queries, keys, 1, 1)
    ko = _offsets(keys)
    at = {ko[b]: ko[b + 1] for b, n in enumerate(queries) if n == 0 and keys[b]}
    for _q, _r, rows, first, n, part, *_ in idle:
        assert rows == 0 and part < 0 and 1 <= n <= 4096 and n * 32 < 1 << 31
        at_now = [k for k in at if k == first]
        assert at_now, first  # starts where the range before it ended
        end = at.pop(first)
        if first + n < end:
            at[first + n] = end
        else:
            assert first + n == end
    assert not at


def test_plan_refusals(capi) -> None:
    plan = capi.AttentionPlan()

    def rc(qo, ko, graphs, nq, nk, heads, kv_heads):
        return capi.lib().relm_mp_attention_plan_build(_i64(qo), _i64(ko), graphs, nq, nk, heads, kv_heads, None, 0,
                                                       ctypes.byref(plan))

    assert rc([0, 2], [0, 3], 1, 2, 3, 2, 1) == capi.OK
    for bad in (([1, 2], [0, 3], 1, 2, 3, 1, 1), ([0, 2], [0, 3], 1, 3, 3, 1, 1), ([0, 2, 1], [0, 1, 1], 2, 1, 1, 1, 1),
                ([0, 2], [0, 3], 1, 2, 3, 3, 2), ([0, 2], [0, 3], 1, 2, 3, 0, 0), ([0, 2], [0, 3], 1, 2, 3, 8192, 1),
                ([0, 1 << 31], [0, 3], 1, 1 << 31, 3, 1, 1), ([0, 1 << 30], [0, 3], 1, 1 << 30, 3, 4, 1)):
        assert rc(*bad) == capi.ERR_INVALID_ARGUMENT, bad
        assert "attention plan" in capi.last_error()
    assert capi.lib().relm_mp_attention_plan_build(None, None, 1, 1, 1, 1, 1, None, 0, ctypes.byref(plan)) == \
        capi.ERR_INVALID_ARGUMENT
    small = (ctypes.c_int32 * 8)()
    assert capi.lib().relm_mp_attention_plan_build(_i64([0, 2]), _i64([0, 3]), 1, 2, 3, 1, 1, small, 32,
                                                   ctypes.byref(plan)) == capi.ERR_WORKSPACE


def test_plans_past_the_table_are_refused_before_they_are_laid_out() -> None:
    """The longest lengths, whose pairs do not count in 64 bits: refused by their counts, in little memory."""

    import subprocess
    import sys

    code = """
import ctypes, resource
from relmo_amd import capi
lib = capi.lib()
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (256 << 20), resource.getrlimit(resource.RLIMIT_AS)[1]))
most = (1 << 31) - 2
plan = capi.AttentionPlan()
for nq, nk, heads, kv_heads in ((most, most, 4096, 4096), (most, most, 1, 1), (most, 1, 1, 1), (0, most, 1, 1), (most // 4096, most, 4096, 1)):
    o = [(ctypes.c_int64 * 2)(0, n) for n in (nq, nk)]
    rc = lib.relm_mp_attention_plan_build(o[0], o[1], 1, nq, nk, heads, kv_heads, None, 0, ctypes.byref(plan))
    print(rc, capi.last_error())
"""
    from pathlib import Path

    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100,
                         cwd=Path(__file__).resolve().parent.parent)
    assert run.returncode == 0, run.stderr[-2000:]
    lines = run.stdout.strip().splitlines()
    assert len(lines) == 5
    for line in lines:
        assert line.startswith("1 ") and "too many queries and keys" in line, lines


@pytest.mark.parametrize("struct", ["relm_mp_attention_plan", "relm_mp_head_rows", "relm_mp_update"])
def test_readout_struct_layouts_match_header(tmp_path, capi, struct) -> None:
    import subprocess
    from pathlib import Path

    include = Path(__file__).resolve().parent.parent / "include"
    mirror = {"relm_mp_attention_plan": capi.AttentionPlan, "relm_mp_head_rows": capi.HeadRows,
              "relm_mp_update": capi.Update}[struct]
    fields = [(name, "in" if name == "src" else name) for name, _ in mirror._fields_]
    body = "\n".join(f'    printf("{f} %zu\\n", offsetof({struct}, {c}));' for f, c in fields)
    prog = tmp_path / "layout.c"
    prog.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"relm_mp.h\"\n"
                    f"int main(void) {{\n    printf(\"sizeof %zu\\n\", sizeof({struct}));\n{body}\n    return 0;\n}}\n")
    subprocess.run(["gcc", "-std=c11", f"-I{include}", str(prog), "-o", str(tmp_path / "layout")], check=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                                                        check=True).stdout.splitlines())
    assert int(out["sizeof"]) == ctypes.sizeof(mirror)
    for f, _ in fields:
        assert int(out[f]) == getattr(mirror, f).offset, f
