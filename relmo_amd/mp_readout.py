"""The readout ops of the facade: what a program runs on the object states.

``add_rms_norm`` (a residual stream's norm, also with an 8-bit output),
``cross_attention`` (per-graph queries to the graphs' objects) and ``orthogonalise``
(the weight updates of what they train), without counterparts in relmo.  GPU tensors of float32, bfloat16 or float16 run the library's ops, which check
their arguments and make their own autograd nodes (reverse mode once; forward mode raises); CPU tensors (and the policy's fallback)
run the ATen formulations below, which autograd differentiates.
"""

from __future__ import annotations

from .mp_dispatch import library_op
from .mp_runtime import torch

FP8_MAX = 448.0
FLOAT_MAX = 3.4028234663852886e38  # the library's constants are float32
ORTHO_STEPS = 64


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- residual norm ---------------------------------------------------------------


def _eps_check(op_name: str, eps: float) -> None:
    if not 0.0 <= eps <= FLOAT_MAX:
        raise RuntimeError(f"{op_name}: eps must be finite and not negative.")


def _norm_checks(op_name: str, x, residual, weight, eps: float) -> None:
    if x.dim() < 1 or weight.dim() != 1 or weight.size(0) != x.size(-1):
        raise ValueError(f"{op_name} expects x [..., width] and weight [width].")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"{op_name} expects residual to have the shape of x.")
    for name, t in (("residual", residual), ("weight", weight)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{op_name} expects {name} to have the dtype and device of x.")
    _eps_check(op_name, eps)


def _norm_float(x, residual, weight, eps: float):
    """(y, h) unrounded, at least in float32."""

    wide = torch.promote_types(x.dtype, torch.float32)
    h = x.to(wide) if residual is None else x.to(wide) + residual.to(wide)
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * weight.to(wide), h


def add_rms_norm(x, residual, weight, eps: float):
    if residual is None:
        return rms_norm(x, weight, eps), x
    op = library_op("add_rms_norm", tensor=x, gpu_only=True)
    if op is not None:
        return op(x, residual, weight, eps)
    _norm_checks("add_rms_norm", x, residual, weight, eps)
    y, h = _norm_float(x, residual, weight, eps)
    return y.to(x.dtype), h.to(x.dtype)


def rms_norm(x, weight, eps: float):
    op = library_op("rms_norm", tensor=x, gpu_only=True)
    if op is not None:
        return op(x, weight, eps)
    _norm_checks("rms_norm", x, None, weight, eps)
    return _norm_float(x, None, weight, eps)[0].to(x.dtype)


def add_rms_norm_fp8(x, residual, weight, eps: float):
    if _wants_grad(x, residual, weight):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad(), or add_rms_norm to train.")
    op = library_op("add_rms_norm_fp8", tensor=x, gpu_only=True)
    if op is not None:
        q, scale, h = op(x, residual, weight, eps)
        return q, scale, x if residual is None else h
    _norm_checks("add_rms_norm_fp8", x, residual, weight, eps)
    y, h = _norm_float(x, residual, weight, eps)
    scale = (y.abs().amax(-1) if x.size(-1) else y.new_zeros(x.shape[:-1])) / FP8_MAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale).to(torch.float32)
    q = (y / scale.unsqueeze(-1).to(y.dtype)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, scale, x if residual is None else h.to(x.dtype)


# ---- cross attention ---------------------------------------------------------------


class AttentionPlan:
    """The lengths of a batch's graphs and, on the GPU, how their attention is laid over the device.

    ``q_offsets`` and ``k_offsets`` are the plan's own, in host memory."""

    def __init__(self, q_offsets, k_offsets, heads: int, kv_heads: int, ref=None, number: int | None = None):
        self.q_offsets, self.k_offsets = q_offsets, k_offsets
        self.heads, self.kv_heads = heads, kv_heads
        self._ref = ref        # keeps the library's plan, which the op finds by its number
        self.number = number


def attention_plan(q_offsets, k_offsets, heads: int, kv_heads: int | None) -> AttentionPlan:
    heads = int(heads)
    kv_heads = heads if kv_heads is None else int(kv_heads)
    if heads < 1 or kv_heads < 1 or heads % kv_heads != 0:
        raise ValueError("attention_plan expects heads to be a multiple of kv_heads.")
    for name, t in (("q_offsets", q_offsets), ("k_offsets", k_offsets)):
        if t.dim() != 1 or t.dtype != torch.int64 or t.numel() < 1 or t.numel() != q_offsets.numel():
            raise ValueError(f"attention_plan expects {name} to be int64 [graphs + 1].")
    op = library_op("attention_plan", tensor=q_offsets, gpu_only=True)
    if op is not None:
        ref, number, own = op(q_offsets, k_offsets, heads, kv_heads)
        return AttentionPlan(own[0], own[1], heads, kv_heads, ref, number)
    q_offsets, k_offsets = (t.detach().to("cpu", copy=True) for t in (q_offsets, k_offsets))
    for name, t in (("q_offsets", q_offsets), ("k_offsets", k_offsets)):
        if int(t[0]) != 0 or bool((t[1:] < t[:-1]).any()):
            raise RuntimeError(f"relm_mp attention plan: {name} must ascend from 0.")
    return AttentionPlan(q_offsets, k_offsets, heads, kv_heads)


def _attention_checks(q, k, v, plan, key_mask, scale: float) -> None:
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.size(2) != k.size(2):
        raise ValueError("cross_attention expects q [queries, heads, head_dim] and k, v [keys, kv_heads, head_dim].")
    if q.size(1) != plan.heads or k.size(1) != plan.kv_heads:
        raise ValueError("cross_attention expects the plan's heads and kv_heads.")
    for name, t in (("k", k), ("v", v)):
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"cross_attention expects {name} to have the dtype and device of q.")
    if key_mask is not None and (key_mask.dtype != torch.bool or key_mask.shape != k.shape[:1] or key_mask.device != q.device):
        raise ValueError("cross_attention expects key_mask to be bool [keys] on the device of q.")
    if not 0.0 < scale < float("inf"):
        raise ValueError("cross_attention expects a finite, positive scale.")


def cross_attention_python(q, k, v, plan, key_mask, scale: float):
    """Graph by graph in ATen, in at least float32: the facade's formulation for CPU tensors."""

    group, dim = plan.heads // plan.kv_heads, q.size(2)
    wide = torch.promote_types(q.dtype, torch.float32)
    qo, ko = plan.q_offsets.tolist(), plan.k_offsets.tolist()
    if qo[-1] != q.size(0) or ko[-1] != k.size(0):
        raise ValueError("cross_attention expects the plan's numbers of queries and keys.")
    outs = [q.new_zeros(0, plan.heads, dim, dtype=wide)]
    for b in range(len(qo) - 1):
        n = qo[b + 1] - qo[b]
        qb = q[qo[b]:qo[b + 1]].to(wide).view(n, plan.kv_heads, group, dim).permute(1, 2, 0, 3)
        kb, vb = (t[ko[b]:ko[b + 1]] for t in (k, v))
        if key_mask is not None:
            kept = key_mask[ko[b]:ko[b + 1]]
            kb, vb = kb[kept], vb[kept]
        kb, vb = (t.to(wide).permute(1, 0, 2).unsqueeze(1) for t in (kb, vb))
        if kb.size(2) == 0:
            outs.append(q.new_zeros(n, plan.heads, dim, dtype=wide))
            continue
        p = torch.softmax(qb.matmul(kb.transpose(2, 3)) * scale, 3)
        outs.append(p.matmul(vb).permute(2, 0, 1, 3).reshape(n, plan.heads, dim))
    return torch.cat(outs).to(q.dtype)


def cross_attention(q, k, v, plan, key_mask, scale: float | None):
    if scale is None:
        scale = max(q.size(-1), 1) ** -0.5
    op = library_op("cross_attention", tensor=q, gpu_only=True)
    if op is None:
        _attention_checks(q, k, v, plan, key_mask, scale)
        return cross_attention_python(q, k, v, plan, key_mask, scale)
    if plan.number is None:
        raise ValueError("cross_attention expects a plan made from offsets on the GPU.")
    return op(q, k, v, plan.number, key_mask, scale)


# ---- orthogonalised update ---------------------------------------------------------


def _orthogonalise_checks(steps: int, coefficients, eps: float) -> None:
    """What the library refuses: among it polynomials that take values of [0, 1] past 2, on the same grid of them."""

    if not 1 <= steps <= ORTHO_STEPS:
        raise RuntimeError(f"orthogonalise: steps must be in [1, {ORTHO_STEPS}].")
    _eps_check("orthogonalise", eps)
    a, b, c = coefficients
    x = torch.linspace(0.0, 1.0, 1025, dtype=torch.float64)
    within = torch.ones((), dtype=torch.bool)
    for _ in range(steps):
        square = x.square()
        x = (a + b * square + c * square.square()) * x
        within = within & (x.abs() <= 2.0).all()
    if not bool(within):
        raise RuntimeError("orthogonalise: these coefficients take singular values past 2.")


def _orthogonalise_float(update, steps: int, coefficients, eps: float):
    a, b, c = coefficients
    x = update.to(torch.promote_types(update.dtype, torch.float32))
    tall = x.size(-2) > x.size(-1)
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if tall else x).to(update.dtype).contiguous()


def orthogonalise(updates, steps: int, coefficients, eps: float):
    one = torch.is_tensor(updates)
    parts = [updates] if one else list(updates)
    coefficients = [float(v) for v in coefficients]
    if len(coefficients) != 3:
        raise ValueError("orthogonalise expects three coefficients.")
    for u in parts:
        if u.dim() < 2:
            raise ValueError("orthogonalise expects matrices or stacks of them.")
        if u.dtype != parts[0].dtype or u.device != parts[0].device:
            raise ValueError("orthogonalise expects updates of one dtype on one device.")
    op = library_op("orthogonalise", tensor=parts[0], gpu_only=True) if parts else None
    with torch.no_grad():
        if op is not None:
            results = op(parts, int(steps), coefficients, float(eps))
        else:
            if parts:
                _orthogonalise_checks(int(steps), coefficients, eps)
            results = [_orthogonalise_float(u, int(steps), coefficients, eps) for u in parts]
    return results[0] if one else results


__all__ = ["AttentionPlan", "add_rms_norm", "add_rms_norm_fp8", "attention_plan", "cross_attention",
           "orthogonalise", "rms_norm"]
