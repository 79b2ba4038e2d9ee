"""The readout ops of the facade: what a program runs on the object states.

``add_rms_norm`` (a residual stream's norm, also with an 8-bit output) without a
counterpart in relmo.  GPU tensors of float32, bfloat16 or float16 run the
library's kernels through autograd functions; CPU tensors (and the policy's
fallback) run the ATen formulations below, which autograd differentiates.
"""

from __future__ import annotations

from .mp_dispatch import library_op
from .mp_runtime import ops_namespace, torch

FP8_MAX = 448.0


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- residual norm ---------------------------------------------------------------


def _norm_checks(op_name: str, x, residual, weight) -> None:
    if x.dim() < 1 or weight.dim() != 1 or weight.size(0) != x.size(-1):
        raise ValueError(f"{op_name} expects x [..., width] and weight [width].")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"{op_name} expects residual to have the shape of x.")
    for name, t in (("residual", residual), ("weight", weight)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{op_name} expects {name} to have the dtype and device of x.")


def _norm_float(x, residual, weight, eps: float):
    """(y, h) unrounded, at least in float32."""

    wide = torch.promote_types(x.dtype, torch.float32)
    h = x.to(wide) if residual is None else x.to(wide) + residual.to(wide)
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * weight.to(wide), h


if torch is not None:

    class _AddRmsNormFunction(torch.autograd.Function):
        """(y, h); the backward reads h, rounded as it was stored, and the rows' 1 / root."""

        @staticmethod
        def forward(ctx, x, residual, weight, eps):
            y, h, rstd = ops_namespace().add_rms_norm(x, residual, weight, eps, True)
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(h, weight, rstd)
            return y, h

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad_y, grad_h):
            h, weight, rstd = ctx.saved_tensors
            if grad_y is None:
                return grad_h, grad_h, None, None
            dx, dw = ops_namespace().add_rms_norm_backward(grad_y, grad_h, h, weight, rstd)
            return dx, dx, dw, None

    class _RmsNormFunction(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, eps):
            y, _h, rstd = ops_namespace().add_rms_norm(x, None, weight, eps, True)
            ctx.save_for_backward(x, weight, rstd)
            return y

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad_y):
            x, weight, rstd = ctx.saved_tensors
            dx, dw = ops_namespace().add_rms_norm_backward(grad_y, None, x, weight, rstd)
            return dx, dw, None

else:  # pragma: no cover - torch missing
    _AddRmsNormFunction = _RmsNormFunction = None


def add_rms_norm(x, residual, weight, eps: float):
    if residual is None:
        return rms_norm(x, weight, eps), x
    _norm_checks("add_rms_norm", x, residual, weight)
    op = library_op("add_rms_norm", tensor=x, gpu_only=True)
    if op is None:
        y, h = _norm_float(x, residual, weight, eps)
        return y.to(x.dtype), h.to(x.dtype)
    if _wants_grad(x, residual, weight):
        return _AddRmsNormFunction.apply(x, residual, weight, float(eps))
    y, h, _rstd = op(x, residual, weight, float(eps), False)
    return y, h


def rms_norm(x, weight, eps: float):
    _norm_checks("rms_norm", x, None, weight)
    op = library_op("add_rms_norm", tensor=x, gpu_only=True)
    if op is None:
        return _norm_float(x, None, weight, eps)[0].to(x.dtype)
    if _wants_grad(x, weight):
        return _RmsNormFunction.apply(x, weight, float(eps))
    return op(x, None, weight, float(eps), False)[0]


def add_rms_norm_fp8(x, residual, weight, eps: float):
    _norm_checks("add_rms_norm_fp8", x, residual, weight)
    if _wants_grad(x, residual, weight):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad(), or add_rms_norm to train.")
    op = library_op("add_rms_norm_fp8", tensor=x, gpu_only=True)
    if op is not None:
        q, scale, h = op(x, residual, weight, float(eps))
        return q, scale, x if residual is None else h
    y, h = _norm_float(x, residual, weight, eps)
    scale = (y.abs().amax(-1) if x.size(-1) else y.new_zeros(x.shape[:-1])) / FP8_MAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale).to(torch.float32)
    q = (y / scale.unsqueeze(-1).to(y.dtype)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, scale, x if residual is None else h.to(x.dtype)


__all__ = ["add_rms_norm", "add_rms_norm_fp8", "rms_norm"]
