"""rmsnorm / rmsnorm_residual with autograd; interface of primus_turbo/pytorch/ops/normalization.py of the reference.
qk_norm_rope, which the reference lacks: the norm of every query and key head and the position rotation in one pass."""
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from ..kernels.normalization.qk_norm_rope_impl import qk_norm_rope_args, qk_norm_rope_bwd_impl, qk_norm_rope_fwd_impl

from ..kernels.normalization.rmsnorm_impl import (
    rmsnorm_bwd_impl,
    rmsnorm_bwd_residual_impl,
    rmsnorm_fwd_impl,
    rmsnorm_fwd_residual_impl,
)
from .utils import _forward_ad_active

__all__ = ["rmsnorm", "rmsnorm_residual", "qk_norm_rope"]


class _RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, eps=1e-6, zero_centered=False):
        assert x.is_cuda and gamma.is_cuda, "rmsnorm: x and gamma must be CUDA tensors"
        H = gamma.shape[0]
        assert x.shape[-1] == H, f"rmsnorm: last dim of x ({x.shape[-1]}) must equal gamma.shape[0] ({H})"
        y, x2, rstd = rmsnorm_fwd_impl(x, gamma, eps, zero_centered)
        ctx.save_for_backward(x2, gamma, rstd)
        ctx.zero_centered, ctx.orig_shape = zero_centered, x.shape
        return y.reshape(x.shape)

    @staticmethod
    def backward(ctx, grad_out):
        x2, gamma, rstd = ctx.saved_tensors
        dx, dg = rmsnorm_bwd_impl(grad_out, x2, gamma, rstd, ctx.zero_centered)
        return dx.reshape(ctx.orig_shape), dg, None, None


class _RMSNormResidualFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gamma, eps=1e-6):
        assert x.is_cuda and residual.is_cuda and gamma.is_cuda, "rmsnorm_residual: x, residual and gamma must be CUDA tensors"
        assert x.shape == residual.shape, f"rmsnorm_residual: shape mismatch {tuple(x.shape)} vs {tuple(residual.shape)}"
        assert x.shape[-1] == gamma.shape[0]
        y, x_plus_r, rstd = rmsnorm_fwd_residual_impl(x, residual, gamma, eps)
        ctx.save_for_backward(x_plus_r, gamma, rstd)
        ctx.orig_shape = x.shape
        return y.reshape(x.shape), x_plus_r.reshape(x.shape)

    @staticmethod
    def backward(ctx, grad_y, grad_xpr):
        x_plus_r, gamma, rstd = ctx.saved_tensors
        dx, dg = rmsnorm_bwd_residual_impl(grad_y, grad_xpr, x_plus_r, gamma, rstd)
        dx = dx.reshape(ctx.orig_shape)
        return dx, dx, dg, None   # the add sends the same gradient to x and to the residual


def rmsnorm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6, zero_centered: bool = False) -> torch.Tensor:
    """y = x * rsqrt(mean(x^2, -1) + eps) * (gamma, or 1 + gamma when zero_centered); statistics in fp32."""
    return _RMSNormFunction.apply(x, gamma, eps, zero_centered)


def rmsnorm_residual(x: torch.Tensor, residual: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(rmsnorm(x + residual), x + residual) in one pass over the row."""
    return _RMSNormResidualFunction.apply(x, residual, gamma, eps)


class _QKNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_gamma, k_gamma, cos, sin, positions, eps, interleaved, zero_centered):
        ctx.save_for_backward(q, k, q_gamma, k_gamma, cos, sin, positions)
        ctx.options = (eps, interleaved, zero_centered)
        return qk_norm_rope_fwd_impl(q, k, q_gamma, k_gamma, cos, sin, positions, eps, interleaved, zero_centered)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, q_gamma, k_gamma, cos, sin, positions = ctx.saved_tensors
        dq, dk = (d.to(q.dtype) if d.stride(-1) == 1 else d.to(q.dtype).contiguous() for d in (dq, dk))
        return (*qk_norm_rope_bwd_impl(dq, dk, q, k, q_gamma, k_gamma, cos, sin, positions, *ctx.options),) + (None,) * 6


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_gamma: torch.Tensor, k_gamma: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                 zero_centered: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head, then the position rotation: (q_out, k_out), contiguous, in one pass.

    q [..., tokens, Hq, D] and k [..., tokens, Hk, D]: bf16, fp16 or fp32, any strides with a contiguous last dimension (views
    into a packed projection are read in place).  q_gamma, k_gamma [D] in the same dtype; cos, sin fp32 [P, R / 2].
    n = x * rsqrt(mean(x^2, -1) + eps) * (gamma, or 1 + gamma when zero_centered); the first R elements of n are rotated in pairs
    (i, i + R / 2), or (2 i, 2 i + 1) when interleaved, by cos / sin of the token's position; elements from R on pass through.
    positions: int32 / int64 of the shape [..., tokens]; None: 0, 1, ... along the token dimension.  A position outside of
    [0, P) gives zeros for its token and an error at a following call.  Differentiable in q, k and the gains."""
    args = (*qk_norm_rope_args(q, k, q_gamma, k_gamma, cos, sin, positions), eps, interleaved, zero_centered)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_gamma.requires_grad or k_gamma.requires_grad or
                                     cos.requires_grad or sin.requires_grad)) or _forward_ad_active():
        assert not (cos.requires_grad or sin.requires_grad), "qk_norm_rope: the tables are not differentiated"
        q_out, k_out = _QKNormRopeFunction.apply(*args)
    else:
        q_out, k_out = qk_norm_rope_fwd_impl(*args)
    return (q_out, k_out) if q.dim() <= 4 else (q_out.view(q.shape), k_out.view(k.shape))
