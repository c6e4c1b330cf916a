"""gemm: BF16 / FP16 GEMM with autograd, on the tcgen05 kernels of the FP8 path run with 16-bit operands.

Operator surface and data flow follow primus_turbo/pytorch/ops/gemm.py of the reference (GemmFunction, gemm).  gemm_bias_act, which
the reference lacks, adds bias, activation and residual in the product's epilogue and serves single tokens as well as prompts.
"""
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from ..kernels.gemm.gemm_impl import (
    act_bias_bwd_impl,
    bias_act_dgrad_impl,
    bias_act_wgrad_impl,
    check_gemm_bias_act,
    gemm_accum_impl,
    gemm_bias_act_impl,
    gemm_impl,
)
from .utils import _forward_ad_active, _get_dummy_wgrad, _setup_fused_grad_accum

__all__ = ["gemm", "gemm_bias_act"]


class GemmFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, trans_a, trans_b, out_dtype, fuse_bgrad_accum_pattern=None):
        assert a.dim() == 2 and b.dim() == 2, "Only 2D GEMM is supported"
        fuse, main_grad = _setup_fused_grad_accum(b, fuse_bgrad_accum_pattern)
        out = gemm_impl(a, trans_a, b, trans_b, out_dtype, False)
        ctx.save_for_backward(a, b)
        ctx.trans_a, ctx.trans_b, ctx.fuse, ctx.main_grad = trans_a, trans_b, fuse, main_grad
        return out

    @staticmethod
    def backward(ctx, grad_out):
        a, b = ctx.saved_tensors
        grad_out = grad_out.contiguous()
        if grad_out.dtype != a.dtype:
            grad_out = grad_out.to(a.dtype)
        grad_a = gemm_impl(grad_out, False, b, not ctx.trans_b, a.dtype, ctx.trans_a)      # grad_out . b^T
        if ctx.fuse:
            gemm_accum_impl(a, not ctx.trans_a, grad_out, False, b.dtype, ctx.trans_b, out=ctx.main_grad)
            grad_b = _get_dummy_wgrad(b.shape, b.dtype, device=b.device)
        else:
            grad_b = gemm_impl(a, not ctx.trans_a, grad_out, False, b.dtype, ctx.trans_b)  # a^T . grad_out
        return grad_a, grad_b, None, None, None, None


def gemm(a: torch.Tensor, b: torch.Tensor, trans_a: bool = False, trans_b: bool = False, out_dtype: Optional[torch.dtype] = None,
         fuse_bgrad_accum_pattern: Union[None, str] = None) -> torch.Tensor:
    """out = op(a) . op(b) for 2-D bf16 / fp16 tensors; fp32 accumulate."""
    if out_dtype is None:
        out_dtype = torch.result_type(a, b)
    return GemmFunction.apply(a, b, trans_a, trans_b, out_dtype, fuse_bgrad_accum_pattern)


class GemmBiasActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, bias, residual, trans_b, act, out_dtype, fuse_bgrad_accum_pattern):
        fuse, main_grad = _setup_fused_grad_accum(b, fuse_bgrad_accum_pattern)
        out, z = gemm_bias_act_impl(a, b, trans_b, bias, act, residual, out_dtype, act is not None and any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(a, b, z)
        ctx.trans_b, ctx.act, ctx.fuse, ctx.main_grad = trans_b, act, fuse, main_grad
        ctx.bias_dtype = None if bias is None else bias.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        a, b, z = ctx.saved_tensors
        need_a, need_b, need_bias, need_residual = ctx.needs_input_grad[:4]
        grad_a = grad_b = grad_bias = None
        if need_a or need_b or need_bias:
            dz, grad_bias = act_bias_bwd_impl(grad_out, z, ctx.act, a.dtype, ctx.bias_dtype if need_bias else None, need_a or need_b)
        # an empty contraction (no columns for grad_a, no rows for grad_b) is a sum of nothing
        if need_a:                                                                         # dz . op(b)^T
            grad_a = bias_act_dgrad_impl(dz, b, ctx.trans_b) if dz.shape[1] else torch.zeros_like(a)
        if need_b and ctx.fuse:
            if a.shape[0]:
                bias_act_wgrad_impl(a, dz, ctx.trans_b, out=ctx.main_grad)
            grad_b = _get_dummy_wgrad(b.shape, b.dtype, device=b.device)
        elif need_b:                                                                       # a^T . dz
            grad_b = bias_act_wgrad_impl(a, dz, ctx.trans_b) if a.shape[0] else torch.zeros_like(b)
        return grad_a, grad_b, grad_bias, (grad_out if need_residual else None), None, None, None, None


def gemm_bias_act(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                  residual: Optional[torch.Tensor] = None, trans_b: bool = False, out_dtype: Optional[torch.dtype] = None,
                  fuse_bgrad_accum_pattern: Union[None, str] = None) -> torch.Tensor:
    """out = act(a . op(b) + bias) + residual for 2-D bf16 / fp16 tensors in one kernel; fp32 accumulate, rounded once.

    activation: None, "relu", "silu", "gelu" (erf form) or "gelu_tanh".  bias [N] in a's dtype or fp32; residual [M, N] in out_dtype
    (a's dtype by default).  Few rows (a decoding batch) run on a kernel that streams the weight over all SMs.  A contraction that is
    not a multiple of 8 is padded first (copies of a and b), as in gemm.  Differentiable in a, b, bias and residual.  When an activation
    needs it the pre-activation is kept for the backward in a's dtype, half of fp32's memory: the slope is taken at the rounded value (in
    fp16 a positive one below 2^-25 is kept as zero, where ReLU's slope is zero), and the gradient behind the activation is rounded once to
    a's dtype, the operand type of the two products that follow."""
    out_dtype = a.dtype if out_dtype is None else out_dtype
    check_gemm_bias_act(a, b, trans_b, bias, activation, residual, out_dtype)
    grad = a.requires_grad or b.requires_grad or (bias is not None and bias.requires_grad) or (residual is not None and residual.requires_grad)
    if (grad and torch.is_grad_enabled()) or _forward_ad_active():
        return GemmBiasActFunction.apply(a, b, bias, residual, trans_b, activation, out_dtype, fuse_bgrad_accum_pattern)
    return gemm_bias_act_impl(a, b, trans_b, bias, activation, residual, out_dtype, False)[0]
