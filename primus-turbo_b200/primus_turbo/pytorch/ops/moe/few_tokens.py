"""moe_few_tokens: a whole mixture-of-experts layer (gate, up, gated activation, down, weighted sum) for few tokens.

The reference composes the layer from token_permute, grouped_gemm, swiglu_with_probs and token_unpermute
(primus_turbo/pytorch/ops/moe/permutation.py, ops/grouped_gemm.py, ops/activation.py), which is the way to train it and to run long
prompts.  For a decoding batch those steps cost more than reading the weights; here the layer is two kernels that stream the chosen
experts' weights once.
"""
import torch
from torch.autograd import forward_ad

from ...kernels.moe.few_tokens_impl import moe_few_tokens_impl
from ..utils import _forward_ad_active

__all__ = ["moe_few_tokens"]


def moe_few_tokens(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, topk_indices: torch.Tensor, topk_probs: torch.Tensor,
                   act_type: str = "silu") -> torch.Tensor:
    """out[t] = sum over j of topk_probs[t, j] * down[e] . (act(gate[e] . x[t]) * (up[e] . x[t])) with e = topk_indices[t, j].

    x [T, H], gate_up [E, 2 I, H] (gate rows first), down [E, H, I], bf16 or fp16, the weights starting on 16-byte boundaries (views into
    a larger buffer that do not are refused; copying all experts would cost more than the layer); topk_indices int32 / int64 and
    topk_probs fp32 [T, K].  An index outside of [0, E), such as -1 for an expert of another shard, adds nothing.  H and I are multiples
    of 8; T at most 128, E 1024, K 32, T * K 2048: longer inputs go through token_permute and grouped_gemm.  Forward only (no gradient).
    act(gate) * up * prob is rounded to x's dtype between the two products, as swiglu_with_probs rounds it: the second product's operand
    type.  In fp16 a value of it beyond 65504 is therefore an infinity, also where the layer's output would be finite.  The weights must be
    finite: the down product multiplies the rows of an expert's weight with zeros for tokens that did not choose it, and an infinity
    would reach them.  act_type: "silu" or "gelu" (erf form)."""
    if torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad or down.requires_grad or topk_probs.requires_grad):
        raise RuntimeError("moe_few_tokens has no backward: call it under torch.no_grad(), or train through token_permute and grouped_gemm")
    if _forward_ad_active() and any(forward_ad.unpack_dual(t).tangent is not None for t in (x, gate_up, down, topk_probs)):
        raise RuntimeError("moe_few_tokens has no forward-mode derivative either")
    return moe_few_tokens_impl(x, gate_up, down, topk_indices, topk_probs, act_type)
