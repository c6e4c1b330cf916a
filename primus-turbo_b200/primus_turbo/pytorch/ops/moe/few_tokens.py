"""moe_few_tokens: a whole mixture-of-experts layer (gate, up, gated activation, down, weighted sum) for few tokens.

The reference composes the layer from token_permute, grouped_gemm, swiglu_with_probs and token_unpermute
(primus_turbo/pytorch/ops/moe/permutation.py, ops/grouped_gemm.py, ops/activation.py), which is the way to train it and to run long
prompts.  For a decoding batch those steps cost more than reading the weights; here the layer is two kernels that stream the chosen
experts' weights once.
"""
import torch

from ...kernels.moe.few_tokens_impl import MAX_EXPERTS, MAX_SLOTS, MAX_TOKENS, MAX_TOP_K, moe_few_tokens_impl
from ..activation import SUPPORTED_ACT_TYPES

__all__ = ["moe_few_tokens"]


def moe_few_tokens(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, topk_indices: torch.Tensor, topk_probs: torch.Tensor,
                   act_type: str = "silu") -> torch.Tensor:
    """out[t] = sum over j of topk_probs[t, j] * down[e] . (act(gate[e] . x[t]) * (up[e] . x[t])) with e = topk_indices[t, j].

    x [T, H], gate_up [E, 2 I, H] (gate rows first), down [E, H, I], bf16 or fp16; topk_indices int32 / int64 and topk_probs fp32
    [T, K].  An index outside of [0, E), such as -1 for an expert of another shard, adds nothing.  H and I are multiples of 8;
    T at most 128, E 1024, K 32, T * K 2048: longer inputs go through token_permute and grouped_gemm.  Forward only (no gradient);
    act(gate) * up * prob is rounded to x's dtype between the two products.  The weights must be finite: the down product multiplies
    the rows of an expert's weight with zeros for tokens that did not choose it, and an infinity would reach them.  act_type: "silu" or "gelu" (erf form)."""
    assert act_type in SUPPORTED_ACT_TYPES, f"Unsupported act_type: {act_type}. Supported types: {SUPPORTED_ACT_TYPES}"
    assert x.dim() == 2 and gate_up.dim() == 3 and down.dim() == 3, "moe_few_tokens: x must be [T, H], gate_up [E, 2I, H], down [E, H, I]"
    T, H = x.shape
    E, I = down.shape[0], down.shape[2]
    assert tuple(gate_up.shape) == (E, 2 * I, H) and down.shape[1] == H, \
        f"moe_few_tokens: x {tuple(x.shape)}, gate_up {tuple(gate_up.shape)} and down {tuple(down.shape)} do not fit each other"
    assert x.dtype == gate_up.dtype == down.dtype and x.dtype in (torch.bfloat16, torch.float16), "moe_few_tokens: x and weights must all be bf16 or fp16"
    assert topk_indices.dim() == 2 and topk_indices.shape[0] == T and topk_indices.shape == topk_probs.shape, \
        "moe_few_tokens: topk_indices and topk_probs must be [T, K]"
    K = topk_indices.shape[1]
    assert topk_indices.dtype in (torch.int32, torch.int64), "moe_few_tokens: topk_indices must be int32 or int64"
    assert topk_probs.dtype == torch.float32, "probs must be float32"
    assert H >= 8 and I >= 8 and H % 8 == 0 and I % 8 == 0, f"moe_few_tokens: hidden and expert width must be multiples of 8 (got {H}, {I})"
    assert T <= MAX_TOKENS and 1 <= E <= MAX_EXPERTS and 1 <= K <= MAX_TOP_K and T * K <= MAX_SLOTS, \
        f"moe_few_tokens: takes at most {MAX_TOKENS} tokens, {MAX_EXPERTS} experts, {MAX_TOP_K} per token and {MAX_SLOTS} slots (got {T}, {E}, {K}); " \
        "longer inputs go through token_permute and grouped_gemm"
    index = x.get_device()
    assert gate_up.get_device() == index and down.get_device() == index and topk_indices.get_device() == index and topk_probs.get_device() == index, \
        "moe_few_tokens: all tensors must be on one device"
    if torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad or down.requires_grad or topk_probs.requires_grad):
        raise RuntimeError("moe_few_tokens has no backward: call it under torch.no_grad(), or train through token_permute and grouped_gemm")
    return moe_few_tokens_impl(x.contiguous(), gate_up.contiguous(), down.contiguous(), topk_indices.contiguous(), topk_probs.contiguous(), act_type)
