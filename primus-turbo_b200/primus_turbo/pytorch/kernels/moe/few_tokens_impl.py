"""A whole mixture-of-experts layer for few tokens over the C ABI (two launches)."""
import torch

from .. import _native as nv
from ..activation.glu_impl import ACT_CODES

MAX_TOKENS, MAX_EXPERTS, MAX_TOP_K, MAX_SLOTS = 128, 1024, 32, 2048


def check_moe_few_tokens(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, topk_indices: torch.Tensor, topk_probs: torch.Tensor,
                         act: str) -> None:
    """Refuses what the kernels do not take: everything that they trust, but for the layout, which the call below makes."""
    assert act in ACT_CODES, f"Unsupported act_type: {act}. Supported types: {list(ACT_CODES)}"
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


def moe_few_tokens_impl(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, topk_indices: torch.Tensor, topk_probs: torch.Tensor,
                        act: str) -> torch.Tensor:
    check_moe_few_tokens(x, gate_up, down, topk_indices, topk_probs, act)
    nv.require_cuda(x, gate_up, down, topk_indices, topk_probs)
    x, gate_up, down = x.contiguous(), gate_up.contiguous(), down.contiguous()
    topk_indices, topk_probs = topk_indices.contiguous(), topk_probs.contiguous()
    T, H = x.shape
    E, I = down.shape[0], down.shape[2]
    K = topk_indices.shape[1]
    if x.data_ptr() % 16:      # a view into a larger buffer; TMA reads from 16-byte boundaries
        x = x.clone()
    out = x.new_empty((T, H))
    lib = nv.lib()
    nbytes = lib.pt_moe_few_tokens_scratch_bytes(T, K, I)
    scratch = torch.empty((nbytes,), dtype=torch.uint8, device=x.device)
    with nv.on_device(x.device):
        nv.check(lib.pt_moe_few_tokens(nv.ptr(x), nv.ptr(gate_up), nv.ptr(down), nv.src_code(x.dtype), nv.ptr(topk_indices),
                                       topk_indices.element_size(), nv.ptr(topk_probs), T, E, K, H, I, ACT_CODES[act], nv.ptr(scratch), nbytes,
                                       nv.ptr(out), nv.mapped_status(x.device), nv.stream(x.device)), "moe_few_tokens")
    nv.launched(x.device)
    return out
