"""A whole mixture-of-experts layer for few tokens over the C ABI (two launches)."""
import torch

from .. import _native as nv
from ..activation.glu_impl import ACT_CODES

MAX_TOKENS, MAX_EXPERTS, MAX_TOP_K, MAX_SLOTS = 128, 1024, 32, 2048


def moe_few_tokens_impl(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, topk_indices: torch.Tensor, topk_probs: torch.Tensor,
                        act: str) -> torch.Tensor:
    nv.require_cuda(x, gate_up, down, topk_indices, topk_probs)
    T, H = x.shape
    E, I = down.shape[0], down.shape[2]
    K = topk_indices.shape[1]
    if x.data_ptr() % 16:      # a view into a larger buffer; TMA reads from 16-byte boundaries
        x = x.clone()
    out = torch.empty_like(x)
    lib = nv.lib()
    nbytes = lib.pt_moe_few_tokens_scratch_bytes(T, K, I)
    scratch = torch.empty((nbytes,), dtype=torch.uint8, device=x.device)
    with nv.on_device(x.device):
        nv.check(lib.pt_moe_few_tokens(nv.ptr(x), nv.ptr(gate_up), nv.ptr(down), nv.src_code(x.dtype), nv.ptr(topk_indices),
                                       topk_indices.element_size(), nv.ptr(topk_probs), T, E, K, H, I, ACT_CODES[act], nv.ptr(scratch), nbytes,
                                       nv.ptr(out), nv.mapped_status(x.device), nv.stream(x.device)), "moe_few_tokens")
    return out
