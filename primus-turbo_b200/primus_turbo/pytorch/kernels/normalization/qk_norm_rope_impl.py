"""Per-head RMS norm and position rotation of queries and keys over the C ABI.  Tensors come as [B, S, heads, D] views with a
contiguous last dimension; the kernels take their strides."""
import ctypes
from typing import Optional, Tuple

import torch

from .. import _native as nv

_Strides = ctypes.c_int64 * 3


def _strides(t):
    # the stride of an extent of one is never used, but would decide the alignment of the vector accesses
    return _Strides(*(st if n > 1 else 0 for n, st in zip(t.shape[:3], t.stride()[:3])))


def _pos(positions):
    return (None, 0) if positions is None else (nv.ptr(positions), positions.element_size())


def qk_norm_rope_fwd_impl(q: torch.Tensor, k: torch.Tensor, q_gamma: torch.Tensor, k_gamma: torch.Tensor, cos: torch.Tensor,
                          sin: torch.Tensor, positions: Optional[torch.Tensor], eps: float, interleaved: bool,
                          zero_centered: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (q_out, k_out), contiguous."""
    B, S, Hq, D = q.shape
    Hk, R = k.shape[2], 2 * cos.shape[1]
    q_out = torch.empty((B, S, Hq, D), dtype=q.dtype, device=q.device)
    k_out = torch.empty((B, S, Hk, D), dtype=q.dtype, device=q.device)
    nv.poll_host_status(q.device)
    with nv.on_device(q.device):
        nv.check(nv.lib().pt_qk_norm_rope_fwd(nv.ptr(q), nv.ptr(k), nv.src_code(q.dtype), nv.ptr(q_gamma), nv.ptr(k_gamma), nv.ptr(cos),
                                              nv.ptr(sin), *_pos(positions), B, S, cos.shape[0], Hq, Hk, D, R, _strides(q), _strides(k),
                                              eps, int(interleaved), int(zero_centered), nv.ptr(q_out), nv.ptr(k_out),
                                              nv.host_status(q.device)[2], nv.stream(q.device)), "qk_norm_rope_fwd")
    return q_out, k_out


def qk_norm_rope_bwd_impl(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, q_gamma: torch.Tensor,
                          k_gamma: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor], eps: float,
                          interleaved: bool, zero_centered: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (gradient of q, of k, of q_gamma, of k_gamma)."""
    B, S, Hq, D = q.shape
    Hk, R = k.shape[2], 2 * cos.shape[1]
    q_in = torch.empty((B, S, Hq, D), dtype=q.dtype, device=q.device)
    k_in = torch.empty((B, S, Hk, D), dtype=q.dtype, device=q.device)
    dqg, dkg = torch.empty_like(q_gamma), torch.empty_like(k_gamma)
    lib = nv.lib()
    nv.poll_host_status(q.device)
    with nv.on_device(q.device):
        parts = lib.pt_qk_norm_rope_bwd_parts(B * S, Hq, Hk)
        partial = torch.empty((parts, D), dtype=torch.float32, device=q.device)
        nv.check(lib.pt_qk_norm_rope_bwd(nv.ptr(dq), nv.ptr(dk), nv.ptr(q), nv.ptr(k), nv.src_code(q.dtype), nv.ptr(q_gamma),
                                         nv.ptr(k_gamma), nv.ptr(cos), nv.ptr(sin), *_pos(positions), B, S, cos.shape[0], Hq, Hk, D, R,
                                         _strides(dq), _strides(dk), _strides(q), _strides(k), eps, int(interleaved), int(zero_centered),
                                         nv.ptr(q_in), nv.ptr(k_in), nv.ptr(dqg), nv.ptr(dkg), nv.ptr(partial), parts,
                                         nv.host_status(q.device)[2], nv.stream(q.device)), "qk_norm_rope_bwd")
    return q_in, k_in, dqg, dkg
