"""Per-head RMS norm and position rotation of queries and keys over the C ABI.  Tensors come as [S, heads, D] or [B, S, heads, D]
views with a contiguous last dimension; the kernels take their strides."""
import struct
from typing import Optional, Tuple

import torch

from .. import _native as nv

_pack3 = struct.Struct("3q").pack


def _strides(t):
    """(batch, token, head) strides as the int64[3] the C ABI reads."""
    return _pack3(*t.stride()[:3]) if t.dim() == 4 else _pack3(0, *t.stride()[:2])


def _extents(q):
    return q.shape[:2] if q.dim() == 4 else (1, q.shape[0])


def qk_norm_rope_fwd_impl(q: torch.Tensor, k: torch.Tensor, q_gamma: torch.Tensor, k_gamma: torch.Tensor, cos: torch.Tensor,
                          sin: torch.Tensor, positions: Optional[torch.Tensor], eps: float, interleaved: bool,
                          zero_centered: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (q_out, k_out), contiguous."""
    device, dtype = q.device, q.dtype
    B, S = _extents(q)
    (Hq, D), Hk = q.shape[-2:], k.shape[-2]
    P, half = cos.shape
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    status = nv.mapped_status(device)
    with nv.on_device(device):
        nv.check(nv.lib().pt_qk_norm_rope_fwd(q.data_ptr(), k.data_ptr(), nv.src_code(dtype), q_gamma.data_ptr(), k_gamma.data_ptr(),
                                              cos.data_ptr(), sin.data_ptr(), nv.ptr(positions), 0 if positions is None else positions.element_size(),
                                              B, S, P, Hq, Hk, D, 2 * half, _strides(q), _strides(k), eps, interleaved, zero_centered,
                                              q_out.data_ptr(), k_out.data_ptr(), status, nv.stream(device)), "qk_norm_rope_fwd")
    return q_out, k_out


def qk_norm_rope_bwd_impl(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, q_gamma: torch.Tensor,
                          k_gamma: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor], eps: float,
                          interleaved: bool, zero_centered: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (gradient of q, of k, of q_gamma, of k_gamma)."""
    device, dtype = q.device, q.dtype
    B, S = _extents(q)
    (Hq, D), Hk = q.shape[-2:], k.shape[-2]
    P, half = cos.shape
    q_in = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_in = torch.empty_like(k, memory_format=torch.contiguous_format)
    dqg, dkg = torch.empty_like(q_gamma), torch.empty_like(k_gamma)
    lib = nv.lib()
    status = nv.mapped_status(device)
    with nv.on_device(device):
        parts = lib.pt_qk_norm_rope_bwd_parts(B * S, Hq, Hk)
        partial = torch.empty((parts, D), dtype=torch.float32, device=device)
        nv.check(lib.pt_qk_norm_rope_bwd(dq.data_ptr(), dk.data_ptr(), q.data_ptr(), k.data_ptr(), nv.src_code(dtype), q_gamma.data_ptr(),
                                         k_gamma.data_ptr(), cos.data_ptr(), sin.data_ptr(), nv.ptr(positions),
                                         0 if positions is None else positions.element_size(), B, S, P, Hq, Hk, D, 2 * half, _strides(dq),
                                         _strides(dk), _strides(q), _strides(k), eps, interleaved, zero_centered, q_in.data_ptr(),
                                         k_in.data_ptr(), dqg.data_ptr(), dkg.data_ptr(), partial.data_ptr(), parts,
                                         status, nv.stream(device)), "qk_norm_rope_bwd")
    return q_in, k_in, dqg, dkg
