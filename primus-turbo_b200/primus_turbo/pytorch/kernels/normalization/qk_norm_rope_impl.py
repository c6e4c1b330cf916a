"""Per-head RMS norm and position rotation of queries and keys over the C ABI.  qk_norm_rope_args checks a call's tensors and lays them
out as the two functions below it take them: [S, heads, D] or [B, S, heads, D] views with a contiguous last dimension, whose strides the
kernels read, and contiguous gains, tables and positions."""
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


def _as_heads(x):
    """x [..., tokens, heads, D] with three or four dimensions and a contiguous last one, without a copy where its strides allow it."""
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    return x if x.dim() <= 4 else x.flatten(0, -4)


def qk_norm_rope_args(q: torch.Tensor, k: torch.Tensor, q_gamma: torch.Tensor, k_gamma: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                      positions: Optional[torch.Tensor]) -> Tuple[Optional[torch.Tensor], ...]:
    """The same seven tensors as qk_norm_rope_fwd_impl and qk_norm_rope_bwd_impl take them; refuses what does not fit together."""
    index, dtype, D = q.get_device(), q.dtype, q.shape[-1]
    for t in (q, k, q_gamma, k_gamma, cos, sin) if positions is None else (q, k, q_gamma, k_gamma, cos, sin, positions):
        if t.get_device() != index or index < 0:
            if not t.is_cuda:
                raise RuntimeError("primus_turbo (B200) operators take CUDA tensors only; there is no CPU path")
            raise AssertionError("qk_norm_rope: all tensors must be on one device")
    assert dtype in (torch.bfloat16, torch.float16, torch.float32), f"qk_norm_rope: unsupported dtype {dtype}"
    assert k.dtype == dtype == q_gamma.dtype == k_gamma.dtype, "qk_norm_rope: q, k and the gains must have one dtype"
    assert q.dim() >= 3, f"qk_norm_rope: q must be [..., tokens, heads, D], got {tuple(q.shape)}"
    lead = q.shape[:-2]
    assert k.dim() == q.dim() and k.shape[:-2] == lead and k.shape[-1] == D, \
        f"qk_norm_rope: q {tuple(q.shape)} and k {tuple(k.shape)} must agree but in their heads"
    assert q_gamma.shape == (D,) and k_gamma.shape == (D,), "qk_norm_rope: the gains must be [D]"
    assert cos.dtype == sin.dtype == torch.float32 and cos.dim() == 2 and cos.shape == sin.shape, \
        "qk_norm_rope: cos and sin must be float32 [positions, R / 2]"
    assert 2 * cos.shape[1] <= D, f"qk_norm_rope: the tables rotate {2 * cos.shape[1]} elements of heads of {D}"
    if positions is not None:
        assert positions.dtype in (torch.int32, torch.int64), "qk_norm_rope: positions must be int32 or int64"
        assert positions.shape == lead, f"qk_norm_rope: positions {tuple(positions.shape)} must be [..., tokens] {tuple(q.shape[:-2])}"
        positions = positions.contiguous()
    else:
        assert q.shape[-3] <= cos.shape[0], f"qk_norm_rope: {q.shape[-3]} tokens need as many rows of cos / sin, got {cos.shape[0]}"
    return _as_heads(q), _as_heads(k), q_gamma.contiguous(), k_gamma.contiguous(), cos.contiguous(), sin.contiguous(), positions


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
    nv.launched(device)
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
    nv.launched(device)
    return q_in, k_in, dqg, dkg
