"""BF16 / FP16 dense GEMM over the C ABI.

Same call shape as primus_turbo::gemm_impl / gemm_accum_impl of the reference
(primus_turbo/pytorch/kernels/gemm/gemm_impl.py).  The CUDA kernel is the FP8 one run with kind::f16 instructions:
C = A . B^T; an operand is read as it is stored, K-major ([rows, K]) or contraction-major ([K, rows]), and the operands swap for
trans_c.  Rows that are not a multiple of 8 elements cannot be read contraction-major in place (a TMA row is a multiple of 16
bytes): those operands are transposed first.
"""
from typing import Optional, Tuple

import torch

from .. import _native as nv
from ..quantization.quantization_impl import transpose_2d


def _k_major16(x, trans):
    """x as [rows, K] with K a multiple of 8 (a 16-byte row pitch): x itself, its transpose, zero padded if ragged."""
    x = x.contiguous()
    y = transpose_2d(x) if trans else x
    K = y.shape[1]
    if K % 8 == 0:
        return y
    z = torch.zeros((y.shape[0], (K + 7) // 8 * 8), dtype=y.dtype, device=y.device)
    z[:, :K] = y
    return z


def _in_place(x, trans, other, other_trans):
    """Whether x, needed as [rows, K] and stored [K, rows] (trans), is read where it lies: see the note above.  A contraction that
    is not a multiple of 8 must be contraction-major on both sides (a K-major operand would be padded)."""
    def fits(t):
        return t.shape[1] % 8 == 0 and t.data_ptr() % 16 == 0
    return trans and x.is_contiguous() and fits(x) and (x.shape[0] % 8 == 0 or (other_trans and other.is_contiguous() and fits(other)))


def _launch(a, a_mn, b, b_mn, out, beta, mapped_status=False):
    (M, K) = a.shape[::-1] if a_mn else a.shape
    (N, Kb) = b.shape[::-1] if b_mn else b.shape
    assert Kb == K, f"contraction mismatch: {tuple(a.shape)} vs {tuple(b.shape)}"
    st = nv.mapped_status(out.device) if mapped_status else nv.ptr(nv.status_word(out.device))
    with nv.on_device(out.device):
        nv.check(nv.lib().pt_gemm_mn(nv.ptr(a), int(a_mn), nv.ptr(b), int(b_mn), nv.src_code(a.dtype), nv.ptr(out), nv.src_code(out.dtype), M, N, K,
                                     float(beta), st, nv.stream(out.device)), "gemm")
    if mapped_status:
        nv.launched(out.device)
    else:
        nv.poll_status(out.device)
    return out


def _gemm(a, trans_a, b, trans_b, out_dtype, trans_c, out=None, mapped_status=False):
    nv.require_cuda(a, b)
    assert a.dim() == 2 and b.dim() == 2, "Only 2D tensors are supported"
    assert a.dtype == b.dtype and a.dtype in (torch.bfloat16, torch.float16), "a and b must both be bf16 or fp16"
    a_mn, b_mn = _in_place(a, trans_a, b, not trans_b), _in_place(b, not trans_b, a, trans_a)
    if not a_mn:
        a = _k_major16(a, trans_a)        # [M, K]
    if not b_mn:
        b = _k_major16(b, not trans_b)    # [N, K]
    M, N = a.shape[1 if a_mn else 0], b.shape[1 if b_mn else 0]
    beta = 0.0 if out is None else 1.0
    if out is None:
        out = torch.empty((N, M) if trans_c else (M, N), dtype=out_dtype, device=a.device)
    else:
        assert out.is_contiguous() and tuple(out.shape) == ((N, M) if trans_c else (M, N))
    if trans_c:
        a, a_mn, b, b_mn = b, b_mn, a, a_mn
    return _launch(a, a_mn, b, b_mn, out, beta, mapped_status)


def gemm_impl(a: torch.Tensor, trans_a: bool, b: torch.Tensor, trans_b: bool, out_dtype: torch.dtype, trans_c: bool,
              default_backend: int = 0) -> torch.Tensor:
    """op(a) . op(b) (transposed when trans_c), fp32 accumulate, output in out_dtype."""
    return _gemm(a, trans_a, b, trans_b, out_dtype, trans_c)


def gemm_accum_impl(a: torch.Tensor, trans_a: bool, b: torch.Tensor, trans_b: bool, out_dtype: torch.dtype, trans_c: bool,
                    out: torch.Tensor, default_backend: int = 0) -> torch.Tensor:
    """out += op(a) . op(b) in place (the fused main_grad accumulation of the wgrad)."""
    return _gemm(a, trans_a, b, trans_b, out.dtype, trans_c, out=out)


EPILOGUE_ACTS = {"silu": 0, "gelu": 1, None: 2, "relu": 3, "gelu_tanh": 4}


def check_gemm_bias_act(a: torch.Tensor, b: torch.Tensor, trans_b: bool, bias: Optional[torch.Tensor], act: Optional[str],
                        residual: Optional[torch.Tensor], out_dtype: torch.dtype) -> None:
    """Refuses what gemm_bias_act_impl, which trusts its arguments but for their strides, does not take."""
    assert a.dim() == 2 and b.dim() == 2, "Only 2D GEMM is supported"
    dtype, index, (M, K) = a.dtype, a.get_device(), a.shape
    assert b.dtype == dtype and dtype in (torch.bfloat16, torch.float16), "a and b must both be bf16 or fp16"
    assert act in EPILOGUE_ACTS, f"Unsupported activation: {act}. Supported: {list(EPILOGUE_ACTS)}"
    N, Kb = b.shape if trans_b else b.shape[::-1]
    assert Kb == K, f"contraction mismatch: {tuple(a.shape)} vs {tuple(b.shape)} (trans_b={trans_b})"
    assert K > 0, "gemm_bias_act: the contraction must not be empty"
    assert out_dtype in (torch.bfloat16, torch.float16, torch.float32), f"gemm_bias_act: unsupported out_dtype {out_dtype}"
    assert b.get_device() == index, "gemm_bias_act: all tensors must be on one device"
    if bias is not None:
        assert bias.shape == (N,) and bias.dtype in (dtype, torch.float32), f"gemm_bias_act: bias must be [{N}] in a's dtype or float32"
        assert bias.get_device() == index, "gemm_bias_act: all tensors must be on one device"
    if residual is not None:
        assert residual.shape == (M, N) and residual.dtype == out_dtype, f"gemm_bias_act: residual must be [{M}, {N}] in {out_dtype}"
        assert residual.get_device() == index, "gemm_bias_act: all tensors must be on one device"


def gemm_bias_act_impl(a: torch.Tensor, b: torch.Tensor, trans_b: bool, bias: Optional[torch.Tensor], act: Optional[str],
                       residual: Optional[torch.Tensor], out_dtype: torch.dtype, want_z: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(act(a . op(b) + bias) + residual, the pre-activation in a's type or None) in one kernel."""
    nv.require_cuda(a, b, bias, residual)
    device, dtype, (M, K) = a.device, a.dtype, a.shape
    b_mn = not trans_b and _in_place(b, True, a, False)
    N = b.shape[0 if trans_b else 1]
    if K % 8 or not a.is_contiguous():
        a = _k_major16(a, False)                         # [M, K]
    if not b_mn and (K % 8 or not trans_b or not b.is_contiguous()):
        b = _k_major16(b, not trans_b)                   # [N, K]
    if a.data_ptr() % 16:                                # a view into a larger buffer; TMA reads from 16-byte boundaries
        a = a.clone()
    if b.data_ptr() % 16:
        b = b.clone()
    out = a.new_empty((M, N)) if out_dtype == dtype else torch.empty((M, N), dtype=out_dtype, device=device)
    z = a.new_empty((M, N)) if want_z else None
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    with nv.on_device(device):
        nv.check(nv.lib().pt_gemm_bias_act(a.data_ptr(), b.data_ptr(), b_mn, nv.src_code(dtype), nv.ptr(bias),
                                           0 if bias is None else nv.src_code(bias.dtype), nv.ptr(residual), out.data_ptr(),
                                           nv.src_code(out_dtype), nv.ptr(z), EPILOGUE_ACTS[act], M, N, (K + 7) // 8 * 8,
                                           nv.mapped_status(device), nv.stream(device)), "gemm_bias_act")
    nv.launched(device)
    return out, z


def act_bias_bwd_impl(grad_out: torch.Tensor, z: Optional[torch.Tensor], act: Optional[str], dtype: torch.dtype,
                      bias_dtype: Optional[torch.dtype], want_dz: bool = True) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(grad_out * act'(z) in the operands' type, its column sums in bias_dtype or None) in one pass.  Without an activation the
    first is grad_out itself where the types agree."""
    nv.require_cuda(grad_out, z)
    grad_out = grad_out.contiguous()
    if grad_out.dtype not in (dtype, torch.float32):
        grad_out = grad_out.to(torch.float32)
    device, (M, N) = grad_out.device, grad_out.shape
    same = act is None and grad_out.dtype == dtype
    dz = torch.empty((M, N), dtype=dtype, device=device) if want_dz and not same else None
    if dz is None and bias_dtype is None:
        return (grad_out if same else None), None
    lib = nv.lib()
    with nv.on_device(device):
        dbias = partial = None
        parts = 0
        if bias_dtype is not None:
            parts = lib.pt_act_bias_bwd_parts(M, N)
            dbias = torch.empty((N,), dtype=bias_dtype, device=device)
            if parts > 1:
                partial = torch.empty((parts, N), dtype=torch.float32, device=device)
        nv.check(lib.pt_act_bias_bwd(grad_out.data_ptr(), nv.src_code(grad_out.dtype), nv.ptr(z), nv.src_code(dtype), EPILOGUE_ACTS[act], M, N,
                                     nv.ptr(dz), nv.ptr(dbias), 0 if dbias is None else nv.src_code(bias_dtype), nv.ptr(partial), parts,
                                     nv.stream(device)), "act_bias_bwd")
    return (grad_out if same else dz), dbias


def bias_act_dgrad_impl(dz: torch.Tensor, b: torch.Tensor, trans_b: bool) -> torch.Tensor:
    """dz . op(b)^T: the product again, on the kernel that suits its rows."""
    return gemm_bias_act_impl(dz, b, not trans_b, None, None, None, dz.dtype, False)[0]


def bias_act_wgrad_impl(a: torch.Tensor, dz: torch.Tensor, trans_b: bool, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a^T . dz in the layout of b; added to `out` when it is given."""
    return _gemm(a, True, dz, False, dz.dtype if out is None else out.dtype, trans_b, out=out, mapped_status=True)
