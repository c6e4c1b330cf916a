"""Refusals of the operators around a decoder layer's products.  They come before any launch, so fake CUDA tensors and null
pointers reach them on a machine without a GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

bf16 = torch.bfloat16


def _e(*shape, dt=bf16):
    return torch.empty(shape, dtype=dt, device="cuda")


# ------------------------------------------------------------------------------------------------ qk_norm_rope
def _qk_args(**change):
    a = dict(q=_e(5, 4, 64), k=_e(5, 2, 64), q_gamma=_e(64), k_gamma=_e(64), cos=_e(16, 32, dt=torch.float32),
             sin=_e(16, 32, dt=torch.float32), positions=None)
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (lambda: dict(k=_e(5, 2, 32)), "agree but in their heads"),
    (lambda: dict(k=_e(4, 2, 64)), "agree but in their heads"),
    (lambda: dict(k=_e(5, 2, 64, dt=torch.float16)), "one dtype"),
    (lambda: dict(q_gamma=_e(64, dt=torch.float32)), "one dtype"),
    (lambda: dict(k_gamma=_e(32)), "gains must be"),
    (lambda: dict(cos=_e(16, 32)), "float32"),
    (lambda: dict(sin=_e(16, 16, dt=torch.float32)), "float32"),
    (lambda: dict(cos=_e(16, 40, dt=torch.float32), sin=_e(16, 40, dt=torch.float32)), "tables rotate"),
    (lambda: dict(cos=_e(4, 32, dt=torch.float32), sin=_e(4, 32, dt=torch.float32)), "as many rows"),
    (lambda: dict(positions=_e(5, dt=torch.float32)), "int32 or int64"),
    (lambda: dict(positions=_e(4, dt=torch.int64)), "must be"),
    (lambda: dict(cos=_e(16, 32, dt=torch.float32).requires_grad_()), "not differentiated"),
    (lambda: dict(q=_e(5, 64), k=_e(5, 64)), "heads, D"),
    (lambda: dict(q=_e(5, 4, 64, dt=torch.float64), k=_e(5, 2, 64, dt=torch.float64)), "unsupported dtype"),
])
def test_qk_norm_rope_refuses(change, match):
    from primus_turbo.pytorch.ops import qk_norm_rope
    with FakeTensorMode(), pytest.raises((AssertionError, TypeError), match=match):
        qk_norm_rope(**_qk_args(**change()))


def test_qk_norm_rope_refuses_cpu_tensors():
    from primus_turbo.pytorch.ops import qk_norm_rope
    z = torch.zeros
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        qk_norm_rope(z(2, 1, 8), z(2, 1, 8), z(8), z(8), z(2, 4), z(2, 4))


def test_qk_norm_rope_abi_refusals():
    from primus_turbo import _clib
    lib = _clib.load()
    st = (ctypes.c_int64 * 3)(0, 0, 0)

    def call(D=64, R=64, dtype=0, pos_bytes=0, S=4, strides=st):
        return lib.pt_qk_norm_rope_fwd(None, None, dtype, None, None, None, None, None, pos_bytes, 1, S, 8, 2, 1, D, R, strides, strides, 1e-6, 0, 0,
                                       None, None, None, None)
    for kw, msg in ((dict(D=2048), b"head size"), (dict(R=7), b"head size"), (dict(R=66), b"head size"), (dict(dtype=5), b"dtype"),
                    (dict(pos_bytes=2), b"positions"), (dict(pos_bytes=8), b"go together"), (dict(), b"null"), (dict(S=-1), b"negative"),
                    (dict(strides=None), b"strides")):
        assert call(**kw) == -1 and msg in lib.pt_last_error(), kw
    assert call(S=0) == 0
    rc = lib.pt_qk_norm_rope_bwd(None, None, None, None, 0, None, None, None, None, None, 0, 1, 4, 8, 0, 0, 64, 0, st, st, st, st, 1e-6, 0, 0, None,
                                 None, None, None, None, 0, None, None)
    assert rc == -1 and b"dgamma buffers" in lib.pt_last_error()


# ------------------------------------------------------------------------------------------------ gemm_bias_act
@pytest.mark.parametrize("change,match", [
    (lambda: dict(a=_e(4, 63)), "contraction mismatch"),
    (lambda: dict(trans_b=False), "contraction mismatch"),
    (lambda: dict(a=_e(2, 4, 64)), "Only 2D"),
    (lambda: dict(a=_e(4, 64, dt=torch.float16)), "both be bf16 or fp16"),
    (lambda: dict(a=_e(4, 64, dt=torch.float32), b=_e(32, 64, dt=torch.float32)), "both be bf16 or fp16"),
    (lambda: dict(a=_e(4, 0), b=_e(32, 0)), "must not be empty"),
    (lambda: dict(activation="swish"), "Unsupported activation"),
    (lambda: dict(bias=_e(64)), "bias must be"),
    (lambda: dict(bias=_e(32, dt=torch.float16)), "bias must be"),
    (lambda: dict(residual=_e(4, 31)), "residual must be"),
    (lambda: dict(residual=_e(4, 32, dt=torch.float32)), "residual must be"),
    (lambda: dict(out_dtype=torch.float64), "unsupported out_dtype"),
    (lambda: dict(bias=torch.empty(32, dtype=bf16, device="cpu")), "one device"),
])
def test_gemm_bias_act_refuses(change, match):
    from primus_turbo.pytorch.ops import gemm_bias_act
    with FakeTensorMode(), pytest.raises(AssertionError, match=match):
        gemm_bias_act(**{**dict(a=_e(4, 64), b=_e(32, 64), trans_b=True), **change()})


def test_gemm_bias_act_refuses_cpu_tensors():
    from primus_turbo.pytorch.ops import gemm_bias_act
    z = lambda *s: torch.zeros(s, dtype=bf16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gemm_bias_act(z(4, 64), z(32, 64), trans_b=True)


def test_gemm_bias_act_abi_refusals():
    from primus_turbo import _clib
    lib = _clib.load()

    def call(ab=0, bias=None, bias_dt=0, cd=0, act=2, M=4, N=8, K=64, b_mn=0):
        return lib.pt_gemm_bias_act(None, None, b_mn, ab, bias, bias_dt, None, None, cd, None, act, M, N, K, None, None)
    for kw, msg in ((dict(ab=2), b"operands"), (dict(cd=7), b"output dtype"), (dict(act=5), b"activation"), (dict(act=-1), b"activation"),
                    (dict(M=-1), b"bad shape"), (dict(K=12), b"multiple of 8"), (dict(K=0), b"multiple of 8"), (dict(), b"null"), (dict(b_mn=1, N=12), b"row count"),
                    (dict(bias=ctypes.c_void_p(16), bias_dt=9), b"bias dtype")):
        assert call(**kw) == -1 and msg in lib.pt_last_error(), kw
    assert call(M=0) == 0 and call(N=0) == 0
    mn = lambda a_mn=1, b_mn=0, M=8, N=8, K=64: lib.pt_gemm_mn(None, a_mn, None, b_mn, 0, None, 0, M, N, K, 0.0, None, None)
    for kw, msg in ((dict(M=12), b"row count"), (dict(b_mn=1, N=12), b"row count"), (dict(K=12), b"multiple of 8"), (dict(), b"null"),
                    (dict(b_mn=1, K=12), b"null")):
        assert mn(**kw) == -1 and msg in lib.pt_last_error(), kw
    bwd = lambda dt=0, act=0, dy=0, dbias=None, parts=0: lib.pt_act_bias_bwd(None, dy, None, dt, act, 4, 8, None, dbias, 0, None, parts, None)
    for kw, msg in ((dict(dt=2), b"operands"), (dict(act=9), b"activation"), (dict(dy=4), b"gradient dtype"), (dict(), b"null"),
                    (dict(dbias=ctypes.c_void_p(16)), b"bias buffers")):
        assert bwd(**kw) == -1 and msg in lib.pt_last_error(), kw


# ------------------------------------------------------------------------------------------------ moe_few_tokens
def _moe_args(**change):
    a = dict(x=_e(3, 64), gate_up=_e(4, 32, 64), down=_e(4, 64, 16), topk_indices=_e(3, 2, dt=torch.int64), topk_probs=_e(3, 2, dt=torch.float32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (lambda: dict(act_type="relu"), "Unsupported act_type"),
    (lambda: dict(x=_e(3, 1, 64)), "must be"),
    (lambda: dict(x=_e(3, 72)), "do not fit"),
    (lambda: dict(gate_up=_e(4, 16, 64)), "do not fit"),
    (lambda: dict(down=_e(3, 64, 16)), "do not fit"),
    (lambda: dict(x=_e(3, 64, dt=torch.float16)), "bf16 or fp16"),
    (lambda: dict(topk_indices=_e(2, 2, dt=torch.int64)), "must be .T, K."),
    (lambda: dict(topk_probs=_e(3, 1, dt=torch.float32)), "must be .T, K."),
    (lambda: dict(topk_indices=_e(3, 2, dt=torch.int16)), "int32 or int64"),
    (lambda: dict(topk_probs=_e(3, 2)), "float32"),
    (lambda: dict(gate_up=_e(4, 24, 64), down=_e(4, 64, 12)), "multiples of 8"),
    (lambda: dict(x=_e(129, 64), topk_indices=_e(129, 2, dt=torch.int64), topk_probs=_e(129, 2, dt=torch.float32)), "at most"),
    (lambda: dict(topk_indices=_e(3, 33, dt=torch.int64), topk_probs=_e(3, 33, dt=torch.float32)), "at most"),
    (lambda: dict(x=_e(100, 64), topk_indices=_e(100, 24, dt=torch.int64), topk_probs=_e(100, 24, dt=torch.float32)), "at most"),
    (lambda: dict(topk_probs=torch.empty(3, 2, device="cpu")), "one device"),
])
def test_moe_few_tokens_refuses(change, match):
    from primus_turbo.pytorch.ops import moe_few_tokens
    with FakeTensorMode(), pytest.raises(AssertionError, match=match):
        moe_few_tokens(**_moe_args(**change()))


def test_moe_few_tokens_refuses_cpu_tensors_and_gradients():
    from primus_turbo.pytorch.ops import moe_few_tokens
    z = lambda *s: torch.zeros(s, dtype=bf16)
    args = (z(3, 64), z(4, 32, 64), z(4, 64, 16), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        moe_few_tokens(*args)
    with FakeTensorMode(), pytest.raises(RuntimeError, match="no backward"):
        moe_few_tokens(**_moe_args(x=_e(3, 64).requires_grad_()))


def test_moe_few_tokens_abi_refusals():
    from primus_turbo import _clib
    lib = _clib.load()

    def call(dt=0, idb=8, T=3, E=4, K=2, H=64, I=16, act=0):
        return lib.pt_moe_few_tokens(None, None, None, dt, None, idb, None, T, E, K, H, I, act, None, 0, None, None, None)
    for kw, msg in ((dict(dt=2), b"bf16 or fp16"), (dict(idb=2), b"int32 or int64"), (dict(T=129), b"at most"), (dict(E=1025), b"at most"),
                    (dict(K=33), b"at most"), (dict(T=128, K=17), b"at most"), (dict(H=60), b"multiples of 8"), (dict(I=12), b"multiples of 8"),
                    (dict(act=2), b"activation"), (dict(I=1 << 21, E=1024), b"32-bit"), (dict(), b"null")):
        assert call(**kw) == -1 and msg in lib.pt_last_error(), kw
    assert call(T=0) == 0
    assert lib.pt_moe_few_tokens_scratch_bytes(3, 2, 16) == 6 * 32


# ------------------------------------------------------------------------------------------------ torch.library
def test_custom_ops_have_fake_implementations():
    import primus_turbo.pytorch  # noqa: F401
    t = torch.ops.primus_turbo
    with FakeTensorMode():
        y = t.gemm_bias_act_impl(_e(5, 64), _e(64, 96), False, _e(96), "silu", None, torch.float32)
        assert tuple(y.shape) == (5, 96) and y.dtype == torch.float32 and y.device.type == "cuda"
        a = _qk_args()
        q, k = t.qk_norm_rope_fwd_impl(a["q"], a["k"], a["q_gamma"], a["k_gamma"], a["cos"], a["sin"], None, 1e-6, False, False)
        assert q.shape == a["q"].shape and k.shape == a["k"].shape and q.dtype == bf16
        m = _moe_args()
        assert t.moe_few_tokens_impl(m["x"], m["gate_up"], m["down"], m["topk_indices"], m["topk_probs"], "silu").shape == m["x"].shape
