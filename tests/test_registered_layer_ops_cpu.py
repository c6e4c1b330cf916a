"""torch.ops.primus_turbo forms of the operators around a decoder layer's products: they refuse what `ops` refuses.  Fake CUDA tensors
reach the refusals on a machine without a GPU; the implementations make the same checks before anything is launched."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

bf16, f16, f32, i64 = torch.bfloat16, torch.float16, torch.float32, torch.int64


def _e(*shape, dt=bf16):
    return torch.empty(shape, dtype=dt, device="cuda")


def _op(name):
    import primus_turbo.pytorch  # noqa: F401
    return getattr(torch.ops.primus_turbo, name)


def _refused(call, match):
    with FakeTensorMode(), pytest.raises(AssertionError, match=match):
        call()


# ------------------------------------------------------------------------------------------------ moe_few_tokens
def _moe(**change):
    a = dict(x=_e(3, 64), gate_up=_e(4, 32, 64), down=_e(4, 64, 16), topk_indices=_e(3, 2, dt=i64), topk_probs=_e(3, 2, dt=f32), act_type="silu")
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (lambda: dict(act_type="relu"), "Unsupported act_type"),
    (lambda: dict(x=_e(3, 72)), "do not fit"),
    (lambda: dict(gate_up=_e(4, 16, 64)), "do not fit"),
    (lambda: dict(gate_up=_e(3, 32, 64)), "do not fit"),
    (lambda: dict(x=_e(3, 64, dt=f16)), "bf16 or fp16"),
    (lambda: dict(topk_indices=_e(2, 2, dt=i64)), "must be .T, K."),
    (lambda: dict(topk_probs=_e(3, 1, dt=f32)), "must be .T, K."),
    (lambda: dict(topk_probs=_e(3, 2)), "float32"),
    (lambda: dict(topk_indices=_e(3, 2, dt=torch.int16)), "int32 or int64"),
    (lambda: dict(topk_probs=torch.empty(3, 2, device="cpu")), "one device"),
])
def test_moe_few_tokens_refuses(change, match):
    from primus_turbo.pytorch.kernels.moe.few_tokens_impl import moe_few_tokens_impl
    _refused(lambda: _op("moe_few_tokens_impl")(**_moe(**change())), match)
    _refused(lambda: moe_few_tokens_impl(*_moe(**change()).values()), match)


def test_moe_few_tokens_output_is_contiguous():
    with FakeTensorMode():
        assert _op("moe_few_tokens_impl")(**_moe(x=_e(64, 3).t())).is_contiguous()


# ------------------------------------------------------------------------------------------------ qk_norm_rope
def _qk(**change):
    a = dict(q=_e(5, 4, 64), k=_e(5, 2, 64), q_gamma=_e(64), k_gamma=_e(64), cos=_e(16, 32, dt=f32), sin=_e(16, 32, dt=f32), positions=None,
             eps=1e-6, interleaved=False, zero_centered=False)
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (lambda: dict(k=_e(4, 2, 64)), "agree but in their heads"),
    (lambda: dict(k=_e(5, 2, 32)), "agree but in their heads"),
    (lambda: dict(k_gamma=_e(32)), "gains must be"),
    (lambda: dict(q_gamma=_e(64, dt=f32)), "one dtype"),
    (lambda: dict(cos=_e(16, 32)), "float32"),
    (lambda: dict(sin=_e(8, 32, dt=f32)), "float32"),
    (lambda: dict(cos=_e(16, 40, dt=f32), sin=_e(16, 40, dt=f32)), "tables rotate"),
    (lambda: dict(cos=_e(4, 32, dt=f32), sin=_e(4, 32, dt=f32)), "as many rows"),
    (lambda: dict(positions=_e(4, dt=i64)), "must be"),
    (lambda: dict(positions=_e(5, dt=torch.int16)), "int32 or int64"),
    (lambda: dict(q=_e(5, 64), k=_e(5, 64)), "heads, D"),
    (lambda: dict(q_gamma=torch.empty(64, dtype=bf16, device="cpu")), "CUDA tensors only"),
])
def test_qk_norm_rope_refuses(change, match):
    with FakeTensorMode(), pytest.raises((AssertionError, RuntimeError), match=match):
        _op("qk_norm_rope_fwd_impl")(**_qk(**change()))


# ------------------------------------------------------------------------------------------------ gemm_bias_act
@pytest.mark.parametrize("change,match", [
    (lambda: dict(a=_e(4, 63)), "contraction mismatch"),
    (lambda: dict(trans_b=False), "contraction mismatch"),
    (lambda: dict(a=_e(2, 4, 64)), "Only 2D"),
    (lambda: dict(a=_e(4, 64, dt=f16)), "both be bf16 or fp16"),
    (lambda: dict(a=_e(4, 0), b=_e(32, 0)), "must not be empty"),
    (lambda: dict(activation="swish"), "Unsupported activation"),
    (lambda: dict(bias=_e(31)), "bias must be"),
    (lambda: dict(bias=_e(32, dt=f16)), "bias must be"),
    (lambda: dict(residual=_e(4, 31)), "residual must be"),
    (lambda: dict(residual=_e(4, 32), out_dtype=f32), "residual must be"),
    (lambda: dict(out_dtype=torch.float64), "unsupported out_dtype"),
    (lambda: dict(bias=torch.empty(32, dtype=bf16, device="cpu")), "one device"),
])
def test_gemm_bias_act_refuses(change, match):
    _refused(lambda: _op("gemm_bias_act_impl")(**{**dict(a=_e(4, 64), b=_e(32, 64), trans_b=True, bias=None, activation=None, residual=None, out_dtype=bf16),
                                                  **change()}), match)
