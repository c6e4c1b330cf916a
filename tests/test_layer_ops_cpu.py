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
