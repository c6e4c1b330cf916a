"""Edges of the operators around a decoder layer's products that need no launch: they reach the C ABI or the Python checks without a GPU."""
import ctypes

import pytest


@pytest.mark.parametrize("pos_bytes", [0, 4, 8])
@pytest.mark.parametrize("B,S", [(1, 0), (0, 5), (3, 0)])
def test_qk_norm_rope_takes_no_tokens_with_positions(pos_bytes, B, S):
    """An empty positions tensor is a null pointer of a known element size."""
    from primus_turbo import _clib
    lib = _clib.load()
    st = (ctypes.c_int64 * 3)(0, 0, 0)
    assert lib.pt_qk_norm_rope_fwd(None, None, 0, None, None, None, None, None, pos_bytes, B, S, 8, 2, 1, 64, 64, st, st, 1e-6, 0, 0, None, None, None,
                                   None) == 0, lib.pt_last_error()
    # the backward goes on to its own buffers, which are missing here
    rc = lib.pt_qk_norm_rope_bwd(None, None, None, None, 0, None, None, None, None, None, pos_bytes, B, S, 8, 2, 1, 64, 64, st, st, st, st, 1e-6, 0, 0, None,
                                 None, None, None, None, 0, None, None)
    assert rc == -1 and b"dgamma buffers" in lib.pt_last_error()


def test_moe_few_tokens_refuses_a_tangent():
    import torch
    from torch.autograd import forward_ad
    from primus_turbo.pytorch.ops import moe_few_tokens
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    x, rest = z(3, 64), (z(4, 32, 64), z(4, 64, 16), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match="forward-mode"):
            moe_few_tokens(forward_ad.make_dual(x, x.clone()), *rest)
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            moe_few_tokens(x, *rest)


@pytest.mark.parametrize("which", ["x", "gate_up", "down", "out"])
def test_moe_few_tokens_abi_refuses_pointers_off_their_boundary(which):
    from primus_turbo import _clib
    lib = _clib.load()
    at = dict(x=1 << 20, gate_up=2 << 20, down=3 << 20, out=4 << 20)
    at[which] += 8 if which != "out" else 4
    rc = lib.pt_moe_few_tokens(at["x"], at["gate_up"], at["down"], 0, 5 << 20, 8, 6 << 20, 3, 4, 2, 64, 16, 0, 7 << 20, 1 << 16, at["out"], None, None)
    assert rc == -1 and b"boundar" in lib.pt_last_error()
