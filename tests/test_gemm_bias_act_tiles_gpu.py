"""gemm_bias_act where its tests of the same file name without "tiles" do not go: the training path at sizes that reach the tile kernels
(their epilogue writes the pre-activation, dgrad and wgrad run on tiles), last blocks of a few tokens on the CTA pairs of the few-row
kernels, and activations alone against tight bounds.  Formulas and tolerances are those of test_gemm_bias_act_gpu.py."""
import math

import pytest
import torch

from test_gemm_bias_act_gpu import U, _check, _few

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", [(9000, 1001, 1000), (8200, 1028, 264), (33000, 130, 1032), (33000, 131, 1032)])
def test_gradients_on_tiles(M, N, K, act):
    """CTA pairs with a ragged and a vector write-out, single CTAs with both; the last row block is short in each."""
    assert not _few(M, N, K)
    _check(M, N, K, BF, act, True, True, grad=True)


@pytest.mark.parametrize("M,N,K", [(9000, 1001, 1000), (8200, 1028, 264), (33000, 130, 1032)])
def test_gradients_on_tiles_other_types_and_layouts(M, N, K):
    assert not _few(M, N, K)
    _check(M, N, K, F16, "silu", True, False, grad=True)
    _check(M, N, K, F16, "gelu", False, True, out_dtype=F32, grad=True)
    _check(M, N, K, BF, "gelu_tanh", True, True, out_dtype=F32, bias_dtype=F32, grad=True)
    _check(M, N, K, BF, "gelu", True, False, trans_b=False, grad=True)


@pytest.mark.parametrize("M,N,K", [(3613, 1021, 72), (3849, 502, 2832)])
def test_last_block_of_a_few_tokens_on_pairs(M, N, K):
    """Blocks of 240 and 256 tokens whose last one holds 13 and 9: each CTA of the pair brings eight of its 16 rows; one share of the
    contraction and two."""
    assert _few(M, N, K)
    for i, act in enumerate((None, "relu", "silu", "gelu", "gelu_tanh")):
        _check(M, N, K, BF, act, with_bias=i % 2 == 0, with_res=i % 3 != 1, seed=10 * i)
    _check(M, N, K, F16, "silu", True, True, out_dtype=F32)
    _check(M, N, K, F16, "gelu", True, True, grad=True)


@pytest.mark.parametrize("M,N", [(2000, 8), (2000, 5), (40000, 257), (9000, 1028)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_sigmoid_forms_in_fp32(act, M, N):
    """Exact pre-activations: y = z / (1 + exp(-v)) with v = z, or 2 sqrt(2 / pi) (z + 0.044715 z^3).  In half steps u of fp32: the
    exponential's argument carries 2 (product with log2 e) or 8 (with the polynomial) of |v|, the exponential 4, sum, division and product 8."""
    from primus_turbo.pytorch.ops import gemm_bias_act
    a, b = torch.zeros(M, 8, dtype=F16, device="cuda"), torch.zeros(N, 8, dtype=F16, device="cuda")
    a[:, 3] = torch.linspace(-12.5, 6.0, M, device="cuda").to(F16)
    b[:, 3] = 2.0 ** -(torch.arange(N, device="cuda") % 5).to(F16)
    z = a[:, 3:4].double() * b[:, 3].double()
    v, steps = (z, 2) if act == "silu" else (2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3), 8)
    y = gemm_bias_act(a, b, activation=act, trans_b=True, out_dtype=F32).double()
    want = z * torch.sigmoid(v)
    tol = (steps * v.abs() + 12) * U * want.abs() + 2e-37      # a denominator beyond 2^126 gives zero
    assert ((y - want).abs() <= tol).all()
