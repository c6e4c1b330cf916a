"""torch.ops.primus_turbo forms of the operators around a decoder layer's products on layouts that the kernels do not read directly:
the bits of `ops` on the same tensors, and of contiguous copies."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _rand(shape, seed, std=1.0, dt=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, std, generator=g).to(dt)


def _turned(t, i=0, j=1):
    """The values of t behind swapped strides."""
    return t.transpose(i, j).contiguous().transpose(i, j)


def test_moe_few_tokens_with_strides():
    from primus_turbo.pytorch import ops
    T, E, H, I, K = 5, 4, 64, 24, 3
    x, gu, dn = _rand((T, H), 1), _rand((E, 2 * I, H), 2, 0.1), _rand((E, H, I), 3, 0.2)
    ids, p = torch.arange(T * K, device="cuda").view(T, K) % E, torch.rand(T, K, device="cuda")
    want = ops.moe_few_tokens(x, gu, dn, ids, p)
    wide = torch.zeros(T, 2 * K, device="cuda")
    wide[:, ::2] = p
    for args in ((_turned(x), gu, dn, ids, p), (x, _turned(gu, 1, 2), dn, ids, p), (x, gu, _turned(dn, 1, 2), ids, p), (x, gu, dn, _turned(ids), p),
                 (x, gu, dn, ids, wide[:, ::2]), (_turned(x), _turned(gu, 1, 2), _turned(dn, 0, 2), _turned(ids).int(), _turned(p))):
        got = torch.ops.primus_turbo.moe_few_tokens_impl(*args, "silu")
        assert got.is_contiguous() and torch.equal(got, want) and torch.equal(ops.moe_few_tokens(*args), want)


def test_qk_norm_rope_with_strides_and_more_dimensions():
    from primus_turbo.pytorch import ops
    T, Hq, Hk, D, R = 6, 4, 2, 32, 24
    q, k, qg, kg = _rand((T, Hq, D), 1), _rand((T, Hk, D), 2), _rand((D,), 3), _rand((D,), 4)
    cos, sin = _rand((16, R // 2), 5, dt=torch.float32), _rand((16, R // 2), 6, dt=torch.float32)
    pos = torch.tensor([3, 0, 15, 2, 2, 9], device="cuda")
    reg = torch.ops.primus_turbo.qk_norm_rope_fwd_impl
    want = ops.qk_norm_rope(q, k, qg, kg, cos, sin, positions=pos)
    gap = lambda t: torch.stack([t, torch.zeros_like(t)], -1).flatten(-2)[..., ::2]      # the values of t, every second element
    for args in ((_turned(q, 1, 2), k, qg, kg, cos, sin, pos), (q, _turned(k, 0, 2), qg, kg, cos, sin, pos), (q, k, gap(qg), kg, cos, sin, pos),
                 (q, k, qg, gap(kg), _turned(cos), sin, pos), (q, k, qg, kg, cos, gap(sin), gap(pos)), (gap(q), gap(k), qg, kg, cos, sin, pos.int())):
        for got in (reg(*args, 1e-6, False, False), ops.qk_norm_rope(*args)):
            assert all(torch.equal(g, w) and g.is_contiguous() for g, w in zip(got, want))
    many = lambda t: t.view(1, 3, 1, 2, *t.shape[1:])
    got = reg(many(q), many(k), qg, kg, cos, sin, pos.view(1, 3, 1, 2), 1e-6, False, False)
    assert all(g.shape == many(t).shape and torch.equal(g, many(w)) for g, t, w in zip(got, (q, k), want))


def test_gemm_bias_act_with_strides():
    from primus_turbo.pytorch import ops
    M, N, K = 9, 40, 24
    a, b, bias, res = _rand((M, K), 1), _rand((N, K), 2), _rand((2 * N,), 3)[::2], _rand((N, M), 4).t()
    want = ops.gemm_bias_act(a, b, bias.contiguous(), "silu", res.contiguous(), trans_b=True)
    for args in ((_turned(a), b), (a, _turned(b)), (_turned(a), _turned(b))):
        assert torch.equal(torch.ops.primus_turbo.gemm_bias_act_impl(*args, True, bias, "silu", res, BF), want)


def test_a_misfit_is_refused_before_any_launch():
    t = torch.ops.primus_turbo
    a, b = _rand((4, 64), 1), _rand((32, 64), 2)
    with pytest.raises(AssertionError, match="bias must be"):
        t.gemm_bias_act_impl(a, b, True, b[0, :16], None, None, BF)
    with pytest.raises(AssertionError, match="gains must be"):
        t.qk_norm_rope_fwd_impl(a.view(4, 1, 64), a.view(4, 1, 64), b[0], b[0, :32], torch.ones(4, 32, device="cuda"), torch.ones(4, 32, device="cuda"), None, 1e-6,
                                False, False)
    with pytest.raises(AssertionError, match="must be float32"):
        t.moe_few_tokens_impl(a, b.view(2, 16, 64), _rand((2, 64, 8), 3), torch.zeros(4, 1, dtype=torch.int64, device="cuda"), a[:, :1], "silu")
