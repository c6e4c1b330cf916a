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
