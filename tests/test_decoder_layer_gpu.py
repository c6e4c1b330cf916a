"""gemm_bias_act, qk_norm_rope and moe_few_tokens together, as a decoder layer uses them: projection with bias -> per-head norm and
rotation -> attention (written out in torch here) -> output projection added to the residual -> rmsnorm -> experts or a dense MLP.

Accuracy: against the layer in 64 bits, relative in the Frobenius norm.  Every rounding to bf16 adds at most half a step, 2^-8, of its
tensor; a layer has about ten in sequence and no map in it amplifies a relative error by more than about two (unit-scale weights,
normalised inputs): 20 x 2^-8 = 0.08 bounds outputs, twice that gradients (which pass the layer's roundings both ways)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
H, HEADS, KV, D, E, I, K, FFN = 512, 8, 2, 64, 8, 256, 2, 1024
BOUND = 20 * 2.0 ** -8


def _rand(shape, seed, std=1.0, dt=BF):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dt).cuda()


def _weights():
    w = {"wqkv": _rand(((HEADS + 2 * KV) * D, H), 1, H ** -0.5), "bqkv": _rand(((HEADS + 2 * KV) * D,), 2, 0.1),
         "qg": 1 + _rand((D,), 3, 0.1), "kg": 1 + _rand((D,), 4, 0.1), "wo": _rand((H, HEADS * D), 5, (HEADS * D) ** -0.5), "bo": _rand((H,), 6, 0.1),
         "gamma": 1 + _rand((H,), 7, 0.1), "router": _rand((E, H), 8, H ** -0.5), "gate_up": _rand((E, 2 * I, H), 9, H ** -0.5),
         "down": _rand((E, H, I), 10, I ** -0.5), "up": _rand((FFN, H), 11, H ** -0.5), "bup": _rand((FFN,), 12, 0.1), "w2": _rand((H, FFN), 13, FFN ** -0.5)}
    ang = torch.arange(512, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)[None, :]
    w["cos"], w["sin"] = ang.cos().float().cuda(), ang.sin().float().cuda()
    return w


def _attend(q, k, v, first):
    """q [S, HEADS, D] at positions first .., k, v [T, KV, D] from 0: causal, in q's precision."""
    S, T = q.shape[0], k.shape[0]
    k, v = (t.repeat_interleave(HEADS // KV, dim=1) for t in (k, v))
    s = torch.einsum("shd,thd->hst", q, k) / math.sqrt(D)
    s = s.masked_fill(torch.arange(T, device=q.device)[None, :] > torch.arange(first, first + S, device=q.device)[:, None], float("-inf"))
    return torch.einsum("hst,thd->shd", s.softmax(-1), v).reshape(S, HEADS * D)


def _layer(x, w, first=0, cache=None, experts=True, sync=False):
    from primus_turbo.pytorch import ops
    barrier = torch.cuda.synchronize if sync else (lambda: None)
    S = x.shape[0]
    qkv = ops.gemm_bias_act(x, w["wqkv"], bias=w["bqkv"], trans_b=True).view(S, HEADS + 2 * KV, D)
    barrier()
    pos = torch.arange(first, first + S, device="cuda")
    q, k = ops.qk_norm_rope(qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV], w["qg"], w["kg"], w["cos"], w["sin"], positions=pos)
    barrier()
    v = qkv[:, HEADS + KV:]
    if cache is not None:
        k, v = torch.cat([cache[0], k]), torch.cat([cache[1], v])
    att = _attend(q.float(), k.float(), v.float(), first).to(BF)
    x = ops.gemm_bias_act(att, w["wo"], bias=w["bo"], residual=x, trans_b=True)
    barrier()
    n = ops.rmsnorm(x, w["gamma"])
    barrier()
    if experts:
        probs, ids = (n.float() @ w["router"].float().t()).softmax(-1).topk(K)
        out = x + torch.cat([ops.moe_few_tokens(n[i:i + 128], w["gate_up"], w["down"], ids[i:i + 128], probs[i:i + 128]) for i in range(0, S, 128)])
        return out, (k, v), ids, probs
    h = ops.gemm_bias_act(n, w["up"], bias=w["bup"], activation="silu", trans_b=True)
    return ops.gemm_bias_act(h, w["w2"], residual=x, trans_b=True), (k, v), None, None


def _layer64(x, w, experts, ids=None):
    """The whole prompt in 64 bits from the same weights; the routing of the bf16 layer (a rounding may swap near-equal experts)."""
    w = {n: t.double() for n, t in w.items()}
    S = x.shape[0]
    qkv = (x @ w["wqkv"].t() + w["bqkv"]).view(S, HEADS + 2 * KV, D)

    def head(t, g):
        n = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * g
        a, b, c, s = n[..., :D // 2], n[..., D // 2:], w["cos"][:S, None], w["sin"][:S, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    att = _attend(head(qkv[:, :HEADS], w["qg"]), head(qkv[:, HEADS:HEADS + KV], w["kg"]), qkv[:, HEADS + KV:], 0)
    x = x + att @ w["wo"].t() + w["bo"]
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w["gamma"]
    if not experts:
        h = n @ w["up"].t() + w["bup"]
        return x + (h * torch.sigmoid(h)) @ w["w2"].t()
    p = (n @ w["router"].t()).softmax(-1).gather(1, ids)
    out = x.clone()
    for j in range(K):
        z = torch.einsum("sh,sih->si", n, w["gate_up"][ids[:, j]])
        out = out + p[:, j:j + 1] * torch.einsum("si,shi->sh", z[:, :I] * torch.sigmoid(z[:, :I]) * z[:, I:], w["down"][ids[:, j]])
    return out


def _rel(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("S", [1, 7, 61, 200])
def test_prompt(S):
    from primus_turbo.pytorch.kernels import _native as nv
    w, x = _weights(), _rand((S, H), 20)
    with torch.no_grad():
        out, _, ids, _ = _layer(x, w)
        assert _rel(out, _layer64(x.double(), w, True, ids)) <= BOUND
        dense = _layer(x, w, experts=False)[0]
        assert _rel(dense, _layer64(x.double(), w, False)) <= BOUND
    nv.check_status(out.device)


def test_tokens_one_by_one_follow_the_prompt():
    w, x = _weights(), _rand((24, H), 21)
    with torch.no_grad():
        out, cache, ids, _ = _layer(x[:16], w)
        got = [out]
        for t in range(16, 24):
            o, cache, i, _ = _layer(x[t:t + 1], w, first=t, cache=cache)
            got.append(o)
            ids = torch.cat([ids, i])
        assert _rel(torch.cat(got), _layer64(x.double(), w, True, ids)) <= BOUND


@pytest.mark.parametrize("S", [1, 33])
def test_back_to_back_launches_and_graph_give_the_bits_of_separate_ones(S):
    """The kernels start while their predecessors finish; with a synchronisation after each, on another stream and in a graph the
    bits are the same."""
    w, x = _weights(), _rand((S, H), 22)
    with torch.no_grad():
        want = [_layer(x, w, sync=True)[0], _layer(x, w, experts=False, sync=True)[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(10):
                got = [_layer(x, w)[0], _layer(x, w, experts=False)[0]]
            side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = [_layer(x, w)[0], _layer(x, w, experts=False)[0]]
        for _ in range(5):
            for h in held:
                h.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize("S", [5, 300])
def test_gradients_of_a_dense_layer(S):
    w = _weights()
    names = ["wqkv", "bqkv", "qg", "kg", "wo", "bo", "gamma", "up", "bup", "w2"]
    x = _rand((S, H), 23).requires_grad_()
    for n in names:
        w[n] = w[n].requires_grad_()
    dy = _rand((S, H), 24)
    out = _layer(x, w, experts=False)[0]
    grads = torch.autograd.grad(out, [x] + [w[n] for n in names], dy)
    w64 = {n: t.detach().double().requires_grad_(n in names) for n, t in w.items()}
    x64 = x.detach().double().requires_grad_()
    want = torch.autograd.grad(_layer64(x64, w64, False), [x64] + [w64[n] for n in names], dy.double())
    for n, a, b in zip(["x"] + names, grads, want):
        assert a.shape == b.shape and _rel(a, b) <= 2 * BOUND, n


def test_second_derivatives_are_refused():
    from primus_turbo.pytorch import ops
    w, x = _weights(), _rand((5, H), 25).requires_grad_()
    dy = _rand((5, FFN), 26).requires_grad_()
    (g,) = torch.autograd.grad(ops.gemm_bias_act(x, w["up"], activation="silu", trans_b=True), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
    q = _rand((5, 4, D), 27).requires_grad_()
    dq = _rand((5, 4, D), 28).requires_grad_()
    (g,) = torch.autograd.grad(ops.qk_norm_rope(q, q[:, :1], w["qg"], w["kg"], w["cos"], w["sin"])[0], q, dq, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()


def test_first_call_of_a_process_inside_a_capture():
    """The operators need no warm-up call: a fresh process captures them first."""
    import os
    import subprocess
    import sys
    code = """
import torch, sys
sys.path.insert(0, 'primus-turbo_b200')
from primus_turbo.pytorch import ops
b = torch.bfloat16
x, w, g = torch.ones(4, 64, device='cuda', dtype=b), torch.ones(96, 64, device='cuda', dtype=b), torch.ones(16, device='cuda', dtype=b)
big = torch.ones(9000, 64, device='cuda', dtype=b); wide = torch.ones(2048, 64, device='cuda', dtype=b)
t = torch.ones(8, 8, device='cuda'); gu, dn = torch.ones(2, 32, 64, device='cuda', dtype=b), torch.ones(2, 64, 16, device='cuda', dtype=b)
ids, p = torch.zeros(4, 1, device='cuda', dtype=torch.int64), torch.ones(4, 1, device='cuda')
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.gemm_bias_act(x, w, trans_b=True)
    z = ops.gemm_bias_act(big, wide, activation='relu', trans_b=True)
    q, k = ops.qk_norm_rope(x.view(4, 4, 16), x.view(4, 4, 16), g, g, t, t)
    m = ops.moe_few_tokens(x, gu, dn, ids, p)
graph.replay()
torch.cuda.synchronize()
assert (y == 64).all() and (z == 64).all() and q.isfinite().all() and (m == m[0, 0]).all() and m[0, 0] > 0
print('captured')
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_registered_ops_are_the_operators():
    from primus_turbo.pytorch import ops
    w, x, t = _weights(), _rand((5, H), 29), torch.ops.primus_turbo
    assert torch.equal(t.gemm_bias_act_impl(x, w["up"], True, w["bup"], "gelu", None, BF), ops.gemm_bias_act(x, w["up"], bias=w["bup"], activation="gelu", trans_b=True))
    q = _rand((5, 4, D), 30)
    got = t.qk_norm_rope_fwd_impl(q, q[:, :1], w["qg"], w["kg"], w["cos"], w["sin"], None, 1e-6, True, False)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.qk_norm_rope(q, q[:, :1], w["qg"], w["kg"], w["cos"], w["sin"], interleaved=True)))
    p, ids = torch.rand(5, E, device="cuda").topk(K)
    assert torch.equal(t.moe_few_tokens_impl(x, w["gate_up"], w["down"], ids, p, "gelu"), ops.moe_few_tokens(x, w["gate_up"], w["down"], ids, p, act_type="gelu"))
