"""moe_few_tokens against the formula in 64 bits: routings with gaps, repeats and foreign experts, ragged widths, full slots.

Tolerances as for gemm_bias_act: a contraction of length K leaves (K / 8 + 32) 2 u sum|a||b| (u = 2^-24); the gated activation at most
1.13 times the gate's error, 128 u of its own and half a step of the type when it is rounded between the products; the second
contraction carries those errors through |down|; the result adds its half step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def _make(shape, dt, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, std, generator=g).to(dt)


def _routing(T, K, all_experts, seed, idt=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    v, ids = torch.empty((T, all_experts), device="cuda").normal_(generator=g).topk(K, dim=1)
    return ids.to(idt), v.softmax(1)


def _oracle(x, gu, dn, ids, probs, act):
    """Output and its error bound, expert by expert in 64 bits."""
    dt, (T, H), (E, _, I) = x.dtype, x.shape, dn.shape
    X = x.double()
    out, tol = torch.zeros_like(X), torch.zeros_like(X)
    for e in range(E):
        p = torch.where(ids == e, probs, torch.zeros_like(probs)).double().sum(1)
        rows = (ids == e).any(1).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        xr, p = X[rows], p[rows][:, None]
        G, Up, D = gu[e, :I].double(), gu[e, I:].double(), dn[e].double()
        g, u = xr @ G.t(), xr @ Up.t()
        eg, eu = [(H / 8 + 32) * 2 * U * (xr.abs() @ w.abs().t()) for w in (G, Up)]
        a = g * torch.sigmoid(g) if act == "silu" else 0.5 * g * torch.erfc(-g / math.sqrt(2))
        ea = 1.13 * eg + 128 * U * (g.abs() + a.abs())
        h = p * a * u
        eh = p.abs() * (ea * (u.abs() + eu) + a.abs() * eu) + 4 * U * h.abs()
        eh = eh + HALF[dt] * (h.abs() + eh) + TINY[dt]
        out[rows] += h @ D.t()
        tol[rows] += eh @ D.abs().t() + (ids.shape[1] * I / 8 + 64) * 2 * U * (h.abs() @ D.abs().t())
    return out, tol + (HALF[dt] + U) * (out.abs() + tol) + TINY[dt]


def _check(T, E, K, H, I, dt, act="silu", ids=None, probs=None, shards=1, seed=0, idt=torch.int64):
    from primus_turbo.pytorch.kernels import _native as nv
    from primus_turbo.pytorch.ops import moe_few_tokens
    x, gu, dn = _make((T, H), dt, seed + 1), _make((E, 2 * I, H), dt, seed + 2, H ** -0.5), _make((E, H, I), dt, seed + 3, I ** -0.5)
    if ids is None:
        ids, probs = _routing(T, K, E * shards, seed + 4, idt)
        ids = torch.where(ids < E, ids, torch.full_like(ids, -1))
    if probs is None:
        probs = torch.rand(ids.shape, generator=torch.Generator(device="cuda").manual_seed(seed + 5), device="cuda")
    out = moe_few_tokens(x, gu, dn, ids, probs, act_type=act)
    nv.check_status(out.device)
    want, tol = _oracle(x, gu, dn, ids, probs, act)
    err = (out.double() - want).abs()
    bad = (err > tol) | err.isnan()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst {float((err / tol.clamp(min=1e-30)).max()):.2f} x tolerance"
    return out


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,K,H,I", [
    (1, 1, 1, 8, 8), (1, 8, 2, 256, 128), (2, 4, 4, 136, 72), (3, 16, 6, 512, 712), (7, 8, 2, 1024, 256), (16, 32, 8, 256, 64),
    (17, 5, 3, 264, 136), (33, 12, 4, 128, 200), (64, 60, 8, 512, 96), (65, 3, 2, 640, 320), (128, 16, 8, 384, 128), (128, 1, 1, 64, 1024),
    (128, 64, 16, 64, 64), (1, 64, 32, 128, 128), (5, 1024, 8, 64, 16)])
def test_against_the_formula(dt, T, E, K, H, I):
    _check(T, E, K, H, I, dt, act="silu" if T % 2 else "gelu")


@pytest.mark.parametrize("T", [1, 5, 40, 128])
def test_experts_of_other_shards(T):
    _check(T, 8, 4, 256, 128, torch.bfloat16, shards=8, idt=torch.int32)


def test_routings_with_gaps_and_repeats():
    dt = torch.bfloat16
    t = lambda rows: torch.tensor(rows, device="cuda")
    none = _check(3, 4, 2, 128, 64, dt, ids=t([[-1, -1], [4, 99], [-5, 2 ** 33]]))            # nobody chose a local expert
    assert not none.any()
    part = _check(3, 4, 2, 128, 64, dt, ids=t([[-1, -1], [3, -1], [-1, 0]]))
    assert not part[0].any() and part[1].any()
    _check(3, 4, 3, 128, 64, dt, ids=t([[2, 2, 2], [1, 2, 1], [-1, 3, 3]]))                   # the same expert twice
    _check(20, 4, 1, 128, 64, dt, ids=t([[3]] * 20))                                          # everybody the same one
    _check(128, 4, 2, 256, 72, dt, ids=t([[0, 3]] * 127 + [[1, 1]]))
    _check(40, 64, 1, 128, 64, dt, ids=torch.arange(40, device="cuda")[:, None])              # everybody another one
    _check(2, 4, 2, 128, 64, dt, ids=t([[0, 1], [2, 3]]), probs=torch.tensor([[0.0, 1.0], [-0.5, 2.0]], device="cuda"))


def test_wide_and_long():
    _check(4, 6, 2, 4096, 1024, torch.bfloat16)
    _check(70, 8, 2, 2056, 1416, torch.float16)


def test_strided_inputs_and_views():
    from primus_turbo.pytorch.ops import moe_few_tokens
    x, gu, dn = _make((6, 300), torch.bfloat16, 1), _make((4, 128, 256), torch.bfloat16, 2, 0.06), _make((4, 256, 64), torch.bfloat16, 3, 0.1)
    ids, probs = _routing(6, 2, 4, 4)
    want = moe_few_tokens(x[:, 3:259].contiguous(), gu, dn, ids, probs)
    assert torch.equal(moe_few_tokens(x[:, 3:259], gu, dn, ids, probs), want)
    odd = torch.empty(6 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 256).copy_(x[:, 3:259])
    assert torch.equal(moe_few_tokens(odd, gu, dn, ids.repeat(1, 2)[:, :2], probs.t().contiguous().t()), want)
    assert torch.equal(moe_few_tokens(x[:, 3:259], gu.transpose(1, 2).contiguous().transpose(1, 2), dn, ids, probs), want)


def test_no_tokens_and_bad_rows():
    from primus_turbo.pytorch.ops import moe_few_tokens
    x, gu, dn = _make((5, 128), torch.bfloat16, 1), _make((4, 128, 128), torch.bfloat16, 2, 0.06), _make((4, 128, 64), torch.bfloat16, 3, 0.1)
    ids, probs = _routing(5, 2, 4, 4)
    assert moe_few_tokens(x[:0], gu, dn, ids[:0], probs[:0]).shape == (0, 128)
    want = moe_few_tokens(x, gu, dn, ids, probs)
    x[2, 5], x[4, 0] = float("nan"), float("inf")
    got = moe_few_tokens(x, gu, dn, ids, probs)
    assert torch.equal(got[[0, 1, 3]], want[[0, 1, 3]]) and got[2].isnan().all()


def test_gradients_are_refused():
    from primus_turbo.pytorch.ops import moe_few_tokens
    x, gu, dn = _make((5, 128), torch.bfloat16, 1).requires_grad_(), _make((4, 128, 128), torch.bfloat16, 2), _make((4, 128, 64), torch.bfloat16, 3)
    ids, probs = _routing(5, 2, 4, 4)
    with pytest.raises(RuntimeError, match="no backward"):
        moe_few_tokens(x, gu, dn, ids, probs)
    with torch.no_grad():
        moe_few_tokens(x, gu, dn, ids, probs)


@pytest.mark.parametrize("T,E,K", [(1, 8, 2), (24, 16, 4)])
def test_same_bits_on_streams_and_in_graphs(T, E, K):
    from primus_turbo.pytorch.ops import moe_few_tokens
    H, I = 512, 256
    gu, dn = _make((E, 2 * I, H), torch.bfloat16, 2, 0.04), _make((E, H, I), torch.bfloat16, 3, 0.06)
    ins = [(_make((T, H), torch.bfloat16, i), *_routing(T, K, E, i)) for i in range(2)]
    call = lambda v: moe_few_tokens(v[0], gu, dn, v[1], v[2])
    want = [call(v) for v in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        got = []
        for v, s in zip(ins, streams):
            with torch.cuda.stream(s):
                got.append(call(v))
        torch.cuda.synchronize()
        assert all(torch.equal(g, t) for g, t in zip(got, want))
    graphs, held = [], []
    for v in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(call(v))
        graphs.append(g)
    for _ in range(10):
        for h in held:
            h.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(h, t) for h, t in zip(held, want))
    # other tokens and another routing through the captured call
    ins[0][0].copy_(ins[1][0]); ins[0][1].copy_(ins[1][1]); ins[0][2].copy_(ins[1][2])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], want[1])


def test_weights_beyond_32_bits():
    """The last of 150 experts of 7168 x 1024: its gate rows start past 2^31 elements."""
    from primus_turbo.pytorch.ops import moe_few_tokens
    E, H, I = 150, 7168, 1024
    gu, dn = _make((1, 2 * I, H), torch.bfloat16, 1, H ** -0.5), _make((1, H, I), torch.bfloat16, 2, I ** -0.5)
    big_gu, big_dn = torch.zeros((E, 2 * I, H), dtype=torch.bfloat16, device="cuda"), torch.zeros((E, H, I), dtype=torch.bfloat16, device="cuda")
    assert (E - 1) * 2 * I * H > 2 ** 31
    big_gu[-1], big_dn[-1] = gu[0], dn[0]
    x, p = _make((3, H), torch.bfloat16, 3), torch.rand(3, 1, device="cuda")
    ids = torch.full((3, 1), E - 1, device="cuda")
    want, tol = _oracle(x, gu, dn, torch.zeros_like(ids), p, "silu")
    assert ((moe_few_tokens(x, big_gu, big_dn, ids, p).double() - want).abs() <= tol).all()
