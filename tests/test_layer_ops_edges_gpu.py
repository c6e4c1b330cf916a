"""Edges of the operators around a decoder layer's products: empty inputs, values at the ends of the types' ranges, tails of the
activations, sizes at which a block of tokens holds next to nothing."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _rand(shape, seed, std=1.0, dt=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, std, generator=g).to(dt)


# ------------------------------------------------------------------------------------------------ qk_norm_rope
@pytest.mark.parametrize("idt", [None, torch.int32, torch.int64])
@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3)])
def test_qk_norm_rope_without_tokens(idt, lead):
    """Empty outputs and gradients of zero for the gains, with positions and without."""
    from primus_turbo.pytorch.ops import qk_norm_rope
    q, k = (torch.empty((*lead, h, 64), dtype=BF, device="cuda", requires_grad=True) for h in (4, 2))
    qg, kg = _rand((64,), 1).requires_grad_(), _rand((64,), 2).requires_grad_()
    cos = sin = torch.ones(8, 32, device="cuda")
    pos = None if idt is None else torch.empty(lead, dtype=idt, device="cuda")
    q_out, k_out = qk_norm_rope(q, k, qg, kg, cos, sin, positions=pos)
    assert q_out.shape == q.shape and k_out.shape == k.shape
    dq, dk, dqg, dkg = torch.autograd.grad([q_out, k_out], [q, k, qg, kg], [torch.empty_like(q_out), torch.empty_like(k_out)])
    assert dq.shape == q.shape and dk.shape == k.shape and not dqg.any() and not dkg.any()


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
@pytest.mark.parametrize("enabled", [True, False])
def test_forward_mode_derivatives_are_refused(enabled):
    """None of the operators has them: a tangent is refused, not dropped, under torch.no_grad too; without one nothing changes."""
    from torch.autograd import forward_ad
    from primus_turbo.pytorch import ops
    x, w, h, g, t = _rand((4, 64), 1), _rand((16, 64), 2), _rand((4, 2, 32), 3), _rand((32,), 4), torch.ones(4, 16, device="cuda")
    gu, dn, ids, p = _rand((2, 16, 64), 5), _rand((2, 64, 8), 6), torch.zeros(4, 1, dtype=torch.int64, device="cuda"), torch.ones(4, 1, device="cuda")
    calls = [(lambda a, b: ops.gemm_bias_act(a, b, trans_b=True), (x, w)), (lambda a, b: ops.gemm_bias_act(x, w, bias=a, residual=b, trans_b=True), (w[:, 0], _rand((4, 16), 7))),
             (lambda a, b: ops.qk_norm_rope(a, h, b, g, t, t)[0], (h, g)), (lambda a, b: ops.qk_norm_rope(h, a, g, g, b, t)[1], (h, t)),
             (lambda a, b: ops.moe_few_tokens(a, gu, dn, ids, b), (x, p)), (lambda a, b: ops.moe_few_tokens(x, a, b, ids, p), (gu, dn))]
    with torch.set_grad_enabled(enabled):
        for call, args in calls:
            want = call(*args)
            with forward_ad.dual_level():
                assert torch.equal(call(*args), want)
                for i in range(2):
                    dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
                    with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                        call(*dual)
            assert torch.equal(call(*args), want)


# ------------------------------------------------------------------------------------------------ PT_CHECK_STATUS
def test_check_status_variable_raises_at_the_launch(monkeypatch):
    """With PT_CHECK_STATUS=1 the call whose kernel reports raises, forward and backward; without it a following call does."""
    from primus_turbo.pytorch import ops
    from primus_turbo.pytorch.kernels import _native as nv
    q, g, t = _rand((3, 2, 32), 1).requires_grad_(), _rand((32,), 2), torch.ones(4, 16, device="cuda")
    good, bad = torch.tensor([0, 1, 3], device="cuda"), torch.tensor([0, 4, 1], device="cuda")
    call = lambda pos: ops.qk_norm_rope(q, q, g, g, t, t, positions=pos)
    nv.check_status(q.device)
    monkeypatch.setenv("PT_CHECK_STATUS", "1")
    for _ in range(2):
        with pytest.raises(RuntimeError, match="outside of its table"):
            call(bad)
        call(good)
    pos = good.clone()
    y = call(pos)
    pos.data.copy_(bad)
    with pytest.raises(RuntimeError, match="outside of its table"):
        torch.autograd.grad(y[0].float().sum(), q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):      # nothing waits inside a capture
        call(good)
    graph.replay()
    monkeypatch.setenv("PT_CHECK_STATUS", "0")
    call(bad)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside of its table"):
        call(good)
    nv.check_status(q.device)


@pytest.mark.parametrize("name", ["gemm_bias_act", "moe_few_tokens", "backward"])
def test_check_status_variable_reaches_every_operator(monkeypatch, name):
    """A code that stands in the mapped word when the launch is over, put there by the host after the call has looked at it."""
    from primus_turbo.pytorch import ops
    from primus_turbo.pytorch.kernels import _native as nv
    x, w = _rand((4, 64), 1), _rand((16, 64), 2)
    gu, dn, ids, p = _rand((2, 16, 64), 3), _rand((2, 64, 8), 4), torch.zeros(4, 1, dtype=torch.int64, device="cuda"), torch.ones(4, 1, device="cuda")
    calls = {"gemm_bias_act": lambda: ops.gemm_bias_act(x, w, trans_b=True), "moe_few_tokens": lambda: ops.moe_few_tokens(x, gu, dn, ids, p)}
    y = ops.gemm_bias_act(x.requires_grad_(name == "backward"), w, trans_b=True)
    calls["backward"] = lambda: y.backward(torch.ones_like(y))
    word, look = nv._host_status[x.device.index][1], nv.mapped_status
    if name == "moe_few_tokens":
        calls[name]()
    monkeypatch.setenv("PT_CHECK_STATUS", "1")

    def leave_a_code(device):
        address = look(device)
        word.value = -4      # PT_ERR_TIMEOUT
        return address
    monkeypatch.setattr(nv, "mapped_status", leave_a_code)
    monkeypatch.setattr(nv, "check_status", lambda device: look(device))
    with pytest.raises(RuntimeError, match="gave up waiting"):
        calls[name]()
    assert word.value == 0


# ------------------------------------------------------------------------------------------------ gemm_bias_act at the ends of the range
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt,av,bv", [(F16, 200.0, 100.0), (BF, 2.0 ** 50, 2.0 ** 20)])
def test_slopes_of_large_pre_activations(dt, av, bv, act):
    """Pre-activations of +-8 av bv: beyond fp16's range, or with a square beyond fp32's.  Every slope is 1 or 0 there, and all sums are
    exact in the operands' type."""
    from primus_turbo.pytorch.ops import gemm_bias_act
    M, N, K = 3, 24, 8
    a = torch.full((M, K), av, dtype=dt, device="cuda").requires_grad_()
    sign = torch.where(torch.arange(N, device="cuda") % 3 == 0, -1.0, 1.0)
    b = (bv * sign)[:, None].expand(N, K).to(dt).contiguous().requires_grad_()
    bias = torch.zeros(N, dtype=dt, device="cuda").requires_grad_()
    y = gemm_bias_act(a, b, bias=bias, activation=act, trans_b=True, out_dtype=F32)
    assert torch.equal(y, (8 * av * bv * sign.clamp(min=0)).float().expand(M, N))
    da, db, dbias = torch.autograd.grad(y, (a, b, bias), torch.ones_like(y))
    open_ = sign.clamp(min=0)
    assert torch.equal(da.float(), torch.full((M, K), 16 * bv, device="cuda"))
    assert torch.equal(db.float(), (M * av * open_)[:, None].expand(N, K)) and torch.equal(dbias.float(), M * open_)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradients_of_nan_stay_nan(act):
    from primus_turbo.pytorch.ops import gemm_bias_act
    a, b = _rand((3, 16), 1), _rand((24, 16), 2)
    a[1, 3] = float("nan")
    a.requires_grad_()
    (da,) = torch.autograd.grad(gemm_bias_act(a, b, activation=act, trans_b=True).sum(), a)
    assert da[1].isnan().all() and da[[0, 2]].isfinite().all()


# ------------------------------------------------------------------------------------------------ the GELU of the epilogues
@pytest.mark.parametrize("M,N", [(2000, 8), (2000, 5), (40000, 260), (40000, 257), (9000, 1028), (9000, 1001)])
def test_gelu_in_fp32_is_right_in_its_tail(M, N):
    """Exact pre-activations (one product of an fp16 value with a power of two) through both kernels, vector and ragged write-out.  The
    result is max(z, 0) - x R exp(-x^2 / 2), x = |z|; in half steps u of fp32 the second term may be off by 3 for the fit of R, 8 + 8 for the
    polynomial's roundings and its argument (conditioned by at most 2), 4 for the hardware exponential, 1.5 x^2 for the three roundings of its
    argument, 5 for the products: (45 + 1.5 x^2) u; the difference adds one more."""
    from primus_turbo.pytorch.kernels import _native as nv
    from primus_turbo.pytorch.ops import gemm_bias_act
    assert bool(nv.lib().pt_gemm_bias_act_few_rows(M, N, 8)) == (M == 2000)
    a, b = torch.zeros(M, 8, dtype=F16, device="cuda"), torch.zeros(N, 8, dtype=F16, device="cuda")
    a[:, 3] = torch.linspace(-12.5, 6.0, M, device="cuda").to(F16)
    b[:, 3] = 2.0 ** -(torch.arange(N, device="cuda") % 5).to(F16)
    z = a[:, 3:4].double() * b[:, 3].double()
    y = gemm_bias_act(a, b, activation="gelu", trans_b=True, out_dtype=F32).double()
    tail = 0.5 * z.abs() * torch.erfc(z.abs() / math.sqrt(2))
    err = (y - (z.clamp(min=0) - tail)).abs()
    tol = (45 + 1.5 * z * z) * U * tail + U * y.abs() + 1e-44
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f} x tolerance"


# ------------------------------------------------------------------------------------------------ moe_few_tokens
@pytest.mark.parametrize("which", ["gate_up", "down"])
def test_moe_few_tokens_refuses_weights_off_the_16_byte_boundary(which):
    from primus_turbo.pytorch.ops import moe_few_tokens
    shapes = dict(gate_up=(4, 48, 64), down=(4, 64, 24))
    w = {n: _rand((math.prod(s) + 8,), i, 0.1)[4 if n == which else 0:][:math.prod(s)].view(s) for i, (n, s) in enumerate(shapes.items())}
    x, ids, p = _rand((3, 64), 5), torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, 1, device="cuda")
    with pytest.raises((RuntimeError, ValueError), match="16-byte boundaries"):
        moe_few_tokens(x, w["gate_up"], w["down"], ids, p)
    w[which] = w[which].clone()
    assert moe_few_tokens(x, w["gate_up"], w["down"], ids, p).isfinite().all()


@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_moe_few_tokens_reads_the_routing_of_this_call(idt):
    """The routing is rewritten in place by the kernel just ahead of every call, eagerly and in a replayed graph: the second product, which
    starts before the first has finished, must see the new one."""
    from primus_turbo.pytorch.ops import moe_few_tokens
    T, E, K, H, I, rounds = 6, 8, 2, 512, 264, 24
    x, gu, dn, p = _rand((T, H), 1), _rand((E, 2 * I, H), 2, 0.05), _rand((E, H, I), 3, 0.06), torch.rand(T, K, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    tables = torch.rand((rounds, T, E), generator=g, device="cuda").topk(K, dim=2).indices.to(idt)
    want = []
    for t in tables:
        torch.cuda.synchronize()
        want.append(moe_few_tokens(x, gu, dn, t.clone(), p))
    torch.cuda.synchronize()
    ids, got = tables[0].clone(), []

    def steps():
        for t in tables:
            ids.copy_(t)
            got.append(moe_few_tokens(x, gu, dn, ids, p))
    steps()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps()
    for _ in range(3):
        for y in got:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ host threads
@pytest.mark.parametrize("shared_stream", [False, True])
def test_same_bits_from_several_threads(shared_stream):
    """Four host threads, each on a stream of its own or all on one, forward and backward: the bits of the same calls one after another."""
    import threading
    from primus_turbo.pytorch import ops
    t = torch.ones(64, 32, device="cuda")
    cases = []
    for i in range(4):
        x, w, b = _rand((3 + 40 * i, 256), i), _rand((264, 256), 10 + i, 0.06), _rand((264,), 20 + i)
        q, g = _rand((5 + i, 6, 64), 30 + i), _rand((64,), 40 + i)
        gu, dn, p = _rand((4, 96, 256), 50 + i, 0.06), _rand((4, 256, 48), 60 + i, 0.1), torch.rand(3, 2, device="cuda")
        ids = (torch.arange(6, device="cuda").view(3, 2) + i) % 4

        def run(x=x, w=w, b=b, q=q, g=g, gu=gu, dn=dn, p=p, ids=ids):
            a, v, h = x.detach().requires_grad_(), w.detach().requires_grad_(), q.detach().requires_grad_()
            y = ops.gemm_bias_act(a, v, bias=b, activation="gelu", trans_b=True)
            z = ops.qk_norm_rope(h, h[:, :2], g, g, t, t)
            return [y.detach(), *torch.autograd.grad(y, (a, v), y.detach()), z[0].detach(), *torch.autograd.grad(z, h, [z[0].detach(), z[1].detach()]),
                    ops.moe_few_tokens(x[:3], gu, dn, ids, p)]
        cases.append(run)
    want = [run() for run in cases]
    torch.cuda.synchronize()
    common, wrong = torch.cuda.Stream(), []

    def work(i):
        stream = common if shared_stream else torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(25):
                got = cases[i]()
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


# ------------------------------------------------------------------------------------------------ captured training steps
@pytest.mark.parametrize("M,N,K", [(3, 264, 96), (300, 264, 96), (8200, 1028, 264)])
@pytest.mark.parametrize("fused", [False, True])
def test_captured_training_step_follows_new_inputs(M, N, K, fused):
    """Forward and backward of a product and of the head norm in one graph, replayed on inputs that changed: the bits of eager calls on them,
    also where the weight's gradient is added to main_grad."""
    from primus_turbo.pytorch import ops
    a, b, bias = (t.requires_grad_() for t in (_rand((M, K), 1), _rand((N, K), 2, 0.1), _rand((N,), 3)))
    q, g, t = _rand((M, 3, 64), 4).requires_grad_(), _rand((64,), 5).requires_grad_(), torch.linspace(-1, 1, 16 * 32, device="cuda").view(16, 32)
    pos, dy, dq = torch.arange(M, device="cuda") % 16, _rand((M, N), 6), _rand((M, 3, 64), 7)
    if fused:
        b.main_grad, b.grad_added_to_main_grad = torch.zeros(N, K, device="cuda"), False

    def step():
        y = ops.gemm_bias_act(a, b, bias=bias, activation="gelu", trans_b=True, fuse_bgrad_accum_pattern="megatron" if fused else None)
        u, _ = ops.qk_norm_rope(q, q.detach()[:, :1], g, g.detach(), t, t, positions=pos)
        grads = torch.autograd.grad([y, u], [a, b, bias, q, g], [dy, dq])
        return [y.detach(), u.detach(), grads[0], b.main_grad if fused else grads[1], *grads[2:]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (11, 12):
        with torch.no_grad():
            for i, x in enumerate((a, b, bias, q, g, dy, dq)):
                x.copy_(_rand(x.shape, seed * 10 + i))
            pos.copy_(torch.randint(0, 16, (M,), generator=torch.Generator().manual_seed(seed)).cuda())
        if fused:
            b.main_grad.fill_(0.5)
        want = [w.clone() for w in step()]
        if fused:
            b.main_grad.fill_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, w) for x, w in zip(held, want))
