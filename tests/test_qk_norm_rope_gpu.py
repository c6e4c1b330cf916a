"""qk_norm_rope against the formulas in 64 bits: forward, gradients (formula and central differences), layouts, edge rows.

Tolerances.  With u = 2^-24 the kernel's fp32 arithmetic leaves, to first order, a relative error of at most (D + 16) u on a
normalised element (the sum of D squares contributes D u at worst, rsqrt and the products the rest), which the rotation spreads
over the pair: (D + 16) u (|n_a| + |n_b|).  The rounding of the result adds half a step of its type, and fp16 results below its
normal range half of 2^-24.  The backward has one more sum of D terms and a few more products: (2 D + 48) u times the sum of the
magnitudes that enter; dgamma adds its sum over the rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step relative to the value
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def _tables(P, R, base=1e4):
    ang = torch.arange(P, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))[None, :]
    return ang.cos().float().cuda(), ang.sin().float().cuda()


def _rotate(v, c, s, il, sign=1.0, absolute=False):
    """Rotation of the first R elements of v [..., H, D] in 64 bits; absolute: the sum of the magnitudes instead."""
    R = 2 * c.shape[-1]
    c, s = c[..., None, :], sign * s[..., None, :]
    head, rest = v[..., :R], v[..., R:]
    a, b = (head[..., 0::2], head[..., 1::2]) if il else (head[..., :R // 2], head[..., R // 2:])
    if absolute:
        x = y = a + b
    else:
        x, y = a * c - b * s, b * c + a * s
    head = torch.stack([x, y], -1).flatten(-2) if il else torch.cat([x, y], -1)
    return torch.cat([head, rest], -1)


def _oracle(x, g, c, s, il, zc, eps):
    x, g = x.double(), g.double() + (1.0 if zc else 0.0)
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * g
    return _rotate(n, c, s, il), _rotate(n.abs(), c, s, il, absolute=True)


def _oracle_bwd(x, g, dy, c, s, il, zc, eps):
    """dx, dgamma and the magnitudes that their bounds multiply."""
    x, g, dy = x.double(), g.double() + (1.0 if zc else 0.0), dy.double()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    xh = x * r
    dn, dn_mag = _rotate(dy, c, s, il, -1.0), _rotate(dy.abs(), c, s, il, absolute=True)
    w, w_mag = dn * g, dn_mag * g.abs()
    dx = (w - xh * (w * xh).mean(-1, keepdim=True)) * r
    mag = (w_mag + xh.abs() * (w_mag * xh.abs()).mean(-1, keepdim=True)) * r
    dims = tuple(range(x.dim() - 1))
    return dx, mag, (dn * xh).sum(dims), (dn_mag * xh.abs()).sum(dims)


def _within(got, want, mag, factor, dt, what):
    err = (got.double() - want).abs()
    tol = HALF[dt] * (want.abs() + factor * U * mag) + factor * U * mag + TINY[dt]
    bad = (err > tol) | err.isnan()
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err - tol).max()):.3e} over"


def _check(q, k, qg, kg, cos, sin, pos, il, zc, eps, dq=None, dk=None):
    from primus_turbo.pytorch.kernels import _native as nv
    from primus_turbo.pytorch.ops import qk_norm_rope
    D, dt = q.shape[-1], q.dtype
    grad = dq is not None
    leaves = [t.detach().requires_grad_(grad) for t in (q, k, qg, kg)]
    qo, ko = qk_norm_rope(*leaves, cos, sin, positions=pos, eps=eps, interleaved=il, zero_centered=zc)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == dt and qo.is_contiguous() and ko.is_contiguous()
    idx = torch.arange(q.shape[-3], device="cuda").expand(q.shape[:-2]) if pos is None else pos.long()
    c, s = cos.double()[idx], sin.double()[idx]
    for x, g, o, name in ((q, qg, qo, "q"), (k, kg, ko, "k")):
        want, mag = _oracle(x, g, c, s, il, zc, eps)
        _within(o.detach(), want, mag, D + 16, dt, f"{name} forward")
    if grad:
        grads = torch.autograd.grad([qo, ko], leaves, [dq, dk])
        for x, g, dy, dx, dg, name in ((q, qg, dq, grads[0], grads[2], "q"), (k, kg, dk, grads[1], grads[3], "k")):
            want, mag, wg, mg = _oracle_bwd(x, g, dy, c, s, il, zc, eps)
            assert dx.shape == x.shape and dg.shape == g.shape
            _within(dx, want, mag, 2 * D + 48, dt, f"d{name}")
            _within(dg, wg, mg, x.numel() // D + 2 * D + 48, dt, f"d{name}_gamma")
    nv.check_status(q.device)


def _make(shape, dt, seed, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std + mean).to(dt).cuda()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R", [
    (1, 32, 8, 128, 128), (1, 1, 1, 64, 64), (37, 5, 3, 128, 128), (19, 33, 1, 64, 32), (8, 4, 4, 256, 256), (5, 7, 2, 80, 80),
    (6, 9, 2, 96, 44), (4, 3, 2, 192, 92), (3, 2, 2, 512, 512), (3, 2, 1, 50, 14), (2, 3, 1, 37, 6), (2, 2, 1, 1000, 500),
    (9, 2, 2, 128, 0), (130, 16, 2, 64, 28), (2, 1, 1, 8, 8), (3, 2, 2, 2, 2), (3, 2, 2, 1, 0), (4, 2, 0, 64, 64), (4, 0, 2, 64, 64)])
def test_forward_and_gradients(dt, il, T, Hq, Hk, D, R):
    cos, sin = _tables(300, R)
    q, k = _make((T, Hq, D), dt, 1, 1.5), _make((T, Hk, D), dt, 2, 0.3)
    qg, kg = _make((D,), dt, 3, 0.2, 1.0), _make((D,), dt, 4, 0.2, 1.0)
    dq, dk = _make((T, Hq, D), dt, 5), _make((T, Hk, D), dt, 6)
    pos = torch.randint(0, 300, (T,), generator=torch.Generator().manual_seed(7)).cuda()
    _check(q, k, qg, kg, cos, sin, pos, il, False, 1e-6, dq, dk)


@pytest.mark.parametrize("il", [False, True])
def test_many_rows_and_zero_centered_gains(il):
    cos, sin = _tables(2100, 64)
    q, k = _make((2051, 12, 128), torch.bfloat16, 1), _make((2051, 4, 128), torch.bfloat16, 2)
    qg, kg = _make((128,), torch.bfloat16, 3, 0.1), _make((128,), torch.bfloat16, 4, 0.1)
    dq, dk = _make(q.shape, torch.bfloat16, 5), _make(k.shape, torch.bfloat16, 6)
    _check(q, k, qg, kg, cos, sin, None, il, True, 1e-5, dq, dk)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layouts(dt):
    """Views into a packed projection, batches, heads-first storage, odd strides, gradients that are expanded or transposed."""
    D, R, B, S, Hq, Hk = 64, 64, 3, 11, 6, 2
    cos, sin = _tables(64, R)
    qg, kg = _make((D,), dt, 3, 0.2, 1.0), _make((D,), dt, 4, 0.2, 1.0)
    pos32 = torch.randint(0, 64, (B, S), generator=torch.Generator().manual_seed(8)).to(torch.int32).cuda()
    packed = _make((B, S, (Hq + 2 * Hk) * D), dt, 1)
    q, k = packed[..., :Hq * D].view(B, S, Hq, D), packed[..., Hq * D:(Hq + Hk) * D].view(B, S, Hk, D)
    dq, dk = _make((B, Hq, S, D), dt, 5).transpose(1, 2), _make((B, S, 1, D), dt, 6).expand(B, S, Hk, D)
    _check(q, k, qg, kg, cos, sin, pos32, False, False, 1e-6, dq, dk)
    _check(q, k, qg, kg, cos, sin, None, True, False, 1e-6, dq, dk)
    q, k = _make((B, Hq, S, D), dt, 1).transpose(1, 2), _make((B, Hk, S, D), dt, 2).transpose(1, 2)
    _check(q, k, qg, kg, cos, sin, pos32.long(), False, False, 1e-6, dq, dk)
    odd = _make((B, S, Hq * (D + 1) + 1), dt, 9)[..., 1:].view(B, S, Hq, D + 1)[..., :D]      # rows that start at odd elements
    _check(odd, k, qg, kg, cos, sin, pos32, False, False, 1e-6, dq, dk)
    even = _make((S, Hq, D + 2), dt, 9)[..., 2:]                                              # ... at even, unaligned ones
    _check(even, _make((S, Hk, D), dt, 2), qg, kg, cos, sin, None, False, False, 1e-6, _make((S, Hq, D), dt, 5), _make((S, Hk, D), dt, 6))
    five = _make((2, 2, 3, Hq, D), dt, 9)
    _check(five, five[..., :1, :], qg, kg, cos, sin, None, False, False, 1e-6, five, five[..., :1, :])
    last = _make((S, D, Hq), dt, 9).transpose(1, 2)                                           # last dimension not contiguous
    _check(last, last, qg, kg, cos, sin, None, False, False, 1e-6, last, last)


def test_gradient_against_central_differences():
    """Differences of the formula in 64 bits (step 1e-5: their own error is far below the fp32 bound) against the kernel's fp32
    gradient along random directions."""
    from primus_turbo.pytorch.ops import qk_norm_rope
    T, H, D, R = 5, 3, 32, 16
    cos, sin = _tables(T, R)
    q, k = _make((T, H, D), torch.float32, 1), _make((T, 1, D), torch.float32, 2)
    qg, kg = _make((D,), torch.float32, 3, 0.2, 1.0), _make((D,), torch.float32, 4, 0.2, 1.0)
    w = [_make((T, H, D), torch.float32, 5), _make((T, 1, D), torch.float32, 6)]
    leaves = [t.clone().requires_grad_() for t in (q, k, qg, kg)]
    grads = torch.autograd.grad(list(qk_norm_rope(*leaves, cos, sin)), leaves, w)
    c, s = cos.double(), sin.double()

    def loss(q, k, qg, kg):
        return float((_oracle(q, qg, c, s, False, False, 1e-6)[0] * w[0]).sum() + (_oracle(k, kg, c, s, False, False, 1e-6)[0] * w[1]).sum())

    base = [t.double() for t in (q, k, qg, kg)]
    for i in range(4):
        v = _make(base[i].shape, torch.float64, 20 + i)
        up, down = [t.clone() for t in base], [t.clone() for t in base]
        up[i] += 1e-5 * v
        down[i] -= 1e-5 * v
        diff = (loss(*up) - loss(*down)) / 2e-5
        # magnitudes entering <grad, v>: at most |grad's bound| |v|; 64-bit difference error ~ 1e-9 of the loss terms
        if i < 2:
            _, mag, _, _ = _oracle_bwd(base[i], base[2 + i], w[i], c, s, False, False, 1e-6)
            bound = (2 * D + 48) * U * mag
        else:
            _, _, _, mg = _oracle_bwd(base[i - 2], base[i], w[i - 2], c, s, False, False, 1e-6)
            bound = (2 * D + 48 + T * H) * U * mg
        tol = float(((bound + U * grads[i].double().abs()) * v.abs()).sum()) + 1e-7
        assert abs(float((grads[i].double() * v).sum()) - diff) <= tol


def test_rows_of_zeros_infinities_and_nan_stay_in_their_row():
    from primus_turbo.pytorch.ops import qk_norm_rope
    cos, sin = _tables(8, 64)
    q, k = _make((8, 4, 64), torch.bfloat16, 1), _make((8, 2, 64), torch.bfloat16, 2)
    g = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    clean = [t.clone() for t in qk_norm_rope(q, k, g, g, cos, sin)]
    q[1, 2] = 0
    q[2, 1, 5] = float("nan")
    q[3, 0, 7] = float("inf")
    out = qk_norm_rope(q, k, g, g, cos, sin)
    assert torch.equal(out[0][1, 2], torch.zeros(64, dtype=torch.bfloat16, device="cuda"))
    assert out[0][2, 1].isnan().all() and out[0][3, 0].isnan().any()
    same = torch.ones(8, 4, dtype=torch.bool)
    same[1, 2] = same[2, 1] = same[3, 0] = False
    assert torch.equal(out[0][same.cuda()], clean[0][same.cuda()]) and torch.equal(out[1], clean[1])


def test_position_outside_of_the_tables():
    """Its token comes out as zeros with zero gradients, the others are untouched, and the error surfaces."""
    from primus_turbo.pytorch.kernels import _native as nv
    from primus_turbo.pytorch.ops import qk_norm_rope
    cos, sin = _tables(16, 64)
    q, k = _make((3, 4, 64), torch.bfloat16, 1).requires_grad_(), _make((3, 1, 64), torch.bfloat16, 2)
    g = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for bad in (16, -1, 2 ** 40):
        good = torch.tensor([3, 4, 5], device="cuda")
        pos = torch.tensor([3, bad, 5], device="cuda")
        want = qk_norm_rope(q, k, g, g, cos, sin, positions=good)[0].detach()
        got = qk_norm_rope(q, k, g, g, cos, sin, positions=pos)[0]
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside of its table"):
            nv.check_status(q.device)
        assert torch.equal(got[[0, 2]], want[[0, 2]]) and not got[1].any()
        dq = torch.autograd.grad(got.sum(), q)[0]
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside of its table"):
            qk_norm_rope(q, k, g, g, cos, sin, positions=good)
        assert not dq[1].any() and dq[0].any()
    nv.check_status(q.device)


def test_no_tokens():
    from primus_turbo.pytorch.ops import qk_norm_rope
    cos, sin = _tables(16, 64)
    q, k = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    g = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    qo, ko = qk_norm_rope(q, k, g, g, cos, sin)
    assert qo.shape == q.shape and ko.shape == k.shape
    (dg,) = torch.autograd.grad(qo.sum() + ko.sum(), g)
    assert torch.equal(dg, torch.zeros_like(dg))


def test_same_bits_every_run_on_another_stream_and_in_a_graph():
    from primus_turbo.pytorch.ops import qk_norm_rope
    cos, sin = _tables(600, 128)
    q, k = _make((600, 8, 128), torch.bfloat16, 1).requires_grad_(), _make((600, 2, 128), torch.bfloat16, 2).requires_grad_()
    qg, kg = _make((128,), torch.bfloat16, 3).requires_grad_(), _make((128,), torch.bfloat16, 4).requires_grad_()
    dq, dk = _make(q.shape, torch.bfloat16, 5), _make(k.shape, torch.bfloat16, 6)

    def step():
        out = qk_norm_rope(q, k, qg, kg, cos, sin)
        return [o.detach() for o in out] + list(torch.autograd.grad(list(out), [q, k, qg, kg], [dq, dk]))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            again = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_offsets_beyond_32_bits():
    """Tokens more than 2^31 elements apart, read in place and written beyond 2^31 elements of the output."""
    from primus_turbo.pytorch.ops import qk_norm_rope
    cos, sin = _tables(4, 64)
    g = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    wide = torch.empty(3, 2 ** 30 + 128, dtype=torch.bfloat16, device="cuda")
    q, k = wide[:, 64:64 + 4 * 64].view(3, 4, 64), wide[:, -128:].view(3, 2, 64)
    q.copy_(_make((3, 4, 64), torch.bfloat16, 1))
    k.copy_(_make((3, 2, 64), torch.bfloat16, 2))
    _check(q, k, g, g, cos, sin, None, False, False, 1e-6, _make((3, 4, 64), torch.bfloat16, 3), _make((3, 2, 64), torch.bfloat16, 4))
    del wide
    T = 2 ** 31 // (8 * 128) + 5
    big = torch.empty(T, 8, 128, dtype=torch.bfloat16, device="cuda")
    big[-3:].copy_(_make((3, 8, 128), torch.bfloat16, 5))
    g = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    cos, sin = _tables(8, 128)
    pos = torch.arange(T, device="cuda") % 8
    out = qk_norm_rope(big, big[:, :1], g, g, cos, sin, positions=pos)
    want = qk_norm_rope(big[-3:], big[-3:, :1], g, g, cos, sin, positions=pos[-3:])
    assert torch.equal(out[0][-3:], want[0]) and torch.equal(out[1][-3:], want[1])
