"""gemm_bias_act against the formula in 64 bits: both kernels (few rows, tiles), every activation, layouts, gradients.

Tolerances, u = 2^-24.  The products of 16-bit operands are exact in fp32; the tensor core adds 16 of them per instruction to the
accumulator, at worst one truncation (2 u) per instruction and inside it a few bits more: |z error| <= (K / 8 + 32) 2 u sum|a||b| +
u |z|.  The activations have slopes of at most 1.13 and second derivatives of at most 0.9; their evaluation (hardware exponential
of an argument of up to some tens, approximate division) stays within 128 u (|z| + |act|).  Each result adds half a step of its
type.  The backward evaluates act' at z rounded to the operands' type and rounds dz once to it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def _make(shape, dt, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, std, generator=g).to(dt)


def _act(z, name):
    return {None: lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2)),
            "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}[name](z)


def _mm_bound(x, y, K):
    return (K / 8 + 32) * 2 * U * (x.abs() @ y.abs())


def _assert_within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = (err > tol) | err.isnan()
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / tol).max()):.2f} x tolerance"


def _few(M, N, K):
    """Whether the rule sends this size to the few-row kernels."""
    from primus_turbo.pytorch.kernels import _native as nv
    return bool(nv.lib().pt_gemm_bias_act_few_rows(M, N, (K + 7) // 8 * 8))


def _check(M, N, K, dt, act, with_bias, with_res, trans_b=True, out_dtype=None, bias_dtype=None, grad=False, seed=0, a=None):
    from primus_turbo.pytorch.kernels import _native as nv
    from primus_turbo.pytorch.ops import gemm_bias_act
    od = out_dtype or dt
    a = _make((M, K), dt, seed + 1) if a is None else a
    b = _make((N, K) if trans_b else (K, N), dt, seed + 2, K ** -0.5)
    bias = _make((N,), bias_dtype or dt, seed + 3) if with_bias else None
    res = _make((M, N), od, seed + 4, 2.0) if with_res else None
    leaves = [t.requires_grad_(grad) for t in (a, b, bias, res) if t is not None]
    y = gemm_bias_act(a, b, bias=bias, activation=act, residual=res, trans_b=trans_b, out_dtype=out_dtype)
    assert y.shape == (M, N) and y.dtype == od and y.is_contiguous()
    A, B = a.detach().double(), (b.detach().double().t() if trans_b else b.detach().double())
    z = A @ B + (0 if bias is None else bias.detach().double())
    ez = _mm_bound(A, B, K) + U * z.abs()
    want = _act(z, act)
    ey = 1.13 * ez + 128 * U * (z.abs() + want.abs())
    if res is not None:
        want = want + res.detach().double()
    _assert_within(y.detach(), want, ey + (HALF[od] + U) * (want.abs() + ey) + TINY[od], "y")
    if grad:
        dy = _make((M, N), od, seed + 5)
        got = dict(zip([n for n, t in zip("a b bias res".split(), (a, b, bias, res)) if t is not None], torch.autograd.grad(y, leaves, dy)))
        zz = z.clone().requires_grad_()
        (slope,) = torch.autograd.grad(_act(zz, act).sum(), zz)
        D = dy.double()
        dz = D * slope
        # slope at the rounded, inexact z; relu jumps where z may change sign
        es = {None: 0 * z, "relu": (z.abs() <= 2 * ez).double()}.get(act, 0.9 * (ez + HALF[dt] * (z.abs() + ez)) + 128 * U * (1 + z.abs()))
        ed = D.abs() * es + 2 * U * dz.abs()
        edr = ed + HALF[dt] * (dz.abs() + ed) + TINY[dt]
        da, db = dz @ B.t(), A.t() @ dz
        ta = edr @ B.t().abs() + _mm_bound(dz, B.t(), N)
        tb = A.t().abs() @ edr + _mm_bound(A.t(), dz, M)
        _assert_within(got["a"], da, ta + (HALF[dt] + U) * (da.abs() + ta) + TINY[dt], "da")
        if not trans_b:
            _assert_within(got["b"], db, tb + (HALF[dt] + U) * (db.abs() + tb) + TINY[dt], "db")
        else:
            _assert_within(got["b"], db.t(), (tb + (HALF[dt] + U) * (db.abs() + tb) + TINY[dt]).t(), "db")
        if bias is not None:
            wb, bt = dz.sum(0), bias.dtype
            tbias = ed.sum(0) + (M + 16) * U * dz.abs().sum(0)
            _assert_within(got["bias"], wb, tbias + (HALF[bt] + U) * (wb.abs() + tbias) + TINY[bt], "dbias")
        if res is not None:
            assert torch.equal(got["res"], dy)
    nv.check_status(y.device)
    return y


ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 128, 64), (1, 1, 8), (2, 129, 72), (3, 1000, 512), (7, 256, 4096), (16, 4101, 1024), (17, 64, 2048),
                                   (31, 333, 264), (32, 128, 128), (33, 640, 136), (64, 257, 320), (65, 96, 1096), (100, 2049, 64), (128, 130, 512), (129, 128, 64), (200, 257, 520), (300, 1001, 72),
                                   (513, 512, 1024), (1030, 4, 16), (777, 1028, 256), (2000, 130, 1024), (40000, 8, 72)])
def test_few_rows(dt, M, N, K):
    assert _few(M, N, K)
    for i, act in enumerate(ACTS):
        _check(M, N, K, dt, act, with_bias=i % 2 == 0, with_res=i % 3 != 1, seed=10 * i)


@pytest.mark.parametrize("M,N,K", [(65, 100, 1024), (129, 100, 1024), (192, 520, 2056), (200, 2056, 1024), (513, 4101, 64), (500, 3976, 1544),
                                   (300, 3976, 1544), (300, 4101, 1544), (222, 2049, 4104), (200, 2056, 4096), (130, 4096, 128), (700, 512, 200)])
def test_wide_blocks(M, N, K):
    """Blocks of more than 128 tokens, with one to eight shares of the contraction, single CTAs and pairs, even and odd numbers of weight
    blocks, and the write-out of several tokens at once with everything that may join it."""
    assert _few(M, N, K)
    _check(M, N, K, torch.bfloat16, "gelu", True, True)
    _check(M, N, K, torch.float16, "silu", False, True, out_dtype=torch.float32)
    if N % 8 == 0:
        _check(M, N, K, torch.bfloat16, None, True, False, trans_b=False)
    _check(M, N, K, torch.float16, "gelu_tanh", True, True, grad=True)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(33000, 130, 1032), (40000, 257, 2048), (9000, 1001, 1000)])
def test_tiles(dt, M, N, K):
    """Enough tiles for the tile kernels: single CTAs below 512 columns, CTA pairs from there on."""
    assert not _few(M, N, K)
    for i, act in enumerate(ACTS):
        _check(M, N, K, dt, act, with_bias=i % 2 == 0, with_res=i % 3 != 1, seed=10 * i)


@pytest.mark.parametrize("M,N,K,act", [(4100, 4104, 192, "gelu"), (4097, 4101, 64, "silu"), (8192, 4096, 64, None)])
def test_cta_pairs(M, N, K, act):
    assert not _few(M, N, K)
    _check(M, N, K, torch.bfloat16, act, True, True)


@pytest.mark.parametrize("M", [5, 300])
def test_types_layouts_and_ragged_contractions(M):
    bf, f32 = torch.bfloat16, torch.float32
    _check(M, 200, 96, bf, "silu", True, True, out_dtype=f32)
    _check(M, 200, 96, bf, "silu", True, True, out_dtype=torch.float16, bias_dtype=f32)
    _check(M, 201, 96, torch.float16, "gelu", True, True, out_dtype=f32, bias_dtype=f32)
    _check(M, 200, 96, bf, "gelu", True, False, trans_b=False)
    _check(M, 203, 100, bf, "gelu_tanh", True, True, trans_b=False)      # K not a multiple of 8: padded
    _check(M, 200, 3, bf, None, True, True)
    wide = _make((M, 300), bf, 1)
    _check(M, 200, 96, bf, None, True, True, a=wide[:, 100:196])           # strided rows
    flat = _make((M * 96 + 1,), bf, 1)
    _check(M, 200, 96, bf, None, True, True, a=flat[1:].view(M, 96))       # rows that start off the 16-byte boundary


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 136, 64), (40, 129, 200), (300, 256, 264), (513, 1000, 96)])
@pytest.mark.parametrize("act", ACTS)
def test_gradients(dt, M, N, K, act):
    _check(M, N, K, dt, act, True, True, grad=True)


def test_gradients_without_bias_other_layouts_and_types():
    bf = torch.bfloat16
    _check(200, 264, 128, bf, "silu", False, False, grad=True)
    _check(200, 264, 128, bf, None, False, True, grad=True)
    _check(200, 264, 128, bf, "gelu", True, True, trans_b=False, grad=True)
    _check(200, 261, 128, bf, "gelu", True, True, out_dtype=torch.float32, bias_dtype=torch.float32, grad=True)
    _check(200, 264, 128, bf, None, True, False, out_dtype=torch.float32, grad=True)


@pytest.mark.parametrize("M", [4, 300])
@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("off", [1, 2, 4])
def test_views_off_the_16_byte_boundary(M, trans_b, off):
    """Every tensor a view that starts `off` elements into a buffer: the bits of aligned copies, forward and backward."""
    from primus_turbo.pytorch.ops import gemm_bias_act
    N, K, bf = 264, 96, torch.bfloat16
    shapes = [(M, K), (N, K) if trans_b else (K, N), (N,), (M, N), (M, N)]

    def run(shift):
        ts = []
        for i, s in enumerate(shapes):
            buf = torch.zeros(math.prod(s) + 8, dtype=bf, device="cuda")
            v = buf[shift:shift + math.prod(s)].view(s)
            v.copy_(_make(s, bf, i + 1, 0.5))
            ts.append(v)
        a, b, bias, res = (t.requires_grad_() for t in ts[:4])
        y = gemm_bias_act(a, b, bias=bias, activation="silu", residual=res, trans_b=trans_b)
        return (y, *torch.autograd.grad(y, (a, b, bias, res), ts[4]))

    for got, want in zip(run(off), run(0)):
        assert torch.equal(got, want)


def test_expanded_and_strided_inputs():
    """Broadcast and transposed tensors are the values that they show; a broadcast leaf gets the sum over its copies."""
    from primus_turbo.pytorch.ops import gemm_bias_act
    M, N, K, bf = 40, 136, 64, torch.bfloat16
    row, col, b0, r0 = _make((1, K), bf, 1), _make((N, 1), bf, 2), _make((1,), bf, 3), _make((M,), bf, 4)
    a, b, bias, res = row.expand(M, K), col.expand(N, K), b0.expand(N), r0[:, None].expand(M, N)
    plain = [t.contiguous() for t in (a, b, bias, res)]
    assert torch.equal(gemm_bias_act(a, b, bias, "gelu", res, trans_b=True), gemm_bias_act(plain[0], plain[1], plain[2], "gelu", plain[3], trans_b=True))
    w = _make((K, N), bf, 5)
    assert torch.equal(gemm_bias_act(a, w.t(), bias, "gelu", res, trans_b=True), gemm_bias_act(plain[0], w.t().contiguous(), bias, "gelu", res, trans_b=True))
    big = _make((2 * M, 2 * N), bf, 6)
    assert torch.equal(gemm_bias_act(a, w, residual=big[::2, ::2]), gemm_bias_act(plain[0], w, residual=big[::2, ::2].contiguous()))
    res_leaf = r0.clone().requires_grad_()
    dy = _make((M, N), bf, 7)
    gemm_bias_act(a, w, residual=res_leaf[:, None].expand(M, N)).backward(dy)
    assert torch.equal(res_leaf.grad, dy.sum(1, keepdim=True)[:, 0])
    x = plain[0].clone().requires_grad_()
    gemm_bias_act(x, w, activation="silu").sum().backward()            # the gradient arrives with strides of zero
    y = plain[0].clone().requires_grad_()
    gemm_bias_act(y, w, activation="silu").backward(torch.ones(M, N, dtype=bf, device="cuda"))
    assert torch.equal(x.grad, y.grad)


def test_gradients_that_are_not_asked_for():
    from primus_turbo.pytorch.ops import gemm_bias_act
    a, b, bias = _make((40, 64), torch.bfloat16, 1), _make((96, 64), torch.bfloat16, 2), _make((96,), torch.bfloat16, 3)
    dy = _make((40, 96), torch.bfloat16, 4)
    full = torch.autograd.grad(gemm_bias_act(*[t.requires_grad_() for t in (a, b, bias)][:2], bias=bias, activation="silu", trans_b=True), [a, b, bias], dy)
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((a, b, bias))]
        y = gemm_bias_act(leaves[0], leaves[1], bias=leaves[2], activation="silu", trans_b=True)
        (g,) = torch.autograd.grad(y, leaves[i], dy)
        assert torch.equal(g, full[i])
    res = dy.clone().requires_grad_()
    (g,) = torch.autograd.grad(gemm_bias_act(a.detach(), b.detach(), residual=res, activation="relu", trans_b=True), res, dy)
    assert torch.equal(g, dy)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradient_against_central_differences(act):
    """Differences of the 64-bit formula along a random direction of every input against the kernel's gradient; the tolerance sums
    the element bounds of _check over the direction, dominated by the half steps of the 16-bit operands and results."""
    from primus_turbo.pytorch.ops import gemm_bias_act
    M, N, K, dt = 24, 40, 48, torch.float16
    ts = [_make((M, K), dt, 1), _make((N, K), dt, 2, K ** -0.5), _make((N,), dt, 3), _make((M, N), dt, 4)]
    w = _make((M, N), dt, 5)
    leaves = [t.clone().requires_grad_() for t in ts]
    grads = torch.autograd.grad(gemm_bias_act(leaves[0], leaves[1], bias=leaves[2], activation=act, residual=leaves[3], trans_b=True), leaves, w)
    base, W = [t.double() for t in ts], w.double()
    loss = lambda a, b, bias, res: float(((_act(a @ b.t() + bias, act) + res) * W).sum())
    z = base[0] @ base[1].t() + base[2]
    ez = _mm_bound(base[0], base[1].t(), K) + U * z.abs()
    ed = W.abs() * (0.9 * (ez + HALF[dt] * (z.abs() + ez)) + 128 * U * (1 + z.abs()) + 1.13 * HALF[dt]) + TINY[dt]
    dz = 1.13 * W.abs()
    bounds = [ed @ base[1].abs() + _mm_bound(dz, base[1], N), ed.t() @ base[0].abs() + _mm_bound(dz.t(), base[0], M), ed.sum(0) + M * U * dz.sum(0), 0 * W]
    for i in range(4):
        v = _make(base[i].shape, torch.float64, 20 + i)
        up, down = [t.clone() for t in base], [t.clone() for t in base]
        up[i] += 1e-5 * v
        down[i] -= 1e-5 * v
        diff = (loss(*up) - loss(*down)) / 2e-5
        g = grads[i].double()
        tol = float(((bounds[i] + (HALF[dt] + U) * (g.abs() + bounds[i]) + TINY[dt]) * v.abs()).sum()) + 1e-6
        assert abs(float((g * v).sum()) - diff) <= tol


@pytest.mark.parametrize("M", [9, 200])
def test_bad_values_stay_in_their_row_and_column(M):
    from primus_turbo.pytorch.ops import gemm_bias_act
    a, b = _make((M, 200), torch.bfloat16, 1), _make((140, 200), torch.bfloat16, 2)
    want = gemm_bias_act(a, b, activation="silu", trans_b=True)
    a[4, 7], b[9, 3] = float("nan"), float("inf")
    got = gemm_bias_act(a, b, activation="silu", trans_b=True)
    keep_r, keep_c = torch.arange(M, device="cuda") != 4, torch.arange(140, device="cuda") != 9
    assert torch.equal(got[keep_r][:, keep_c], want[keep_r][:, keep_c]) and got[4].isnan().all() and not got[:, 9].isfinite().all()


def test_nothing_to_do():
    from primus_turbo.pytorch.ops import gemm_bias_act
    e = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")
    assert gemm_bias_act(e(0, 64), e(32, 64), trans_b=True).shape == (0, 32)
    assert gemm_bias_act(e(4, 64), e(0, 64), trans_b=True).shape == (4, 0)
    a, b, bias = e(0, 64).requires_grad_(), _make((32, 64), torch.bfloat16, 1).requires_grad_(), _make((32,), torch.bfloat16, 1).requires_grad_()
    ga, gbias = torch.autograd.grad(gemm_bias_act(a, b, bias=bias, activation="silu", trans_b=True).sum(), [a, bias])
    assert ga.shape == a.shape and not gbias.any()


def test_main_grad_accumulation():
    from primus_turbo.pytorch.ops import gemm_bias_act
    a, b = _make((200, 64), torch.bfloat16, 1), _make((96, 64), torch.bfloat16, 2).requires_grad_()
    dy = _make((200, 96), torch.bfloat16, 3)
    (want,) = torch.autograd.grad(gemm_bias_act(a, b, activation="silu", trans_b=True, out_dtype=torch.bfloat16), b, dy)
    b.main_grad, b.grad_added_to_main_grad = torch.ones(96, 64, device="cuda"), False
    gemm_bias_act(a, b, activation="silu", trans_b=True, fuse_bgrad_accum_pattern="megatron").backward(dy)
    assert b.grad_added_to_main_grad
    err = (b.main_grad.double() - 1.0 - want.double()).abs()      # want is rounded to bf16, main_grad is not
    assert (err <= HALF[torch.bfloat16] * want.double().abs() * 1.01 + 4 * U * b.main_grad.double().abs() + 1e-6).all()


@pytest.mark.parametrize("M", [3, 40, 300])
def test_same_bits_on_streams_and_in_graphs(M):
    """Two streams at once and two graphs replayed at once give the eager call's bits (nothing is shared between calls)."""
    from primus_turbo.pytorch.ops import gemm_bias_act
    xs = [_make((M, 4096), torch.bfloat16, i) for i in range(2)]
    w, bias = _make((512, 4096), torch.bfloat16, 5, 0.02), _make((512,), torch.bfloat16, 6)
    call = lambda x: gemm_bias_act(x, w, bias=bias, activation="gelu", trans_b=True)
    want = [call(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(call(x))
        torch.cuda.synchronize()
        assert all(torch.equal(g, t) for g, t in zip(got, want))
    graphs, held = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(call(x))
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


@pytest.mark.parametrize("M,N,K", [(128, 128, 64), (200, 264, 72), (1032, 520, 1000), (4096, 4104, 200), (64, 8, 16), (2048, 4096, 33), (8, 16, 130)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_operands_read_contraction_major_give_the_bits_of_transposed_ones(M, N, K, dt):
    """pt_gemm_mn on operands stored [K, rows] against the same call on their transposed copies: the tensor core sees the same
    products in the same order."""
    from primus_turbo.pytorch.kernels.gemm import gemm_impl as g
    a, b = _make((M, K), dt, 1), _make((N, K), dt, 2)
    want = torch.empty(M, N, dtype=torch.float32, device="cuda")
    ak, bk = g._k_major16(a, False), g._k_major16(b, False)      # padded where K is not a multiple of 8
    g._launch(ak, False, bk, False, want, 0.0)
    _assert_within(want, a.double() @ b.double().t(), _mm_bound(a.double(), b.double().t(), K) + U * want.double().abs() + 1e-30, "product")
    for a_mn, b_mn in ((True, True), (True, False), (False, True)):
        if K % 8 and not (a_mn and b_mn):
            continue
        got = torch.empty_like(want)
        g._launch(a.t().contiguous() if a_mn else a, a_mn, b.t().contiguous() if b_mn else b, b_mn, got, 0.0)
        assert torch.equal(got, want), (a_mn, b_mn)


@pytest.mark.parametrize("M", [1, 20, 100, 300, 4200])
def test_weight_read_contraction_major(M):
    """trans_b=False reads a [K, N] weight in place, with the bits of the transposed call."""
    from primus_turbo.pytorch.ops import gemm_bias_act
    for N, K in ((4200, 264), (136, 1000)):
        a, b, bias = _make((M, K), torch.bfloat16, 1), _make((K, N), torch.bfloat16, 2, K ** -0.5), _make((N,), torch.bfloat16, 3)
        y = _check(M, N, K, torch.bfloat16, "silu", True, True, trans_b=False)
        assert y.shape == (M, N)
        assert torch.equal(gemm_bias_act(a, b, bias=bias, activation="gelu"), gemm_bias_act(a, b.t().contiguous(), bias=bias, activation="gelu", trans_b=True))


@pytest.mark.parametrize("M,N", [(66000, 33000), (40, 2 ** 26)])
def test_outputs_beyond_32_bits(M, N):
    from primus_turbo.pytorch.ops import gemm_bias_act
    a, b, res = _make((M, 64), torch.bfloat16, 1), _make((N, 64), torch.bfloat16, 2, 0.125), None
    assert M * N > 2 ** 31
    y = gemm_bias_act(a, b, activation="relu", trans_b=True)
    A, B = a[-3:].double(), b[-500:].double()
    want = (A @ B.t()).relu()
    _assert_within(y[-3:, -500:], want, _mm_bound(A, B.t(), 64) + (HALF[torch.bfloat16] + U) * (want + 1e-3) + 1e-6, "last rows and columns")
