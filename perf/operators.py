"""What is measured of the operators around a decoder layer's products.

Three operators, each in its plain form (elementary torch operations in 32 bits, rounded once at the end) and through the
package's public entry points:

  gemm_bias_act    y = act(a . b^T + bias) + residual, forward or forward + backward
  qk_norm_rope     RMS norm of every query / key head followed by the position rotation, forward or forward + backward
  moe_few_tokens   a whole mixture-of-experts layer (gate, up, gated activation, down, weighted sum) for few tokens

`listed()` gives the measured cases, `draw()` more of the same ranges, `prepare()` what a program has in hand before the
call, `run()` one pass, `work()` the bytes and operations a pass cannot do without, `exact()` the outputs in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one token through the up projection of an 8B model's MLP: latency and the weight's bytes
        {"name": "linear_token_gelu", "op": "gemm", "M": 1, "N": 14336, "K": 4096, "act": "gelu", "bias": True, "residual": False,
         "dtype": "bf16", "train": False},
        # a small decoding batch through the down projection, added to the residual stream
        {"name": "linear_batch24_residual", "op": "gemm", "M": 24, "N": 4096, "K": 14336, "act": "none", "bias": True, "residual": True,
         "dtype": "fp16", "train": False},
        # a short prompt of odd length and an output width that no tile divides
        {"name": "linear_odd_silu", "op": "gemm", "M": 333, "N": 4101, "K": 4096, "act": "silu", "bias": True, "residual": False,
         "dtype": "bf16", "train": False},
        # a long prompt through the up projection: the largest product
        {"name": "linear_prompt_gelu_tanh", "op": "gemm", "M": 8192, "N": 14336, "K": 4096, "act": "gelu_tanh", "bias": True,
         "residual": False, "dtype": "bf16", "train": False},
        # a training step of the same layer with a residual: output and four gradients
        {"name": "linear_train_silu", "op": "gemm", "M": 4096, "N": 14336, "K": 4096, "act": "silu", "bias": True, "residual": True,
         "dtype": "bf16", "train": True},
        # one token at a far position of a long context
        {"name": "qk_token", "op": "qk", "T": 1, "Hq": 32, "Hk": 8, "D": 128, "R": 128, "P": 131072, "interleaved": False,
         "zero_centered": False, "dtype": "bf16", "train": False},
        # a long prompt, heads of a 70B model, read in place out of the packed projection
        {"name": "qk_prompt", "op": "qk", "T": 8192, "Hq": 64, "Hk": 8, "D": 128, "R": 128, "P": 131072, "interleaved": False,
         "zero_centered": False, "dtype": "bf16", "train": False},
        # a training step on an odd number of tokens, half of each head rotated, neighbouring pairs, (1 + gamma) gains
        {"name": "qk_train_partial", "op": "qk", "T": 8191, "Hq": 32, "Hk": 8, "D": 128, "R": 64, "P": 8192, "interleaved": True,
         "zero_centered": True, "dtype": "fp16", "train": True},
        # one token through eight of 32 experts of a large mixture
        {"name": "moe_token_top8", "op": "moe", "T": 1, "E": 32, "all": 32, "K": 8, "H": 7168, "I": 2048, "act": "silu", "dtype": "bf16"},
        # 64 tokens of a decoding batch on one of eight expert shards (32 of 256 experts; slots of other shards are -1)
        {"name": "moe_shard_batch64", "op": "moe", "T": 64, "E": 32, "all": 256, "K": 8, "H": 7168, "I": 2048, "act": "silu",
         "dtype": "bf16"},
        # seven tokens, two of eight wide experts
        {"name": "moe_wide_experts_batch7", "op": "moe", "T": 7, "E": 8, "all": 8, "K": 2, "H": 4096, "I": 14336, "act": "silu",
         "dtype": "fp16"},
        # three tokens, many narrow experts of an odd width, GELU gate: the smallest layer
        {"name": "moe_narrow_batch3", "op": "moe", "T": 3, "E": 64, "all": 64, "K": 6, "H": 2048, "I": 712, "act": "gelu",
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gemm", "qk", "moe"])
    if op == "gemm":
        train = rng.random() < 0.35
        M = _log_int(rng, 1, 8192)
        N = _log_int(rng, 256, 16384)
        if rng.random() < 0.6:
            N = max(8, N // 8 * 8)
        K = max(128, _log_int(rng, 256, 14336) // 8 * 8)      # hidden sizes: rows of 16 bytes
        while M * N * K > 8192 * 14336 * 4096 // (3 if train else 1):
            M = max(1, M // 2)
        return {"op": op, "M": M, "N": N, "K": K, "act": rng.choice(["none", "silu", "gelu", "gelu_tanh"] + ([] if train else ["relu"])),
                "bias": rng.random() < 0.75, "residual": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "train": train}
    if op == "qk":
        train = rng.random() < 0.5
        D = rng.choice([64, 80, 96, 128, 128, 192, 256])
        Hk = rng.choice([1, 2, 4, 8])
        return {"op": op, "T": _log_int(rng, 1, 4096 if train else 8192), "Hq": Hk * rng.choice([1, 3, 4, 5, 8]), "Hk": Hk, "D": D,
                "R": rng.choice([D, D, D // 2, D // 4 * 2 - 4]), "P": 8192 * rng.choice([1, 4, 16]), "interleaved": rng.random() < 0.4,
                "zero_centered": rng.random() < 0.3, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "train": train}
    E = rng.choice([4, 8, 16, 32, 60])
    shards = rng.choice([1, 1, 2, 8])
    H = _log_int(rng, 512, 7168) // 8 * 8
    I = max(64, _log_int(rng, 128, 8192) // 8 * 8)
    while E * 3 * H * I * 2 > 6 * 10 ** 9:
        I = max(64, I // 2 // 8 * 8)
    return {"op": op, "T": _log_int(rng, 1, 128), "E": E, "all": E * shards, "K": rng.choice([1, 2, 4, min(8, E)]), "H": H, "I": I,
            "act": rng.choice(["silu", "silu", "gelu"]), "dtype": rng.choice(["bf16", "bf16", "fp16"])}


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed, device="cuda"):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device=device).manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(shape, std, mean=0.0, dtype=dt):
        return torch.empty(shape, dtype=torch.float32, device=device).normal_(mean, std, generator=g).to(dtype)

    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        a = normal((M, K), 1.0)
        a[:, 0] *= 20.0      # one hidden unit far above the others, as residual streams have
        s = {"a": a, "b": normal((N, K), 1.0 / math.sqrt(K)), "bias": normal((N,), 0.5) if case["bias"] else None,
             "residual": normal((M, N), 2.0) if case["residual"] else None}
        if case["train"]:
            s["dy"] = normal((M, N), 1e-2)
        return s
    if case["op"] == "qk":
        T, Hq, Hk, D, R, P = (case[n] for n in ("T", "Hq", "Hk", "D", "R", "P"))
        packed = normal((T, (Hq + 2 * Hk) * D), 1.5)
        base = 0.0 if case["zero_centered"] else 1.0
        angle = torch.arange(P, device=device, dtype=torch.float64)[:, None] * \
            (1e6 ** (-torch.arange(0, R, 2, device=device, dtype=torch.float64) / R))[None, :]
        s = {"packed": packed, "q_gamma": normal((D,), 0.2, base), "k_gamma": normal((D,), 0.2, base),
             "cos": angle.cos().float(), "sin": angle.sin().float()}
        first = int(torch.randint(0, max(1, P - T + 1), (1,), generator=g, device=device))
        s["positions"] = torch.arange(first, first + T, device=device) % P       # a chunk of a prompt, or one far token
        if case["train"]:
            s["dq"], s["dk"] = normal((T, Hq, D), 1e-2), normal((T, Hk, D), 1e-2)
        return s
    T, E, K, H, I = (case[n] for n in ("T", "E", "K", "H", "I"))
    x = normal((T, H), 1.0)
    gate_up = torch.empty((E, 2 * I, H), dtype=dt, device=device).normal_(0.0, 1.0 / math.sqrt(H), generator=g)
    down = torch.empty((E, H, I), dtype=dt, device=device).normal_(0.0, 1.0 / math.sqrt(I), generator=g)
    logits = torch.empty((T, case["all"]), dtype=torch.float32, device=device).normal_(0.0, 1.0, generator=g)
    values, ids = logits.topk(K, dim=1)
    probs = values.softmax(dim=1)
    ids = torch.where(ids < E, ids, torch.full_like(ids, -1))      # experts of the other shards
    return {"x": x, "gate_up": gate_up, "down": down, "ids": ids, "probs": probs}


def _qk_views(case, packed):
    T, Hq, Hk, D = (case[n] for n in ("T", "Hq", "Hk", "D"))
    return packed[:, :Hq * D].view(T, Hq, D), packed[:, Hq * D:(Hq + Hk) * D].view(T, Hk, D)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "qk":
        s["q"], s["k"] = _qk_views(case, s.pop("packed"))
    if own:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "primus-turbo_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import primus_turbo.pytorch as turbo
        s["ops"] = turbo.ops
        if case.get("train"):
            leaves = ("a", "b", "bias", "residual") if case["op"] == "gemm" else ("q", "k", "q_gamma", "k_gamma")
            s["leaves"] = [s[n].requires_grad_(True) if s[n].is_leaf else s[n].detach().requires_grad_(True)
                           for n in leaves if s[n] is not None]
            for n, t in zip([n for n in leaves if s[n] is not None], s["leaves"]):
                s[n] = t
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))


def _act_grad(z, name):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)


def _plain_gemm(s):
    case, dt = s["case"], s["a"].dtype
    a, b = s["a"].float(), s["b"].float()
    z = a @ b.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not case["train"]:
        return [y.to(dt)]
    dy = s["dy"].float()
    dz = dy * _act_grad(z, case["act"])
    out = [y.to(dt), (dz @ b).to(dt), (dz.t() @ a).to(dt)]
    if s["bias"] is not None:
        out.append(dz.sum(0).to(dt))
    if s["residual"] is not None:
        out.append(s["dy"].clone())
    return out


def _rotate(v, cos, sin, R, interleaved, inverse=False):
    """v [T, H, D]; cos / sin [T, 1, R / 2].  The rotation of the first R elements, or its transpose."""
    if inverse:
        sin = -sin
    r, rest = v[..., :R], v[..., R:]
    if interleaved:
        x0, x1 = r[..., 0::2], r[..., 1::2]
        r = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], dim=-1).flatten(-2)
    else:
        x0, x1 = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], dim=-1)
    return torch.cat([r, rest], dim=-1)


def _plain_qk(s):
    case = s["case"]
    dt, R, il = s["q"].dtype, case["R"], case["interleaved"]
    cos, sin = s["cos"][s["positions"]][:, None, :], s["sin"][s["positions"]][:, None, :]
    outs, grads, gammas = [], [], []
    for x, gamma, dy in ((s["q"], s["q_gamma"], s.get("dq")), (s["k"], s["k_gamma"], s.get("dk"))):
        x, g = x.float(), gamma.float() + (1.0 if case["zero_centered"] else 0.0)
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        outs.append(_rotate(x * rstd * g, cos, sin, R, il).to(dt))
        if case["train"]:
            dn = _rotate(dy.float(), cos, sin, R, il, inverse=True)
            xh = x * rstd
            gammas.append((dn * xh).sum((0, 1)).to(dt))
            dn = dn * g
            grads.append(((dn - xh * (dn * xh).mean(-1, keepdim=True)) * rstd).to(dt))
    return outs + grads + gammas


def _plain_moe(s):
    case, x, ids, probs = s["case"], s["x"].float(), s["ids"], s["probs"]
    T, E, K, I = case["T"], case["E"], case["K"], case["I"]
    out = torch.zeros_like(x)
    if T * K <= E:      # few slots: gather each slot's expert
        for t in range(T):
            e = ids[t].clamp(min=0)
            p = torch.where(ids[t] >= 0, probs[t], torch.zeros_like(probs[t]))
            for j in range(K):
                z = s["gate_up"][e[j:j + 1]][0].float() @ x[t]
                h = _act(z[:I], case["act"]) * z[I:]
                out[t] += p[j] * (s["down"][e[j:j + 1]][0].float() @ h)
        return [out.to(s["x"].dtype)]
    weight = torch.zeros((T, E + 1), dtype=torch.float32, device=x.device)
    weight.scatter_add_(1, torch.where(ids >= 0, ids, torch.full_like(ids, E)), probs)
    for e in range(E):
        z = x @ s["gate_up"][e].float().t()
        h = _act(z[:, :I], case["act"]) * z[:, I:]
        out += weight[:, e:e + 1] * (h @ s["down"][e].float().t())
    return [out.to(s["x"].dtype)]


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s, case = state, state["case"]
    if not own:
        return {"gemm": _plain_gemm, "qk": _plain_qk, "moe": _plain_moe}[case["op"]](s)
    ops = s["ops"]
    if case["op"] == "gemm":
        y = ops.gemm_bias_act(s["a"], s["b"], bias=s["bias"], activation=None if case["act"] == "none" else case["act"],
                              residual=s["residual"], trans_b=True)
        if not case["train"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])]
    if case["op"] == "qk":
        q, k = ops.qk_norm_rope(s["q"], s["k"], s["q_gamma"], s["k_gamma"], s["cos"], s["sin"], positions=s["positions"], eps=1e-6,
                                interleaved=case["interleaved"], zero_centered=case["zero_centered"])
        if not case["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad([q, k], s["leaves"], [s["dq"], s["dk"]])]
    return [ops.moe_few_tokens(s["x"], s["gate_up"], s["down"], s["ids"], s["probs"], act_type=case["act"])]


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        bias, res = (N if case["bias"] else 0), (M * N if case["residual"] else 0)
        nbytes, flops = e * (M * K + N * K + M * N + bias + res), 2 * M * N * K
        if case["train"]:      # the output's gradient read; the gradients of a, b, bias and residual written
            nbytes += e * (M * N + M * K + N * K + bias + res)
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "qk":
        T, D, R, heads = case["T"], case["D"], case["R"], case["Hq"] + case["Hk"]
        nbytes = 2 * e * T * heads * D + 2 * e * D + 4 * R * T + 8 * T
        flops = T * heads * (4 * D + 3 * R)
        if case["train"]:
            nbytes += 2 * e * T * heads * D + 2 * e * D
            flops += T * heads * (8 * D + 3 * R)
        return {"bytes": nbytes, "flops": flops}
    T, E, K, H, I = (case[n] for n in ("T", "E", "K", "H", "I"))
    experts = E * (1.0 - (1.0 - K / case["all"]) ** T)      # expected number of local experts that some token chose
    slots = T * K * E / case["all"]
    return {"bytes": int(experts * 3 * H * I * e + 2 * T * H * e + 12 * T * K), "flops": int(slots * 6 * H * I)}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    f = torch.float64
    if case["op"] == "gemm":
        train = case["train"]
        leaf = {n: (None if s[n] is None else s[n].to(f).requires_grad_(train)) for n in ("a", "b", "bias", "residual")}
        z = torch.mm(leaf["a"], leaf["b"].transpose(0, 1))
        if leaf["bias"] is not None:
            z = z + leaf["bias"][None, :]
        y = {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
             "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2.0)),
             "gelu_tanh": lambda v: v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))}[case["act"]](z)
        if leaf["residual"] is not None:
            y = y + leaf["residual"]
        if not train:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, [t for t in leaf.values() if t is not None], s["dy"].to(f))]
    if case["op"] == "qk":
        train, R = case["train"], case["R"]
        q, k = _qk_views(case, s["packed"].to(f))
        leaf = [t.detach().requires_grad_(train) for t in (q, k, s["q_gamma"].to(f), s["k_gamma"].to(f))]
        phase = torch.complex(s["cos"].to(f), s["sin"].to(f))[s["positions"]].unsqueeze(1)
        outs = []
        for x, gamma in ((leaf[0], leaf[2]), (leaf[1], leaf[3])):
            n = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["D"] + 1e-6) * (gamma + 1.0 if case["zero_centered"] else gamma)
            first, second = (n[..., 0:R:2], n[..., 1:R:2]) if case["interleaved"] else (n[..., :R // 2], n[..., R // 2:R])
            turned = torch.view_as_real(torch.complex(first.contiguous(), second.contiguous()) * phase)
            rot = turned.reshape(*turned.shape[:-2], R) if case["interleaved"] else turned.transpose(-1, -2).reshape(*turned.shape[:-2], R)
            outs.append(torch.cat((rot, n[..., R:]), -1))
        if not train:
            return outs
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaf, [s["dq"].to(f), s["dk"].to(f)]))
    T, K, I = case["T"], case["K"], case["I"]
    x, ids, probs = s["x"].to(f), s["ids"].tolist(), s["probs"].to(f)
    out = torch.zeros_like(x)
    for e in range(case["E"]):
        slots = [(t, j) for t in range(T) for j in range(K) if ids[t][j] == e]
        if not slots:
            continue
        rows = torch.tensor([t for t, _ in slots], device=x.device)
        p = torch.stack([probs[t, j] for t, j in slots])
        gate, up = s["gate_up"][e, :I].to(f), s["gate_up"][e, I:].to(f)
        gv = torch.einsum("th,ih->ti", x[rows], gate)
        gv = gv * torch.sigmoid(gv) if case["act"] == "silu" else gv * 0.5 * torch.erfc(-gv / math.sqrt(2.0))
        y = torch.einsum("ti,hi->th", gv * torch.einsum("th,ih->ti", x[rows], up), s["down"][e].to(f))
        out.index_add_(0, rows, y * p[:, None])
    return [out]
