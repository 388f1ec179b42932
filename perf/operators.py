"""The state space layer's operators, measured: the short causal convolution, the selective scan (prompts, training steps and
single tokens) and the linear layer with bias, activation and residual.

`run` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the end) or, where `own` is
set, through timeband_amd.ops.  Notation: (B, T, D) are sequences, steps and channels, N the states of a channel, G the groups
of channels that share their input and output vectors, K the taps of the convolution."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token for each of 16 streams: the convolution in front of the scan, latency alone
        dict(name="conv_step_bf16", op="conv_step", type="bf16", B=16, D=1024, K=4, act="silu"),
        # a prompt batch, padded to its longest member, in the framework's own type; 515 channels leave no aligned rows
        dict(name="conv_prompt_fp32_ragged", op="conv", type="fp32", B=6, T=1013, D=515, K=3, act="none", ragged=True, carry=True),
        # a training step's convolution, forward and backward, of a wide layer
        dict(name="conv_train_bf16", op="conv_train", type="bf16", B=8, T=2048, D=2048, K=4, act="silu", ragged=False),
        # one token for each of 64 streams through the state update
        dict(name="scan_step_bf16", op="scan_step", type="bf16", B=64, D=2048, N=16, G=1, gate=True),
        # one long prompt: few rows, so the work has to be split over the steps
        dict(name="scan_prompt_bf16_long", op="scan", type="bf16", B=1, T=16384, D=2048, N=16, G=1, gate=True, ragged=False, carry=False),
        # a padded batch of prompts that goes on from earlier states, two groups, eight states, 130 channels a group
        dict(name="scan_prompt_fp32_ragged", op="scan", type="fp32", B=5, T=1021, D=260, N=8, G=2, gate=False, ragged=True, carry=True),
        # a training step of a wide layer
        dict(name="scan_train_bf16", op="scan_train", type="bf16", B=4, T=2048, D=2048, N=16, G=1, gate=True, ragged=False),
        # a training step at the window length and hidden size that the LSTM layers are trained with, 64 windows
        dict(name="scan_train_fp32_window", op="scan_train", type="fp32", B=64, T=128, D=256, N=16, G=1, gate=True, ragged=False),
        # the output projection of eight streams' single tokens: reads the weights once
        dict(name="linear_step_bf16", op="linear", type="bf16", M=8, K=2048, N=4096, act="silu", residual=True),
        # a prompt batch through a wide projection
        dict(name="linear_prompt_bf16", op="linear", type="bf16", M=16384, K=2048, N=8192, act="gelu", residual=True),
        # a training step with rows and widths that fill no tile
        dict(name="linear_train_fp16_odd", op="linear_train", type="fp16", M=4099, K=1000, N=1500, act="silu", residual=True),
        # a training step over 512 windows of 128 steps at hidden size 256, in the framework's own type
        dict(name="linear_train_fp32_window", op="linear_train", type="fp32", M=65536, K=256, N=256, act="tanh", residual=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "conv_train", "conv_step", "scan", "scan_train", "scan_step", "linear", "linear_train"])
    kind = rng.choice(["bf16", "fp16", "fp32"])
    if op.startswith("conv"):
        D = _log(rng, 16, 4096)
        B = _log(rng, 1, 128 if op == "conv_step" else 32)
        case = dict(op=op, type=kind, B=B, D=D, K=rng.choice([2, 3, 4, 4, 7]), act=rng.choice(["silu", "none"]))
        if op != "conv_step":
            case.update(T=_log(rng, 1, max(1, min(16384, 33_000_000 // (B * D)))), ragged=rng.random() < 0.4)
        if op == "conv":
            case.update(carry=rng.random() < 0.5)
        return case
    if op.startswith("scan"):
        G = rng.choice([1, 1, 1, 2, 3])
        D = G * _log(rng, 16, 2400 // G)
        N = rng.choice([4, 8, 11, 16, 16, 16, 32])
        B = _log(rng, 1, 128 if op == "scan_step" else 64)
        case = dict(op=op, type=kind, B=B, D=D, N=N, G=G, gate=rng.random() < 0.7)
        if op != "scan_step":
            most = (500_000_000 if op == "scan" else 260_000_000) // (B * D * N)
            case.update(T=_log(rng, 1, max(1, min(16384, most))), ragged=rng.random() < 0.4)
        if op == "scan":
            case.update(carry=rng.random() < 0.5)
        return case
    K, N = _log(rng, 24, 4096), _log(rng, 24, 4096)
    most = (500_000_000_000 if op == "linear" else 60_000_000_000) // (2 * K * N)
    # relu's gradient jumps at 0, where two roundings of the same sum can fall on either side: forward only
    acts = ["none", "tanh", "sigmoid", "silu", "gelu"] + (["relu"] if op == "linear" else [])
    return dict(op=op, type=kind, M=_log(rng, 1, min(65536, most)), K=K, N=N, act=rng.choice(acts), residual=rng.random() < 0.6)


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = TYPES[case["type"]]

    def normal(*shape, scale=1.0, type=dt):
        return (torch.randn(shape, generator=g, device=dev) * scale).to(type)

    def uniform(lo, hi, *shape):
        return torch.rand(shape, generator=g, device=dev) * (hi - lo) + lo

    s = dict(case=case)
    op = case["op"]
    if op.startswith("conv"):
        B, D, K = case["B"], case["D"], case["K"]
        s["weight"] = normal(D, K, scale=K ** -0.5)
        s["bias"] = normal(D, scale=0.1)
        if op == "conv_step":
            s["x"], s["state"] = normal(B, D), normal(B, K - 1, D)
            return s
        s["x"] = normal(B, case["T"], D)
        if case.get("carry"):
            s["state"] = normal(B, K - 1, D)
    elif op.startswith("scan"):
        B, D, N, G = case["B"], case["D"], case["N"], case["G"]
        lead = (B,) if op == "scan_step" else (B, case["T"])
        s["u"], s["dt"] = normal(*lead, D), normal(*lead, D, scale=0.7)
        s["Bm"], s["Cm"] = normal(*lead, G, N), normal(*lead, G, N)
        if case["gate"]:
            s["z"] = normal(*lead, D)
        # decay rates as such layers start with: -1 ... -N, spread; step sizes between 1e-3 and 1e-1 before the input acts
        s["A"] = -(torch.arange(1, N + 1, device=dev, dtype=torch.float32) * uniform(0.8, 1.25, D, N)).contiguous()
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), D))
        s["dt_bias"] = torch.log(torch.expm1(step))
        s["D"] = uniform(0.5, 1.5, D)
        if op == "scan_step":
            s["state"] = normal(B, D, N, scale=0.3, type=torch.float32)
            return s
        if case.get("carry"):
            s["h0"] = normal(B, D, N, scale=0.3, type=torch.float32)
    else:
        M, K, N = case["M"], case["K"], case["N"]
        s["x"], s["W"], s["b"] = normal(M, K), normal(N, K, scale=K ** -0.5), normal(N, scale=0.1)
        if case["residual"]:
            s["r"] = normal(M, N)
        if op == "linear_train":
            s["dy"] = normal(M, N)
            for k in ("x", "W", "b", "r"):
                if k in s:
                    s[k].requires_grad_(True)
        return s
    if case.get("ragged"):
        # a padded batch: as long as its longest member, others down to nothing
        s["lengths"] = torch.randint(0, case["T"] + 1, (case["B"],), generator=g, device=dev, dtype=torch.int32)
        s["lengths"][0] = case["T"]
    if op.endswith("train"):
        s["dy"] = normal(B, case["T"], D)
        for k in ("x", "weight", "bias", "u", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias"):
            if k in s:
                s[k].requires_grad_(True)
    return s


# ---- the framework's operators ----------------------------------------------------------------------------------------
def _run_own(s):
    from timeband_amd import ops
    case, op = s["case"], s["case"]["op"]
    act = {"none": ops.ACT_NONE, "tanh": ops.ACT_TANH, "sigmoid": ops.ACT_SIGMOID, "relu": ops.ACT_RELU, "silu": ops.ACT_SILU,
           "gelu": ops.ACT_GELU}[case.get("act", "none")]
    if op == "conv_step":
        return [ops.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], act), s["state"]]
    if op == "conv":
        r = ops.causal_conv(s["x"], s["weight"], s["bias"], act, state=s.get("state"), lengths=s.get("lengths"),
                            return_state=case["carry"])
        return list(r) if case["carry"] else [r]
    if op == "conv_train":
        y = ops.causal_conv(s["x"], s["weight"], s["bias"], act, lengths=s.get("lengths"))
        return [y, *torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["dy"])]
    if op == "scan_step":
        y = ops.selective_scan_step(s["state"], s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s.get("z"),
                                    dt_bias=s["dt_bias"], softplus=True)
        return [y, s["state"]]
    if op.startswith("scan"):
        r = ops.selective_scan(s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s.get("z"), dt_bias=s["dt_bias"],
                               softplus=True, h0=s.get("h0"), lengths=s.get("lengths"), return_state=op == "scan" and case["carry"])
        if op == "scan":
            return list(r) if case["carry"] else [r]
        wrt = [s[k] for k in ("u", "dt", "A", "Bm", "Cm", "D", "dt_bias", "z") if k in s]
        return [r, *torch.autograd.grad(r, wrt, s["dy"])]
    y = ops.linear_residual(s["x"], s["W"], s["b"], act, residual=s.get("r"))
    if op == "linear":
        return [y]
    wrt = [s[k] for k in ("x", "W", "b", "r") if k in s]
    return [y, *torch.autograd.grad(y, wrt, s["dy"])]


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _act(x, kind):
    if kind == "tanh":
        return torch.tanh(x)
    if kind == "sigmoid":
        return torch.sigmoid(x)
    if kind == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if kind == "silu":
        return x * torch.sigmoid(x)
    if kind == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
    return x


def _act_grad(x, kind):
    if kind == "tanh":
        return 1 - torch.tanh(x).square()
    if kind == "sigmoid":
        return torch.sigmoid(x) * (1 - torch.sigmoid(x))
    if kind == "relu":
        return (x > 0).to(x.dtype)
    if kind == "silu":
        q = torch.sigmoid(x)
        return q * (1 + x * (1 - q))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    return torch.ones_like(x)


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))


def _valid(s, T):
    """(B, T, 1): the steps inside each sequence's length; None where all are."""
    if s.get("lengths") is None:
        return None
    return (torch.arange(T, device=s["lengths"].device)[None, :] < s["lengths"][:, None])[..., None]


def _conv_plain(s):
    case = s["case"]
    K, kind = case["K"], case["act"]
    w, b, x = s["weight"].detach().float(), s["bias"].detach().float(), s["x"].detach().float()
    if case["op"] == "conv_step":
        xs = torch.cat([s["state"].float(), x[:, None]], 1)
        y = _act((xs * w.t()[None]).sum(1) + b, kind)
        s["state"].copy_(xs[:, 1:])
        return [y.to(s["x"].dtype), s["state"]]
    B, T, D = x.shape
    ok = _valid(s, T)
    if ok is not None:
        x = torch.where(ok, x, torch.zeros_like(x))
    past = s["state"].float() if s.get("state") is not None else x.new_zeros(B, K - 1, D)
    xp = torch.cat([past, x], 1)
    taps = xp.unfold(1, K, 1)                      # (B, T, D, K)
    pre = (taps * w).sum(-1) + b
    y = _act(pre, kind)
    if ok is not None:
        y = torch.where(ok, y, torch.zeros_like(y))
    y = y.to(s["x"].dtype)
    if case["op"] == "conv":
        if not case["carry"]:
            return [y]
        end = s["lengths"].long() if ok is not None else torch.full((B,), T, device=x.device)
        at = end[:, None] + torch.arange(K - 1, device=x.device)[None]
        return [y, torch.gather(xp, 1, at[..., None].expand(B, K - 1, D)).to(s["x"].dtype)]
    dpre = s["dy"].float() * _act_grad(pre, kind)
    if ok is not None:
        dpre = torch.where(ok, dpre, torch.zeros_like(dpre))
    dx = (torch.cat([dpre, dpre.new_zeros(B, K - 1, D)], 1).unfold(1, K, 1) * w.flip(1)).sum(-1)
    dw = (dpre[..., None] * taps).sum((0, 1))
    return [y, dx.to(s["x"].dtype), dw.to(s["weight"].dtype), dpre.sum((0, 1)).to(s["bias"].dtype)]


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, by doubling: after each round an entry holds twice as many steps."""
    n, T = 1, a.shape[1]
    while n < T:
        b = torch.cat([b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _scan_plain(s):
    case = s["case"]
    G, op = case["G"], case["op"]
    of = s["u"].dtype
    u, raw = s["u"].detach().float(), s["dt"].detach().float() + s["dt_bias"].detach()
    A, Dp = s["A"].detach(), s["D"].detach()
    rep = u.shape[-1] // G
    Bm, Cm = (s[k].detach().float().repeat_interleave(rep, dim=-2) for k in ("Bm", "Cm"))    # (..., D, N)
    z = s["z"].detach().float() if "z" in s else None
    delta = _softplus(raw)
    if op == "scan_step":
        h = torch.exp(delta[..., None] * A) * s["state"] + (delta * u)[..., None] * Bm
        s["state"].copy_(h)
        y = (h * Cm).sum(-1) + Dp * u
        return [(y * _act(z, "silu") if z is not None else y).to(of), s["state"]]
    T = u.shape[1]
    ok = _valid(s, T)
    if ok is not None:
        delta = torch.where(ok, delta, torch.zeros_like(delta))
    a = torch.exp(delta[..., None] * A)                                # (B, T, D, N)
    b = (delta * u)[..., None] * Bm
    if s.get("h0") is not None:
        b = torch.cat([b[:, :1] + a[:, :1] * s["h0"][:, None], b[:, 1:]], 1)
    h = _recurrence(a, b)
    y = (h * Cm).sum(-1) + Dp * u
    out = y * _act(z, "silu") if z is not None else y
    if ok is not None:
        out = torch.where(ok, out, torch.zeros_like(out))
    out = out.to(of)
    if op == "scan":
        return [out, h[:, -1].contiguous()] if case["carry"] else [out]
    dout = s["dy"].float()
    if ok is not None:
        dout = torch.where(ok, dout, torch.zeros_like(dout))
    dy = dout * _act(z, "silu") if z is not None else dout
    one = torch.ones_like(a[:, :1])
    g = _recurrence(torch.cat([a[:, 1:], one], 1).flip(1), (dy[..., None] * Cm).flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    gah = g * a * before
    gB = (g * Bm).sum(-1)
    ddelta = (gah * A).sum(-1) + u * gB
    draw_ = ddelta * torch.sigmoid(raw)
    if ok is not None:
        draw_ = torch.where(ok, draw_, torch.zeros_like(draw_))
    shared = (u.shape[0], T, G, rep, A.shape[1])
    grads = [(delta * gB + Dp * dy).to(of), draw_.to(of), (gah * delta[..., None]).sum((0, 1)),
             (g * (delta * u)[..., None]).reshape(shared).sum(3).to(of), (h * dy[..., None]).reshape(shared).sum(3).to(of),
             (dy * u).sum((0, 1)), draw_.sum((0, 1))]
    if z is not None:
        grads.append((dout * y * _act_grad(z, "silu")).to(of))
    return [out, *grads]


def _linear_plain(s):
    kind, of = s["case"]["act"], s["x"].dtype
    x, W, b = s["x"].detach().float(), s["W"].detach().float(), s["b"].detach().float()
    pre = x @ W.t() + b
    y = _act(pre, kind)
    if "r" in s:
        y = y + s["r"].detach().float()
    y = y.to(of)
    if s["case"]["op"] == "linear":
        return [y]
    dpre = s["dy"].float() * _act_grad(pre, kind)
    out = [y, (dpre @ W).to(of), (dpre.t() @ x).to(of), dpre.sum(0).to(of)]
    return out + [s["dy"].clone()] if "r" in s else out


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _conv_plain(state) if op.startswith("conv") else _scan_plain(state) if op.startswith("scan") else _linear_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "fp32" else 2
    op = case["op"]
    if op.startswith("conv"):
        B, D, K = case["B"], case["D"], case["K"]
        if op == "conv_step":
            return {"bytes": e * (B * D * (2 + 2 * (K - 1)) + D * (K + 1)), "flops": 2.0 * B * D * K}
        n = B * case["T"] * D
        if op == "conv":
            return {"bytes": e * (2 * n + D * (K + 1) + (2 * B * (K - 1) * D if case["carry"] else 0)), "flops": 2.0 * n * K}
        return {"bytes": e * (4 * n + 2 * D * (K + 1)), "flops": 6.0 * n * K}          # x, y, dy, dx
    if op.startswith("scan"):
        B, D, N, G = case["B"], case["D"], case["N"], case["G"]
        z = 1 if case["gate"] else 0
        n = B * (1 if op == "scan_step" else case["T"])
        par = 4 * D * (N + 2)
        if op == "scan_step":
            return {"bytes": e * n * (D * (3 + z) + 2 * G * N) + 8 * B * D * N + par, "flops": 7.0 * n * D * N}
        if op == "scan":
            return {"bytes": e * n * (D * (3 + z) + 2 * G * N) + par + (8 * B * D * N if case["carry"] else 0), "flops": 7.0 * n * D * N}
        return {"bytes": e * n * (D * (6 + 2 * z) + 4 * G * N) + 2 * par, "flops": 21.0 * n * D * N}   # u, dt, z, out, dout and three gradients
    M, K, N = case["M"], case["K"], case["N"]
    r = 1 if case["residual"] else 0
    if op == "linear":
        return {"bytes": e * (M * K + N * K + N + (1 + r) * M * N), "flops": 2.0 * M * N * K}
    return {"bytes": e * (2 * M * K + 2 * N * K + 2 * N + (2 + 2 * r) * M * N), "flops": 6.0 * M * N * K}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------
def _d(t):
    return None if t is None else t.detach().double()


def _f(x, kind):
    """(value, derivative) of an activation in 64 bits."""
    if kind == "none":
        return x, torch.ones_like(x)
    if kind == "relu":
        return x.clamp(min=0), (x > 0).double()
    if kind == "tanh":
        y = x.tanh()
        return y, 1 / x.cosh().square()
    p = 1 / (1 + torch.exp(-x))
    if kind == "sigmoid":
        return p, torch.exp(-x) * p * p
    if kind == "silu":
        return x * p, p + x * torch.exp(-x) * p * p
    cdf = 0.5 * torch.erfc(-x / math.sqrt(2.0))
    return x * cdf, cdf + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"].startswith("conv"):
            return _conv_exact(case, s)
        if case["op"].startswith("scan"):
            return _scan_exact(case, s)
        x, W, b = _d(s["x"]), _d(s["W"]), _d(s["b"])
        v, dv = _f(torch.addmm(b, x, W.t()), case["act"])
        y = v + _d(s["r"]) if "r" in s else v
        if case["op"] == "linear":
            return [y]
        q = _d(s["dy"]) * dv
        return [y, q.mm(W), q.t().mm(x), q.sum(0)] + ([_d(s["dy"])] if "r" in s else [])


def _conv_exact(case, s):
    K = case["K"]
    w, b = _d(s["weight"]), _d(s["bias"])
    x = _d(s["x"])
    if case["op"] == "conv_step":
        hist = [_d(s["state"])[:, k] for k in range(K - 1)] + [x]
        pre = b + sum(w[:, k] * hist[k] for k in range(K))
        return [_f(pre, case["act"])[0], torch.stack(hist[1:], 1)]
    B, T, D = x.shape
    ends = s["lengths"].tolist() if "lengths" in s else [T] * B
    ys, dxs, news = [], [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for i, n in enumerate(ends):
        row = torch.cat([_d(s["state"])[i] if "state" in s else x.new_zeros(K - 1, D), x[i, :n]])     # one sequence, its past first
        pre = b + sum(w[:, k] * row[k:k + n] for k in range(K))
        v, dv = _f(pre, case["act"])
        ys.append(torch.cat([v, x.new_zeros(T - n, D)]))
        news.append(row[n:])
        if case["op"] == "conv_train":
            q = _d(s["dy"])[i, :n] * dv
            back = torch.zeros_like(row)
            for k in range(K):
                back[k:k + n] += w[:, k] * q
                dw[:, k] += (q * row[k:k + n]).sum(0)
            db += q.sum(0)
            dxs.append(torch.cat([back[K - 1:], x.new_zeros(T - n, D)]))
    if case["op"] == "conv":
        return [torch.stack(ys), torch.stack(news)] if case["carry"] else [torch.stack(ys)]
    return [torch.stack(ys), torch.stack(dxs), dw, db]


def _scan_exact(case, s):
    """Step by step; the gradients by the adjoint recurrence, step by step backwards."""
    op, G = case["op"], case["G"]
    A, Dp, bias = _d(s["A"]), _d(s["D"]), _d(s["dt_bias"])
    Dn, N = A.shape
    lead = (lambda t: _d(t)[:, None]) if op == "scan_step" else _d
    u, raw, Bm, Cm = lead(s["u"]), lead(s["dt"]) + bias, lead(s["Bm"]), lead(s["Cm"])
    z = lead(s["z"]) if "z" in s else None
    B, T = u.shape[:2]
    ends = s["lengths"].long() if "lengths" in s else torch.full((B,), T, device=u.device)
    wide = lambda v: v[:, :, None, :].expand(B, G, Dn // G, N).reshape(B, Dn, N)  # noqa: E731
    delta = torch.nn.functional.softplus(raw, threshold=40.0)
    on = torch.arange(T, device=u.device)[None] < ends[:, None]
    h = _d(s["h0"]) if "h0" in s else _d(s["state"]) if op == "scan_step" else u.new_zeros(B, Dn, N)
    keep = torch.empty(T + 1, B, Dn, N, dtype=torch.float64, device=u.device) if op == "scan_train" else None
    if keep is not None:
        keep[0] = h
    y = torch.empty_like(u)
    for t in range(T):
        new = torch.exp(delta[:, t, :, None] * A).mul_(h).addcmul_((delta[:, t] * u[:, t])[..., None], wide(Bm[:, t]))
        h = torch.where(on[:, t, None, None], new, h)
        if keep is not None:
            keep[t + 1] = h
        y[:, t] = (h * wide(Cm[:, t])).sum(-1) + Dp * u[:, t]
    gate, dgate = _f(z, "silu") if z is not None else (None, None)
    zero = u.new_zeros(())
    mask = lambda v: torch.where(on[..., None], v, zero)  # noqa: E731
    out = mask(y * gate if gate is not None else y)
    if op == "scan_step":
        return [out[:, 0], h]
    if op == "scan":
        return [out, h] if case["carry"] else [out]
    dout = mask(_d(s["dy"]))
    dy = dout * gate if gate is not None else dout
    g = torch.zeros_like(h)
    du, ddt, dA = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(A)
    dB, dC = torch.zeros_like(Bm), torch.zeros_like(Cm)
    parts = (B, G, Dn // G, N)
    for t in range(T - 1, -1, -1):
        g = g + dy[:, t, :, None] * wide(Cm[:, t])
        dC[:, t] = (keep[t + 1] * dy[:, t, :, None]).reshape(parts).sum(2)
        a = torch.exp(delta[:, t, :, None] * A)
        gah = torch.where(on[:, t, None, None], g * a * keep[t], zero)
        gB = (g * wide(Bm[:, t])).sum(-1)
        dA += (gah * delta[:, t, :, None]).sum(0)
        du[:, t] = delta[:, t] * gB + Dp * dy[:, t]
        ddt[:, t] = (gah * A).sum(-1) + u[:, t] * gB
        dB[:, t] = torch.where(on[:, t, None, None], g * (delta[:, t] * u[:, t])[..., None], zero).reshape(parts).sum(2)
        g = torch.where(on[:, t, None, None], g * a, g)
    du, ddt = mask(du), mask(ddt) * torch.sigmoid(raw)
    grads = [du, ddt, dA, dB, dC, (dy * mask(u)).sum((0, 1)), ddt.sum((0, 1))]
    if z is not None:
        grads.append(dout * mask(y) * dgate)
    return [out, *grads]
