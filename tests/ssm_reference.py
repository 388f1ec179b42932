"""Plain 64-bit forms of the state space layer's operators, with bounds on what 32-bit arithmetic may be off by.

Every form takes `mag`: with it, every product and sum is formed of magnitudes, so that its results bound the sizes of the sums that the
kernels round in.  A 32-bit sum of n products is off by at most n 2^-24 times the sum of magnitudes, to first order."""
import math

import torch

F64 = torch.float64
U = 2.0 ** -24          # half a step of fp32, relative


def d(t):
    return None if t is None else t.detach().to("cpu", F64)


def act(x, kind):
    """(value, derivative); kinds are the ACT_* numbers."""
    if kind == 0:
        return x, torch.ones_like(x)
    if kind == 1:
        return torch.tanh(x), 1 / torch.cosh(x) ** 2
    if kind == 3:
        return x.clamp(min=0), (x > 0).to(F64)
    s = torch.sigmoid(x)
    if kind == 2:
        return s, s * torch.sigmoid(-x)
    if kind == 4:
        return x * s, s + x * s * torch.sigmoid(-x)
    c = 0.5 * torch.erfc(-x / math.sqrt(2))
    return x * c, c + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


def conv(x, w, b=None, kind=0, state=None, lengths=None, dy=None, mag=False):
    """y, new state, dx, dw, db (the last three with dy) by loops over sequences and taps."""
    f = torch.abs if mag else (lambda t: t)
    x, w, dy = d(x), d(w), d(dy)
    B, T, D = x.shape
    K = w.shape[1]
    b = torch.zeros(D, dtype=F64) if b is None else d(b)
    st = torch.zeros(B, K - 1, D, dtype=F64) if state is None else d(state)
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    new = torch.zeros(B, K - 1, D, dtype=F64)
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for i in range(B):
        n = T if lengths is None else min(max(int(lengths[i]), 0), T)
        row = torch.cat([st[i], x[i, :n]])
        pre, size = b.expand(n, D).clone(), b.abs().expand(n, D).clone()
        for k in range(K):
            pre += w[:, k] * row[k:k + n]
            size += (w[:, k] * row[k:k + n]).abs()
        v, dv = act(pre, kind)
        y[i, :n] = size if mag else v
        new[i] = row[n:n + K - 1]
        if dy is not None:
            q = dy[i, :n] * dv
            # the derivative is off by what pre is off by (its own slope is below 1) besides its own size
            if mag:
                q = dy[i, :n].abs() * (dv.abs() + (size if kind else 0) + 1)
            back = torch.zeros(n + K - 1, D, dtype=F64)
            for k in range(K):
                back[k:k + n] += f(w[:, k]) * q
                dw[:, k] += (q * f(row[k:k + n])).sum(0)
            db += q.sum(0)
            dx[i, :n] = back[K - 1:]
    return y, new, dx, dw, db


def scan(u, dt, A, Bm, Cm, D=None, z=None, bias=None, softplus=True, h0=None, lengths=None, dout=None, dhT=None, mag=False):
    """dict(out, hT, and with dout: du, ddt, dA, dB, dC, dD, dz, dbias, dh0), step by step."""
    f = torch.abs if mag else (lambda t: t)
    u, dt, A, Bm, Cm, D, z, bias, h0, dout, dhT = (d(t) for t in (u, dt, A, Bm, Cm, D, z, bias, h0, dout, dhT))
    B, T, Dn = u.shape
    G, N = Bm.shape[2:]
    rep = Dn // G
    raw = dt if bias is None else dt + bias
    delta = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30)))) if softplus else raw
    on = torch.ones(B, T, dtype=torch.bool) if lengths is None else torch.arange(T)[None] < lengths.cpu().long()[:, None]
    delta = torch.where(on[..., None], delta, torch.zeros((), dtype=F64))
    wide = lambda v: f(v)[:, :, None, :].expand(B, G, rep, N).reshape(B, Dn, N)
    Dp = torch.zeros(Dn, dtype=F64) if D is None else f(D)
    h = torch.zeros(B, Dn, N, dtype=F64) if h0 is None else f(h0)
    uu, dd = f(u), f(delta)
    hs, y = [h], torch.zeros_like(u)
    zero = torch.zeros((), dtype=F64)
    for t in range(T):
        x = torch.where(on[:, t, None], dd[:, t] * uu[:, t], zero)
        Bt, Ct = (torch.where(on[:, t, None, None], wide(v[:, t]), zero) for v in (Bm, Cm))
        h = torch.exp(delta[:, t, :, None] * A) * h + x[..., None] * Bt
        hs.append(h)
        y[:, t] = (h * Ct).sum(-1) + Dp * uu[:, t]
    gate, dgate = act(z, 4) if z is not None else (torch.ones_like(u), None)
    if mag and z is not None:
        gate, dgate = z.abs(), 1 + z.abs()
    m = lambda v: torch.where(on[..., None], v, zero)
    r = dict(out=m(y * gate), hT=h)
    if dout is None:
        return r
    dout = m(f(dout))
    dy = dout * gate
    g = torch.zeros(B, Dn, N, dtype=F64) if dhT is None else f(dhT)
    du, ddl = torch.zeros_like(u), torch.zeros_like(u)
    dA = torch.zeros_like(A)
    dB, dC = torch.zeros_like(Bm), torch.zeros_like(Cm)
    for t in range(T - 1, -1, -1):
        o = on[:, t, None, None]
        Bt, Ct = (torch.where(o, wide(v[:, t]), zero) for v in (Bm, Cm))
        g = g + dy[:, t, :, None] * Ct
        dC[:, t] = torch.where(o, hs[t + 1] * dy[:, t, :, None], zero).reshape(B, G, rep, N).sum(2)
        x = torch.where(on[:, t, None], dd[:, t] * uu[:, t], zero)
        dB[:, t] = torch.where(o, g * x[..., None], zero).reshape(B, G, rep, N).sum(2)
        a = torch.exp(delta[:, t, :, None] * A)
        q = torch.where(o, g * a * hs[t], zero)
        gB = (g * Bt).sum(-1)
        dA += (q * dd[:, t, :, None]).sum(0)
        du[:, t] = dd[:, t] * gB + Dp * dy[:, t]
        ddl[:, t] = (q * f(A)).sum(-1) + uu[:, t] * gB
        g = g * a
    ddt = m(ddl) * (torch.sigmoid(raw) if softplus else 1.0)
    r.update(du=m(du), ddt=ddt, dA=dA, dB=dB, dC=dC, dD=(dy * m(uu)).sum((0, 1)), dbias=ddt.sum((0, 1)), dh0=g)
    if z is not None:
        r["dz"] = dout * m(y) * dgate
    return r


def linear(x, W, b=None, kind=0, res=None, dy=None, mag=False):
    """y, dx, dW, db.  x (M, K)."""
    f = torch.abs if mag else (lambda t: t)
    x, W, b, res, dy = (d(t) for t in (x, W, b, res, dy))
    pre = x @ W.t() + (0 if b is None else b)
    size = x.abs() @ W.t().abs() + (0 if b is None else b.abs())
    v, dv = act(pre, kind)
    y = size if mag else v
    if res is not None:
        y = y + f(res)
    if dy is None:
        return y
    q = dy.abs() * (dv.abs() + (size if kind else 0) + 1) if mag else dy * dv
    return y, q @ f(W), q.t() @ f(x), q.sum(0)


def near(got, want, size, steps, what=""):
    """|got - want| is within one rounding to got's type of the true value, plus `steps` 32-bit roundings of sums of size `size`."""
    fi = torch.finfo(got.dtype)
    g, w = got.detach().to("cpu", F64), want
    assert g.shape == w.shape, (what, g.shape, w.shape)
    own = 0.0 if got.dtype == torch.float32 else fi.eps / 2
    err = steps * U * size
    tol = err * (1 + own) + own * w.abs() + fi.tiny * fi.eps
    off = (g - w).abs()
    bad = ~(off <= tol)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, off / tol.clamp(min=1e-300), torch.zeros_like(off))))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst at {i}: got {g.reshape(-1)[i]:.9g}, want "
                             f"{w.reshape(-1)[i]:.9g}, may be off by {tol.reshape(-1)[i]:.3g}")
