"""CPU: the plain forms' gradients against differences, and what the state space layer's operators refuse before any launch."""
import ctypes

import pytest
import torch

import ssm_reference as R

F64 = torch.float64


def _differences(loss, t, at, eps=1e-5):
    flat = t.reshape(-1)
    out = []
    for i in at:
        v = float(flat[i])
        flat[i] = v + eps
        up = float(loss())
        flat[i] = v - eps
        dn = float(loss())
        flat[i] = v
        out.append((up - dn) / (2 * eps))
    return torch.tensor(out, dtype=F64)


@pytest.mark.parametrize("kind", [0, 4])
@pytest.mark.parametrize("lengths", [None, [5, 0, 2]])
def test_conv_formula_against_differences(kind, lengths):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, dtype=F64)
    x, w, b, st, dy = r(3, 5, 4), r(4, 3), r(4), r(3, 2, 4), r(3, 5, 4)
    ln = None if lengths is None else torch.tensor(lengths)
    loss = lambda: (R.conv(x, w, b, kind, st, ln)[0] * dy).sum()
    _, _, dx, dw, db = R.conv(x, w, b, kind, st, ln, dy)
    for t, dt in ((x, dx), (w, dw), (b, db)):
        at = range(0, t.numel(), 3)
        # central differences at 1e-5: third derivatives of order ten give 1e-9, 64-bit rounding 1e-15 / 1e-5
        assert torch.allclose(_differences(loss, t, at), dt.reshape(-1)[list(at)], rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("gate,softplus,lengths,groups", [(True, True, None, 1), (False, True, [4, 0], 2), (True, False, [2, 4], 2)])
def test_scan_formula_against_differences(gate, softplus, lengths, groups):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(s, generator=g, dtype=F64)
    B, T, D, N = 2, 4, 4, 3
    t = dict(u=r(B, T, D), dt=r(B, T, D) * 0.3, A=-torch.rand(D, N, generator=g, dtype=F64) - 0.2, Bm=r(B, T, groups, N), Cm=r(B, T, groups, N),
             D=r(D), bias=r(D), h0=r(B, D, N))
    if gate:
        t["z"] = r(B, T, D)
    dout, dhT = r(B, T, D), r(B, D, N)
    ln = None if lengths is None else torch.tensor(lengths)

    def loss():
        q = R.scan(**t, softplus=softplus, lengths=ln)
        return (q["out"] * dout).sum() + (q["hT"] * dhT).sum()

    got = R.scan(**t, softplus=softplus, lengths=ln, dout=dout, dhT=dhT)
    for k, v in t.items():
        grad = got["d" + k[0] if k in ("Bm", "Cm") else "d" + k]
        at = range(0, v.numel(), 2)
        assert torch.allclose(_differences(loss, v, at), grad.reshape(-1)[list(at)], rtol=1e-6, atol=1e-7), k


@pytest.mark.parametrize("kind", [0, 1, 2, 4, 5])
def test_linear_formula_against_differences(kind):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, dtype=F64)
    x, W, b, res, dy = r(3, 4), r(5, 4), r(5), r(3, 5), r(3, 5)
    loss = lambda: (R.linear(x, W, b, kind, res) * dy).sum()
    _, dx, dW, db = R.linear(x, W, b, kind, res, dy)
    for t, dt in ((x, dx), (W, dW), (b, db)):
        at = range(t.numel())
        assert torch.allclose(_differences(loss, t, at), dt.reshape(-1), rtol=1e-6, atol=1e-7)


def test_cpu_tensors_are_refused():
    from timeband_amd import ops
    x = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.causal_conv_step(x[:, 0], torch.zeros(2, 3, 8), torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.selective_scan(x, x, torch.zeros(8, 4), torch.zeros(2, 3, 4), torch.zeros(2, 3, 4))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.selective_scan_step(torch.zeros(2, 8, 4), x[:, 0], x[:, 0], torch.zeros(8, 4), torch.zeros(2, 4), torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.linear_residual(x, torch.zeros(5, 8))


def test_library_refuses_bad_calls_before_launching():
    """Return codes of the C entries (1 argument, 3 unsupported, 4 workspace), without a GPU and with no pointer followed."""
    from timeband_amd import _lib
    lib = _lib.load()
    p, ls = 4096, (ctypes.c_long * 14)()
    conv = lambda **k: lib.tb_conv_fwd(*(k.get(n, v) for n, v in dict(
        x=p, xb=64, xs=8, w=p, bias=0, wf=0, state=0, lengths=0, y=p, out=0, B=2, T=8, D=8, K=4, act=0, dtype=0, stream=0).items()))
    assert conv(K=9) == 3 and b"9 taps" in lib.tb_last_error()
    assert conv(K=0) == 3 and conv(act=1) == 3 and conv(act=5) == 3
    assert conv(dtype=3) == 1 and conv(D=0) == 1 and conv(B=-1) == 1 and conv(x=0) == 1 and conv(y=0) == 1
    assert conv(B=0) == 0                                       # nothing to do, nothing launched
    assert lib.tb_conv_bwd(p, p, 64, 8, p, 0, 0, 0, 0, p, p, p, 2, 8, 8, 4, 0, 0, p, 16, 0) == 4
    assert lib.tb_conv_bwd(p, p, 64, 8, p, 0, 0, 0, 0, p, p, p, 0, 8, 8, 4, 0, 0, p, 1 << 30, 0) == 1
    assert lib.tb_conv_step(p, 8, 0, 24, p, 0, 0, p, 2, 8, 4, 0, 0, 0) == 1
    scan = lambda **k: lib.tb_scan_fwd(*(k.get(n, v) for n, v in dict(
        u=p, dt=p, z=0, B=p, C=p, st=ls, A=p, D=0, bias=0, sp=1, h0=0, lengths=0, out=p, hT=0, states=0, Bn=2, T=8, Dn=8, N=4, G=1,
        dtype=0, ws=p, wsb=1 << 30, stream=0).items()))
    assert scan(N=65) == 3 and scan(N=0) == 1 and scan(G=3) == 1 and scan(G=0) == 1 and scan(dtype=-1) == 1
    assert scan(T=0) == 1 and scan(Bn=0) == 1 and scan(u=0) == 1 and scan(wsb=0) == 4 and scan(ws=0) == 1
    back = lambda **k: lib.tb_scan_bwd(*(k.get(n, v) for n, v in dict(
        dout=p, u=p, dt=p, z=0, B=p, C=p, st=ls, A=p, D=0, bias=0, sp=1, lengths=0, states=p, dhT=0, du=p, ddt=p, dz=0, dB=p, dC=p, dA=p,
        dD=0, dbias=0, dh0=0, Bn=2, T=8, Dn=8, N=4, G=1, dtype=0, ws=p, wsb=1 << 30, stream=0).items()))
    assert back(states=0) == 1 and back(wsb=64) == 4 and back(N=100) == 3
    assert lib.tb_scan_step(p, 32, p, p, 0, p, p, ls, p, 0, 0, 1, p, 2, 8, 65, 1, 0, 0) == 3
    assert lib.tb_scan_step(0, 32, p, p, 0, p, p, ls, p, 0, 0, 1, p, 2, 8, 4, 1, 0, 0) == 1
    lin = lambda **k: lib.tb_linres_fwd(*(k.get(n, v) for n, v in dict(
        x=p, xs=8, W=p, ws_=8, b=0, r=0, rs=0, y=p, z=0, M=100, K=8, N=8, act=0, dtype=0, ws=p, wsb=1 << 30, stream=0).items()))
    assert lin(act=6) == 3 and lin(act=-1) == 3 and lin(K=0) == 1 and lin(N=0) == 1 and lin(M=-1) == 1 and lin(dtype=7) == 1
    assert lin(wsb=0) == 4 and lin(W=0) == 1 and lin(M=0) == 0
    assert lib.tb_linres_bwd(p, 8, p, 8, p, 8, 0, 4, p, p, p, 100, 8, 8, 0, p, 1 << 30, 0) == 1        # no pre-activation kept
    assert lib.tb_linres_bwd(p, 8, p, 8, p, 8, 0, 0, p, p, p, 100, 8, 8, 0, p, 16, 0) == 4


def test_library_refuses_sizes_past_its_indexes():
    """Steps whose sums with a run pass 32 bits, and launches of 2^32 threads: refused (3) before anything is launched."""
    from timeband_amd import _lib
    lib = _lib.load()
    p, ls, wide = 4096, (ctypes.c_long * 14)(), 1 << 62
    top = 2 ** 31 - 1
    assert lib.tb_conv_fwd(p, top, 1, p, 0, 0, 0, 0, p, 0, 1, top, 1, 4, 0, 1, 0) == 3
    assert lib.tb_conv_bwd(p, p, top, 1, p, 0, 0, 0, 0, p, p, p, 1, top, 1, 4, 0, 1, p, wide, 0) == 3
    assert lib.tb_conv_step(p, 4097, p, 4097 * 3, p, 0, 0, p, 1 << 20, 4097, 4, 0, 1, 0) == 3        # element by element
    assert lib.tb_conv_step(p, 1 << 15, p, 3 << 15, p, 0, 0, p, 1 << 20, 1 << 15, 4, 0, 1, 0) == 3    # eight a thread
    fwd = lambda B, T, D, N: lib.tb_scan_fwd(p, p, 0, p, p, ls, p, 0, 0, 1, 0, 0, p, 0, 0, B, T, D, N, 1, 1, p, wide, 0)
    bwd = lambda B, T, D, N: lib.tb_scan_bwd(p, p, p, 0, p, p, ls, p, 0, 0, 1, 0, p, 0, p, p, 0, p, p, p, 0, 0, 0, B, T, D, N, 1, 1, p, wide, 0)
    assert fwd(1, top, 1, 16) == 3 and bwd(1, top, 1, 16) == 3
    assert fwd(1 << 20, 1, 1024, 16) == 3 and bwd(1 << 20, 1, 1024, 16) == 3
    assert bwd(1 << 10, 1 << 17, 1, 16) == 3                     # the sums of dB and dC
    assert lib.tb_scan_step(p, 1 << 14, p, p, 0, p, p, ls, p, 0, 0, 1, p, 1 << 20, 1024, 16, 1, 1, 0) == 3
    lin = lambda M, K, N: lib.tb_linres_fwd(p, K, p, K, 0, 0, 0, p, 0, M, K, N, 0, 0, p, wide, 0)
    back = lambda M, K, N: lib.tb_linres_bwd(p, N, p, K, p, K, 0, 0, p, p, p, M, K, N, 0, p, wide, 0)
    assert lin(2 ** 30 + 64, 4, 4) == 3 and back(2 ** 30 + 64, 4, 4) == 3
    assert lin(1 << 28, 65, 4) == 3 and lin(100, 4000001, 4) == 3 and lin(100, 4, 4000001) == 3
