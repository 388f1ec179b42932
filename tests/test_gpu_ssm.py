"""GPU: causal convolution, selective scan and linear with residual against their plain 64-bit forms (tests/ssm_reference.py).

Tolerances: one rounding to the output's type, and a count of 32-bit roundings times the sum of magnitudes that the output is
a sum of (ssm_reference.near).  The counts, to first order:
  convolution   K + 1 products and sums; SiLU on the hardware exp: its argument x log2 e carries |x| U, |x| < 8 here, besides a
                few U of its own: K + 32.  Sums over all steps: + B T.
  scan          a step multiplies the state by exp2(delta A log2 e): three roundings of the exponent, which is below 8 here, and
                the exp's own, the fused sum: below 40 U of what is kept, which shrinks with the decay; over T steps at most
                40 T when nothing decays.  softplus, gate, sums over N states: + 64 + N; over the channels of a group: + D;
                over all steps: + B T.
  linear        K + 2 sums, the activation's own error (8 U, or |z| U for the exponent, |z| < 16): K + 64.  Backward: dz is
                rounded to the operands' type before the products, eps / 2 of its size, besides N or M + 64.
"""
import itertools

import pytest
import torch

import ssm_reference as R

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
NAN = float("nan")
near = R.near


@pytest.fixture(autouse=True)
def poisoned():
    """Memory that the allocator hands out again holds NaN: what a kernel does not write, or reads unwritten, shows."""
    for n in (1 << 24, 1 << 20, 1 << 12, 256):
        torch.full((n // 4,), NAN, device="cuda")
    yield


def rnd(seed, *shape, type=FP, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(type).cuda()


def ints(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")


def req(*ts):
    for t in ts:
        if t is not None:
            t.requires_grad_(True)
    return ts


# ---- convolution ---------------------------------------------------------------------------------------------------------
CONV = [  # B, T, D, K, state, lengths
    (1, 1, 1, 4, False, None), (2, 1, 8, 4, True, None), (3, 2, 7, 4, True, [0, 1, 2]), (2, 5, 16, 1, False, None),
    (2, 9, 24, 2, True, [9, 3]), (1, 40, 64, 3, False, None), (2, 33, 65, 5, True, [33, 20]), (1, 17, 515, 6, False, [12]),
    (2, 70, 40, 7, True, None), (1, 19, 136, 8, True, [19]), (5, 64, 512, 4, True, [64, 0, 1, 2, 63]), (1, 700, 3, 4, False, [699]),
    (40, 3, 16, 4, True, None), (2, 0, 8, 4, True, None), (0, 4, 8, 4, False, None),
]


@pytest.mark.parametrize("type,wtype", [(FP, FP), (BF, BF), (HF, HF), (BF, FP)])
@pytest.mark.parametrize("B,T,D,K,has_state,lengths", CONV)
def test_conv(B, T, D, K, has_state, lengths, type, wtype):
    from timeband_amd import ops
    kind = ops.ACT_SILU if (T + D) % 2 else ops.ACT_NONE
    x, w, b = rnd(1, B, T, D, type=type), rnd(2, D, K, type=wtype, scale=K ** -0.5), rnd(3, D, type=wtype, scale=0.3)
    st = rnd(4, B, K - 1, D, type=type) if has_state else None
    dy, ln = rnd(5, B, T, D, type=type), ints(lengths)
    clean = x.clone()
    if ln is not None:                       # what lies behind a sequence's end must not be read, whatever it is
        for i, n in enumerate(lengths):
            x[i, n:], dy[i, n:], clean[i, n:] = NAN, NAN, 0
    req(x, w, b)
    y, new = ops.causal_conv(x, w, b, kind, state=st, lengths=ln, return_state=True)
    dyc = torch.nan_to_num(dy)
    want = R.conv(clean, w, b, kind, st, ln, dyc)
    size = R.conv(clean, w, b, kind, st, ln, dyc, mag=True)
    near(y, want[0], size[0], K + 32, "y")
    assert not new.requires_grad
    near(new, want[1], 0 * want[1], 0, "state")
    got = torch.autograd.grad(y, (x, w, b), dy)
    near(got[0], want[2], size[2], K + 48, "dx")
    near(got[1], want[3], size[3], B * T + 48, "dw")
    near(got[2], want[4], size[4], B * T + 48, "db")


@pytest.mark.parametrize("type", [FP, BF, HF])
def test_conv_views_without_bias(type):
    """A view with gaps between rows and an odd first element, no bias; a transposed view; an expanded batch."""
    from timeband_amd import ops
    big = rnd(1, 3, 21, 101, type=type)
    w = rnd(2, 64, 4, type=type, scale=0.5)
    for x in (big[:, :20, 5:69], big[:, ::2, 8:72], rnd(3, 3, 64, 20, type=type).transpose(1, 2), big[:1, :, 3:67].expand(3, 21, 64)):
        leaf = x.detach()
        req(leaf, w)
        y = ops.causal_conv(leaf, w, None, ops.ACT_SILU)
        dy = rnd(4, *y.shape, type=type)
        want, size = R.conv(leaf, w, None, 4, dy=dy), R.conv(leaf, w, None, 4, dy=dy, mag=True)
        got = torch.autograd.grad(y, (leaf, w), dy.transpose(1, 2).contiguous().transpose(1, 2))
        near(y, want[0], size[0], 36, "y")
        near(got[0], want[2], size[2], 52, "dx")
        near(got[1], want[3], size[3], 3 * 21 + 48, "dw")


@pytest.mark.parametrize("type", [FP, BF, HF])
@pytest.mark.parametrize("B,D,K", [(1, 1, 4), (3, 8, 4), (5, 37, 3), (2, 64, 1), (16, 1024, 4), (2, 40, 8), (0, 8, 4)])
def test_conv_step_continues_the_prompt(B, D, K, type):
    """A prompt, then steps: the same values as one call over all of it, bit for bit (the sums run in the same order)."""
    from timeband_amd import ops
    T, more = 6, 5
    x, w, b = rnd(1, B, T + more, D, type=type), rnd(2, D, K, type=type), rnd(3, D, type=type)
    whole = ops.causal_conv(x, w, b, ops.ACT_SILU)
    y, state = ops.causal_conv(x[:, :T], w, b, ops.ACT_SILU, return_state=True)
    assert torch.equal(y, whole[:, :T])
    pool = torch.full((B, K + 2, D), NAN, dtype=type, device="cuda")     # rows of state inside a larger buffer
    pool[:, :K - 1] = state
    for i in range(more):
        assert torch.equal(ops.causal_conv_step(x[:, T + i], pool[:, :K - 1], w, b, ops.ACT_SILU), whole[:, T + i])
    assert torch.equal(pool[:, :K - 1], x[:, T + more - (K - 1):]) and torch.isnan(pool[:, K - 1:]).all()


# ---- scan ----------------------------------------------------------------------------------------------------------------
def scan_inputs(B, T, D, N, G, type, gate, h0, seed=10):
    t = dict(u=rnd(seed, B, T, D, type=type), dt=rnd(seed + 1, B, T, D, type=type, scale=0.7),
             A=-(torch.rand(D, N, generator=torch.Generator().manual_seed(seed)) * 4 + 0.05).cuda(),
             Bm=rnd(seed + 2, B, T, G, N, type=type), Cm=rnd(seed + 3, B, T, G, N, type=type), D=rnd(seed + 4, D),
             bias=rnd(seed + 5, D) - 2)
    if gate:
        t["z"] = rnd(seed + 6, B, T, D, type=type)
    if h0:
        t["h0"] = rnd(seed + 7, B, D, N)
    return t


def call_scan(t, **k):
    from timeband_amd import ops
    return ops.selective_scan(t["u"], t["dt"], t["A"], t["Bm"], t["Cm"], D=t.get("D"), z=t.get("z"), dt_bias=t.get("bias"),
                              h0=t.get("h0"), **k)


SCAN = [  # B, T, D, N, G, gate, h0, lengths, softplus
    (1, 1, 1, 1, 1, False, False, None, True), (2, 1, 8, 16, 1, True, True, None, True), (2, 2, 5, 3, 1, True, False, [0, 2], True),
    (1, 31, 64, 4, 1, False, True, None, True), (2, 32, 65, 5, 1, True, True, [32, 7], True), (1, 33, 130, 8, 2, True, False, None, True),
    (2, 64, 48, 11, 3, False, True, [64, 33], True), (1, 65, 72, 16, 1, True, True, None, False), (3, 40, 129, 16, 1, True, False, [40, 0, 39], True),
    (1, 50, 24, 17, 1, True, True, None, True), (2, 35, 32, 32, 2, False, True, [35, 16], True), (1, 30, 40, 33, 1, True, True, None, True),
    (2, 23, 66, 64, 1, True, True, [23, 8], True), (1, 300, 70, 16, 1, True, True, None, True), (2, 400, 40, 6, 2, True, True, [400, 130], True),
    (1, 260, 24, 40, 1, False, False, [257], True), (1, 700, 8, 2, 1, True, True, [640], True),
]


@pytest.mark.parametrize("type", [FP, BF, HF])
@pytest.mark.parametrize("B,T,D,N,G,gate,h0,lengths,softplus", SCAN)
def test_scan(B, T, D, N, G, gate, h0, lengths, softplus, type):
    t = scan_inputs(B, T, D, N, G, type, gate, h0)
    if not softplus:
        t["dt"], t["bias"] = t["dt"].abs() * 0.1, t["bias"] * 0 + 0.01
    dout, dhT, ln = rnd(30, B, T, D, type=type), rnd(31, B, D, N), ints(lengths)
    plain = {k: v.clone() for k, v in t.items()}
    if ln is not None:
        for i, n in enumerate(lengths):
            dout[i, n:] = NAN
            for k in ("u", "dt", "Bm", "Cm", "z"):
                if k in t:
                    t[k][i, n:], plain[k][i, n:] = NAN, 0
    req(*t.values())
    out, hT = call_scan(t, softplus=softplus, lengths=ln, return_state=True)
    k = dict(softplus=softplus, lengths=ln, dout=torch.nan_to_num(dout), dhT=dhT)
    want, size = R.scan(**plain, **k), R.scan(**plain, **k, mag=True)
    n = 40 * T + 64 + N
    near(out, want["out"], size["out"], n, "out")
    near(hT, want["hT"], size["hT"], n, "hT")
    names = [q for q in t]
    got = dict(zip(names, torch.autograd.grad((out, hT), [t[q] for q in names], (dout, dhT))))
    for q in names:
        key = "d" + q[0] if q in ("Bm", "Cm") else "d" + q
        near(got[q], want[key], size[key], 2 * n + D + B * T, key)
    if ln is not None:
        for i, m in enumerate(lengths):
            assert not out[i, m:].any()


@pytest.mark.parametrize("type", [FP, BF])
def test_scan_views_and_optional_parts(type):
    """Slices of one projection's output (as a layer makes them), B and C without the axis of groups, no D, no bias, no gradient
    for some."""
    from timeband_amd import ops
    B, T, D, N = 2, 37, 48, 16
    proj = rnd(1, B, T, 3 * D + 2 * N + 5, type=type, scale=0.7)
    u, dt, z, Bm, Cm = (proj[..., 5:5 + D], proj[..., 5 + D:5 + 2 * D], proj[..., 5 + 2 * D:5 + 3 * D], proj[..., 5 + 3 * D:5 + 3 * D + N],
                        proj[..., 5 + 3 * D + N:])
    A = -(torch.rand(D, N, generator=torch.Generator().manual_seed(2)) + 0.1).cuda()
    leaf = proj.requires_grad_(True)
    cut = [leaf[..., 5:5 + D], leaf[..., 5 + D:5 + 2 * D], leaf[..., 5 + 3 * D:5 + 3 * D + N], leaf[..., 5 + 3 * D + N:], leaf[..., 5 + 2 * D:5 + 3 * D]]
    out = ops.selective_scan(cut[0], cut[1], A, cut[2], cut[3], z=cut[4])
    dout = rnd(3, B, T, D, type=type)
    got, = torch.autograd.grad(out, leaf, dout)
    k = dict(u=u, dt=dt, A=A, Bm=Bm[:, :, None], Cm=Cm[:, :, None], z=z, dout=dout)
    want, size = R.scan(**k), R.scan(**k, mag=True)
    n = 40 * T + 64 + N
    near(out, want["out"], size["out"], n, "out")
    for key, at in (("du", slice(5, 5 + D)), ("ddt", slice(5 + D, 5 + 2 * D)), ("dz", slice(5 + 2 * D, 5 + 3 * D))):
        near(got[..., at], want[key], size[key], 2 * n + D + B * T, key)
    near(got[..., 5 + 3 * D:5 + 3 * D + N], want["dB"][:, :, 0], size["dB"][:, :, 0], 2 * n + D + B * T, "dB")
    near(got[..., 5 + 3 * D + N:], want["dC"][:, :, 0], size["dC"][:, :, 0], 2 * n + D + B * T, "dC")
    assert not got[..., :5].any()


def test_scan_small_and_large_step_sizes():
    """softplus over its whole range: far below 0 (delta = e^x, down to where 1 + e^x rounds to 1) and far above (delta = x)."""
    B, T, D, N = 1, 64, 16, 4
    t = scan_inputs(B, T, D, N, 1, FP, False, False)
    t["dt"] = torch.linspace(-30, 30, T, device="cuda")[None, :, None].expand(B, T, D).contiguous()
    t["bias"] = torch.zeros(D, device="cuda")
    t["A"] = t["A"] * 0.01
    req(*t.values())
    out = call_scan(t)
    dout = rnd(5, B, T, D)
    want, size = R.scan(**t, dout=dout), R.scan(**t, dout=dout, mag=True)
    near(out, want["out"], size["out"], 40 * T + 68, "out")
    got = dict(zip(t, torch.autograd.grad(out, list(t.values()), dout)))
    for q in ("u", "dt", "Bm", "Cm"):
        key = "d" + q[0] if q in ("Bm", "Cm") else "d" + q
        near(got[q], want[key], size[key], 100 * T, key)


def test_scan_empty_sequences_and_batches():
    from timeband_amd import ops
    t = scan_inputs(2, 0, 8, 4, 1, BF, True, True)
    req(*t.values())
    out, hT = call_scan(t, return_state=True)
    assert out.shape == (2, 0, 8) and torch.equal(hT, t["h0"])
    g = torch.autograd.grad((out, hT), (t["h0"], t["A"]), (out.detach(), torch.ones_like(hT)))
    assert torch.equal(g[0], torch.ones_like(hT)) and not g[1].any()
    t = scan_inputs(0, 5, 8, 4, 1, FP, False, False)
    out, hT = call_scan(t, return_state=True)
    assert out.shape == (0, 5, 8) and hT.shape == (0, 8, 4)
    y = ops.causal_conv(rnd(1, 2, 0, 8).requires_grad_(True), rnd(2, 8, 4))
    assert y.shape == (2, 0, 8)


@pytest.mark.parametrize("type", [FP, BF, HF])
@pytest.mark.parametrize("B,D,N,G,gate", [(1, 1, 1, 1, False), (3, 8, 16, 1, True), (2, 66, 5, 2, True), (16, 129, 16, 3, False), (2, 40, 33, 1, True),
                                          (1, 64, 64, 1, True), (0, 8, 16, 1, True)])
def test_scan_step(B, D, N, G, gate, type):
    from timeband_amd import ops
    t = scan_inputs(B, 1, D, N, G, type, gate, True)
    want, size = R.scan(**t), R.scan(**t, mag=True)
    pool = torch.full((B, D * N + 3), NAN, device="cuda")
    state = pool[:, 1:1 + D * N].unflatten(1, (D, N))                    # rows inside a larger buffer, off 16 bytes
    state.copy_(t["h0"])
    args = dict(D=t["D"], z=t["z"][:, 0] if gate else None, dt_bias=t["bias"])
    out = ops.selective_scan_step(state, t["u"][:, 0], t["dt"][:, 0], t["A"], t["Bm"][:, 0], t["Cm"][:, 0], **args)
    near(out, want["out"][:, 0], size["out"][:, 0], 104 + N, "out")
    near(state, want["hT"], size["hT"], 104, "state")
    assert torch.isnan(pool[:, 0]).all() and torch.isnan(pool[:, 1 + D * N:]).all()


# ---- linear --------------------------------------------------------------------------------------------------------------
LINEAR = [  # M, K, N
    (1, 1, 1), (1, 8, 16), (3, 7, 5), (16, 64, 33), (17, 200, 48), (32, 65, 20), (33, 16, 16), (40, 63, 17), (100, 64, 130), (129, 72, 127),
    (257, 200, 256), (130, 1000, 36), (300, 1, 3), (64, 4096, 40), (1000, 40, 8), (2049, 24, 132),
]


@pytest.mark.parametrize("type", [FP, BF, HF])
@pytest.mark.parametrize("M,K,N", LINEAR)
def test_linear(M, K, N, type):
    from timeband_amd import ops
    kind = (M + K + N) % 6
    has_b, has_r = (M + N) % 3 != 0, K % 2 == 0
    x, W = rnd(1, M, K, type=type), rnd(2, N, K, type=type, scale=K ** -0.5)
    b, res, dy = rnd(3, N, type=type) if has_b else None, rnd(4, M, N, type=type) if has_r else None, rnd(5, M, N, type=type)
    leaves = [t for t in req(x, W, b, res) if t is not None]
    y = ops.linear_residual(x, W, b, kind, residual=res)
    want, size = R.linear(x, W, b, kind, res, dy), R.linear(x, W, b, kind, res, dy, mag=True)
    near(y, want[0], size[0], K + 64, "y")
    got = torch.autograd.grad(y, leaves, dy)
    if kind == 3:                      # relu's derivative jumps where z is 0: only rows and columns away from it are compared
        z = R.linear(x, W, b, 0)
        if (z.abs() <= (K + 4) * R.U * R.linear(x, W, b, 0, mag=True)).any():
            return
    round_dz = 0 if type == FP or kind == 0 else torch.finfo(type).eps / 2 / R.U
    near(got[0], want[1], size[1], N + K + 64 + round_dz, "dx")
    near(got[1], want[2], size[2], M + K + 64 + round_dz, "dW")
    if has_b:
        near(got[2], want[3], size[3], M + K + 64, "db")
    if has_r:
        assert torch.equal(got[-1], dy)


@pytest.mark.parametrize("type", [FP, BF, HF])
def test_linear_large_tiles(type):
    """Enough output for the 256 x 256 tiles, with rows, columns and k that do not fill the last ones; every activation."""
    from timeband_amd import ops
    M, K, N = 4100, 88, 4092
    x, W, b, res = rnd(1, M, K, type=type), rnd(2, N, K, type=type, scale=K ** -0.5), rnd(3, N, type=type), rnd(4, M, N, type=type)
    for kind in range(6):
        y = ops.linear_residual(x, W, b, kind, residual=res)
        near(y, R.linear(x, W, b, kind, res), R.linear(x, W, b, kind, res, mag=True), K + 64, f"act {kind}")


@pytest.mark.parametrize("type", [FP, BF])
def test_linear_views(type):
    """Rows with gaps, off 16 bytes, leading axes, an expanded row, a transposed input; one row of one axis."""
    from timeband_amd import ops
    K, N = 48, 40
    big = rnd(1, 3, 50, 77, type=type)
    W = rnd(2, N + 3, 64, type=type, scale=0.2)[1:N + 1, 5:5 + K]
    for x in (big[..., 8:56], big[..., 3:51], big[:, ::7, 8:56], big[:1, :1, :48].expand(3, 50, 48), rnd(3, 48, 90, type=type).t(), rnd(4, 48, type=type)):
        res = rnd(5, *x.shape[:-1], N + 9, type=type)[..., 4:4 + N]
        x, Wl, res = x.detach().requires_grad_(True), W.detach().requires_grad_(True), res.detach().requires_grad_(True)
        y = ops.linear_residual(x, Wl, None, ops.ACT_SILU, residual=res)
        assert y.shape == (*x.shape[:-1], N)
        dy = rnd(6, *y.shape, type=type)
        flat = lambda t, n: t.detach().reshape(-1, n)
        want = R.linear(flat(x, K), W, None, 4, flat(res, N), flat(dy, N))
        size = R.linear(flat(x, K), W, None, 4, flat(res, N), flat(dy, N), mag=True)
        near(y.reshape(-1, N), want[0], size[0], K + 64, "y")
        got = torch.autograd.grad(y, (x, Wl, res), dy)
        extra = 0 if type == FP else torch.finfo(type).eps / 2 / R.U
        near(got[0].reshape(-1, K), want[1], size[1], N + K + 64 + extra, "dx")
        near(got[1], want[2], size[2], 150 + K + 64 + extra, "dW")
        assert torch.equal(got[2], dy)


def test_linear_infinities_and_nan_stay_in_their_rows():
    from timeband_amd import ops
    for type, M in itertools.product((FP, BF, HF), (5, 200)):
        x, W = rnd(1, M, 40, type=type), rnd(2, 24, 40, type=type)
        clean = ops.linear_residual(x, W)
        x[2, 3], x[3, 7] = float("inf"), NAN
        y = ops.linear_residual(x, W)
        keep = [i for i in range(M) if i not in (2, 3)]
        assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[3]).all()
        assert torch.isinf(y[2]).all() and torch.equal(torch.sign(y[2].float()), torch.sign(W[:, 3].float()))


def test_linear_no_rows():
    from timeband_amd import ops
    x, W, b = rnd(1, 2, 0, 8).requires_grad_(True), rnd(2, 5, 8).requires_grad_(True), rnd(3, 5).requires_grad_(True)
    y = ops.linear_residual(x, W, b, ops.ACT_SILU)
    assert y.shape == (2, 0, 5)
    g = torch.autograd.grad(y, (x, W, b), torch.empty_like(y))
    assert g[0].shape == x.shape and not g[1].any() and not g[2].any()


def test_what_lies_between_rows_is_not_used():
    """NaN in the gaps between rows (and behind the last columns of a tile's k): the same results as from dense tensors."""
    from timeband_amd import ops
    for type, M, K, N in itertools.product((FP, BF, HF), (5, 200), (24, 40, 45), (24,)):
        x, W, res, dy = rnd(1, M, K, type=type), rnd(2, N, K, type=type), rnd(3, M, N, type=type), rnd(4, M, N, type=type)
        gap = lambda t: torch.cat([t, torch.full((t.shape[0], 16), NAN, dtype=type, device="cuda")], 1)[:, :t.shape[1]]
        out = []
        for f in (lambda t: t.clone(), gap):
            a = [f(t).detach().requires_grad_(True) for t in (x, W, res)]
            y = ops.linear_residual(a[0], a[1], None, ops.ACT_GELU, residual=a[2])
            out.append([y, *torch.autograd.grad(y, a, f(dy))])
        assert all(torch.equal(p, q) for p, q in zip(*out)), (type, M, K)
        x, w = rnd(5, 2, 37, K, type=type), rnd(6, K, 4, type=type)
        wide = torch.full((2, 37, K + 16), NAN, dtype=type, device="cuda")
        wide[..., :K] = x
        out = []
        for v in (x, wide[..., :K]):
            v = v.detach().requires_grad_(True)
            y = ops.causal_conv(v, w, None, ops.ACT_SILU)
            t = scan_inputs(2, 37, K, 6, 1, type, False, False)
            h = ops.selective_scan(v, v, t["A"], t["Bm"], t["Cm"], z=v)
            out.append([y, h, *torch.autograd.grad((y, h), v, (x, x))])
        assert all(torch.equal(p, q) for p, q in zip(*out)), (type, K)


def test_lengths_outside_the_steps_are_taken_as_the_nearest():
    from timeband_amd import ops
    x, w = rnd(1, 3, 10, 16), rnd(2, 16, 4)
    t = scan_inputs(3, 10, 16, 4, 1, FP, True, True)
    for f in (lambda ln: ops.causal_conv(x, w, lengths=ln, return_state=True), lambda ln: call_scan(t, lengths=ln, return_state=True)):
        assert all(torch.equal(p, q) for p, q in zip(f(ints([-3, 99, 4])), f(ints([0, 10, 4]))))


def test_tensors_of_more_than_2_31_elements():
    """Offsets behind 2^31 elements: the last rows of one large call against a call on those rows alone."""
    from timeband_amd import ops
    D, T = 32768, 70000                     # 2.3 G elements
    x = torch.zeros(1, T, D, dtype=BF, device="cuda")
    x[:, -40:] = rnd(1, 1, 40, D, type=BF)
    w = rnd(2, D, 4, type=BF)
    y, st = ops.causal_conv(x, w, None, ops.ACT_SILU, return_state=True)
    assert torch.equal(y[:, -30:], ops.causal_conv(x[:, -40:], w, None, ops.ACT_SILU)[:, -30:]) and torch.equal(st, x[:, -3:])
    del y
    A = torch.full((D, 4), -0.5, device="cuda")
    B = rnd(3, 1, T, 4, type=BF)
    y, h = ops.selective_scan(x, x, A, B, B, return_state=True)
    # the steps before are of zeros: they leave the state at 0
    y2, h2 = ops.selective_scan(x[:, -40:], x[:, -40:], A, B[:, -40:], B[:, -40:], return_state=True)
    assert float((y[:, -40:].float() - y2.float()).norm() / y2.float().norm()) < 2.0 ** -7 and float((h - h2).norm() / h2.norm()) < 1e-4
    del y
    W = rnd(4, 40, D, type=BF, scale=D ** -0.5)
    flat = x[0]
    y = ops.linear_residual(flat, W)
    y2 = ops.linear_residual(flat[-64:], W)
    assert not y[:-40].any() and float((y[-64:].float() - y2.float()).norm() / y2.float().norm()) < 2.0 ** -7


def test_gradients_into_a_flat_buffer():
    """Parameters of a FlatParams module (what the trainer's optimizer works on): the gradients land in its buffer, added up."""
    from timeband_amd import ops, optim
    lin = torch.nn.Linear(24, 40).cuda()
    flat = optim.FlatParams(lin)
    x, dy = rnd(1, 50, 24), rnd(2, 50, 40)
    want = torch.autograd.grad(ops.linear_residual(x, lin.weight, lin.bias, ops.ACT_SILU), (lin.weight, lin.bias), dy)
    for _ in range(2):
        ops.linear_residual(x, lin.weight, lin.bias, ops.ACT_SILU).backward(dy)
    assert torch.equal(flat.grad[:960].view(40, 24), want[0] + want[0]) and torch.equal(flat.grad[960:], want[1] + want[1])


def test_captured_steps_move_their_states():
    """A token's path captured once and replayed: each replay reads the input buffer and moves the states, as eager calls do."""
    p = layer(type=BF)
    with torch.no_grad():
        x = rnd(95, 6, 3, 40, type=BF)
        _, cs, h = run_layer(p, rnd(94, 3, 9, 40, type=BF))
        cs2, h2, buf = cs.clone(), h.clone(), x[0].clone()
        step_layer(p, buf, cs.clone(), h.clone())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step_layer(p, buf, cs2, h2)
        for i in range(6):
            buf.copy_(x[i])
            g.replay()
            want = step_layer(p, x[i], cs, h)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(cs, cs2) and torch.equal(h, h2)


# ---- all of them ---------------------------------------------------------------------------------------------------------
def layer(D=64, N=16, R_=8, model=40, K=4, type=FP, seed=50):
    """The weights of one state space layer: in-projection, convolution, what makes dt, B and C, scan, out-projection."""
    A = -(torch.rand(D, N, generator=torch.Generator().manual_seed(seed)) * 2 + 0.1).cuda()
    return dict(w_in=rnd(seed, 2 * D, model, type=type, scale=model ** -0.5), b_in=rnd(seed + 1, 2 * D, type=type, scale=0.1),
                w_conv=rnd(seed + 2, D, K, type=type, scale=0.5), b_conv=rnd(seed + 3, D, type=type, scale=0.1),
                w_x=rnd(seed + 4, D + 2 * N, D, type=type, scale=D ** -0.5), A=A, D=rnd(seed + 5, D), dt_bias=rnd(seed + 6, D) - 2,
                w_out=rnd(seed + 7, model, D, type=type, scale=D ** -0.5), b_out=rnd(seed + 8, model, type=type, scale=0.1))


def run_layer(p, x, lengths=None, conv_state=None, h0=None):
    from timeband_amd import ops
    D, N = p["A"].shape
    xz = ops.linear_residual(x, p["w_in"], p["b_in"])
    u, cs = ops.causal_conv(xz[..., :D], p["w_conv"], p["b_conv"], ops.ACT_SILU, state=conv_state, lengths=lengths, return_state=True)
    q = ops.linear_residual(u, p["w_x"])
    y, h = ops.selective_scan(u, q[..., :D], p["A"], q[..., D:D + N], q[..., D + N:], D=p["D"], z=xz[..., D:], dt_bias=p["dt_bias"], h0=h0,
                              lengths=lengths, return_state=True)
    return ops.linear_residual(y, p["w_out"], p["b_out"], residual=x), cs, h


def step_layer(p, x, cs, h):
    from timeband_amd import ops
    D, N = p["A"].shape
    xz = ops.linear_residual(x, p["w_in"], p["b_in"])
    u = ops.causal_conv_step(xz[..., :D], cs, p["w_conv"], p["b_conv"], ops.ACT_SILU)
    q = ops.linear_residual(u, p["w_x"])
    y = ops.selective_scan_step(h, u, q[..., :D], p["A"], q[..., D:D + N], q[..., D + N:], D=p["D"], z=xz[..., D:], dt_bias=p["dt_bias"])
    return ops.linear_residual(y, p["w_out"], p["b_out"], residual=x)


def layer_64(p, x):
    """The layer in 64 bits, from the plain forms' formulas, differentiable."""
    D, N = p["A"].shape
    xz = x @ p["w_in"].t() + p["b_in"]
    K = p["w_conv"].shape[1]
    pad = torch.cat([torch.zeros_like(xz[:, :K - 1, :D]), xz[..., :D]], 1)
    pre = p["b_conv"] + sum(p["w_conv"][:, k] * pad[:, k:k + x.shape[1]] for k in range(K))
    u = pre * torch.sigmoid(pre)
    q = u @ p["w_x"].t()
    delta = torch.log1p(torch.exp(q[..., :D] + p["dt_bias"]))
    h = torch.zeros(x.shape[0], D, N, dtype=x.dtype, device=x.device)
    ys = []
    for t in range(x.shape[1]):
        h = torch.exp(delta[:, t, :, None] * p["A"]) * h + (delta[:, t] * u[:, t])[..., None] * q[:, t, None, D:D + N]
        ys.append((h * q[:, t, None, D + N:]).sum(-1) + p["D"] * u[:, t])
    z = xz[..., D:]
    return (torch.stack(ys, 1) * z * torch.sigmoid(z)) @ p["w_out"].t() + p["b_out"] + x


def test_layer_trains_as_its_formula_says():
    """Output and every weight's gradient of a whole layer, fp32, against the formula in 64 bits (norms: the bound is a few
    hundred 32-bit roundings of sums whose parts are of the results' own size)."""
    p = layer()
    x = rnd(99, 3, 50, 40)
    req(x, *p.values())
    y = run_layer(p, x)[0]
    dy = rnd(98, *y.shape)
    got = torch.autograd.grad(y, [x, *p.values()], dy)
    q = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    x64 = x.detach().double().requires_grad_(True)
    y64 = layer_64(q, x64)
    want = torch.autograd.grad(y64, [x64, *q.values()], dy.double())
    for name, a, b in zip(["y", "x", *p], [y, *got], [y64, *want]):
        off = float(((a.double() - b).norm() / b.norm()).detach())
        assert off < 400 * R.U, (name, off)


@pytest.mark.parametrize("type,tol", [(FP, 400 * R.U), (BF, 24 * 2.0 ** -8)])
def test_layer_prompt_then_tokens(type, tol):
    """A padded batch of prompts and tokens one by one give what one call over each whole sequence gives.  bf16: the layer
    rounds four tensors between its operators on either path, and a difference of one step is carried on."""
    p = layer(type=type)
    lens, more = [9, 1, 23], 6
    x = rnd(97, 3, 40, 40, type=type)
    with torch.no_grad():
        ln = ints(lens)
        y, cs, h = run_layer(p, x[:, :23], lengths=ln)
        steps = []
        for i in range(more):
            tok = torch.stack([x[b, lens[b] + i] for b in range(3)])
            steps.append(step_layer(p, tok, cs, h))
        for b, n in enumerate(lens):
            whole = run_layer(p, x[b:b + 1, :n + more])[0][0]
            got = torch.cat([y[b, :n], torch.stack([s[b] for s in steps])])
            assert float((got.float() - whole.float()).norm() / whole.float().norm()) < tol


def test_layer_in_two_pieces_equals_one():
    p = layer()
    x = rnd(96, 2, 70, 40)
    with torch.no_grad():
        whole, cs, h = run_layer(p, x)
        a, cs1, h1 = run_layer(p, x[:, :33])
        b, cs2, h2 = run_layer(p, x[:, 33:], conv_state=cs1, h0=h1)
    assert float((torch.cat([a, b], 1) - whole).norm() / whole.norm()) < 100 * R.U
    assert float((h2 - h).norm() / h.norm()) < 100 * R.U and float((cs2 - cs).norm() / cs.norm()) < 100 * R.U


def all_outputs(seed, type=BF):
    """One call of everything, forward and backward, at sizes that take the split paths: what it returns, in a list."""
    from timeband_amd import ops
    t = scan_inputs(1, 300, 40, 16, 1, type, True, True, seed=seed)
    x, w, b = rnd(seed, 2, 50, 64, type=type), rnd(seed + 1, 64, 4, type=type), rnd(seed + 2, 64, type=type)
    lx, lw, lb, lr = rnd(seed + 3, 150, 1030, type=type), rnd(seed + 4, 72, 1030, type=type, scale=0.03), rnd(seed + 5, 72, type=type), rnd(seed + 6, 150, 72, type=type)
    req(*t.values(), x, w, b, lx, lw, lb, lr)

    def run():
        o = list(call_scan(t, return_state=True))
        o += torch.autograd.grad(o[0], list(t.values()), t["u"].detach())
        y = ops.causal_conv(x, w, b, ops.ACT_SILU)
        o += [y, *torch.autograd.grad(y, (x, w, b), x.detach())]
        y = ops.linear_residual(lx, lw, lb, ops.ACT_GELU, residual=lr)
        return o + [y, *torch.autograd.grad(y, (lx, lw, lb, lr), lr.detach())]

    return run


def test_same_inputs_same_bits():
    run = all_outputs(70)
    first = [o.clone() for o in run()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_on_another_stream_while_the_first_is_busy():
    one, two = all_outputs(71), all_outputs(72)
    want = [[o.clone() for o in f()] for f in (one, two)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s):
            b = two()
        a = one()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want[0], a)) and all(torch.equal(p, q) for p, q in zip(want[1], b))


def test_two_captured_graphs_with_eager_work_between():
    """Forward and backward captured twice with other inputs; replays in turn, eager calls of other sizes between."""
    runs = [all_outputs(73), all_outputs(74)]
    want = [[o.detach().clone() for o in f()] for f in runs]      # detached: no eager graph of the leaves may live
    graphs, outs = [], []
    s = torch.cuda.Stream()
    for f in runs:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            f()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    other = all_outputs(75, FP)
    for _ in range(4):
        for g in graphs:
            g.replay()
        other()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, w))


def test_capture_over_a_live_eager_graph_is_refused():
    from timeband_amd import ops
    x, W = rnd(1, 40, 8).requires_grad_(True), rnd(2, 6, 8).requires_grad_(True)
    held = ops.linear_residual(x, W)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.linear_residual(x * 2, W)
    del held
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.linear_residual(x * 2, W)
        d, = torch.autograd.grad(y, W, torch.ones_like(y))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(d, torch.autograd.grad(ops.linear_residual(x * 2, W), W, torch.ones_like(y))[0])


def test_double_backward_is_refused():
    from timeband_amd import ops
    x, W = rnd(1, 40, 8).requires_grad_(True), rnd(2, 6, 8).requires_grad_(True)
    g, = torch.autograd.grad(ops.linear_residual(x, W, act=ops.ACT_SILU).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), W)


def test_refusals():
    from timeband_amd import ops
    x, w = rnd(1, 2, 5, 8), rnd(2, 8, 4)
    ok = dict(u=x, dt=x, A=-torch.ones(8, 4, device="cuda"), B=rnd(3, 2, 5, 4), C=rnd(4, 2, 5, 4))

    def refused(match, f, *a, **k):
        with pytest.raises(RuntimeError, match=match):
            f(*a, **k)

    refused("weight must be", ops.causal_conv, x, rnd(2, 7, 4))
    refused("9 taps", ops.causal_conv, x, rnd(2, 8, 9))
    refused("activation", ops.causal_conv, x, w, None, ops.ACT_TANH)
    refused("expected shape", ops.causal_conv, x, w, rnd(2, 7))
    refused("expected shape", ops.causal_conv, x, w, state=rnd(3, 2, 4, 8))
    refused("throughout", ops.causal_conv, x, w, state=rnd(3, 2, 3, 8, type=BF))
    refused("must both be", ops.causal_conv, x, w.to(BF))
    refused("not supported", ops.causal_conv, x.double(), w)
    refused("lengths", ops.causal_conv, x, w, lengths=torch.zeros(2, dtype=torch.int64, device="cuda"))
    refused("lengths", ops.causal_conv, x, w, lengths=ints([1, 2, 3]))
    refused("no gradient runs", ops.causal_conv, x, w, state=rnd(3, 2, 3, 8).requires_grad_(True))
    refused("no_grad", ops.causal_conv_step, x[:, 0].clone().requires_grad_(True), rnd(3, 2, 3, 8), w)
    refused("dense", ops.causal_conv_step, x[:, 0], rnd(3, 2, 8, 3).transpose(1, 2), w)
    refused("overlap", ops.causal_conv_step, x[:, 0], rnd(3, 1, 3, 8).expand(2, 3, 8), w)
    refused("dt", ops.selective_scan, **{**ok, "dt": rnd(1, 2, 4, 8)})
    refused("throughout", ops.selective_scan, **{**ok, "dt": x.to(BF)})
    refused("groups", ops.selective_scan, **{**ok, "B": rnd(3, 2, 5, 3, 4), "C": rnd(3, 2, 5, 3, 4)})
    refused("float32", ops.selective_scan, **{**ok, "A": ok["A"].to(BF)})
    refused("float32", ops.selective_scan, **ok, h0=rnd(3, 2, 8, 5))
    refused("must be", ops.selective_scan, **{**ok, "C": rnd(3, 2, 5, 5)})
    refused("65 states", ops.selective_scan, **{**ok, "A": -torch.ones(8, 65, device="cuda"), "B": rnd(3, 2, 5, 65), "C": rnd(3, 2, 5, 65)})
    st = dict(u=x[:, 0], dt=x[:, 0], A=ok["A"], B=ok["B"][:, 0], C=ok["C"][:, 0])
    refused("state must be", ops.selective_scan_step, rnd(3, 2, 8, 4, type=BF), **st)
    refused("dense", ops.selective_scan_step, rnd(3, 2, 4, 8).transpose(1, 2), **st)
    refused("overlap", ops.selective_scan_step, rnd(3, 1, 8, 4).expand(2, 8, 4), **st)
    refused("no_grad", ops.selective_scan_step, rnd(3, 2, 8, 4), **{**st, "A": ok["A"].clone().requires_grad_(True)})
    refused("does not match", ops.linear_residual, x, rnd(2, 6, 7))
    refused("expected shape", ops.linear_residual, x, rnd(2, 6, 8), rnd(3, 5))
    refused("expected shape", ops.linear_residual, x, rnd(2, 6, 8), residual=rnd(3, 2, 1, 6))
    refused("activation", ops.linear_residual, x, rnd(2, 6, 8), act=6)
    refused("throughout", ops.linear_residual, x, rnd(2, 6, 8, type=BF))


def test_step_marks_its_state_as_changed():
    """A state that a recorded call saved and a step then changes: its backward pass is refused, not computed from the new state."""
    from timeband_amd import ops
    x, w, state = rnd(3, 2, 5, 8).requires_grad_(True), rnd(4, 8, 4), rnd(5, 2, 3, 8)
    y = ops.causal_conv(x, w, None, ops.ACT_SILU, state=state)
    before = state._version
    with torch.no_grad():
        ops.causal_conv_step(rnd(6, 2, 8), state, w, None, ops.ACT_SILU)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    h = rnd(7, 2, 8, 4)
    before = h._version
    with torch.no_grad():
        ops.selective_scan_step(h, rnd(8, 2, 8), rnd(9, 2, 8), -torch.ones(8, 4, device="cuda"), rnd(10, 2, 4), rnd(11, 2, 4))
    assert h._version > before
    with torch.inference_mode():                      # tensors without a version are stepped as before
        s = torch.zeros(2, 3, 8, device="cuda")
        ops.causal_conv_step(rnd(6, 2, 8), s, w)
    with torch.no_grad():
        ops.causal_conv_step(rnd(6, 2, 8), s, w)
    assert bool((s != 0).any())
