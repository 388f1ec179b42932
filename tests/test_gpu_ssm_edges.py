"""GPU: the state space layer's operators where they went wrong once, or could unseen: gradients through 16-bit products, infinities,
long and uncut walks, every dispatch branch of the linear layer's backward pass.  Plain forms and `near`: ssm_reference."""
import pytest
import torch

import ssm_reference as R

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")
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


def req(*ts):
    return [t.requires_grad_(True) for t in ts]


def rounded_once(got, want, what):
    """got is the 64-bit `want` with an error far below its type's step, rounded once: its distance is that of want's own rounding.
    Over n values that distance's square scatters by 0.9 / sqrt(n) of itself; 25000 values leave 0.3 % on the distance, and 3 % is
    ten times that.  A second rounding of the same size gives 41 %."""
    g = got.detach().to("cpu", torch.float64)
    assert g.numel() >= 25000 and torch.isfinite(g).all(), what
    ratio = float((g - want).norm() / (want.to(got.dtype).double() - want).norm())
    assert ratio < 1.03, (what, ratio)


# ---- linear: dz of 16-bit types --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", [BF, HF])
@pytest.mark.parametrize("kind", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("M,K,N", [(257, 200, 256), (2049, 132, 200), (300, 90, 1501), (1500, 301, 84)])
def test_linear_gradients_of_16_bits_are_rounded_once(M, K, N, kind, type):
    """dz = dy act'(z) must not be rounded to the operands' type before the products: that doubles the gradients' error.  relu:
    dz is dy or 0, exact; z's sign is clear of its rounding errors (|z| > 0.5 by the bias)."""
    from timeband_amd import ops
    x, W, b, dy = rnd(1, M, K, type=type), rnd(2, N, K, type=type, scale=K ** -0.5), rnd(3, N, type=type), rnd(5, M, N, type=type)
    if kind == 3:
        W, b = W * 0.05, torch.where(b > 0, b + 1, b - 1)
    req(x, W, b)
    got = torch.autograd.grad(ops.linear_residual(x, W, b, kind), (x, W, b), dy)
    _, dx, dW, _ = R.linear(x, W, b, kind, None, dy)
    rounded_once(got[0], dx, "dx")
    rounded_once(got[1], dW, "dW")


def test_linear_gradients_at_the_ends_of_fp16():
    """dy near the largest value where the activation's slope is above 1: dz is past the type, the gradients are not.  dy among the
    smallest values: dz is below the type's steps, its sums over many rows are not."""
    from timeband_amd import ops
    M, K, N = 80, 320, 330
    x, W, b = rnd(1, M, K, type=HF, scale=1e-3), rnd(2, N, K, type=HF, scale=5e-3), torch.full((N,), 1.4, dtype=HF, device="cuda")
    dy = (65504 * torch.sign(rnd(3, M, N))).to(HF)
    req(x, W, b)
    for kind in (4, 5):
        got = torch.autograd.grad(ops.linear_residual(x, W, b, kind), (x, W), dy)
        _, dx, dW, _ = R.linear(x, W, b, kind, None, dy)
        assert float(dx.abs().max()) < 60000 and float(dW.abs().max()) < 60000
        rounded_once(got[0], dx, "dx")
        rounded_once(got[1], dW, "dW")
    M, K, N = 6000, 200, 200
    x, W, dy = rnd(4, M, K, type=HF), rnd(5, N, K, type=HF, scale=K ** -0.5), rnd(6, M, N, type=HF, scale=2.0 ** -21)
    req(x, W)
    for kind in (1, 2, 4, 5):
        got = torch.autograd.grad(ops.linear_residual(x, W, None, kind), (x, W), dy)
        _, dx, dW, _ = R.linear(x, W, None, kind, None, dy)
        rounded_once(got[1], dW, "dW")
        rounded_once(got[0], dx, "dx")


def test_linear_infinite_gradients_stay_in_their_rows():
    """An infinite or NaN dy: the infinities and NaN that the formula gives, in its row of dx and its column of dW alone."""
    from timeband_amd import ops
    for type in (FP, BF, HF):
        x, W, dy = rnd(1, 90, 40, type=type), rnd(2, 48, 40, type=type), rnd(3, 90, 48, type=type)
        req(x, W)
        y = ops.linear_residual(x, W, None, ops.ACT_SIGMOID)
        clean = torch.autograd.grad(y, (x, W), dy, retain_graph=True)
        dy[7, 5], dy[8, 6] = INF, NAN
        dx, dW = torch.autograd.grad(y, (x, W), dy)
        rows, cols = [i for i in range(90) if i not in (7, 8)], [i for i in range(48) if i not in (5, 6)]
        assert torch.equal(dx[rows], clean[0][rows]) and torch.equal(dW[cols], clean[1][cols])
        assert torch.equal(dx[7].float(), INF * torch.sign(W[5].float())) and torch.isnan(dx[8]).all()
        assert torch.equal(dW[5].float(), INF * torch.sign(x[7].float())) and torch.isnan(dW[6]).all()


# ---- modes of differentiation ------------------------------------------------------------------------------------------------
def test_forward_mode_is_refused():
    from test_ssm_edges_host import check_forward_mode_is_refused
    check_forward_mode_is_refused("cuda")


# ---- scan: infinities ------------------------------------------------------------------------------------------------------------
def scan_case(B, T, D, N, G=1, type=FP, seed=10, positive=False):
    t = dict(u=rnd(seed, B, T, D, type=type), dt=rnd(seed + 1, B, T, D, type=type, scale=0.7),
             A=-(torch.rand(D, N, generator=torch.Generator().manual_seed(seed)) * 2 + 0.05).cuda(),
             Bm=rnd(seed + 2, B, T, G, N, type=type), Cm=rnd(seed + 3, B, T, G, N, type=type), D=rnd(seed + 4, D), bias=rnd(seed + 5, D) - 2,
             z=rnd(seed + 6, B, T, D, type=type), h0=rnd(seed + 7, B, D, N))
    if positive:
        for k in ("Bm", "Cm", "D", "h0"):
            t[k] = t[k].abs()
    return t


def call_scan(t, **k):
    from timeband_amd import ops
    return ops.selective_scan(t["u"], t["dt"], t["A"], t["Bm"], t["Cm"], D=t.get("D"), z=t.get("z"), dt_bias=t.get("bias"), h0=t.get("h0"), **k)


def grads(t, out, hT, dout, dhT):
    return dict(zip(["d" + (k[0] if k in ("Bm", "Cm") else k) for k in t], torch.autograd.grad((out, hT), list(t.values()), (dout, dhT))))


def like(got, want, size, steps, what):
    """Infinities and NaN where the 64-bit form has them, of the same sign; what is finite, and of finite parts, is near."""
    g, w = got.detach().to("cpu", torch.float64), want
    assert torch.equal(torch.isnan(g), torch.isnan(w)), (what, "NaN", int(torch.isnan(g).sum()), int(torch.isnan(w).sum()))
    assert torch.equal(torch.where(torch.isinf(g), g, 0), torch.where(torch.isinf(w), w, 0)), (what, "infinities")
    fine = torch.isfinite(w) & torch.isfinite(size)
    near(got.detach().cpu()[fine], w[fine], size[fine], steps, what)


def scan_like(t, dout, dhT, lengths=None, names=None, **k):
    """A call forward and backward like the 64-bit form.  Counts of 32-bit roundings: 40 T for a decay over T steps, 64 + N for the
    functions and the sum over states, D and B T for the sums over channels and steps."""
    plain = {n: v.detach().clone() for n, v in t.items()}
    req(*t.values())
    out, hT = call_scan(t, lengths=lengths, return_state=True, **k)
    got = dict(grads(t, out, hT, dout, dhT), out=out, hT=hT)
    want = R.scan(**plain, lengths=lengths, dout=dout, dhT=dhT, **k)
    size = R.scan(**plain, lengths=lengths, dout=dout, dhT=dhT, mag=True, **k)
    B, T, D = t["u"].shape
    for n in names or got:
        like(got[n], want[n], size[n], 2 * (40 * T + 64 + t["A"].shape[1]) + D + B * T, n)
    return got, want


@pytest.mark.parametrize("type", [FP, BF])
@pytest.mark.parametrize("N", [1, 3, 6, 11, 16, 17, 33, 40])
def test_scan_infinities_with_any_number_of_states(N, type):
    """An infinite u, delta or dy: the infinities of the definition, also where N does not fill the lanes' states."""
    B, T, D = 2, 64, 6
    dhT = rnd(31, B, D, N)
    for where in ("u", "dt", "dout"):
        t, dout = scan_case(B, T, D, N, type=type, positive=True), rnd(30, B, T, D, type=type)
        if where == "dout":
            dout[0, 40, 1], dout[1, 9, 2] = INF, -INF
        else:
            t[where][0, 37, 1] = INF
            t[where][1, 5, 2] = INF if where == "dt" else -INF
        scan_like(t, dout, dhT)
    t = scan_case(B, T, D, N, type=type, positive=True)
    t["u"][0, 37, 1] = INF
    t["z"] = None
    y, h = call_scan(t, return_state=True)
    assert (y[0, 37:, 1] == INF).all() and (h[0, 1] == INF).all()


@pytest.mark.parametrize("N", [1, 3, 6, 11, 16, 17, 33])
def test_scan_step_infinities_with_any_number_of_states(N):
    from timeband_amd import ops
    t = scan_case(3, 1, 10, N, positive=True)
    t["u"][0, 0, 4], t["dt"][1, 0, 7] = INF, INF
    want, state = R.scan(**t), t["h0"].clone()
    out = ops.selective_scan_step(state, *(t[k][:, 0] if k != "A" else t[k] for k in ("u", "dt", "A", "Bm", "Cm")), D=t["D"], z=t["z"][:, 0], dt_bias=t["bias"])
    size = R.scan(**t, mag=True)
    like(out, want["out"][:, 0], size["out"][:, 0], 104 + N, "out")
    like(state, want["hT"], size["hT"], 104, "state")


@pytest.mark.parametrize("N", [4, 11])
def test_scan_infinities_without_the_skip_term(N):
    """No D: neither u nor dy is multiplied by a 0 in its place, and with positive B and C an infinite u gives infinite outputs, an
    infinite dy infinite du, not NaN."""
    B, T, D = 1, 40, 5
    t = scan_case(B, T, D, N, positive=True)
    del t["D"]
    t["u"][0, 20, 1] = INF
    t["z"] = t["z"].abs() + 0.1
    req(*t.values())
    out, hT = call_scan(t, return_state=True)
    dout = rnd(30, B, T, D)
    clean = torch.autograd.grad(out, t["u"], dout, retain_graph=True)[0]
    assert (out[0, 20:, 1] == INF).all() and torch.isfinite(out[0, :20]).all() and torch.isfinite(out[0, :, [0, 2, 3, 4]]).all()
    du, dz = torch.autograd.grad(out, (t["u"], t["z"]), dout.index_put((torch.tensor(0), torch.tensor(30), torch.tensor(2)), torch.tensor(INF, device="cuda")))
    assert (du[0, :31, 2] == INF).all() and torch.equal(du[0, 31:, 2], clean[0, 31:, 2]) and torch.equal(du[..., [0, 1, 3, 4]], clean[..., [0, 1, 3, 4]])
    assert torch.equal(dz[0, 20:, 1], INF * torch.sign(dout[0, 20:, 1]))


@pytest.mark.parametrize("type", [FP, BF])
@pytest.mark.parametrize("N,T,lengths", [(4, 50, None), (16, 40, [40, 33]), (11, 300, [258, 300]), (40, 9, [1, 9]), (16, 70, [0, 70])])
def test_scan_infinite_last_state_leaves_dA_alone(N, T, lengths, type):
    """An infinite u at a sequence's last step makes its end state infinite.  dA has no part of that state, and the steps that fill the
    walk's last tile, or lie behind `lengths`, must not add 0 times it."""
    B, D = 2, 6
    t, dout, dhT = scan_case(B, T, D, N, type=type, positive=True), rnd(30, B, T, D, type=type), rnd(31, B, D, N)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ends = lengths or [T] * B
    for b, n in enumerate(ends):
        if n:
            t["u"][b, n - 1, 1 + b] = INF
        else:
            t["h0"][b, 3, :] = INF
    scan_like(t, dout, dhT, lengths=ln)
    t = scan_case(B, T, D, N, type=type, positive=True)
    for b, n in enumerate(ends):
        if n:
            t["u"][b, n - 1, 1 + b] = INF
    req(*t.values())
    out, hT = call_scan(t, lengths=ln, return_state=True)
    assert torch.isfinite(torch.autograd.grad(out, t["A"], dout)[0]).all()


@pytest.mark.parametrize("N", [4, 11, 16])
def test_scan_states_past_the_range_of_a_chunk_s_decay(N):
    """Walks that are cut: states that grow by more than fp32's range over a chunk but start small enough, or at 0; and an infinite
    state that decays by more than its range.  Step by step none of them leaves the range (or infinity)."""
    B, D = 1, 4
    big = 3.4e38
    for T, step, A0, h0 in ((36, 2.9, 1.0, 1e-30), (300, 2.9, 1.0, 0.0), (36, 2.9, 1.0, -1e-32), (300, 3.0, -1.0, INF), (300, 0.01, -1.0, INF)):
        t = dict(u=torch.zeros(B, T, D, device="cuda"), dt=torch.full((B, T, D), step, device="cuda"), A=torch.full((D, N), A0, device="cuda"),
                 Bm=rnd(1, B, T, 1, N).abs(), Cm=rnd(2, B, T, 1, N).abs() + 0.1, h0=torch.full((B, D, N), h0, device="cuda"))
        out, hT = call_scan(t, softplus=False, return_state=True)
        want = R.scan(**t, softplus=False)
        assert h0 == INF or (float(want["hT"].abs().max()) < big and float(want["out"].abs().max()) < big)
        n = 40 * T + 64 + N
        like(out, want["out"], want["out"].abs(), n, "out")
        like(hT, want["hT"], want["hT"].abs(), n, "hT")
        # backward: the state's gradient runs the same way from the end
        t = {k: v.detach().clone() for k, v in t.items()}
        t["u"] = rnd(3, B, T, D) * 1e-30
        t["h0"] = torch.zeros_like(t["h0"])
        dhT = torch.full((B, D, N), h0, device="cuda")
        plain = {k: v.clone() for k, v in t.items()}
        req(*t.values())
        out, hT = call_scan(t, softplus=False, return_state=True)
        dh0, = torch.autograd.grad((out, hT), t["h0"], (torch.zeros_like(out), dhT))
        want = R.scan(**plain, softplus=False, dout=torch.zeros(B, T, D), dhT=dhT)["dh0"]
        like(dh0, want, want.abs(), 2 * n, "dh0")


# ---- convolution -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", [FP, BF])
@pytest.mark.parametrize("T,lengths,at", [(40, None, 6), (40, None, 39), (23, [23, 17], 16), (5, [4, 5], 3)])
def test_conv_infinite_x_in_dw(T, lengths, at, type):
    """An infinite x makes the taps' gradients infinite, by the signs of dy, not NaN: steps that do not count, or that belong to
    another run of steps, must not add 0 times it."""
    from timeband_amd import ops
    B, D, K = 2, 16, 4
    x, w, dy = rnd(1, B, T, D, type=type), rnd(2, D, K, type=type), rnd(3, B, T, D, type=type).abs() + 0.1
    x[:, at, 3], x[:, at, 5] = INF, -INF
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    req(x, w)
    y = ops.causal_conv(x, w, None, ops.ACT_NONE, lengths=ln)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want, size = R.conv(x, w, None, 0, lengths=ln, dy=dy), R.conv(x, w, None, 0, lengths=ln, dy=dy, mag=True)
    assert torch.isinf(want[3]).any()
    like(y, want[0], size[0], K + 32, "y")
    like(dx, want[2], size[2], K + 48, "dx")
    like(dw, want[3], size[3], B * T + 48, "dw")


@pytest.mark.parametrize("type", [FP, BF])
@pytest.mark.parametrize("B,T,D,K,run", [(6, 4100, 512, 4, 12), (2, 9001, 2063, 3, 32), (4, 8200, 2064, 4, 64)])
def test_conv_in_long_runs(B, T, D, K, run, type):
    """Enough steps and channels for runs of more than eight steps, which do not divide T: some channels against the formula."""
    from timeband_amd import ops
    assert T % run and min(64, (B * T * ((D + 3) // 4)) >> 18) // 4 * 4 == run
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(B, T, D, device="cuda", generator=g).to(type) for _ in range(2))
    w, b = rnd(2, D, K, type=type, scale=0.5), rnd(3, D, type=type, scale=0.3)
    ln = torch.tensor([T, T - run - 1, 5, T - 1][:B], dtype=torch.int32, device="cuda")
    if B > 4:
        ln = torch.tensor([T, T - run - 1, 5, T - 1, 0, T // 2], dtype=torch.int32, device="cuda")
    req(x, w, b)
    y = ops.causal_conv(x, w, b, ops.ACT_SILU, lengths=ln)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    c = [0, 1, 3, 4, 7, D // 2, D - 5, D - 4, D - 1]
    part = [v.detach()[..., c] for v in (x, dy)] + [w.detach()[c], b.detach()[c]]
    want, size = (R.conv(part[0], part[2], part[3], 4, None, ln, part[1], mag=m) for m in (False, True))
    # |pre| < 8 puts K + 32 roundings on y and K + 48 on dx, as for short ones; a thread sums its run, a block 4 to 64 runs, and
    # sixteen threads the blocks: fewer than B T additions in a row
    near(y[..., c], want[0], size[0], K + 32, "y")
    near(dx[..., c], want[2], size[2], K + 48, "dx")
    near(dw[c], want[3], size[3], B * T + 48, "dw")
    near(db[c], want[4], size[4], B * T + 48, "db")


# ---- scan: walks of many tiles ---------------------------------------------------------------------------------------------------
LONG = [  # B, T, G, channels a group, N, lengths: by the number of channel blocks B G the steps are cut into
    (32, 70, 12, 2, 16, False),      # 384 blocks: one walk of several tiles
    (32, 200, 12, 8, 4, True),       # the same, aligned, states of 32 steps a tile
    (32, 333, 12, 1, 32, False),     # tiles of eight steps
    (33, 130, 12, 2, 64, True),
    (10, 300, 8, 3, 16, True),       # 80 blocks: chunks of 128 steps, the last of 44
    (10, 300, 8, 8, 11, False),
    (16, 1000, 10, 2, 8, True),      # 160 blocks: six chunks of 192 and less
    (16, 1000, 10, 1, 16, False),
    (12, 385, 8, 70, 16, False),     # two channel blocks a group, the second of six channels
]


@pytest.mark.parametrize("type", [FP, BF, HF])
@pytest.mark.parametrize("B,T,G,C,N,ragged", LONG)
def test_scan_gradients_over_many_tiles(B, T, G, C, N, ragged, type):
    t, dout, dhT = scan_case(B, T, G * C, N, G=G, type=type), rnd(30, B, T, G * C, type=type), rnd(31, B, G * C, N)
    ln = None
    if ragged:
        ln = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
        ln[0], ln[1], ln[2] = T, 0, 129
        ln = ln.cuda()
    got, want = scan_like(t, dout, dhT, lengths=ln)
    if type != FP:      # the counts allow 40 T roundings of sums that mostly decay; their norm is far below the type's own step
        for k in ("out", "du", "ddt", "dz", "dB", "dC"):
            if want[k].numel() >= 25000:
                rounded_once(got[k], want[k], k)


# ---- linear: every branch of the backward pass ---------------------------------------------------------------------------------
def linear_like(M, K, N, kind, type, need="xWbr", seed=1):
    from timeband_amd import ops
    x, W, b, res = rnd(seed, M, K, type=type), rnd(seed + 1, N, K, type=type, scale=K ** -0.5), rnd(seed + 2, N, type=type), rnd(seed + 3, M, N, type=type)
    dy = rnd(seed + 4, M, N, type=type)
    if kind == 3:                      # where z is within its rounding errors of 0, dy is 0: relu's derivative does not count there
        z, size = R.linear(x, W, b, 0), R.linear(x, W, b, 0, mag=True)
        close = z.abs() <= (K + 4) * R.U * size
        assert close.float().mean() < 0.01
        dy[close.cuda()] = 0
    leaves = dict(zip("xWbr", (x, W, b, res)))
    req(*(leaves[k] for k in need))
    y = ops.linear_residual(x, W, b, kind, residual=res)
    got = dict(zip(need, torch.autograd.grad(y, [leaves[k] for k in need], dy)))
    want, size = R.linear(x, W, b, kind, res, dy), R.linear(x, W, b, kind, res, dy, mag=True)
    near(y, want[0], size[0], K + 64, "y")
    # dz in two parts of 16 bits: within 2^-16 (bf16) of itself, 2^8 roundings of 32 bits, and twice the sums
    two = 0 if type == FP or kind in (0, 3) else 256
    for k, steps, name in (("x", 2 * N + K, "dx"), ("W", 2 * M + K, "dW"), ("b", M + K, "db")):
        if k in need:
            near(got[k], want["xWb".index(k) + 1], size["xWb".index(k) + 1], steps + 64 + two, name)
    if "r" in need:
        assert torch.equal(got["r"], dy)


@pytest.mark.parametrize("type", [FP, BF, HF])
@pytest.mark.parametrize("M,K,N", [(2049, 24, 132), (129, 72, 127), (33, 16, 16), (7, 40, 30), (300, 88, 1100)])
def test_linear_relu_gradients(M, K, N, type):
    linear_like(M, K, N, 3, type)


@pytest.mark.parametrize("type", [FP, BF, HF])
@pytest.mark.parametrize("kind", [0, 4])
@pytest.mark.parametrize("M,K,N", [
    (65500, 200, 40),        # dx in 256 x 256 tiles, dW in a launch of its own (fp32: from x as it lies)
    (65500, 201, 36),        # the same with rows off 16 bytes
    (100, 4099, 4000),       # dW in 256 x 256 tiles
    (100, 72, 2056),         # dx split over k
    (100, 72, 2051),
    (5000, 72, 90),          # dW split over k
])
def test_linear_backward_branches(M, K, N, kind, type):
    linear_like(M, K, N, kind, type)


@pytest.mark.parametrize("type", [FP, BF, HF])
@pytest.mark.parametrize("kind", [0, 5])
@pytest.mark.parametrize("need", ["x", "W", "b", "r", "xb", "Wb", "xr", "xW"])
def test_linear_some_gradients(need, kind, type):
    for M, K, N in ((150, 72, 136), (150, 75, 131), (20, 72, 1100)):
        linear_like(M, K, N, kind, type, need)


def test_linear_activations_to_their_stated_precision():
    """One input and a weight of 1: z is x itself.  fp32, relative: tanh 2^-20, sigmoid and SiLU |z| + 4 roundings (the exponent's, the
    exponential's, the sum's and the reciprocal's), GELU 2^-20 + 2.5 z^2 2^-24 below 0 and 2^-20 above."""
    from timeband_amd import ops
    one = torch.ones(1, 1, device="cuda")
    for lo, hi in ((1e-6, 0.3), (0.3, 3), (3, 13)):
        for sign in (1, -1):
            z = (torch.linspace(lo, hi, 500009) * sign).cuda()[:, None]
            z64 = z.double().cpu()
            allowed = {1: 2.0 ** -20 + 0 * z64, 2: (z64.abs() + 4) * 2 * R.U, 4: (z64.abs() + 5) * 2 * R.U,
                       5: 2.0 ** -20 + 2.5 * R.U * z64.clamp(max=0) ** 2}
            for kind, tol in allowed.items():
                got, want = ops.linear_residual(z, one, None, kind).double().cpu(), R.act(z64, kind)[0]
                off = ((got - want) / want).abs() / tol
                assert float(off.max()) <= 1, (kind, float(z[int(off.argmax())]), float(off.max()))


def test_linear_takes_the_memory_that_it_uses():
    """Aligned operands are read in place: a call's peak is its outputs and what it lays out."""
    from timeband_amd import ops
    MB = 1 << 20

    def peak(f):
        f()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        r = f()
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before

    x, W = rnd(1, 8192, 1024, type=BF), rnd(2, 2048, 1024, type=BF)
    assert peak(lambda: ops.linear_residual(x, W)) <= 32 * MB + MB
    x, W, dy = rnd(1, 32768, 256), rnd(2, 256, 256), rnd(3, 32768, 256)
    req(x, W)
    y = ops.linear_residual(x, W)
    # dx (32 MB), dW, W across, dW's split sums (up to 64 of 1/4 MB); dy and x as they lie
    assert peak(lambda: torch.autograd.grad(y, (x, W), dy, retain_graph=True)) <= 50 * MB
