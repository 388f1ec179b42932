"""CPU: what the state space layer's operators refuse before they look at a tensor's device."""
import pytest
import torch
from torch.autograd import forward_ad


def forward_mode_calls(device):
    """(name, call of one dual tensor, that tensor's primal) for every tensor of every operator."""
    from timeband_amd import ops
    z = lambda *s: torch.zeros(s, device=device)
    calls = {
        "causal_conv": (ops.causal_conv, dict(x=z(2, 5, 8), weight=z(8, 4), bias=z(8), state=z(2, 3, 8))),
        "causal_conv_step": (ops.causal_conv_step, dict(x=z(2, 8), state=z(2, 3, 8), weight=z(8, 4), bias=z(8))),
        "selective_scan": (ops.selective_scan, dict(u=z(2, 5, 8), dt=z(2, 5, 8), A=z(8, 4), B=z(2, 5, 4), C=z(2, 5, 4), D=z(8), z=z(2, 5, 8),
                                                    dt_bias=z(8), h0=z(2, 8, 4))),
        "selective_scan_step": (ops.selective_scan_step, dict(state=z(2, 8, 4), u=z(2, 8), dt=z(2, 8), A=z(8, 4), B=z(2, 4), C=z(2, 4), D=z(8),
                                                              z=z(2, 8), dt_bias=z(8))),
        "linear_residual": (ops.linear_residual, dict(x=z(40, 8), W=z(6, 8), b=z(6), residual=z(40, 6))),
    }
    for name, (f, args) in calls.items():
        for k in args:
            yield name, (lambda t, f=f, args=args, k=k: f(**{**args, k: t})), args[k]


def check_forward_mode_is_refused(device):
    for name, call, primal in forward_mode_calls(device):
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match=name + ": forward-mode"):
                call(forward_ad.make_dual(primal, torch.ones_like(primal)))


def test_forward_mode_is_refused():
    """Without the refusal the result has no tangent, and x + f(x) would have that of x alone."""
    check_forward_mode_is_refused("cpu")


def test_linear_refuses_more_tiles_than_a_launch():
    """Tiles of a product that one launch cannot hold (their count would wrap): refused (3) before anything is launched."""
    from timeband_amd import _lib
    lib = _lib.load()
    p, wide = 4096, 1 << 62
    lin = lambda M, K, N: lib.tb_linres_fwd(p, K, p, K, 0, 0, 0, p, 0, M, K, N, 0, 1, p, wide, 0)
    back = lambda M, K, N: lib.tb_linres_bwd(p, N, p, K, p, K, 0, 0, p, p, p, M, K, N, 1, p, wide, 0)
    assert lin(10 ** 9, 8, 4 * 10 ** 6) == 3 and back(10 ** 9, 8, 4 * 10 ** 6) == 3 and back(10 ** 9, 4 * 10 ** 6, 8) == 3
    assert back(100, 4 * 10 ** 6, 4 * 10 ** 6) == 3


def test_linear_workspaces_hold_what_a_call_lays_out():
    """The size for given operands: never above the size for any operands, next to nothing where all are read in place, and checked."""
    import itertools
    from timeband_amd import _lib
    lib = _lib.load()
    fwd, bwd, any_ = lib.tb_linres_fwd_workspace_bytes, lib.tb_linres_bwd_workspace_bytes, lib.tb_linres_workspace_bytes
    sizes = [(1, 8, 16), (32, 8, 16), (33, 16, 16), (100, 72, 2056), (100, 75, 2051), (4099, 1000, 1500), (65536, 256, 256), (300, 4096, 40), (70000, 1030, 3)]
    for (M, K, N), dtype, at in itertools.product(sizes, (0, 1, 2), (4096, 4098)):
        assert fwd(at, K, at, K, M, K, N, dtype) <= any_(M, K, N, dtype, 0)
        for act, dx, dW, db in itertools.product((0, 3, 4), (0, 1), (0, 1), (0, 1)):
            assert bwd(at, N, at, K, act, dx, dW, db, M, K, N, dtype) <= any_(M, K, N, dtype, 1)
    p, slack = 4096, 4096
    assert fwd(p, 2048, p, 2048, 16384, 2048, 8192, 1) <= slack                                 # 16384 x 2048 x 8192 bf16, nothing copied
    assert bwd(p, 256, p, 256, 0, 1, 0, 0, 65536, 256, 256, 0) <= 256 * 256 * 4 + slack          # fp32 dx: W across
    assert bwd(p, 256, p, 256, 0, 0, 1, 0, 65536, 256, 256, 0) <= 65 * 256 * 256 * 4 + slack     # fp32 dW: its split sums
    one = bwd(p, 1024, p, 1024, 0, 1, 0, 0, 8192, 1024, 1024, 2)
    assert bwd(p, 1024, p, 1024, 3, 1, 0, 0, 8192, 1024, 1024, 2) == one + 8192 * 1024 * 2          # relu: dz in one part
    assert bwd(p, 1024, p, 1024, 4, 1, 0, 0, 8192, 1024, 1024, 2) == one + 2 * 8192 * 1024 * 2      # SiLU: in two
    need = fwd(4098, 75, p, 75, 100, 75, 2051, 1)
    assert lib.tb_linres_fwd(4098, 75, p, 75, 0, 0, 0, p, 0, 100, 75, 2051, 0, 1, p, need - 1, 0) == 4
    need = bwd(p, 2051, p, 75, 4, 1, 1, 1, 100, 75, 2051, 1)
    assert lib.tb_linres_bwd(p, 2051, p, 75, p, 75, p, 4, p, p, p, 100, 75, 2051, 1, p, need - 1, 0) == 4
