"""Refusals of the training-step entry points that need no GPU: negative codes before any HIP call."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from metal_kans import device
    return device.load_library()


def adamw(lib, **kw):
    a = dict(dtype=0, bits=32, n=1, params=None, grads=None, numel=4, block=0, step=1, m=64, v=64, ms=None, vs=None,
             master=None, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0)
    a.update(kw)
    V, L = ctypes.c_void_p, ctypes.c_long
    one = lambda t, v: ctypes.cast((t * 1)(v), V)  # noqa: E731
    return lib.kans_adamw_step(a["dtype"], a["bits"], a["n"], one(V, a["params"] or 0), one(V, a["grads"] or 0),
                               one(L, a["numel"]), one(L, a["block"]), one(L, a["step"]), a["m"], a["v"], a["ms"], a["vs"],
                               a["master"], a["lr"], a["b1"], a["b2"], a["eps"], a["wd"], None)


def test_adamw_refusals(lib):
    ok = dict(params=64, grads=64)
    for bad in (dict(), dict(ok, dtype=3), dict(ok, bits=16), dict(ok, n=-1), dict(ok, numel=-1), dict(ok, block=-1),
                dict(ok, step=0), dict(ok, m=None), dict(ok, m=65), dict(ok, bits=8), dict(ok, dtype=1),
                dict(ok, lr=-1.0), dict(ok, lr=float("nan")), dict(ok, b1=1.0), dict(ok, b2=-0.1),
                dict(ok, eps=float("inf")), dict(ok, wd=-1.0)):
        assert adamw(lib, **bad) == -1, bad
        assert lib.kans_last_error()
    assert adamw(lib, **ok, numel=1 << 40) == -5
    assert adamw(lib, numel=0, m=None, v=None) == 0
    assert adamw(lib, n=0) == 0
    assert lib.kans_adamw_values(None, None, None, None, None, None, 1, None) == -1
    assert lib.kans_adamw_values(64, 64, 64, 64, 72, 64, 1, None) == -1
    assert lib.kans_adamw_values(None, None, None, None, None, None, 0, None) == 0


def test_residual_norm_refusals(lib):
    def fwd(res=0, dt=0, kind=0, x=64, block=64, gate=None, group=4, post=None, eps=1e-6, y=64, h=64, rows=4, d=8):
        return lib.kans_residual_norm_forward(res, dt, kind, x, block, gate, group, post, None, None, 1.0, eps, y, h, None,
                                              rows, d, None)

    def bwd(stats=64, gate=None, dgate=None, f32=0, ws=64, size=1 << 20, block=64, dblock=None):
        return lib.kans_residual_norm_backward(0, 0, 0, 64, block, gate, 4, None, None, None, 1.0, 1e-6, stats, 64, 64, 64, dblock,
                                               dgate, f32, None, None, None, 4, 8, ws, size, None)
    for bad in (dict(res=1), dict(dt=3), dict(res=3), dict(res=2, dt=1), dict(kind=2), dict(x=None), dict(block=None, gate=64),
                dict(block=None, post=64), dict(eps=-1.0), dict(eps=float("nan")), dict(y=None), dict(h=None), dict(rows=-1),
                dict(d=0), dict(gate=64, group=3), dict(gate=64, group=0), dict(gate=64, group=8)):
        assert fwd(**bad) == -1, bad
    assert fwd(rows=1 << 22) == -5
    assert fwd(rows=0, x=None) == 0
    for bad in (dict(stats=None), dict(dgate=64), dict(ws=None), dict(size=8), dict(block=None, dblock=64),
                dict(gate=64, dgate=64, f32=1)):
        assert bwd(**bad) == -1, bad
    assert lib.kans_residual_norm_workspace(0, 8, 0) == 0
    assert lib.kans_residual_norm_workspace(4, 8, 0) >= 4 * (3 * 8 + 1)


def test_linear_xent_refusals(lib):
    def fwd(dt=0, h=64, w=64, t=64, n=4, d=8, v=10, red=1, loss=64, state=64, ws=64, size=1 << 40):
        return lib.kans_linear_xent_forward(dt, h, w, t, n, d, v, -100, red, loss, state, ws, size, None)

    def bwd(grad=64, dh=64, ws=64, size=1 << 40, n=4):
        return lib.kans_linear_xent_backward(0, 64, 64, 64, n, 8, 10, -100, 1, 64, grad, dh, None, ws, size, None)
    for bad in (dict(dt=3), dict(h=None), dict(w=None), dict(t=None), dict(t=68), dict(n=-1), dict(d=0), dict(v=0), dict(red=3),
                dict(loss=None), dict(state=None), dict(state=66), dict(ws=None), dict(ws=72), dict(size=8)):
        assert fwd(**bad) == -1, bad
    for big in (dict(n=(1 << 22) + 1), dict(d=(1 << 16) + 1), dict(v=(1 << 24) + 1)):
        assert fwd(**big) == -5, big
    assert fwd(n=0) == 0 and bwd(n=0) == 0 and bwd(dh=None) == 0
    for bad in (dict(grad=None), dict(ws=None), dict(size=8)):
        assert bwd(**bad) == -1, bad
    assert lib.kans_linear_xent_workspace(0, 0, 8, 10, 1) == 0
    assert lib.kans_linear_xent_workspace(0, 4, 8, 1 << 25, 1) == -5
    assert lib.kans_linear_xent_workspace(3, 4, 8, 10, 1) == -1
    # no more than a piece of the vocabulary is ever held: below the logits' size
    assert lib.kans_linear_xent_workspace(2, 16384, 4096, 131072, 0) < 16384 * 131072


@pytest.mark.parametrize("d", [64, 4096, 10000])
def test_residual_norm_workspace_of_short_groups(lib, d):
    """Gate groups of few rows need no more partial sums than runs of rows without a gate (and less than twice x)."""
    for rows in (24, 1024, 16384, 1 << 20):
        plain = lib.kans_residual_norm_workspace(rows, d, 0)
        for group in range(1, 65):
            if rows % group == 0 or rows > 1000:
                n = rows // group * group
                assert lib.kans_residual_norm_workspace(n, d, group) <= 2 * plain + 16 * d, (rows, group)


def test_linear_xent_workspace_of_a_reduced_loss(lib):
    """Only a loss of each row may need a second G (fp16): the others' backward takes no more than it did."""
    def bwd(red, size):
        return lib.kans_linear_xent_backward(1, 64, 64, 64, 3001, 777, 50021, -100, red, 64, 64, 64, None, 64, size, None)
    forward, rows, reduced = (lib.kans_linear_xent_workspace(1, 3001, 777, 50021, b) for b in (0, 1, 2))
    g = 3072 * 50176 * 2
    assert forward < reduced and g < reduced < 2 * g and rows >= reduced + g
    for dt in (0, 2):
        assert lib.kans_linear_xent_workspace(dt, 3001, 777, 50021, 1) == lib.kans_linear_xent_workspace(dt, 3001, 777, 50021, 2)
    assert bwd(0, reduced) == -1 and bwd(1, reduced - 1) == -1 and bwd(2, reduced - 1) == -1
