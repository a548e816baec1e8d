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
def test_embedding_refusals(lib):
    def fwd(dt=0, tokens=64, w=64, n=4, d=8, v=5, scale=1.0, out=64):
        return lib.kans_embedding_forward(dt, tokens, w, n, d, v, -100, scale, out, None)

    def bwd(tokens=64, dout=64, n=4, dw=64, ws=64, size=1 << 20):
        return lib.kans_embedding_backward(0, tokens, dout, n, 8, 5, -100, 1.0, dw, ws, size, None)
    for bad in (dict(dt=3), dict(tokens=None), dict(w=None), dict(out=None), dict(n=-1), dict(d=0), dict(v=0),
                dict(scale=float("inf"))):
        assert fwd(**bad) == -1, bad
    for bad in (dict(n=(1 << 23) + 1), dict(d=(1 << 16) + 1), dict(v=(1 << 24) + 1)):
        assert fwd(**bad) == -5, bad
    assert fwd(n=0, tokens=None) == 0
    for bad in (dict(tokens=None), dict(dout=None), dict(dw=None), dict(ws=None), dict(ws=72), dict(size=16), dict(n=-1)):
        assert bwd(**bad) == -1, bad
    assert lib.kans_embedding_workspace(0, -1, 8, 5) == -1
    assert lib.kans_embedding_workspace(0, 4, 8, 1 << 25) == -5
    assert lib.kans_embedding_workspace(0, 4, 8, 5) >= 4 * (2 * 4 + 5 + 1)


def test_dropout_refusals(lib):
    def go(dt=0, x=64, y=64, n=4, p=0.5):
        return lib.kans_dropout(dt, x, y, n, p, 1, None, None, 0, None)
    for bad in (dict(dt=3), dict(x=None), dict(y=None), dict(n=-1), dict(p=-0.1), dict(p=1.1), dict(p=float("nan"))):
        assert go(**bad) == -1, bad
    assert go(n=1 << 34) == -5


def test_causal_conv_refusals(lib):
    def fwd(dt=0, x=64, w=64, y=64, b=2, n=5, d=4, taps=3):
        return lib.kans_causal_conv_forward(dt, x, 20, 4, w, None, None, None, 1, y, b, n, d, taps, None)

    def bwd(x=64, dy=64, bias=None, dbias=None, ws=64, size=1 << 20):
        return lib.kans_causal_conv_backward(0, x, 20, 4, 64, bias, None, 1, dy, 64, 64, dbias, 2, 5, 4, 3, ws, size, None)
    for bad in (dict(dt=3), dict(x=None), dict(w=None), dict(y=None), dict(b=-1), dict(n=-1), dict(d=0)):
        assert fwd(**bad) == -1, bad
    for bad in (dict(taps=0), dict(taps=9), dict(b=1 << 15, n=1 << 25), dict(n=(1 << 30) + 1)):
        assert fwd(**bad) == -5, bad
    assert fwd(b=0, x=None) == 0 and fwd(n=0, x=None) == 0
    for bad in (dict(x=None), dict(dy=None), dict(dbias=64), dict(ws=None), dict(ws=72), dict(size=16)):
        assert bwd(**bad) == -1, bad
    assert lib.kans_causal_conv_workspace(0, 2, 5, 4, 9) == -5
    assert lib.kans_causal_conv_workspace(0, 2, 5, 4, 3) >= 2 * 4 * 4 * 4


def test_selective_scan_refusals(lib):
    def fwd(dt=0, x=64, A=64, bm=64, out=64, state=None, b=2, n=5, d=4, states=16, ws=64, size=1 << 24):
        return lib.kans_selective_scan_forward(dt, x, 20, 4, 64, 20, 4, A, bm, 80, 16, 64, 80, 16, None, None, 0, 0, None, 1, state, None,
                                               out, None, b, n, d, states, ws, size, None)

    def bwd(saved=64, z=None, dz=None, skip=None, dskip=None, dbias=None, ws=64, size=1 << 24, dx=64):
        return lib.kans_selective_scan_backward(0, 64, 20, 4, 64, 20, 4, 64, 64, 80, 16, 64, 80, 16, skip, z, 20, 4, None, 1, None, saved,
                                                64, dx, 64, 64, 64, 64, dskip, dz, dbias, 2, 5, 4, 16, ws, size, None)
    for bad in (dict(dt=3), dict(x=None), dict(A=None), dict(bm=None), dict(out=None), dict(b=-1), dict(n=-1),
                dict(d=0), dict(states=0), dict(n=300, ws=None), dict(n=300, ws=72), dict(n=300, size=16)):
        assert fwd(**bad) == -1, bad
    for bad in (dict(states=65), dict(b=1 << 22), dict(n=(1 << 30) + 1), dict(b=1 << 21, n=1 << 20)):
        assert fwd(**bad) == -5, bad
    assert fwd(b=0, x=None) == 0 and fwd(n=0, x=None) == 0
    for bad in (dict(saved=None), dict(z=64), dict(dz=64), dict(dskip=64), dict(dbias=64), dict(ws=None), dict(ws=72), dict(size=16),
                dict(dx=None)):
        assert bwd(**bad) == -1, bad
    assert lib.kans_selective_scan_workspace(2, 5, 4, 65, 0) == -5 and lib.kans_selective_scan_saved(2, 5, 4, 65) == -5
    assert lib.kans_selective_scan_workspace(2, 5, 4, 16, 0) == 0
    assert lib.kans_selective_scan_workspace(1, 700, 4, 16, 0) > 0
    assert lib.kans_selective_scan_saved(2, 17, 4, 16) == 2 * 2 * 4 * 16 * 4


def test_grids_end_below_2_32_threads(lib):
    """Sizes whose launches would have 2^32 threads or more are refused before anything is launched."""
    assert lib.kans_dropout(0, 64, 64, (1 << 34) - 1023, 0.5, 1, None, None, 0, None) == -5
    for d in ((1 << 27) + 1, 1 << 28):
        assert lib.kans_causal_conv_workspace(0, 1, 1, d, 4) == -5 and lib.kans_causal_conv_workspace(0, 0, 0, d, 4) == -5
    for b, n in ((1, 1), (1, 0), (0, 5)):
        assert lib.kans_selective_scan_workspace(b, n, 1 << 23, 64, 1) == -5


def test_scan_refuses_steps_in_each_others_memory(lib):
    def rows(x=4, dt=4, b=16, c=16, z=4, n=300):   # (more than one step without a workspace: nothing is launched)
        return lib.kans_selective_scan_forward(0, 64, 20, x, 64, 20, dt, 64, 64, 80, b, 64, 80, c, None, 64, 20, z, None, 1, None, None, 64,
                                               None, 2, n, 4, 16, None, 0, None)

    def back(x=4, b=16):
        return lib.kans_selective_scan_backward(0, 64, 20, x, 64, 20, 4, 64, 64, 80, b, 64, 80, 16, None, None, 0, 0, None, 1, None, 64, 64, 64,
                                                64, 64, 64, 64, None, None, None, 2, 300, 4, 16, None, 0, None)
    for good in (dict(), dict(x=0, b=0), dict(x=5, dt=9, z=100, b=17, c=(1 << 23) - 1)):
        assert rows(**good) == -1, good
    assert back() == -1 and back(x=0, b=0) == -1
    for bad in (dict(x=1), dict(x=3), dict(dt=3), dict(b=15), dict(c=1), dict(z=2), dict(c=1 << 23)):
        assert rows(**bad) == -5, bad
    assert back(x=3) == -5 and back(b=15) == -5


def test_conv_sizes_whose_product_passes_64_bits(lib):
    """Threads counted modulo 2^64 would be few, or none."""
    for b, l, d in ((1 << 24, 1 << 30, 1 << 18), (1 << 22, 1 << 27, 1 << 26), ((1 << 31) - 1, 1 << 30, 1 << 27), (1 << 30, 1 << 30, 1 << 20),
                    ((1 << 31) - 1, 1, 1 << 20), (1 << 20, 1 << 30, 4)):
        for dt in (0, 1, 2):
            assert lib.kans_causal_conv_workspace(dt, b, l, d, 4) == -5, (b, l, d)
            assert lib.kans_causal_conv_forward(dt, 64, 0, 0, 64, None, None, None, 1, 64, b, l, d, 4, None) == -5
            assert lib.kans_causal_conv_backward(dt, 64, 0, 0, 64, None, None, 1, 64, 64, 64, None, b, l, d, 4, 64, 1 << 62, None) == -5
    assert lib.kans_causal_conv_workspace(0, (1 << 31) - 1, 0, 1 << 27, 4) == 0    # (no steps, no work)
    # the largest that are taken, and the first beyond: 2^31 threads, of 4 channels and up to 64 steps
    assert lib.kans_causal_conv_workspace(0, 32, 1 << 30, 4, 4) > 0 and lib.kans_causal_conv_workspace(0, 127, 1 << 30, 4, 4) > 0
    assert lib.kans_causal_conv_workspace(0, 128, 1 << 30, 4, 4) == -5
    assert lib.kans_causal_conv_workspace(0, (1 << 31) - 1, 1, 4, 4) > 0
    assert lib.kans_causal_conv_workspace(0, (1 << 31) - 1, 1, 8, 4) == -5


def test_embedding_scales(lib):
    """Scales that fp32 holds with all their digits, and zero."""
    for dt in (0, 1, 2):
        for scale, code in ((0.0, 0), (-0.0, 0), (2.0 ** -126, 0), (-3.4e38, 0), (1e-40, -1), (-1e-300, -1), (3.5e38, -1), (1e300, -1),
                            (float("nan"), -1), (float("-inf"), -1)):
            assert lib.kans_embedding_forward(dt, None, 64, 0, 8, 5, -100, scale, 64, None) == code, scale
            assert lib.kans_embedding_backward(dt, 64, 64, 4, 8, 5, -100, scale, 64, None, 0, None) == -1
