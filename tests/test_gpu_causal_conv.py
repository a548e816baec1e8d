"""causal_conv (run on an MI355X) against its definition in 64 bits.

Tolerances.  u = 2^-24 is one fp32 rounding, t one rounding to the result's type.  The sum before the activation has
W + 1 terms: off by (W + 2) u S, S the sum of the terms' magnitudes.  The sigmoid's exponential has an argument that is
itself rounded (|v| u) and three roundings more: off by (|v| + 6) u of its value.  silu's slope is at most 1.1, its second
derivative at most 0.5:
    y:  1.1 (W + 2) u S + (|v| + 6) u |y|
    du: |dy| (0.5 (W + 2) u S + (|v| + 8) u)                      =: E
    dx: sum |w| E + (W + 1) u sum |w du|,   dw: sum E |x| + k u sum |du x|,   dbias: sum E + k u sum |du|
with k the longest chain of additions: 64 steps of a tile, the tiles of all sequences in 16 runs, and these 16.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEP = {torch.float32: (2.0 ** -24, 2.0 ** -126), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -126)}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def cuda(gpu):
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    return torch.device("cuda:0")


def inputs(b, l, d, w, dt, seed=0, lengths=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dt)  # noqa: E731
    s = dict(x=rnd(b, l, d), weight=rnd(d, w), bias=rnd(d), dy=rnd(b, l, d), state=rnd(b, w - 1, d))
    s["lengths"] = None if lengths is None else torch.tensor(lengths, device="cuda")
    return s


def reference(s, activation, state=False):
    """Results and their bounds without the last rounding, by name."""
    x, w, dy = s["x"].double(), s["weight"].double(), s["dy"].double()
    b, l, d = x.shape
    W = w.shape[1]
    bias = torch.zeros(d, dtype=torch.float64, device="cuda") if s["bias"] is None else s["bias"].double()
    n = torch.full((b,), l, device="cuda") if s["lengths"] is None else s["lengths"].clamp(0, l)
    inside = (torch.arange(l, device="cuda") < n[:, None])[..., None]
    x, dy = torch.where(inside, x, 0.0), torch.where(inside, dy, 0.0)
    before = s["state"].double() if state else torch.zeros(b, W - 1, d, dtype=torch.float64, device="cuda")
    known = torch.cat((before, x), 1)
    v, S = bias.expand(b, l, d).clone(), bias.abs().expand(b, l, d).clone()
    for j in range(W):
        v += w[:, j] * known[:, j:j + l]
        S += (w[:, j] * known[:, j:j + l]).abs()
    sig = torch.sigmoid(v)
    silu = activation == "silu"
    y, g = (v * sig, sig * (1 + v * (1 - sig))) if silu else (v, torch.ones_like(v))
    y = torch.where(inside, y, 0.0)
    off = 1.1 * (W + 2) * U * S + (v.abs() + 6) * U * y.abs()
    R = {"y": (y, torch.where(inside, off, 0.0))}
    R["state"] = (torch.stack([known[i, int(k):int(k) + W - 1] for i, k in enumerate(n)]), torch.zeros((), device="cuda"))
    du = dy * g
    E = dy.abs() * (0.5 * (W + 2) * U * S + (v.abs() + 8) * U)
    dx, dxe = torch.zeros_like(known), torch.zeros_like(known)
    for j in range(W):
        dx[:, j:j + l] += w[:, j] * du
        dxe[:, j:j + l] += w[:, j].abs() * (E + (W + 1) * U * du.abs())
    R["dx"] = (torch.where(inside, dx[:, W - 1:], 0.0), dxe[:, W - 1:])
    k = 64 + b * (l / 8 + 1) / 16 + 20
    R["dweight"] = tuple(torch.stack([t[:, j:j + l].mul(m).sum((0, 1)) for j in range(W)], 1)
                         for t, m in ((known, du), (known.abs(), E + k * U * du.abs())))
    R["dbias"] = (du.sum((0, 1)), (E + k * U * du.abs()).sum((0, 1)))
    return R


def near(got, want, name, dt):
    value, off = want[name]
    t, least = STEP[dt]
    assert got.dtype == dt and got.shape == value.shape, name
    bound = t * value.abs() + off + least
    bad = (got.double() - value).abs() / bound
    assert bad.numel() == 0 or bad.max() <= 1, (name, bad.max().item())


def check(s, activation="silu"):
    import metal_kans as mk
    dt = s["x"].dtype
    leaves = [n for n in ("x", "weight", "bias") if s[n] is not None]
    a = {n: s[n].detach().requires_grad_(True) for n in leaves}
    y = mk.causal_conv(a["x"], a["weight"], a.get("bias"), activation=activation, lengths=s["lengths"])
    grads = dict(zip(leaves, torch.autograd.grad(y, [a[n] for n in leaves], s["dy"])))
    want = reference(s, activation)
    near(y.detach(), want, "y", dt)
    for n in leaves:
        near(grads[n], want, "d" + n, dt)
    # with a state, and with one of zeros
    state = s["state"].clone()
    with torch.no_grad():
        near(mk.causal_conv(s["x"], s["weight"], s["bias"], activation, state, s["lengths"]), reference(s, activation, True), "y", dt)
        assert torch.equal(state.double(), reference(s, activation, True)["state"][0])
        zero = torch.zeros_like(state)
        assert torch.equal(mk.causal_conv(s["x"], s["weight"], s["bias"], activation, zero, s["lengths"]), y)
    return y, grads


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,l,d,w", [(1, 1, 1, 1), (1, 1, 8, 4), (2, 3, 5, 4), (1, 2, 7, 8), (3, 65, 33, 2), (2, 130, 12, 3), (5, 17, 100, 4),
                                     (1, 700, 9, 5), (2, 64, 257, 4), (1, 9, 4, 6), (2, 40, 3, 7)])
def test_sizes(cuda, b, l, d, w, dt):
    check(inputs(b, l, d, w, dt))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lengths", [[0, 1, 2], [40, 33, 0], [-5, 1000, 39]])
@pytest.mark.parametrize("w", [1, 2, 4, 8])
def test_lengths(cuda, w, lengths, dt):
    check(inputs(3, 40, 21, w, dt, lengths=lengths))


@pytest.mark.parametrize("activation", ["silu", None])
@pytest.mark.parametrize("bias", [True, False])
def test_without(cuda, activation, bias):
    s = inputs(2, 70, 24, 4, torch.float32)
    if not bias:
        s["bias"] = None
    check(s, activation)


def test_tiles_and_channels_of_a_large_batch(cuda):
    """Tiles of 64 steps, several workgroups."""
    check(inputs(4, 1000, 520, 4, torch.bfloat16, lengths=[1000, 64, 999, 513]))


@pytest.mark.parametrize("dt", TYPES)
def test_masked_places_are_not_looked_at(cuda, dt):
    import metal_kans as mk
    s = inputs(3, 50, 19, 4, dt, lengths=[0, 20, 50])
    behind = (torch.arange(50, device="cuda") >= s["lengths"][:, None])[..., None]
    y, grads = check({**s, "x": torch.where(behind, 0.0, s["x"]), "dy": torch.where(behind, 0.0, s["dy"])})
    for bad in (float("nan"), float("inf"), torch.finfo(dt).min):
        x = torch.where(behind, bad, s["x"]).requires_grad_(True)
        got = mk.causal_conv(x, s["weight"], s["bias"], lengths=s["lengths"])
        assert torch.equal(got, y)
        dx, = torch.autograd.grad(got, x, torch.where(behind, bad, s["dy"]))
        assert torch.equal(dx, grads["x"])
        state, zero = s["state"].clone(), s["state"].clone()
        with torch.no_grad():
            mk.causal_conv(x, s["weight"], s["bias"], state=state, lengths=s["lengths"])
            mk.causal_conv(torch.where(behind, 0.0, s["x"]), s["weight"], s["bias"], state=zero, lengths=s["lengths"])
        assert torch.equal(state, zero) and torch.equal(state[0], s["state"][0])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_infinities_stay_where_they_belong(cuda, bad):
    """An input reaches the outputs of W steps of its channel, a gradient the inputs of W steps; sums only where a step that
    counts meets it."""
    import metal_kans as mk
    s = inputs(2, 200, 20, 4, torch.float32, lengths=[200, 130])
    y, grads = check(s, None)
    for t, d in ((63, 7), (64, 18), (129, 19)):
        x = s["x"].clone()
        x[1, t, d] = bad
        x.requires_grad_(True)
        w = s["weight"].detach().requires_grad_(True)
        got = mk.causal_conv(x, w, s["bias"], activation=None, lengths=s["lengths"])
        same = torch.ones_like(got, dtype=torch.bool)
        same[1, t:t + 4, d] = False
        assert torch.equal(got[same], y[same]) and not got[1, t, d].isfinite()
        dx, dw = torch.autograd.grad(got, (x, w), s["dy"])
        assert torch.equal(dx, grads["x"])
        keep = torch.arange(20, device="cuda") != d
        assert torch.equal(dw[keep], grads["weight"][keep])
        taps = min(4, 130 - t)     # steps t, t + 1, ... that count see it at the last, the last but one, ... tap
        assert not dw[d, 4 - taps:].isfinite().any() and torch.equal(dw[d, :4 - taps], grads["weight"][d, :4 - taps])
        if bad == float("inf"):    # (one term: no NaN)
            assert dw[d, 4 - taps:].isinf().all()
        dy = s["dy"].clone()
        dy[1, t, d] = bad
        dx, = torch.autograd.grad(mk.causal_conv(x, w, s["bias"], activation=None, lengths=s["lengths"]), x, dy)
        same = torch.ones_like(dx, dtype=torch.bool)
        same[1, t - 3:t + 1, d] = False
        assert torch.equal(dx[same], grads["x"][same])


@pytest.mark.parametrize("dt", TYPES)
def test_pieces_are_the_whole(cuda, dt):
    """A prompt in pieces, then single tokens."""
    import metal_kans as mk
    s = inputs(2, 60, 37, 4, dt)
    with torch.no_grad():
        whole = mk.causal_conv(s["x"], s["weight"], s["bias"])
        state, at, out = torch.zeros(2, 3, 37, device="cuda", dtype=dt), 0, []
        for n in (30, 1, 2, 20, 1, 1, 1, 1, 1, 1, 1):
            version = state._version
            out.append(mk.causal_conv(s["x"][:, at:at + n], s["weight"], s["bias"], state=state))
            assert state._version > version
            at += n
        assert at == 60 and torch.equal(torch.cat(out, 1), whole)
        assert torch.equal(state, s["x"][:, -3:])


def test_orders_of_memory(cuda):
    """Views whose channels lie side by side, odd addresses, and others."""
    import metal_kans as mk
    for dt in TYPES:
        s = inputs(2, 33, 24, 3, dt)
        want, grads = check(s)
        wide = torch.zeros(2, 33, 61, device="cuda", dtype=dt)
        wide[..., 5:29] = s["x"]
        across = s["x"].transpose(0, 1).contiguous().transpose(0, 1)
        apart = s["x"].transpose(1, 2).contiguous().transpose(1, 2)
        for x in (wide[..., 5:29], across, apart):
            x = x.requires_grad_(True)
            y = mk.causal_conv(x, s["weight"].t().contiguous().t(), s["bias"])
            assert torch.equal(y, want)
            dx, = torch.autograd.grad(y, x, s["dy"].transpose(0, 1).contiguous().transpose(0, 1))
            assert torch.equal(dx, grads["x"])
        one = s["x"][:1].expand(2, 33, 24)
        assert torch.equal(mk.causal_conv(one, s["weight"], s["bias"]), mk.causal_conv(one.contiguous(), s["weight"], s["bias"]))
    assert mk.causal_conv(torch.zeros(0, 5, 4, device="cuda"), torch.zeros(4, 2, device="cuda")).shape == (0, 5, 4)
    x, w = torch.zeros(2, 0, 4, device="cuda", requires_grad=True), torch.ones(4, 2, device="cuda", requires_grad=True)
    y = mk.causal_conv(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == dx.shape == (2, 0, 4) and not dw.any()


def test_gradients_are_the_differences(cuda):
    """Against central differences of the 64-bit definition, whose own error is far below the bound."""
    s = inputs(2, 20, 6, 4, torch.float32, lengths=[20, 13])
    _, grads = check(s)
    for name, at in (("x", (0, 3, 2)), ("x", (1, 12, 5)), ("weight", (4, 0)), ("weight", (1, 3)), ("bias", (2,))):
        ends = []
        for e in (1e-4, -1e-4):
            moved = {n: None if t is None else t.double().clone() if t.is_floating_point() else t for n, t in s.items()}
            moved[name][at] += e
            ends.append((reference(moved, "silu")["y"][0] * moved["dy"]).sum())
        slope = (ends[0] - ends[1]) / 2e-4
        assert abs(slope - grads[name][at]) <= 1e-5 * max(1.0, abs(slope))


def test_machinery(cuda):
    """A graph that is replayed, another stream, guarded inputs, no second derivative, no gradients with a state."""
    import metal_kans as mk
    s = inputs(2, 50, 40, 4, torch.float32, lengths=[50, 31])
    for n in ("x", "weight", "bias"):
        s[n].requires_grad_(True)
    state = s["state"].clone()

    def step():
        y = mk.causal_conv(s["x"], s["weight"], s["bias"], lengths=s["lengths"])
        grads = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        with torch.no_grad():
            served = mk.causal_conv(s["x"], s["weight"], s["bias"], state=state, lengths=s["lengths"])
        return [y.detach(), *grads, served, state]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2, 3):
        new = inputs(2, 50, 40, 4, torch.float32, seed=seed)
        with torch.no_grad():
            for n in ("x", "weight", "bias", "dy"):
                s[n].copy_(new[n])
            s["lengths"].copy_(torch.tensor([seed, 50 - seed], device="cuda"))
            state.copy_(new["state"])
        want = [t.clone() for t in step()]
        with torch.no_grad():
            state.copy_(new["state"])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed
    with torch.cuda.stream(side):
        with torch.no_grad():
            state.copy_(new["state"])
        again = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    y = mk.causal_conv(s["x"], s["weight"], s["bias"])
    dx, = torch.autograd.grad(y, s["x"], s["dy"], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()
    y = mk.causal_conv(s["x"], s["weight"], s["bias"])
    with torch.no_grad():
        s["x"].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, s["x"], s["dy"])
    with pytest.raises(RuntimeError, match="no gradients"):
        mk.causal_conv(s["x"], s["weight"], s["bias"], state=state)
    with pytest.raises(RuntimeError, match="no gradients"):
        mk.causal_conv(s["x"].detach(), s["weight"].detach(), state=state.clone().requires_grad_(True))


def test_some_gradients(cuda):
    import metal_kans as mk
    s = inputs(2, 50, 40, 4, torch.float32)
    _, want = check(s)
    for leaves in (["x"], ["weight"], ["bias"], ["x", "bias"]):
        a = {n: s[n].detach().requires_grad_(n in leaves) for n in ("x", "weight", "bias")}
        y = mk.causal_conv(a["x"], a["weight"], a["bias"])
        for n, g in zip(leaves, torch.autograd.grad(y, [a[n] for n in leaves], s["dy"])):
            assert torch.equal(g, want[n])
