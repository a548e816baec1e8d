"""residual_norm (run on an MI355X) against its definition in 64 bits.

Tolerances.  u = 2^-24 is one fp32 rounding, t one rounding to the output's type (2^-11 fp16, 2^-8 bf16 with
its 8-bit significand's half step 2^-9, doubled for results next to a power of two).  Every result is a
sum of products; A is the sum of the products' magnitudes, where a difference counts with the magnitudes
of both sides.  A sum of the lengths here goes through at most some 40 additions one after the other, and its terms
hold some 20 roundings: the error is at most t |result| + 64 u A (and the type's smallest step).
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
C = 64
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEP = {torch.float32: (2.0 ** -24, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 0.0)}


@pytest.fixture(scope="module")
def cuda(gpu):
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    return torch.device("cuda:0")


def rnd(gen, *shape, dt=torch.float32, scale=1.0, shift=0.0):
    return (scale * torch.randn(*shape, generator=gen, device="cuda") + shift).to(dt)


def norm64(a, kind, eps):
    mean = a.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(a[..., :1])
    r = 1 / ((a - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    return (a - mean) * r, mean, r


def grad64(q, n, r, kind):
    return r * (q - n * (q * n).mean(-1, keepdim=True) - (q.mean(-1, keepdim=True) if kind == "layer" else 0))


def bcast(t, like):
    """t, of like's shape, summed over the dimensions in which `like` repeats."""
    while t.dim() > like.dim():
        t = t.sum(0)
    for i, s in enumerate(like.shape):
        if s == 1 and t.shape[i] != 1:
            t = t.sum(i, keepdim=True)
    return t


def reference(x, block, gate, scale, post, pre, dy, dh, kind, eps):
    """Results and the magnitudes A, by name."""
    d = lambda t, one=None: one if t is None else t.detach().double()  # noqa: E731
    one = torch.ones((), dtype=torch.float64, device=x.device)
    x, g, wp, wn = d(x), d(gate, one), d(post, one), d(pre, one)
    s = scale.detach().double() if isinstance(scale, torch.Tensor) else scale * one
    R, A = {}, {}
    if block is not None:
        bn, mb, rb = norm64(d(block), kind, eps)
        ba = (d(block).abs() + mb.abs()) * rb
        u, ua = bn * wp, ba * wp.abs()
        y, ya = x + s * g * u, x.abs() + s.abs() * g.abs() * ua
        R["y"], A["y"] = y, ya
    else:
        y, ya = x, x.abs()
    yn, my, ry = norm64(y, kind, eps)
    yna = (ya + my.abs()) * ry
    R["h"], A["h"] = yn * wn, yna * wn.abs()
    if dy is None and dh is None:
        return R, A
    dy = torch.zeros_like(x) if dy is None else d(dy)
    dh = torch.zeros_like(x) if dh is None else d(dh)
    q = wn * dh
    T = dy + grad64(q, yn, ry, kind)
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    Ta = dy.abs() + ry * (q.abs() + yna * mean(q.abs() * yna) + mean(q.abs()))
    R["x"], A["x"] = T, Ta
    if pre is not None:
        R["pre"], A["pre"] = bcast(dh * yn, pre), bcast(dh.abs() * yna, pre)
    if block is not None:
        if gate is not None:
            R["gate"], A["gate"] = bcast(s * T * u, gate), bcast(s.abs() * Ta * ua, gate)
        R["scale"], A["scale"] = (T * g * u).sum().reshape(1), (Ta * g.abs() * ua).sum().reshape(1)
        du, dua = s * g * T, s.abs() * g.abs() * Ta
        if post is not None:
            R["post"], A["post"] = bcast(du * bn, post), bcast(dua * ba, post)
        R["block"] = grad64(du * wp, bn, rb, kind)
        pa = dua * wp.abs()
        A["block"] = rb * (pa + ba * mean(pa * ba) + mean(pa))
    return R, A


def close(name, got, want, size):
    t, least = STEP[got.dtype]
    err = (got.detach().double() - want).abs()
    bound = t * want.abs() + C * U * size + least
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, (name, worst, err.max().item())


def check(mk, x, block, gate, scale, post, pre, kind, eps=1e-6, gy=True, gh=True, gen=None):
    named = dict(x=x, block=block, gate=gate, scale=scale, post=post, pre=pre)
    leaves = {n: t for n, t in named.items() if isinstance(t, torch.Tensor)}
    with torch.no_grad():
        y0, h0 = mk.residual_norm(x, block, gate, scale, post, pre, kind, eps)
    for t in leaves.values():
        t.requires_grad_(True)
    y, h = mk.residual_norm(x, block, gate, scale, post, pre, kind, eps)
    assert torch.equal(y, y0) and torch.equal(h, h0)
    dy = rnd(gen, *x.shape, dt=x.dtype) if gy else None
    dh = rnd(gen, *x.shape, dt=h.dtype) if gh else None
    R, A = reference(x, block, gate, scale, post, pre, dy, dh, kind, eps)
    close("h", h, R["h"], A["h"])
    if block is not None:
        close("y", y, R["y"], A["y"])
    outs = [(o, g) for o, g in ((y, dy), (h, dh)) if g is not None and o.grad_fn is not None]
    grads = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    for n, g in zip(leaves, grads):
        if n == "x" and block is None and gy:
            continue  # y is x itself: its gradient is tested where there is a block
        if g is None:
            assert n == "pre" and not gh, n
        else:
            close(n, g, R[n].reshape(g.shape), A[n].reshape(g.shape))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 7), (1, 64), (9, 255), (33, 256), (4, 511), (6, 513), (517, 300),
                                    (7, 1000), (3, 1025), (130, 2048), (2, 4095), (65, 4096), (5, 8192), (3, 8193),
                                    (2, 16384), (3, 16391), (2, 20011)])
def test_sizes_and_types(cuda, rows, d, types, kind):
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(rows * 31 + d)
    rt, dt = (DT[t] for t in types)
    check(mk, rnd(gen, rows, d, dt=rt, scale=2.0, shift=0.3), rnd(gen, rows, d, dt=dt, shift=-0.2),
          rnd(gen, d, dt=dt, shift=0.5), torch.full((1,), 0.7, device="cuda"), rnd(gen, d, dt=dt, shift=1.0),
          rnd(gen, d, dt=dt, shift=1.0), kind, gen=gen)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("d", [48, 777, 4096, 17000])
@pytest.mark.parametrize("shape", [None, (1,), "d", (1, 1, "d"), (4, 1, "d"), (4, 9, "d"), (1, 9, "d"), (4, 9, 1), (9, "d")])
def test_gates(cuda, shape, d, types, kind):
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(d)
    rt, dt = (DT[t] for t in types)
    gate = None
    if shape is not None:
        shape = (d,) if shape == "d" else tuple(d if s == "d" else s for s in shape)
        gate = rnd(gen, *shape, dt=dt, shift=0.5)
    check(mk, rnd(gen, 4, 9, d, dt=rt), rnd(gen, 4, 9, d, dt=dt), gate, 0.4, rnd(gen, d, dt=dt, shift=1.0),
          rnd(gen, d, dt=dt, shift=1.0), kind, gen=gen)


@pytest.mark.parametrize("d", [65, 4096, 17000])
@pytest.mark.parametrize("what", ["no block", "no weights", "only y", "only h", "no block, only h"])
def test_parts(cuda, what, d):
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(5)
    block = None if "no block" in what else rnd(gen, 11, d)
    post = None if block is None or what == "no weights" else rnd(gen, d, shift=1.0)
    pre = None if what == "no weights" else rnd(gen, d, shift=1.0)
    for kind in ("rms", "layer"):
        check(mk, rnd(gen, 11, d), block, None, 0.4 if block is not None else 1.0, post, pre, kind, gy=what != "only h" and "no block" not in what,
              gh=what != "only y", gen=gen)


@pytest.mark.parametrize("rows,group", [(24, 2), (600, 3), (1030, 515), (4096, 512)])
def test_groups_of_rows(cuda, rows, group):
    """Runs of rows end inside a group and at its end."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(group)
    d = 130
    check(mk, rnd(gen, rows // group, group, d), rnd(gen, rows // group, group, d), rnd(gen, rows // group, 1, d),
          torch.ones(1, device="cuda"), rnd(gen, d), rnd(gen, d), "rms", gen=gen)


def test_gradients_against_differences(cuda):
    """The loss's change along a random direction of each input, by central differences of the definition in 64 bits."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(1)
    for kind in ("rms", "layer"):
        ins = dict(x=rnd(gen, 6, 37), block=rnd(gen, 6, 37), gate=rnd(gen, 37, shift=0.5),
                   scale=torch.full((1,), 0.6, device="cuda"), post=rnd(gen, 37, shift=1.0), pre=rnd(gen, 37, shift=1.0))
        wy, wh = rnd(gen, 6, 37), rnd(gen, 6, 37)
        leaves = {n: t.clone().requires_grad_(True) for n, t in ins.items()}
        y, h = mk.residual_norm(leaves["x"], leaves["block"], leaves["gate"], leaves["scale"], leaves["post"], leaves["pre"], kind)
        ((y * wy).sum() + (h * wh).sum()).backward()

        def loss(v):
            R, _ = reference(v["x"], v["block"], v["gate"], v["scale"], v["post"], v["pre"], None, None, kind, 1e-6)
            return ((R["y"] * wy).sum() + (R["h"] * wh).sum()).item()
        for n in ins:
            at = {m: t.double() for m, t in ins.items()}
            way = torch.randn(ins[n].shape, generator=gen, device="cuda", dtype=torch.float64)
            e = 1e-5
            up, down = loss({**at, n: at[n] + e * way}), loss({**at, n: at[n] - e * way})
            got = (leaves[n].grad.double() * way).sum().item()
            size = (leaves[n].grad.double() * way).abs().sum().item() + 1.0
            # fp32 gradients (some 64 roundings), differences to the square of the step and the rounding of the loss over it
            assert abs((up - down) / (2 * e) - got) <= size * (64 * U + 1e-6), (kind, n)


def test_strides_alignment_and_streams(cuda):
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(2)
    big = rnd(gen, 70000, dt=torch.bfloat16)
    x, b = big[1:1 + 64 * 300].view(64, 300), rnd(gen, 300, 64, dt=torch.bfloat16).t()
    w = big[3:303]
    want = mk.residual_norm(x.clone(), b.contiguous(), None, 0.5, w.clone(), w.clone())
    got = mk.residual_norm(x, b, None, 0.5, w, w)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        xs = x * 1.0
        got = mk.residual_norm(xs, b, None, 0.5, w, w)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_captured_graph_replays(cuda):
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, b = rnd(gen, 50, 512, dt=torch.bfloat16), rnd(gen, 50, 512, dt=torch.bfloat16)
    mk.residual_norm(x, b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, h = mk.residual_norm(x, b)
    for i in range(3):
        x.copy_(rnd(gen, 50, 512, dt=torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        y1, h1 = mk.residual_norm(x, b)
        assert torch.equal(y, y1) and torch.equal(h, h1), i


def test_same_bits_on_every_run(cuda):
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, b, w = rnd(gen, 3000, 513), rnd(gen, 3000, 513), rnd(gen, 513).requires_grad_(True)
    runs = []
    for _ in range(3):
        y, h = mk.residual_norm(x, b, w, 0.3, w, w)
        runs.append(torch.autograd.grad((y.sum() + h.square().sum()), w)[0])
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


@pytest.mark.parametrize("d", [100, 4096, 17000])
def test_zero_rows_and_values_that_are_not_numbers(cuda, d):
    """A row of zeros stays zero (eps keeps its norm finite); infinities and NaN stay in their row."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(6)
    for kind in ("rms", "layer"):
        x, b = rnd(gen, 9, d), rnd(gen, 9, d)
        x[2], b[2] = 0, 0
        y, h = mk.residual_norm(x, b, kind=kind)
        assert (y[2] == 0).all() and (h[2] == 0).all()
        x1, b1 = x.clone(), b.clone()
        x1[4, d // 2], b1[6, d // 3] = float("nan"), float("inf")
        x1, b1 = x1.requires_grad_(True), b1.requires_grad_(True)
        y1, h1 = mk.residual_norm(x1, b1, kind=kind)
        dx, db = torch.autograd.grad(h1, (x1, b1), torch.ones_like(h1))
        x.requires_grad_(True), b.requires_grad_(True)
        y0, h0 = mk.residual_norm(x, b, kind=kind)
        dx0, db0 = torch.autograd.grad(h0, (x, b), torch.ones_like(h0))
        rest = [0, 1, 2, 3, 5, 7, 8]
        for a, c in ((y1, y0), (h1, h0), (dx, dx0), (db, db0)):
            assert torch.equal(a[rest], c[rest])
        assert torch.isnan(h1[4]).any() and torch.isnan(h1[6]).any()


def test_no_rows(cuda):
    import metal_kans as mk
    x = torch.zeros(0, 5, 40, device="cuda", requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    y, h = mk.residual_norm(x, torch.zeros_like(x), w, 0.5, w, w)
    assert y.shape == h.shape == (0, 5, 40)
    (y.sum() + h.sum()).backward()
    assert (w.grad == 0).all() and x.grad.shape == x.shape


def test_refusals(cuda):
    import metal_kans as mk
    x = torch.zeros(4, 8, device="cuda")
    for bad in (dict(block=torch.zeros(4, 7, device="cuda")), dict(kind="batch"), dict(eps=-1.0), dict(eps=float("nan")),
                dict(gate=x), dict(post_weight=x[0]), dict(pre_weight=torch.zeros(7, device="cuda")),
                dict(block=x, gate=torch.zeros(3, 8, device="cuda")), dict(block=x, gate=torch.zeros(2, 4, 8, device="cuda")),
                dict(block=x.cpu()), dict(pre_weight=torch.zeros(8))):
        with pytest.raises(ValueError):
            mk.residual_norm(x, **bad)
    for bad in (dict(block=x.half(), pre_weight=x[0]), dict(block=x.double()), dict(block=x, gate=x.half()),
                dict(block=x, scale=torch.zeros(2, device="cuda")), dict(block=x, scale=torch.zeros(1, device="cuda").half())):
        with pytest.raises(TypeError):
            mk.residual_norm(x, **bad)
    with pytest.raises(TypeError):
        mk.residual_norm(x.half(), x)
    with pytest.raises(ValueError):
        mk.residual_norm(x.cpu())


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_scale_without_a_block(cuda, kind):
    """A learned scale has no part in a call without a block: no gradient, and those of x and the weight are there."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(21)
    x, w, dh = rnd(gen, 7, 50), rnd(gen, 50, shift=1.0), rnd(gen, 7, 50)
    scale = torch.full((1,), 0.4, device="cuda", requires_grad=True)
    x.requires_grad_(True), w.requires_grad_(True)
    y, h = mk.residual_norm(x, scale=scale, pre_weight=w, kind=kind)
    assert y is x
    dx, dw, ds = torch.autograd.grad(h, (x, w, scale), dh, allow_unused=True)
    h1 = mk.residual_norm(x, pre_weight=w, kind=kind)[1]
    want = torch.autograd.grad(h1, (x, w), dh)
    assert ds is None and torch.equal(h, h1) and torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    # alone it makes no graph
    assert mk.residual_norm(x.detach(), scale=scale, kind=kind)[1].grad_fn is None


@pytest.mark.parametrize("types", [("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("d", [1, 48, 777, 9000])
def test_gate_of_no_dimension(cuda, d, types):
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(d)
    rt, dt = (DT[t] for t in types)
    check(mk, rnd(gen, 4, 9, d, dt=rt), rnd(gen, 4, 9, d, dt=dt), rnd(gen, 1, dt=dt, shift=0.5).reshape(()), 0.4,
          rnd(gen, d, dt=dt, shift=1.0), rnd(gen, d, dt=dt, shift=1.0), "layer", gen=gen)


@pytest.mark.parametrize("shape", [(), (1,), (4, 9, 1)])
def test_gradient_of_a_repeating_gate_is_rounded_once(cuda, shape):
    """Each element's share lies below fp16's smallest number, their sum does not."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(22)
    x, block = rnd(gen, 4, 9, 600), rnd(gen, 4, 9, 600, dt=torch.float16)
    gate = torch.ones(shape, dtype=torch.float16, device="cuda", requires_grad=True)
    y, _ = mk.residual_norm(x, block, gate)
    u, _, _ = norm64(block.double(), "rms", 1e-6)
    dy = 1e-8 * torch.sign(u).float()
    got, = torch.autograd.grad(y, gate, dy)
    want = bcast(dy.double() * u, gate)
    assert got.shape == gate.shape and ((got.double() - want).abs() <= 2.0 ** -11 * want + 2.0 ** -25).all()


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("groups,group,d", [(1, 5, 200), (3, 2, 100), (700, 2, 72), (2000, 3, 130), (5000, 7, 33), (1030, 2, 1000),
                                            (515, 13, 600), (600, 2, 4096), (2, 2, 4096), (90, 6, 8192), (1030, 2, 8000), (40, 2, 9000),
                                            (9, 30, 17000), (1030, 2, 8200)])
def test_short_groups_of_rows(cuda, groups, group, d, types, kind):
    """Gate rows of few rows each, several groups to a run, the last of fewer: a row's results are those of the same gate with a
    row for each row, its gradient their sum (in fp32, and rounded once more), the others' sums in another order."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(group * d)
    rt, dt = (DT[t] for t in types)
    x, block, gate = rnd(gen, groups, group, d, dt=rt), rnd(gen, groups, group, d, dt=dt), rnd(gen, groups, 1, d, dt=dt, shift=0.5)
    scale, post, pre = torch.full((1,), 0.7, device="cuda"), rnd(gen, d, dt=dt, shift=1.0), rnd(gen, d, dt=dt, shift=1.0)
    dy, dh = rnd(gen, groups, group, d, dt=rt), rnd(gen, groups, group, d, dt=dt)
    runs = []
    for g in (gate, gate.expand_as(block).contiguous()):
        t = [v.clone().requires_grad_(True) for v in (x, block, g, scale, post, pre)]
        out = mk.residual_norm(*t, kind=kind)
        runs.append((out, torch.autograd.grad(out, t, (dy, dh))))
    (out0, (dx0, db0, dg0, *sums0)), (out1, (dx1, db1, dg1, *sums1)) = runs
    assert all(torch.equal(a, b) for a, b in zip(out0, out1)) and torch.equal(dx0, dx1) and torch.equal(db0, db1)
    each = dg1.double()
    want, size = each.sum(1, keepdim=True), each.abs().sum(1, keepdim=True)
    t, least = STEP[dt]
    rounded = t * size + group * least if dt != torch.float32 else 0   # of each row's own share
    assert ((dg0.double() - want).abs() <= t * want.abs() + (group + 1) * U * size + rounded + least).all()
    _, A = reference(x, block, gate, scale, post, pre, dy, dh, kind, 1e-6)
    for name, a, b in zip(("scale", "post", "pre"), sums0, sums1):
        close(name, a, b.double(), A[name].reshape(b.shape) + t / (C * U) * b.double().abs())
    again = [v.clone().requires_grad_(True) for v in (x, block, gate, post)]
    y, h = mk.residual_norm(again[0], again[1], again[2], 0.7, again[3], pre, kind)
    for wants, place in (((2,), dg0), ((3,), sums0[1])):           # some gradients alone
        got = torch.autograd.grad((y, h), [again[i] for i in wants], (dy, dh), retain_graph=True)[0]
        assert got.shape == place.shape and torch.isfinite(got).all()


@pytest.mark.parametrize("d", [100, 1000, 4096, 8192, 17000])
def test_gradient_of_the_scale_cancels(cuda, d):
    """Rows in pairs of opposite gradients, far apart: the scale's gradient is 0.  A row's terms are rounded alike in both, so
    only the sums of rows can leave something: those are held in 64 bits."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(d)
    half = 1500 if d < 8192 else 300
    x, block, dy = (rnd(gen, half, d) for _ in range(3))
    scale = torch.ones(1, device="cuda", requires_grad=True)
    y, _ = mk.residual_norm(torch.cat([x, x]), torch.cat([block, block]), scale=scale)
    got, = torch.autograd.grad(y, scale, torch.cat([dy, -dy]))
    u, _, _ = norm64(block.double(), "rms", 1e-6)
    assert got.abs().double().item() <= 2.0 ** -44 * 2 * (dy.double() * u).abs().sum().item()
