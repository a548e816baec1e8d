"""linear_cross_entropy (run on an MI355X) against its definition in 64 bits.

Tolerances.  u = 2^-24; t one rounding to the inputs' type (2^-8 bf16, 2^-11 fp16, u fp32).  A logit is a sum
of D products in runs of 16: off by at most e = (m D / 16 + 20) u sum |h w| with m = 1 MFMA a run (6 for fp32,
whose three-term products are exact to 2 u).  The row's lse is then off by at most max e + 64 u (1 + |lse|), the loss by
that and e.  A probability is off by d p with d twice that; G = c (p - y) is rounded to the type of the
products, t |G|; a gradient is a sum over G of k terms in runs of 16, (m k / 16 + 20) u sum |G x|, rounded once more (to no finer
than half the type's smallest step: gradients of 1e-49 have no fp32 number).
Roundings to the type are independent: the root mean square of the error is held to that of
t sqrt(ref^2 + sum (G x)^2), besides the bounds above.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
T = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the type's smallest step


@pytest.fixture(scope="module")
def cuda(gpu):
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    return torch.device("cuda:0")


def data(n, d, v, dt, seed, spread=2.0, ignored=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(n, d, generator=gen, device="cuda").to(DT[dt])
    w = (torch.randn(v, d, generator=gen, device="cuda") * spread / d ** 0.5).to(DT[dt])
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    if ignored:
        t[torch.rand(n, generator=gen, device="cuda") < ignored] = -100
    return h, w, t, gen


def check(mk, h, w, t, dt, reduction="mean", gen=None, ignore=-100, losses_only=False):
    n, d = h.shape
    v = w.shape[0]
    m = 6 if dt == "f32" else 1
    valid = t != ignore
    h64 = torch.where(valid[:, None], h, torch.zeros_like(h)).double()
    w64 = w.double()
    at = torch.where(valid, t, torch.zeros_like(t))[:, None]
    logits = h64 @ w64.t()
    e = (m * d / 16 + 20) * U * (h64.abs() @ w64.abs().t()).amax(1)
    lse = torch.logsumexp(logits, 1)
    rows = torch.where(valid, lse - logits.gather(1, at)[:, 0], torch.zeros_like(lse))
    row_err = torch.where(valid, 2 * e + 64 * U * (1 + lse.abs()), torch.zeros_like(e))
    count = int(valid.sum())
    want, err = {"none": (rows, row_err), "sum": (rows.sum(), row_err.sum()),
                 "mean": (rows.sum() / max(count, 1), row_err.sum() / max(count, 1))}[reduction]
    err = err + 16 * U * rows.abs().sum() / (count if reduction == "mean" else 1) * (reduction != "none")
    with torch.no_grad():
        got0 = mk.linear_cross_entropy(h, w, t, ignore, reduction)
    hr, wr = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = mk.linear_cross_entropy(hr, wr, t, ignore, reduction)
    assert got.dtype == torch.float32 and got.shape == want.shape and torch.equal(got, got0)
    assert torch.all((got.detach().double() - want).abs() <= err + U * want.abs()), \
        ((got.detach().double() - want).abs() / (err + 1e-300)).max()
    if losses_only:
        return
    grad = torch.randn(n, generator=gen, device="cuda") if reduction == "none" else torch.tensor(1.7, device="cuda")
    dh, dw = torch.autograd.grad(got, (hr, wr), grad)
    c = (grad.double() if reduction == "none" else grad.double() / (count if reduction == "mean" else 1)) * valid
    p = (logits - lse[:, None]).exp_()
    del logits
    g = p.clone()
    g.scatter_add_(1, at, -torch.ones_like(lse)[:, None])
    g *= c[:, None]
    delta = (2 * row_err + 64 * U) * c.abs()
    p *= delta[:, None]            # the error of each G from its probability's
    # (three terms hold G to 2^-24 of itself; the common factor and the products' runs add a few roundings)
    tg = T[dt] if dt != "f32" else 2 * U
    for name, out, G, P, x, k in (("dh", dh, g, p, w64, v), ("dw", dw, g.t(), p.t(), h64, n)):
        ref, size = G @ x, G.abs() @ x.abs()
        bound = T[dt] * ref.abs() + (tg + (m * k / 16 + 20) * U) * size + P @ x.abs() + LEAST[dt]
        diff = (out.double() - ref).abs()
        assert torch.isfinite(out).all() and torch.all(diff <= bound), (name, (diff / (bound + 1e-300)).max().item())
        square = ref.square() + G.square() @ x.square()
        steady = P @ x.abs() + 64 * U * size + LEAST[dt]
        assert diff.square().mean().sqrt() <= tg * square.mean().sqrt() + steady.square().mean().sqrt(), name
    assert (dh[~valid] == 0).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,v", [(1, 1, 2), (1, 64, 1000), (5, 8, 10), (33, 17, 257), (64, 72, 100), (70, 200, 255), (129, 64, 5003),
                                   (256, 128, 256), (300, 777, 1031), (1000, 96, 300), (17, 1024, 4099)])
def test_sizes_and_types(cuda, n, d, v, dt):
    import metal_kans as mk
    h, w, t, gen = data(n, d, v, dt, n + d)
    for reduction in ("mean", "none"):
        check(mk, h, w, t, dt, reduction, gen)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,v", [(300, 64, 25100),      # large tiles of logits
                                   (70, 2050, 6500),      # large tiles of dW
                                   (3300, 4096, 300),     # large tiles of dH
                                   (20, 64, 70001)])      # narrow tiles, dH split over the vocabulary
def test_tile_choices(cuda, n, d, v, dt):
    import metal_kans as mk
    h, w, t, gen = data(n, d, v, dt, v)
    check(mk, h, w, t, dt, "sum", gen)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_vocabulary_in_pieces(cuda, dt):
    """Two pieces, the second of few entries, and the rows' number below its padded one."""
    import metal_kans as mk
    h, w, t, gen = data(4090, 72, 33001, dt, 3, ignored=0.2)
    t[:50] = torch.arange(32990, 33040, device="cuda").clamp_max(33000)
    check(mk, h, w, t, dt, "none", gen)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,v", [(1, 32, 1), (3, 96, 129), (31, 64, 127), (32, 128, 4097), (33, 32, 300), (64, 160, 20001),
                                   (65, 64, 1000), (2, 1024, 700), (24, 30, 1000), (4, 4096, 24000)])
def test_few_rows(cuda, n, d, v, dt):
    """Heads read as they are, in fp32 too, and the borders of the tiles that do it; a head of no aligned rows."""
    import metal_kans as mk
    h, w, t, gen = data(n, d, v, dt, n * v)
    check(mk, h, w, t, dt, "none", gen)
    shifted = torch.empty(v * d + 1, dtype=w.dtype, device="cuda")[1:].view(v, d).copy_(w)
    with torch.no_grad():
        a, b = (mk.linear_cross_entropy(h, x, t, reduction="none") for x in (w, shifted))
    assert (a - b).abs().max() <= 1e-4 * (1 + a.abs().max())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
def test_logits_near_the_largest_number(cuda, dt, sign):
    """One logit stands out by more than any exponential's range, near fp32's largest number or far below all zeros."""
    import metal_kans as mk
    h = torch.tensor([[1.5 * 2.0 ** 63], [1.0]], device="cuda").to(DT[dt]).requires_grad_(True)
    w = torch.full((300, 1), sign * 2.0 ** 63, device="cuda")
    w[7] = w[7] * (1.25 if sign > 0 else 0.75)                          # logits sign 1.5 2^126, 1.875 2^126 or -1.125 2^126
    w = w.to(DT[dt]).requires_grad_(True)
    for target, p_target in ((7, 1.0), (8, 0.0)):
        loss = mk.linear_cross_entropy(h, w, torch.full((2,), target, device="cuda"), reduction="none")
        top, own = (h.detach().double() @ w.detach().double().t()).amax(1), (h.detach().double() * w.detach().double()[target, 0])[:, 0]
        assert ((loss.detach().double() - (top - own)).abs() <= 2 * U * top.abs() + 1e-3).all()
        dh, dw = torch.autograd.grad(loss, (h, w), torch.tensor([1.0, 0.0], device="cuda"))
        want = w.detach().double()[7, 0] - w.detach().double()[target, 0]   # (p - y) W with p = 1 at 7
        assert (dh[0, 0].double() - want).abs() <= 4 * T[dt] * w.detach().double()[7, 0].abs() and dh[1, 0] == 0
        g = torch.zeros(300, dtype=torch.float64, device="cuda")
        g[7] += 1
        g[target] -= 1
        assert ((dw[:, 0].double() - g * h.detach().double()[0, 0]).abs() <= 4 * T[dt] * h.detach().double()[0, 0].abs() * (g != 0)).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n,d,v", [(8180, 72, 33001),     # more than 2^28 logits
                                   (5, 4099, 70001)])     # a head of more than 2^28 values, laid out anew
def test_large_vocabulary_in_pieces(cuda, n, d, v, dt):
    import metal_kans as mk
    h, w, t, gen = data(n, d, v, dt, 4, ignored=0.2)
    last = torch.arange(v - 11, v + 39, device="cuda").clamp_max(v - 1)[-min(n, 50):]
    t[:len(last)] = last
    check(mk, h, w, t, dt, "none", gen)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,v,ignored", [(2100, 800, 9001, 0.9),    # dH's workgroups of rows that do not count
                                           (1300, 300, 20011, 0.5),   # go to more splits of the others
                                           (1000, 2050, 300, 0.97)])
def test_work_shared_out_by_the_rows_that_count(cuda, n, d, v, ignored, dt):
    import metal_kans as mk
    h, w, t, gen = data(n, d, v, dt, 5, ignored=ignored)
    t[1] = 0
    check(mk, h, w, t, dt, "mean", gen)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ignored", [0.1, 0.5, 0.97])
def test_ignored_rows_take_part_in_nothing(cuda, ignored, dt):
    """... even where hidden holds infinities and NaN there."""
    import metal_kans as mk
    h, w, t, gen = data(700, 100, 513, dt, 9, ignored=ignored)
    t[3] = 7
    check(mk, h, w, t, dt, "mean", gen)
    clean = []
    for bad in (None, float("nan"), float("inf")):
        x = h.clone()
        if bad is not None:
            x[t == -100] = bad
        hr, wr = x.requires_grad_(True), w.clone().requires_grad_(True)
        loss = mk.linear_cross_entropy(hr, wr, t)
        clean.append((loss.detach(), *torch.autograd.grad(loss, (hr, wr))))
    for other in clean[1:]:
        assert all(torch.equal(a, b) for a, b in zip(clean[0], other))


def test_no_row_counts(cuda):
    import metal_kans as mk
    h, w, t, _ = data(40, 64, 300, "bf16", 1)
    t[:] = 5
    for reduction in ("mean", "sum", "none"):
        hr, wr = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = mk.linear_cross_entropy(hr, wr, t, ignore_index=5, reduction=reduction)
        dh, dw = torch.autograd.grad(loss.sum(), (hr, wr))
        assert (dh == 0).all() and (dw == 0).all()
        assert torch.isnan(loss) if reduction == "mean" else (loss == 0).all()
    e = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    wr = w.clone().requires_grad_(True)
    loss = mk.linear_cross_entropy(e, wr, t[:0], reduction="sum")
    loss.backward()
    assert loss == 0 and (wr.grad == 0).all()
    assert torch.isnan(mk.linear_cross_entropy(e, w, t[:0]))
    assert mk.linear_cross_entropy(e, w, t[:0], reduction="none").shape == (0,)


def test_targets_outside_the_vocabulary(cuda):
    import metal_kans as mk
    h, w, t, _ = data(100, 64, 300, "f32", 2)
    want = mk.linear_cross_entropy(h, w, t, reduction="none")
    t2 = t.clone()
    t2[10], t2[20], t2[99] = 300, -1, 1 << 40
    got = mk.linear_cross_entropy(h, w, t2, reduction="none")
    bad = torch.isnan(got).nonzero().flatten().tolist()
    assert bad == [10, 20, 99]
    keep = ~torch.isnan(got)
    assert torch.equal(got[keep], want[keep])
    hr = h.clone().requires_grad_(True)
    dh, = torch.autograd.grad(mk.linear_cross_entropy(hr, w, t2), hr)
    assert torch.isnan(dh[10]).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_far_apart_and_equal_logits(cuda, dt):
    """Logits of some hundreds (exp would overflow), one entry far above all others, and rows of zeros, whose
    probabilities of 1 / V lie below fp16's normal numbers."""
    import metal_kans as mk
    h, w, t, gen = data(90, 64, 3000, dt, 4, spread=60.0)
    check(mk, h, w, t, dt, "none", gen)
    h, w, t, gen = data(90, 64, 3000, dt, 5)
    w[1234] = h[7] * 20
    t[7] = 1234
    h[11] = 0
    check(mk, h, w, t, dt, "mean", gen)
    h, w, t, gen = data(40, 64, 60000, dt, 6)
    h[:20] = 0
    check(mk, h, w, t, dt, "mean", gen)


def test_minus_infinity_logits(cuda):
    """Entries of the head that are -inf for a row get probability 0."""
    import metal_kans as mk
    h, w, t, _ = data(50, 8, 700, "f32", 7)
    h = h.abs() + 0.1
    w[5], w[512:600] = float("-inf"), float("-inf")
    t = t % 5
    got = mk.linear_cross_entropy(h, w, t, reduction="none").double()
    logits = (h.double()[:, None, :] * w.double()[None]).sum(-1)
    want = torch.logsumexp(logits, 1) - logits.gather(1, t[:, None])[:, 0]
    assert torch.isfinite(got).all() and (got - want).abs().max() <= 1e-5


def test_gradients_against_differences(cuda):
    import metal_kans as mk
    h, w, t, gen = data(24, 40, 70, "f32", 8, ignored=0.2)
    hr, wr = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dh, dw = torch.autograd.grad(mk.linear_cross_entropy(hr, wr, t), (hr, wr))

    def loss(a, b):
        return torch.nn.functional.cross_entropy(a @ b.t(), t).item()
    for x, grad, which in ((h, dh, 0), (w, dw, 1)):
        way = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
        step = 1e-5
        a = [h.double(), w.double()]
        b = [h.double(), w.double()]
        a[which] = a[which] + step * way
        b[which] = b[which] - step * way
        got = (grad.double() * way).sum().item()
        assert abs((loss(*a) - loss(*b)) / (2 * step) - got) <= 1e-6 * (1 + (grad.double() * way).abs().sum().item())


def test_shapes_strides_and_parts(cuda):
    import metal_kans as mk
    h, w, t, gen = data(60, 72, 500, "bf16", 10)
    want = mk.linear_cross_entropy(h, w, t, reduction="none")
    hs = torch.zeros(60, 80, device="cuda", dtype=torch.bfloat16)
    hs[:, 3:75] = h
    odd = torch.zeros(500 * 72 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(500, 72).copy_(w)
    got = mk.linear_cross_entropy(hs[:, 3:75].reshape(3, 20, 72), odd, t.view(3, 20), reduction="none")
    assert got.shape == (3, 20) and torch.equal(got.flatten(), want)
    wt = w.t().contiguous().t()
    assert torch.equal(mk.linear_cross_entropy(h, wt, t, reduction="none"), want)
    hr, wr = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(mk.linear_cross_entropy(hr, wr, t), (hr, wr))
    assert torch.equal(torch.autograd.grad(mk.linear_cross_entropy(hr, w, t), hr)[0], both[0])
    assert torch.equal(torch.autograd.grad(mk.linear_cross_entropy(h, wr, t), wr)[0], both[1])
    h2, w2 = hr, wr                # aligned but not from the storage's start, D a multiple of 64
    x, y, t2, _ = data(33, 64, 400, "f16", 11)
    z = torch.zeros(400 * 64 + 4, device="cuda", dtype=torch.float16)[4:].view(400, 64).copy_(y)   # 8-byte aligned
    assert torch.equal(mk.linear_cross_entropy(x, y, t2), mk.linear_cross_entropy(x, z, t2))


def test_same_bits_on_every_run_and_stream(cuda):
    import metal_kans as mk
    h, w, t, _ = data(2000, 128, 9000, "bf16", 12, ignored=0.3)
    runs = []
    s = torch.cuda.Stream()
    for i in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(s if i == 1 else torch.cuda.current_stream()):
            hr, wr = (h * 1.0).requires_grad_(True), (w * 1.0).requires_grad_(True)
            loss = mk.linear_cross_entropy(hr, wr, t)
            runs.append((loss.detach(), *torch.autograd.grad(loss, (hr, wr))))
    torch.cuda.synchronize()
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_captured_graph_replays(cuda):
    """Forward and backward in one graph: every replay against the eager result, the rows that count changing."""
    import metal_kans as mk
    h, w, t, gen = data(300, 64, 1000, "bf16", 13, ignored=0.2)
    hr, wr = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    one = torch.ones((), device="cuda")

    def both():
        loss = mk.linear_cross_entropy(hr, wr, t)
        return (loss.detach(), *torch.autograd.grad(loss, (hr, wr), one))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    for i in range(4):
        h2, _, t2, _ = data(300, 64, 1000, "bf16", 20 + i, ignored=0.1 + 0.2 * i)
        with torch.no_grad():
            hr.copy_(h2)
        t.copy_(t2)
        g.replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_refusals(cuda):
    import metal_kans as mk
    h, w, t, _ = data(8, 16, 20, "f32", 14)
    for args in ((h, w[:, :8], t), (h, w[0], t), (h, w, t[:4]), (h, w[:0], t), (h.cpu(), w, t), (h, w.cpu(), t), (h, w, t.cpu())):
        with pytest.raises(ValueError):
            mk.linear_cross_entropy(*args)
    for args in ((h, w.half(), t), (h.double(), w.double(), t), (h, w, t.int())):
        with pytest.raises(TypeError):
            mk.linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        mk.linear_cross_entropy(h, w, t, reduction="max")
    with pytest.raises(mk.device.KansError):   # more columns than the kernels' places hold
        mk.linear_cross_entropy(torch.zeros(1, 65537, device="cuda"), torch.zeros(2, 65537, device="cuda"), t[:1])


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 50, 64, 100])
def test_gradient_of_infinite_entries(cuda, n, dt):
    """An entry that is -inf for every row has probability 0 and so no gradient, however many rows fill up a tile."""
    import metal_kans as mk
    h, w, t, gen = data(n, 8, 700, dt, 15)
    h, t = h.abs() + 0.1, t % 5
    w[5], w[512:600] = float("-inf"), float("-inf")
    wr = w.clone().requires_grad_(True)
    grad = torch.randn(n, generator=gen, device="cuda")
    dw, = torch.autograd.grad(mk.linear_cross_entropy(h, wr, t, reduction="none"), wr, grad)
    logits = (h.double()[:, None, :] * w.double()[None]).sum(-1)
    g = (torch.softmax(logits, 1) - torch.nn.functional.one_hot(t, 700)) * grad.double()[:, None]
    ref, size = g.t() @ h.double(), g.abs().t() @ h.double()
    assert torch.isfinite(dw).all() and (dw[5] == 0).all() and (dw[512:600] == 0).all()
    # G's rounding, dW's own, and some hundred roundings of products and exponentials
    assert ((dw.double() - ref).abs() <= T[dt] * ref.abs() + (2 * T[dt] + 128 * U) * size + LEAST[dt]).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [0, -96, 240, 4096])
@pytest.mark.parametrize("n", [3, 45])
def test_shifted_logits_and_confident_rows(cuda, n, shift, dt):
    """Losses and gradients do not depend on what all logits of a row have in common, and rows whose target has nearly all
    probability keep what is left of it.  All logits here are exact, so what is off is a sum of 300 exponentials (of one
    rounding each and as many in the sum's tree), its logarithm and the differences of logits: 32 u."""
    import metal_kans as mk
    v, rows = 300, torch.arange(n, device="cuda")
    kinds = 9
    gap = torch.tensor([0.0, 3.0, 7.0, 10.0, 13.0, 14.0, 15.5, -2.0, 15.0], device="cuda")
    h, w = torch.zeros(n, 48, device="cuda"), torch.zeros(v, 48, device="cuda")
    h[:, 0], w[:, 0] = 1, shift
    h[:, 40], w[:, 40] = 1, 0.25 * (torch.arange(v, device="cuda") % 5 - 2)
    h[rows, 1 + rows % kinds] = 1
    own = 20 + 31 * torch.arange(kinds, device="cuda")       # the target of each kind of row
    w[own, 1 + torch.arange(kinds, device="cuda")] = gap
    h, w, t = h.to(DT[dt]), w.to(DT[dt]), own[rows % kinds]
    hr, wr = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = mk.linear_cross_entropy(hr, wr, t, reduction="none")
    logits = h.double() @ w.double().t()
    logits -= logits.amax(1, keepdim=True)
    lse = torch.logsumexp(logits, 1)
    want = lse - logits.gather(1, t[:, None])[:, 0]
    assert ((loss.detach().double() - want).abs() <= 32 * U * (1 + want)).all()
    dh, dw = torch.autograd.grad(loss.sum(), (hr, wr))
    p = (logits - lse[:, None]).exp()
    g = p.clone()
    g[rows, t] = torch.expm1(-want)
    tg = T[dt] if dt != "f32" else 2 * U
    m = 6 if dt == "f32" else 1
    for name, out, G, P, x, k in (("dh", dh, g, p, w.double(), v), ("dw", dw, g.t(), p.t(), h.double(), n)):
        ref, size = G @ x, G.abs() @ x.abs()
        bound = T[dt] * ref.abs() + (tg + (m * k / 16 + 20) * U) * size + 32 * U * (P @ x.abs()) + LEAST[dt]
        assert ((out.double() - ref).abs() <= bound).all(), (name, ((out.double() - ref).abs() / bound).max().item())


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_gradients_that_are_not_numbers(cuda, bad, dt):
    """A row whose loss has no finite gradient leaves the other rows' gradients as they are."""
    import metal_kans as mk
    h, w, t, gen = data(50, 64, 300, dt, 17)
    grad = 100 * torch.randn(50, generator=gen, device="cuda")
    rest = torch.arange(50, device="cuda") != 7
    runs = []
    for value in (0.0, bad):
        grad[7] = value
        hr = h.clone().requires_grad_(True)
        runs.append(torch.autograd.grad(mk.linear_cross_entropy(hr, w, t, reduction="none"), hr, grad)[0])
    assert torch.isfinite(runs[0]).all() and torch.equal(runs[0][rest], runs[1][rest])
    assert not torch.isfinite(runs[1][7]).any()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,d,v", [(40, 64, 60000), (300, 72, 20011), (40, 1024, 900)])
@pytest.mark.parametrize("least", [2.0 ** -7, 2.0 ** -12, 2.0 ** 9])
def test_gradients_of_very_different_rows(cuda, least, n, d, v, dt):
    """One row's gradient is 2^12, the others' down to 2^-24 of that: they keep their own small probabilities in dH.  (dW adds
    all rows up: relative to the largest.)"""
    import metal_kans as mk
    h, w, t, gen = data(n, d, v, dt, 16)
    h[::2] = 0                                       # probabilities of 1 / v
    w[:, 0] = 1
    w[t, 0] = 0
    grad = torch.full((n,), least, device="cuda")
    grad[1::4] *= -1.5
    grad[3], grad[n // 2 | 1] = 2.0 ** 12, 0.0
    hr, wr = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dh, dw = torch.autograd.grad(mk.linear_cross_entropy(hr, wr, t, reduction="none"), (hr, wr), grad)
    alone = [torch.autograd.grad(mk.linear_cross_entropy(hr, wr, t, reduction="none"), x, grad)[0] for x in (hr, wr)]
    assert torch.equal(alone[0], dh) and torch.equal(alone[1], dw)
    g = torch.softmax(h.double() @ w.double().t(), 1) - torch.nn.functional.one_hot(t, v)
    g *= grad.double()[:, None]
    tg, m = (2 * U, 6) if dt == "f32" else (T[dt], 1)
    for name, out, G, x, k in (("dh", dh, g, w.double(), v), ("dw", dw, g.t(), h.double(), n)):
        ref, size = G @ x, G.abs() @ x.abs()
        # G and the result rounded; logits of sums of d products, exponentials, sums of k products (as for the other sizes)
        bound = T[dt] * ref.abs() + (tg + (m * k / 16 + m * d / 2 + 500) * U) * size + LEAST[dt]
        if name == "dw" and dt == "f16":             # G below 2^-25 of 2^-14 of the largest gradient has no number
            bound = bound + 2.0 ** -39 * 2.0 ** 12 * x.abs().sum(0)
        assert torch.isfinite(out).all() and ((out.double() - ref).abs() <= bound).all(), (
            name, ((out.double() - ref).abs() / bound).max().item())
    assert (dh[n // 2 | 1] == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("power", [-112, -20, 60])
def test_size_of_the_gradient(cuda, power, reduction, dt):
    """Gradients scale with that of the loss, bit for bit, as far as they are normal numbers: here 2^-112 to 2^60 times those
    of 1, both directions of products included."""
    import metal_kans as mk
    h, w, t, gen = data(70, 96, 500, dt, 18)
    runs = []
    for p in (0, power):
        hr, wr = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = mk.linear_cross_entropy(hr, wr, t, reduction=reduction)
        grad = torch.full_like(loss, 1.2345 * 2.0 ** p)
        runs.append(torch.autograd.grad(loss, (hr, wr), grad))
    for one, other in zip(*runs):
        want = one.double() * 2.0 ** power
        normal = want.abs() >= 2.0 ** -126
        assert normal.any() and torch.equal(other.double()[normal], want[normal])
