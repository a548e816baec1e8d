"""selective_scan (run on an MI355X) against its definition in 64 bits.

Tolerances, from the roundings in the order in which they are made; u = 2^-24, t one rounding to the result's type.
    s (a sum, an exponential, a polynomial, two more): off by 8 u (s + |v| e), e = 1 where softplus is not taken, v = dt + dt_bias:
        the sum's own rounding moves it by |v| u times a slope of at most sigmoid(v); S := s + |v| sigmoid(v)
    a = exp(s A): its exponent has three roundings and s's error, off by c u a with c = 4 |s A| + 8 S |A| + 2
    h: E[t] = a E[t-1] + (c + 2) u a M[t-1] + 12 u S |x B|, M the same recurrence over magnitudes
    y: sum |C| E + (N + 4) u sum |C| M + 2 u |D x|;  out: (that + (|z| + 8) u |y|') |silu(z)|, |y|' the sum of magnitudes
    g, backwards: F[t] = a F[t+1] + (c + 2) u a G[t+1] + (|z| + 10) u |C dy|, G its magnitudes
and the gradients by the product rule, with a rounding for every term and addition: `k` of them along a sequence (16 of a
tile, then the tiles, chunks and sequences), 90 over the channels (16 lanes, 4 waves and up to 64 workgroups).
Exponentials and reciprocals below fp32's smallest normal number 2^-126 =: w become zero, which moves a step size, a decay and a
sigmoid by up to w, and what they multiply by w times its magnitude: h by w (M[t-1] + |x B|), g by w G[t+1], dx by w |g . B|,
ddt by w times the step's gradient, dA by w |k| and dB by w |g x|.
Channels of a sequence whose states or their gradients grow beyond 2^100 (steps that grow states exponentially) are not
compared, nor what sums over them: fp32 ends at 2^128, and a product of two such numbers is not in it.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U, LOW = 2.0 ** -24, 2.0 ** -126
STEP = {torch.float32: (2.0 ** -24, 2.0 ** -126), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -126)}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
LEAVES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


@pytest.fixture(scope="module")
def cuda(gpu):
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    return torch.device("cuda:0")


def inputs(b, l, d, n, dt, seed=0, lengths=None, without=()):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    s = dict(x=rnd(b, l, d).to(dt), dt=rnd(b, l, d).to(dt), A=-torch.exp(rnd(d, n)), B=rnd(b, l, n).to(dt), C=rnd(b, l, n).to(dt),
             D=rnd(d), z=rnd(b, l, d).to(dt), dt_bias=rnd(d) - 2.0, dout=rnd(b, l, d).to(dt), state=rnd(b, d, n))
    for name in without:
        s[name] = None
    s["lengths"] = None if lengths is None else torch.tensor(lengths, device="cuda")
    return s


def reference(s, softplus=True, state=False, backward=True):
    """Results and their bounds without the last rounding, by name."""
    f = lambda t, *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda") if t is None else t.detach().double()  # noqa: E731
    x, A = f(s["x"]), f(s["A"])
    b, l, d = x.shape
    N = A.shape[1]
    n = torch.full((b,), l, device="cuda") if s["lengths"] is None else s["lengths"].clamp(0, l)
    inside = (torch.arange(l, device="cuda") < n[:, None])[..., None]
    clean = lambda t: torch.where(inside, t, 0.0)  # noqa: E731
    x, B, C = clean(x), clean(f(s["B"])), clean(f(s["C"]))
    D, v = f(s["D"], d), clean(f(s["dt"])) + f(s["dt_bias"], d)
    sig_v = torch.sigmoid(v) if softplus else torch.ones_like(v)
    step = clean(torch.logaddexp(v, torch.zeros_like(v)) if softplus else v)
    S = clean(step.abs() + v.abs() * sig_v)
    gate, z = torch.ones_like(x), None
    if s["z"] is not None:
        z = clean(f(s["z"]))
        sig = torch.sigmoid(z)
        gate = z * sig
    zr = 0.0 if z is None else z.abs()
    a = torch.exp(step[..., None] * A)
    c = 4 * (step[..., None] * A).abs() + 8 * S[..., None] * A.abs() + 2
    h = f(s["state"]) if state else torch.zeros(b, d, N, dtype=torch.float64, device="cuda")
    M, E = h.abs(), torch.zeros_like(h)
    hs, Ms, Es = [h], [M], [E]
    for i in range(l):
        u, um = step[:, i] * x[:, i], S[:, i] * x[:, i].abs()
        E = a[:, i] * E + (c[:, i] + 2) * U * a[:, i] * M + 12 * U * um[..., None] * B[:, i, None].abs() \
            + LOW * (M + x[:, i, :, None].abs() * B[:, i, None].abs())
        M = a[:, i] * M + um[..., None] * B[:, i, None].abs()
        h = a[:, i] * h + u[..., None] * B[:, i, None]
        hs.append(h), Ms.append(M), Es.append(E)
    hs, Ms, Es = (torch.stack(t, 1) for t in (hs, Ms, Es))
    fits = (Ms.amax((1, 3)) < 2.0 ** 100)                      # [b, d]
    y = (hs[:, 1:] * C[:, :, None]).sum(-1) + D * x
    ym = (Ms[:, 1:] * C[:, :, None].abs()).sum(-1) + (D * x).abs()
    ye = (C[:, :, None].abs() * (Es[:, 1:] + (N + 4) * U * Ms[:, 1:])).sum(-1) + 2 * U * (D * x).abs()
    R = {"out": (clean(y * gate), clean((ye + (zr + 8) * U * ym) * gate.abs())), "state": (hs[:, -1], Es[:, -1])}
    if not backward:
        return cut(R, fits)
    dout = clean(f(s["dout"]))
    dy, dr = dout * gate, (zr + 10) * U
    g, G, F = (torch.zeros_like(h) for _ in range(3))
    gs, Gs, Fs = [], [], []
    for i in reversed(range(l)):
        Cd = C[:, i, None] * dy[:, i, :, None]
        after = (a[:, i + 1], c[:, i + 1]) if i + 1 < l else (torch.zeros_like(h), torch.zeros_like(h))
        r = dr[:, i, :, None] if z is not None else dr
        F = after[0] * F + (after[1] + 2) * U * after[0] * G + r * Cd.abs() + LOW * G
        G = after[0] * G + Cd.abs()
        g = after[0] * g + Cd
        gs.append(g), Gs.append(G), Fs.append(F)
    gs, Gs, Fs = (torch.stack(t[::-1], 1) for t in (gs, Gs, Fs))
    fits &= Gs.amax((1, 3)) < 2.0 ** 100 if l else True
    k = 16 + l / 4 + b * (l / 64 + 1)
    ab = B[:, :, None].abs()
    gB, gBe, gBm = (gs * B[:, :, None]).sum(-1), (ab * (Fs + (N + 4) * U * Gs)).sum(-1), (ab * Gs).sum(-1)
    if z is not None:
        slope = sig * (1 + z * (1 - sig))
        R["dz"] = (clean(dout * y * slope), clean(dout.abs() * (ye * slope.abs() + (zr + 12) * U * ym * (sig * (1 + zr)))))
    R["dx"] = (clean(step * gB + D * dy), clean(S * (gBe + 12 * U * gBm) + LOW * gBm + (dr + 4 * U) * (D * dy).abs()))
    K = gs * a * hs[:, :-1]
    Km = Gs * a * Ms[:, :-1]
    Ke = a * (Fs * Ms[:, :-1] + Gs * Es[:, :-1]) + (c + 6) * U * Km
    kA, kAe = (K * A).sum(-1), ((Ke + (N + 4) * U * Km) * A.abs()).sum(-1)
    ds, dse = x * gB + kA, x.abs() * (gBe + 4 * U * gBm) + kAe
    dsm = x.abs() * gBm + (Km * A.abs()).sum(-1)
    slope_e = (v.abs() + 8) * U if softplus else 0.0
    R["ddt"] = (clean(ds * sig_v), clean((dse + (slope_e + 4 * U) * dsm) * sig_v + LOW * dsm))
    R["ddt_bias"] = (R["ddt"][0].sum((0, 1)), (R["ddt"][1] + k * U * clean(dsm * sig_v)).sum((0, 1)))
    R["dA"] = ((K * step[..., None]).sum((0, 1)), ((Ke + (k + 12) * U * Km) * S[..., None] + LOW * Km).sum((0, 1)))
    xs, xm = (step * x)[..., None], (S * x.abs())[..., None]
    R["dB"] = ((gs * xs).sum(2), (xm * (Fs + (90 + 12) * U * Gs) + LOW * x.abs()[..., None] * Gs).sum(2))
    drz = dr[..., None] if z is not None else dr
    R["dC"] = ((hs[:, 1:] * dy[..., None]).sum(2), (dy[..., None].abs() * (Es[:, 1:] + (drz + 90 * U) * Ms[:, 1:])).sum(2))
    R["dD"] = ((dy * x).sum((0, 1)), ((dr + k * U) * (dy * x).abs()).sum((0, 1)))
    return cut(R, fits)


def cut(R, fits):
    """Without bounds where a channel's numbers are too large."""
    where = {"out": fits[:, None], "dx": fits[:, None], "ddt": fits[:, None], "dz": fits[:, None], "state": fits[..., None],
             "dA": fits.all(0)[:, None], "dD": fits.all(0), "ddt_bias": fits.all(0), "dB": fits.all(1)[:, None, None],
             "dC": fits.all(1)[:, None, None]}
    return {n: (value, off, where[n].expand_as(value)) for n, (value, off) in R.items()}


def near(got, want, name, dt):
    value, off, fits = want[name]
    t, least = STEP[dt]
    assert got.dtype == dt and got.shape == value.shape, name
    bad = (got.double() - value).abs() / (t * value.abs() + off + least)
    bad = bad[fits]
    assert bad.numel() == 0 or bad.max() <= 1, (name, bad.max().item())


def call(s, softplus=True, **more):
    import metal_kans as mk
    return mk.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], softplus=softplus,
                             lengths=s["lengths"], **more)


def train(s, softplus=True):
    """The output and the gradients, by name."""
    leaves = [n for n in LEAVES if s[n] is not None]
    a = {**s, **{n: s[n].detach().requires_grad_(True) for n in leaves}}
    out = call(a, softplus)
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(leaves, torch.autograd.grad(out, [a[n] for n in leaves], s["dout"]))}}


def check(s, softplus=True):
    dt = s["x"].dtype
    want = reference(s, softplus)
    got = train(s, softplus)
    for n, t in got.items():
        near(t, want, n, torch.float32 if n in ("dA", "dD", "ddt_bias") else dt)
    with torch.no_grad():
        state = s["state"].clone()
        out = call(s, softplus, state=state)
        want = reference(s, softplus, state=True, backward=False)
        near(out, want, "out", dt)
        near(state, want, "state", torch.float32)
        assert torch.equal(call(s, softplus).view(torch.uint8), got["out"].view(torch.uint8))   # (bits: NaN is no NaN's equal)
    return got


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,l,d,n", [(1, 1, 1, 1), (2, 5, 3, 4), (1, 16, 16, 16), (1, 17, 64, 16), (2, 33, 70, 16), (3, 64, 130, 24),
                                     (1, 40, 17, 8), (2, 40, 20, 64), (1, 50, 65, 33), (2, 31, 16, 5), (1, 9, 7, 30), (4, 3, 200, 2)])
def test_sizes(cuda, b, l, d, n, dt):
    check(inputs(b, l, d, n, dt))


@pytest.mark.parametrize("n", [3, 8, 16, 20, 32, 64])
def test_chunks(cuda, n):
    """Long sequences of few channels go in chunks, whose borders are anywhere in the sequence."""
    check(inputs(1, 700, 40, n, torch.float32))
    check(inputs(2, 333, 9, n, torch.float32, lengths=[333, 100]))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lengths", [[0, 1, 2], [60, 33, 0], [-5, 1000, 59]])
def test_lengths(cuda, lengths, dt):
    check(inputs(3, 60, 21, 16, dt, lengths=lengths))


@pytest.mark.parametrize("without", [("z",), ("D",), ("dt_bias",), ("z", "D", "dt_bias")])
@pytest.mark.parametrize("softplus", [True, False])
def test_without(cuda, without, softplus):
    s = inputs(2, 50, 24, 16, torch.float32, without=without)
    if not softplus:
        s["dt"] = s["dt"].abs() * 0.1
    check(s, softplus)


@pytest.mark.parametrize("dt", TYPES)
def test_steps_as_they_are(cuda, dt):
    """No softplus, steps from 0 to 1."""
    s = inputs(2, 150, 24, 16, dt, without=("dt_bias",))
    s["dt"] = s["dt"].abs().clamp(max=1.0)
    check(s, softplus=False)


def test_extreme_steps(cuda):
    """Step sizes from below the smallest to the largest that matter: nothing left of a state, or all of it."""
    s = inputs(1, 40, 32, 16, torch.float32)
    s["dt"] = torch.linspace(-100.0, 60.0, 40 * 32, device="cuda").view(1, 40, 32)
    s["dt_bias"] = None
    check(s)
    s["A"] = -s["A"] * 1e-3       # states that grow
    s["dt"] = s["dt"].clamp(max=3.0)
    check(s)
    s["A"].zero_()                # states that stay
    check(s)


def test_growing_states_in_chunks(cuda):
    """A chunk may multiply a state by more than fp32 holds where there is none yet, or a small one: 700 steps of one,
    growing by up to 2^115 in a chunk (of 48 steps and more), inputs at the end and output gradients at the beginning only."""
    s = inputs(1, 700, 40, 16, torch.float32, without=("dt_bias", "z"))
    s["dt"] = torch.full_like(s["dt"], 1.0)
    s["A"] = s["A"].abs().clamp(max=1.6)
    s["x"][:, :690] = 0.0
    s["dout"][:, 10:] = 0.0
    check(s, softplus=False)
    s["A"][::2] = -1.0
    s["x"].fill_(1e-20)
    s["state"].fill_(1e-35)
    s["lengths"] = torch.tensor([650], device="cuda")
    check(s, softplus=False)


@pytest.mark.parametrize("dt", TYPES)
def test_masked_places_are_not_looked_at(cuda, dt):
    s = inputs(3, 150, 19, 16, dt, lengths=[0, 20, 150])
    behind = (torch.arange(150, device="cuda") >= s["lengths"][:, None])[..., None]
    names = ("x", "dt", "B", "C", "z", "dout")
    want = train({**s, **{n: torch.where(behind, 0.0, s[n]) for n in names}})
    for bad in (float("nan"), float("inf"), torch.finfo(dt).min):
        dirty = {**s, **{n: torch.where(behind, bad, s[n]) for n in names}}
        got = train(dirty)
        for n in want:
            assert torch.equal(got[n], want[n]), n
        for n in ("dx", "ddt", "dz", "dB", "dC", "out"):
            assert not got[n][behind.expand_as(got[n])].any(), n
        state = s["state"].clone()
        with torch.no_grad():
            call(dirty, state=state)
        assert state.isfinite().all() and torch.equal(state[0], s["state"][0])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("n", [16, 30])
def test_infinities_stay_where_they_belong(cuda, n, bad):
    """An infinite or NaN input reaches its own channel (B's and C's: all) from its step on, a gradient its channel up to its
    step, and what sums over them; everything else keeps its bits."""
    s = inputs(2, 150, 20, n, torch.float32, lengths=[150, 90])
    want = train(s)
    for name in ("x", "dt", "z"):
        hurt = {**s, name: s[name].clone()}
        hurt[name][1, 41, 7] = bad
        got = train(hurt)
        assert not got["out"][1, 41, 7].isfinite()
        for a, b in ((got["out"][0], want["out"][0]), (got["out"][1, :41], want["out"][1, :41]), (got["out"][1, :, :7], want["out"][1, :, :7]),
                     (got["out"][1, :, 8:], want["out"][1, :, 8:])):
            assert torch.equal(a, b), name
        others = torch.arange(20, device="cuda") != 7
        for k in ("dx", "ddt", "dz"):
            assert torch.equal(got[k][..., others], want[k][..., others]) and torch.equal(got[k][0], want[k][0]), (name, k)
            assert not got[k][1, 90:].any(), (name, k)
        for k in ("dA", "dD", "ddt_bias"):
            assert torch.equal(got[k][others], want[k][others]), (name, k)
        for k in ("dB", "dC"):
            assert torch.equal(got[k][0], want[k][0]) and not got[k][1, 90:].any(), (name, k)
    for name, at in (("B", 5), ("C", 2)):
        hurt = {**s, name: s[name].clone()}
        hurt[name][1, 41, at] = bad
        got = train(hurt)
        assert torch.equal(got["out"][0], want["out"][0]) and torch.equal(got["out"][1, :41], want["out"][1, :41])
        assert not got["out"][1, 90:].any() and not got["dC"][1, 90:].any() and not got["dB"][1, 90:].any()
    hurt = {**s, "dout": s["dout"].clone()}
    hurt["dout"][1, 41, 7] = bad
    got = train(hurt)
    for k in ("dx", "ddt", "dz", "dB", "dC"):
        assert torch.equal(got[k][0], want[k][0]) and torch.equal(got[k][1, 42:], want[k][1, 42:]), k
    state = s["state"].clone()
    hurt = {**s, "x": s["x"].clone()}
    hurt["x"][1, 41, 7] = bad
    with torch.no_grad():
        call(hurt, state=state)
    other = s["state"].clone()
    with torch.no_grad():
        call(s, state=other)
    assert torch.equal(state[0], other[0]) and torch.equal(state[1, 8:], other[1, 8:]) and not state[1, 7].isfinite().all()


def test_long_padding(cuda):
    """Whole tiles and chunks behind the ends of the sequences."""
    for dt, b, l, d, n, lengths in ((torch.float32, 4, 700, 20, 16, [3, 700, 0, 350]), (torch.bfloat16, 3, 129, 70, 24, [16, 1, 128]),
                                    (torch.float16, 2, 64, 600, 64, [32, 0])):
        check(inputs(b, l, d, n, dt, lengths=lengths))
        s = inputs(b, l, d, n, dt, lengths=lengths)
        used = [torch.full(shape, 7.0, device="cuda", dtype=dt) for shape in ((b, l, d), (b, l, n)) for _ in range(4)]
        del used     # (memory that the results are likely to get holds no zeros)
        got = train(s)
        for i, end in enumerate(lengths):
            for k in ("out", "dx", "ddt", "dz", "dB", "dC"):
                assert not got[k][i, end:].any(), k


def test_odd_addresses_of_the_state(cuda):
    for n in (16, 7):
        s = inputs(3, 1, 33, n, torch.float32)
        space = torch.zeros(3 * 33 * n + 1, device="cuda")
        odd = space[1:].view(3, 33, n)
        for l in (1, 20):
            s = inputs(3, l, 33, n, torch.float32)
            odd.copy_(s["state"])
            state = s["state"].clone()
            with torch.no_grad():
                assert torch.equal(call(s, state=odd), call(s, state=state)) and torch.equal(odd, state) and space[0] == 0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d,n", [(37, 16), (70, 24), (5, 3), (64, 64)])
def test_pieces_are_the_whole(cuda, d, n, dt):
    """A prompt in pieces, then single tokens, against the definition over the whole sequence."""
    s = inputs(2, 60, d, n, dt)
    want = reference(s, state=True, backward=False)
    state, at, out = s["state"].clone(), 0, []
    with torch.no_grad():
        for count in (30, 1, 2, 20, 1, 1, 1, 1, 1, 1, 1):
            piece = {k: v[:, at:at + count] if k in ("x", "dt", "B", "C", "z") else v for k, v in s.items()}
            version = state._version
            out.append(call(piece, state=state))
            assert state._version > version
            at += count
    assert at == 60
    near(torch.cat(out, 1), want, "out", dt)
    near(state, want, "state", torch.float32)


@pytest.mark.parametrize("n", [16, 7])
def test_single_tokens(cuda, n):
    """One token each of many sequences, some of which have none."""
    for dt in TYPES:
        s = inputs(33, 1, 130, n, dt, lengths=[i % 3 for i in range(33)])
        state = s["state"].clone()
        with torch.no_grad():
            out = call(s, state=state)
        want = reference(s, state=True, backward=False)
        near(out, want, "out", dt)
        near(state, want, "state", torch.float32)
        assert torch.equal(state[0], s["state"][0]) and not out[0].any()


def test_orders_of_memory(cuda):
    """Halves of one projection, odd addresses, and channels that do not lie side by side."""
    for dt in TYPES:
        s = inputs(2, 33, 24, 16, dt)
        want = train(s)

        def inside(t, at):
            wide = torch.zeros(*t.shape[:2], 2 * t.shape[2] + 13, device="cuda", dtype=dt)
            wide[..., at:at + t.shape[2]] = t
            return wide[..., at:at + t.shape[2]]
        for move in (lambda t: inside(t, 5), lambda t: inside(t, 16), lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                     lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
            m = {k: move(v) if k in ("x", "dt", "B", "C", "z", "dout") else v for k, v in s.items()}
            m["A"] = torch.cat((s["A"].new_zeros(1), s["A"].flatten()))[1:].view(24, 16)   # (4 bytes past a multiple of 16)
            got = train(m)
            assert all(torch.equal(got[k], want[k]) for k in want)
            state, other = s["state"].clone(), s["state"].clone()
            with torch.no_grad():
                assert torch.equal(call(m, state=state), call(s, state=other)) and torch.equal(state, other)
                one = {k: v[:, 7:8] if k in ("x", "dt", "B", "C", "z") else v for k, v in m.items()}
                same = {k: v[:, 7:8].contiguous() if k in ("x", "dt", "B", "C", "z") else v for k, v in s.items()}
                assert torch.equal(call(one, state=state), call(same, state=other)) and torch.equal(state, other)


def test_far_steps(cuda):
    """Steps 2^23 elements and more apart, batches that repeat, and single steps whose strides mean nothing."""
    s = inputs(1, 3, 24, 16, torch.float16)
    want = train(s)
    far = {}
    for k in ("x", "dt", "B", "C", "z"):
        space = torch.zeros(3 << 23, device="cuda", dtype=torch.float16)
        far[k] = space.as_strided((1, 3, s[k].shape[2]), (1, 1 << 23, 1))
        far[k].copy_(s[k])
    got = train({**s, **far})
    assert all(torch.equal(got[k], want[k]) for k in want)
    two = {k: v.expand(2, *v.shape[1:]) if k in ("x", "dt", "B", "C", "z") else v for k, v in s.items()}
    with torch.no_grad():
        assert torch.equal(call(two), want["out"].expand(2, 3, 24))
        one = {k: v[:, 1:2].as_strided((1, 1, v.shape[2]), (0, 1 << 40, 1), v[:, 1:2].storage_offset())
               if k in ("x", "dt", "B", "C", "z") else v for k, v in s.items()}
        same = {k: v[:, 1:2].contiguous() if k in ("x", "dt", "B", "C", "z") else v for k, v in s.items()}
        assert torch.equal(call(one), call(same))
        assert torch.equal(call(one, state=s["state"].clone()), call(same, state=s["state"].clone()))


def test_more_sums_than_threads(cuda):
    """Partial rows of B's and C's gradients that are more than 2^32 numbers: one channel that forgets at once, 64 states."""
    steps, n = (1 << 25) + 100, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dt, dout = (torch.randn(1, steps, 1, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(3))
    dt.fill_(1.0)
    wide = [torch.empty(1, steps, n, device="cuda", dtype=torch.bfloat16).normal_(generator=g).requires_grad_(True) for _ in range(2)]
    A = torch.full((1, n), -1000.0, device="cuda")
    import metal_kans as mk
    out = mk.selective_scan(x, dt, A, wide[0], wide[1], softplus=False)
    dB, dC = torch.autograd.grad(out, wide, dout)
    # (h = x B in each step, so dB = C dout x and dC = dout x B: two products in fp32 and a rounding)
    for first in (0, steps // 2, steps - (1 << 16)):
        at = slice(first, first + (1 << 16))
        both = dout[:, at].double() * x[:, at].double()
        for got, other in ((dB, wide[1]), (dC, wide[0])):
            want = both * other.detach()[:, at].double()
            assert bool(((got[:, at].double() - want).abs() <= want.abs() * (2 ** -8 + 4 * 2 ** -24) + 2 ** -126).all())


def test_nothing(cuda):
    for b, l in ((0, 5), (2, 0)):
        s = inputs(b, l, 12, 16, torch.float32)
        got = train(s)
        assert got["out"].shape == (b, l, 12) and not got["dA"].any() and not got["dD"].any() and not got["ddt_bias"].any()
        state = s["state"].clone()
        with torch.no_grad():
            call(s, state=state)
        assert torch.equal(state, s["state"])


def test_gradients_are_the_differences(cuda):
    """Against central differences of the 64-bit definition."""
    s = inputs(2, 20, 6, 16, torch.float32, lengths=[20, 13])
    got = train(s)
    for name, at in (("x", (0, 3, 2)), ("dt", (1, 12, 5)), ("dt", (0, 0, 0)), ("A", (4, 9)), ("B", (0, 5, 3)), ("C", (1, 2, 15)), ("D", (2,)),
                     ("z", (0, 19, 1)), ("dt_bias", (3,))):
        ends = []
        for e in (1e-4, -1e-4):
            moved = {n: t.double().clone() if t.is_floating_point() else t for n, t in s.items()}
            moved[name][at] += e
            ends.append((reference(moved, backward=False)["out"][0] * moved["dout"]).sum())
        slope = (ends[0] - ends[1]) / 2e-4
        assert abs(slope - got["d" + name][at]) <= 2e-5 * max(1.0, abs(slope)), name


def test_some_gradients(cuda):
    s = inputs(2, 150, 40, 16, torch.float32)
    want = train(s)
    for leaves in [[n] for n in LEAVES] + [["x", "A", "z"], ["B", "dt_bias"]]:
        a = {**s, **{n: s[n].detach().requires_grad_(True) for n in leaves}}
        out = call(a)
        for n, g in zip(leaves, torch.autograd.grad(out, [a[n] for n in leaves], s["dout"])):
            assert torch.equal(g, want["d" + n]), n


@pytest.mark.parametrize("l", [50, 300])
def test_machinery(cuda, l):
    """The same bits on every run, in a graph that is replayed and on another stream; guarded inputs; no second derivative."""
    s = inputs(2, l, 40, 16, torch.float32, lengths=[l, 31])
    for n in LEAVES:
        s[n].requires_grad_(True)
    state = s["state"].clone()

    def step():
        out = call(s)
        grads = torch.autograd.grad(out, [s[n] for n in LEAVES], s["dout"])
        with torch.no_grad():
            served = call(s, state=state)
        return [out.detach(), *grads, served, state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2, 3):
        new = inputs(2, l, 40, 16, torch.float32, seed=seed)
        with torch.no_grad():
            for n in (*LEAVES, "dout"):
                s[n].copy_(new[n])
            s["lengths"].copy_(torch.tensor([seed, l - seed], device="cuda"))
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
    out = call(s)
    dx, = torch.autograd.grad(out, s["x"], s["dout"], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()
    out = call(s)
    with torch.no_grad():
        s["dt"].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, s["x"], s["dout"])
    with pytest.raises(RuntimeError, match="no gradients"):
        call(s, state=state)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("l,d,n,lengths", [(15, 20, 16, [15, 15]), (16, 20, 16, [16, 13]), (33, 20, 30, [33, 2]), (50, 20, 64, [47, 50]),
                                           (701, 40, 16, [701, 333]), (700, 9, 5, [1, 700])])
def test_the_last_step_may_be_infinite(cuda, l, d, n, lengths, dt, bad):
    """An infinite or NaN input of a sequence's last step is in the state behind it, which no step's decay meets: dA, dx and all that
    belongs to other steps keep their bits."""
    s = inputs(2, l, d, n, dt, lengths=lengths)
    for b, end in enumerate(lengths):
        s["x"][b, end - 1, 7] = 0.0
    want = train(s)
    for b, end in enumerate(lengths):
        s["x"][b, end - 1, 7] = bad
    got = train(s)
    for k in ("dA", "dx"):
        assert got[k].isfinite().all() and torch.equal(got[k], want[k]), k
    for b, end in enumerate(lengths):
        assert not got["out"][b, end - 1, 7].isfinite() and not got["dC"][b, end - 1].isfinite().any()
        for k in ("out", "ddt", "dz", "dB", "dC"):
            assert torch.equal(got[k][b, :end - 1], want[k][b, :end - 1]) and not got[k][b, end:].any(), k


@pytest.mark.parametrize("l,lengths", [(1, None), (1, [0, 1]), (15, None), (40, [17, 0]), (333, None), (333, [100, 333])])
def test_the_largest_decays(cuda, l, lengths):
    """A of the type's lowest value: a step leaves nothing of the state, none (behind a length, or of size zero) all of it.
    Minus infinity is the same for steps of any size."""
    lowest = torch.finfo(torch.float32).min
    for softplus in (True, False):
        s = inputs(2, l, 20, 16, torch.float32, lengths=lengths, without=() if softplus else ("dt_bias",))
        s["A"][3], s["A"][4], s["A"][5, ::2] = lowest, -2.5e38, lowest
        if not softplus:
            s["dt"] = s["dt"].abs()
            s["dt"][0, ::3] = 0.0
        got, want = train(s, softplus), reference(s, softplus)
        for k in got:
            if softplus or k != "ddt":   # (A times a state that a step of size zero leaves is beyond fp32)
                near(got[k], want, k, torch.float32)
        state = s["state"].clone()
        with torch.no_grad():
            out = call(s, softplus, state=state)
            want = reference(s, softplus, state=True, backward=False)
            near(out, want, "out", torch.float32)
            near(state, want, "state", torch.float32)
            if softplus:
                again = s["state"].clone()
                infinite = {**s, "A": torch.where(s["A"] < -2e38, float("-inf"), s["A"])}
                assert torch.equal(call(infinite, state=again), out) and torch.equal(again, state)


def test_steps_that_share_memory(cuda):
    """Steps that lie in each other's memory, an infinite or NaN input among them: it stays with its own steps and channels, though
    what lies behind a length is another step's channel."""
    names = ("x", "B", "C")
    for dt in TYPES:
        for l, lengths in ((40, [21, 9]), (333, [100, 333]), (37, None)):
            for name in names:
                for bad in (float("inf"), float("nan")):
                    s = inputs(2, l, 20, 16, dt, lengths=lengths)
                    gen = torch.Generator("cuda").manual_seed(5)
                    for k in ("x", "dt", "B", "C", "z"):
                        width = s[k].shape[2]
                        long = torch.randn(2, l + width, device="cuda", generator=gen).to(dt)
                        if k == name:    # (the last step's last but two)
                            for b in range(2):
                                long[b, (lengths[b] if lengths else l) - 1 + width - 3] = bad
                        s[k] = long.as_strided((2, l, width), (long.stride(0), 1, 1))
                    apart = {k: v.contiguous() if k in ("x", "dt", "B", "C", "z") else v for k, v in s.items()}
                    want, got = train(apart), train(s)
                    for k in want:
                        assert torch.equal(got[k].nan_to_num(7.0, 8.0, 9.0), want[k].nan_to_num(7.0, 8.0, 9.0)), (name, k)
                    state, other = s["state"].clone(), s["state"].clone()
                    with torch.no_grad():
                        call(s, state=state)
                        call(apart, state=other)
                    assert torch.equal(state.nan_to_num(7.0, 8.0, 9.0), other.nan_to_num(7.0, 8.0, 9.0)), name


# 4 ceil(D / 64) B waves: whole sequences from 1024 on, a grid above 512 workgroups in the second and the last
@pytest.mark.parametrize("b,l,d,n,dt,lengths", [(4, 131, 4099, 4, torch.float32, [131, 70, 17, 0]), (9, 131, 4099, 3, torch.bfloat16, None),
                                                (5, 203, 3300, 8, torch.float16, [203, 202, 96, 1, 150]), (4, 300, 4099, 2, torch.bfloat16, [300, 299, 129, 16]),
                                                (17, 150, 2050, 16, torch.float32, [150 - 9 * i for i in range(17)])])
def test_long_sequences_that_stay_whole(cuda, b, l, d, n, dt, lengths):
    """Large batches are not cut in chunks: many tiles one after the other, ends in the middle of a sequence and of a tile."""
    check(inputs(b, l, d, n, dt, lengths=lengths))
