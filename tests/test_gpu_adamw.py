"""AdamW over many tensors (run on an MI355X).

Against a plain implementation in 64 bits on the same start: each fp32 operation of the step rounds once
(2^-24 relative), so after one step the moments are within 4 roundings of their terms and a parameter
within 2 roundings of itself and 8 of its update.  A 16-bit parameter is the rounding of its master.  The
8-bit codes follow from IEEE operations alone and are compared with an elementwise fp32 restatement, code for code.
"""
import copy

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def cuda(gpu):
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    return torch.device("cuda:0")


def make(shapes, dt, seed, scale=1e-2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda").to(dt)) for s in shapes]
    for p in params:
        p.grad = (scale * torch.randn(p.shape, generator=gen, device="cuda")).to(dt)
    return params


def step64(w, g, m, v, t, lr, b1, b2, eps, wd):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    upd = lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps)
    return w * (1 - lr * wd) - upd, m, v, upd


def blocks(x):
    x = x.reshape(-1)
    return np.concatenate([x, np.zeros(-x.size % 256, x.dtype)]).reshape(-1, 256)


def codes32(m, v):
    """Codes and scales of 8-bit states, operation by operation in fp32."""
    f = np.float32
    mb, vb = blocks(m), blocks(v)
    ms = np.maximum(np.abs(mb).max(1), f(2.0 ** -126))
    vs = np.maximum(vb.max(1), f(2.0 ** -126))
    mq = np.rint(f(127) * np.sqrt(np.abs(mb) * (f(1) / ms)[:, None])) * np.sign(mb)
    vq = np.rint(f(255) * np.sqrt(np.sqrt(vb * (f(1) / vs)[:, None])))
    vq = np.where(vb > 0, np.maximum(vq, 1), 0)
    return mq.astype(np.int8).reshape(-1)[:m.size], ms, vq.astype(np.uint8).reshape(-1)[:v.size], vs


def values32(mq, ms, vq, vs, n):
    f = np.float32
    t = blocks(mq).astype(f) * f(1 / 127)
    m = (ms[:, None] * (t * np.abs(t))).reshape(-1)[:n]
    t = blocks(vq).astype(f) * f(1 / 255)
    t = t * t
    return m, (vs[:, None] * (t * t)).reshape(-1)[:n]


SHAPES = [(1,), (0,), (255,), (256,), (257,), (7, 13), (3, 5, 70), (4096,), (4097,), (33, 1025)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hyper", [(1e-3, (0.9, 0.999), 1e-8, 1e-2), (0.1, (0.0, 0.5), 1e-3, 0.0), (0.0, (0.9, 0.99), 0.0, 0.1)])
def test_states_in_32_bits_against_64(cuda, dt, hyper):
    import metal_kans as mk
    lr, (b1, b2), eps, wd = hyper
    params = make(SHAPES, DT[dt], 1)
    opt = mk.TorchAdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd)
    w = [p.detach().double().cpu().numpy() for p in params]
    m, v = [np.zeros_like(a) for a in w], [np.zeros_like(a) for a in w]
    g = [p.grad.double().cpu().numpy() for p in params]
    for t in range(1, 4):
        opt.step()
        for i, p in enumerate(params):
            w[i], m[i], v[i], upd = step64(w[i], g[i], m[i], v[i], t, lr, b1, b2, eps, wd)
            st = opt.state[p]
            assert st["step"] == t
            got = (st["master"] if dt != "f32" else p).detach().double().cpu().numpy()
            # the roundings of t steps add up; a moment's error moves the update by as much relatively
            assert np.all(np.abs(st["exp_avg"].double().cpu().numpy() - m[i]) <= 4 * t * U * np.abs(g[i]))
            assert np.all(np.abs(st["exp_avg_sq"].double().cpu().numpy() - v[i]) <= 5 * t * U * v[i])
            unit = lr / (1 - b1 ** t) * np.abs(g[i]) / (np.sqrt(v[i] / (1 - b2 ** t)) + eps + 1e-300)
            assert np.all(np.abs(got - w[i]) <= t * U * (2 * np.abs(w[i]) + 12 * t * np.maximum(np.abs(upd), unit)))
            if dt != "f32":
                assert torch.equal(p.detach(), st["master"].to(DT[dt]))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_states_in_8_bits_code_for_code(cuda, dt):
    import metal_kans as mk
    f = np.float32
    lr, b1, b2, eps, wd = 1e-2, 0.9, 0.99, 1e-8, 1e-2
    params = make(SHAPES, DT[dt], 2)
    params[-1].grad[::3] = 0                        # whole blocks without a gradient
    params[-2].grad *= 0
    params[-3].grad[::2] *= 1e-3                    # widely spread magnitudes in a block
    opt = mk.TorchAdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=8)
    w = [p.detach().float().cpu().numpy().reshape(-1) for p in params]
    st = [(np.zeros(p.numel(), np.int8), np.zeros(-(-p.numel() // 256), f), np.zeros(p.numel(), np.uint8),
           np.zeros(-(-p.numel() // 256), f)) for p in params]
    for t in range(1, 4):
        opt.step()
        for i, p in enumerate(params):
            g = p.grad.float().cpu().numpy().reshape(-1)
            m, v = values32(*st[i], g.size)
            m = m * f(b1) + g * f(1 - b1)
            v = v * f(b2) + (g * g) * f(1 - b2)
            size, root = f(lr / (1 - b1 ** t)), f(1 / np.sqrt(1 - b2 ** t))
            w[i] = w[i] * f(1 - lr * wd) - size * (m / (np.sqrt(v) * root + f(eps)))
            if g.size:
                st[i] = codes32(m, v)
            s = opt.state[p]
            got = (s["master"] if dt != "f32" else p).detach().cpu().numpy().reshape(-1)
            np.testing.assert_array_equal(got, w[i])
            for name, want in zip(("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"), st[i]):
                np.testing.assert_array_equal(s[name].cpu().numpy().reshape(-1), want, err_msg=name)
    flat = opt.flat_state()[0]
    at = 0
    for i, p in enumerate(params):
        m, v = values32(*st[i], p.numel())
        np.testing.assert_array_equal(flat["exp_avg"][at:at + p.numel()].cpu().numpy(), m)
        np.testing.assert_array_equal(flat["exp_avg_sq"][at:at + p.numel()].cpu().numpy(), v)
        at += -(-p.numel() // 256) * 256
    assert at == flat["exp_avg"].numel()


def test_8_bit_states_hold_their_moments(cuda):
    """A code's value is within half a step of the moment: |m| within sqrt(s |m|) / 127 and v^(1/4) within
    s^(1/4) / 510 (or, near zero, a whole step), plus the half step's square."""
    import metal_kans as mk
    p = make([(64, 300)], torch.float32, 3)
    opt = mk.TorchAdamW(p, betas=(0.0, 0.0), state_bits=8)
    opt.step()
    g = p[0].grad.double().cpu().numpy().reshape(-1)
    flat = opt.flat_state()[0]
    s = np.repeat(np.abs(blocks(g)).max(1), 256)[:g.size]
    m = flat["exp_avg"][:g.size].double().cpu().numpy()
    v = flat["exp_avg_sq"][:g.size].double().cpu().numpy()
    half = 0.5 / 127
    assert np.all(np.abs(m - g) <= (1 + 1e-5) * (2 * half * np.sqrt(s * np.abs(g)) + half * half * s))
    assert np.all(np.abs(np.sqrt(np.sqrt(v)) - np.sqrt(np.abs(g))) <= np.sqrt(s) / 255 * (1 + 1e-5))


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_groups(cuda, bits):
    """More tensors than one launch holds, two groups, two dtypes, a parameter without a gradient: the same
    as each tensor in an optimizer of its own."""
    import metal_kans as mk
    shapes = [(3 + i % 70, 1 + i % 11) for i in range(210)]
    a = make(shapes, torch.float32, 4) + make(shapes[:20], torch.bfloat16, 5)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    a[7].grad = b[7].grad = None
    groups = [dict(params=a[:100], lr=1e-2), dict(params=a[100:], weight_decay=0.3)]
    opt = mk.TorchAdamW(groups, state_bits=bits)
    singles = [mk.TorchAdamW([q], state_bits=bits, **(dict(lr=1e-2) if i < 100 else dict(weight_decay=0.3)))
               for i, q in enumerate(b)]
    for _ in range(2):
        opt.step()
        for o in singles:
            o.step()
    for i, (p, q) in enumerate(zip(a, b)):
        assert torch.equal(p, q), i
    assert not opt.state.get(a[7])
    a[7].grad = torch.ones_like(a[7])
    opt.step()
    assert opt.state[a[7]]["step"] == 1 and opt.state[a[8]]["step"] == 3


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_alignment_and_strides(cuda, bits, dt):
    """Parameters and gradients at odd addresses, transposed parameters, gradients in another order."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(6)
    base = torch.randn(20000, generator=gen, device="cuda").to(DT[dt])
    grads = torch.randn(20000, generator=gen, device="cuda").to(DT[dt])
    want, got = [], []
    for odd in (0, 1, 3):
        p = torch.nn.Parameter(base[odd:odd + 5000].clone())
        q = base.clone()[odd:odd + 5000].requires_grad_(True)
        p.grad, q.grad = grads[:5000].clone(), grads.clone()[:5000]
        if odd == 3:
            q.grad = torch.cat([grads[:1], grads])[1:5001]
        want.append(p)
        got.append(q)
    p = torch.nn.Parameter(base[:6000].view(60, 100).clone())
    q = base[:6000].clone().view(60, 100).t().contiguous().t().requires_grad_(True)   # strides (1, 60)
    p.grad, q.grad = grads[:6000].view(60, 100).clone(), grads[:6000].view(60, 100).clone()
    a, b = mk.TorchAdamW(want, state_bits=32), mk.TorchAdamW(got, state_bits=32)
    c = mk.TorchAdamW([p], state_bits=32)
    d = mk.TorchAdamW([q], state_bits=32)
    for o in (a, b, c, d):
        o.step()
    for x, y in zip(want + [p], got + [q]):
        assert torch.equal(x, y)
    assert torch.equal(c.state[p]["exp_avg"], d.state[q]["exp_avg"])
    e = mk.TorchAdamW([want[0]], state_bits=bits)
    e.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(cuda, bits):
    import metal_kans as mk
    a = make([(40, 33), (100,)], torch.bfloat16, 7)
    opt = mk.TorchAdamW(a, lr=1e-2, state_bits=bits)
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad
    other = mk.TorchAdamW(b, state_bits=bits)
    other.load_state_dict(sd)
    assert other.param_groups[0]["lr"] == 1e-2
    opt.step()
    other.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for name, t in opt.state[p].items():
            assert torch.equal(t, other.state[q][name]) if isinstance(t, torch.Tensor) else t == other.state[q][name]
    # refused: the other width, a wrong shape; the states stay as they were
    with pytest.raises(ValueError):
        mk.TorchAdamW(b, state_bits=40 - bits).load_state_dict(sd)
    sd["state"][0]["exp_avg"] = sd["state"][0]["exp_avg"][:3]
    before = other.state[b[0]]["exp_avg"].clone()
    with pytest.raises(ValueError):
        other.load_state_dict(sd)
    assert torch.equal(other.state[b[0]]["exp_avg"], before)
    # cleared: the next step starts anew, from the parameter's own value
    other.state.clear()
    other.step()
    assert other.state[b[0]]["step"] == 1
    twin = pickle_copy(opt)
    assert torch.equal(twin.state[twin.param_groups[0]["params"][0]]["exp_avg"], opt.state[a[0]]["exp_avg"])


def pickle_copy(opt):
    return copy.deepcopy(opt)


def test_infinite_gradients_stay_visible(cuda):
    """fp32 states: only the elements concerned; 8-bit states: their block from the next step on."""
    import metal_kans as mk
    for bits in (32, 8):
        p = make([(1024,)], torch.float32, 8)
        p[0].grad[300] = float("inf")
        p[0].grad[301] = float("nan")
        opt = mk.TorchAdamW(p, state_bits=bits)
        opt.step()
        bad = ~torch.isfinite(p[0].detach())
        assert bad.nonzero().flatten().tolist() == [300, 301]
        flat = opt.flat_state()[0]
        lost = ~torch.isfinite(flat["exp_avg"])
        assert lost[300] and lost[301] and int(lost.sum()) == (2 if bits == 32 else 256)
        assert not lost[:256].any() and not lost[512:].any()


def test_module_sees_the_step(cuda):
    """The layer re-tiles its weights after a step (which writes them behind torch's back)."""
    import metal_kans as mk
    np.random.seed(0)
    m = mk.TorchMetalKANLinear(24, 40, degree=5).cuda()
    x = torch.rand(8, 24, device="cuda")
    opt = mk.TorchAdamW(m.parameters(), lr=0.1)
    m(x).square().mean().backward()
    before = m(x).detach().clone()
    opt.step()
    after = m(x).detach()
    m2 = mk.TorchMetalKANLinear(24, 40, degree=5).cuda()
    m2.load_state_dict(m.state_dict())
    assert torch.equal(after, m2(x).detach()) and not torch.equal(before, after)


def test_streams_and_capture(cuda):
    """A step on a side stream follows the gradient made there; a capturing stream is refused."""
    import metal_kans as mk
    p = make([(300000,)], torch.float32, 9)
    q = [torch.nn.Parameter(p[0].detach().clone())]
    a, b = mk.TorchAdamW(p), mk.TorchAdamW(q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(5):
            q[0].grad = p[0].grad * 1.0
            b.step()
    s.synchronize()
    for _ in range(5):
        a.step()
    assert torch.equal(p[0], q[0])
    g = torch.cuda.CUDAGraph()
    with pytest.raises(Exception, match="captur"):
        with torch.cuda.graph(g):
            a.step()
    a.step()
    assert a.state[p[0]]["step"] == 6


def test_refusals(cuda):
    import metal_kans as mk
    p = [torch.nn.Parameter(torch.zeros(4, device="cuda"))]
    for bad in (dict(state_bits=16), dict(lr=-1), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0),
                dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            mk.TorchAdamW(p, **bad)
    with pytest.raises(TypeError):
        mk.TorchAdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64, device="cuda"))])
    with pytest.raises(ValueError):
        mk.TorchAdamW([torch.zeros(4, 4, device="cuda")[:, :2].requires_grad_(True)])
    cpu = [torch.nn.Parameter(torch.zeros(4))]
    cpu[0].grad = torch.zeros(4)
    with pytest.raises(ValueError):
        mk.TorchAdamW(cpu).step()
    empty = torch.nn.Parameter(torch.zeros(0, 3, device="cuda"))
    empty.grad = torch.zeros_like(empty)
    for bits in (8, 32):
        mk.TorchAdamW([empty], state_bits=bits).step()
    p[0].grad = torch.sparse_coo_tensor([[1]], [1.0], (4,), device="cuda")
    with pytest.raises(TypeError):
        mk.TorchAdamW(p).step()
    p[0].grad = None
    opt = mk.TorchAdamW(p)
    opt.step()                     # no gradient anywhere: nothing to do
    assert not opt.state.get(p[0])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_parameter_in_another_order(cuda, dt):
    """A parameter whose elements are put in another order between steps (a change of memory format) keeps its states."""
    import metal_kans as mk
    a, b = make([(30, 50), (2, 3, 4, 5)], DT[dt], 10), make([(30, 50), (2, 3, 4, 5)], DT[dt], 10)
    one, two = mk.TorchAdamW(a, lr=0.1), mk.TorchAdamW(b, lr=0.1)
    for i in range(4):
        one.step()
        two.step()
        for p, q in zip(a, b):
            assert torch.equal(p, q), i
            for name, s in one.state[p].items():
                assert torch.equal(s, two.state[q][name]) if isinstance(s, torch.Tensor) else s == two.state[q][name]
        if i == 0:
            b[0].data = b[0].data.t().contiguous().t()
            b[1].data = b[1].data.contiguous(memory_format=torch.channels_last)
        elif i == 1:
            b[0].grad = b[0].grad.t().contiguous().t()
        elif i == 2:
            b[0].data, b[1].data = b[0].data.contiguous(), b[1].data.permute(3, 0, 2, 1).contiguous().permute(1, 3, 2, 0)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameter_with_gaps_after_a_step(cuda, bits):
    """Elements that do not lie side by side any more are refused, and nothing is written."""
    import metal_kans as mk
    for started in (False, True):
        p = make([(6, 40)], torch.float32, 11)
        opt = mk.TorchAdamW(p, lr=0.1, state_bits=bits)
        if started:
            opt.step()
        states = {n: s.clone() for n, s in opt.state[p[0]].items() if isinstance(s, torch.Tensor)} if started else {}
        big = torch.full((6, 64), 3.0, device="cuda")
        for view in (big[:, :40], big.view(-1)[:1].expand(6, 40), big[:, 4:44]):
            p[0].data = view
            with pytest.raises(ValueError, match="dense"):
                opt.step()
        assert (big == 3.0).all() and len(opt.state.get(p[0], {})) == (len(states) + 1 if started else 0)
        for n, s in states.items():
            assert torch.equal(opt.state[p[0]][n], s)
        p[0].data = torch.zeros(40, 6, device="cuda")    # as many elements in another shape
        if started:
            with pytest.raises(ValueError):
                opt.step()
        p[0].data = torch.zeros(6, 40, device="cuda")
        p[0].grad = torch.ones(6, 40, device="cuda")
        opt.step()
        assert opt.state[p[0]]["step"] == (2 if started else 1)


def test_8_bit_states_belong_to_an_order(cuda):
    """The scales are those of blocks in the parameter's order of memory: in another one the codes mean nothing."""
    import metal_kans as mk
    p = make([(30, 50)], torch.float32, 12)
    opt = mk.TorchAdamW(p, state_bits=8)
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    p[0].data = p[0].data.t().contiguous().t()
    before = p[0].detach().clone()
    with pytest.raises(ValueError, match="order"):
        opt.step()
    assert torch.equal(p[0].detach(), before) and opt.state[p[0]]["step"] == 1
    q = [torch.nn.Parameter(before.clone(memory_format=torch.preserve_format))]
    assert q[0].stride() == (1, 30)
    with pytest.raises(ValueError, match="order"):
        mk.TorchAdamW(q, state_bits=8).load_state_dict(sd)
    opt.state.clear()
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    twin = mk.TorchAdamW(q, state_bits=8)
    twin.load_state_dict(sd)
    q[0].data.copy_(p[0].data)
    q[0].grad = p[0].grad
    opt.step()
    twin.step()
    assert torch.equal(p[0], q[0]) and twin.state[q[0]]["step"] == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_assigned_states_are_taken(cuda, bits):
    """A state tensor that a program puts in the place of the optimizer's own counts from then on."""
    import metal_kans as mk
    a, b = make([(40, 33), (100,)], torch.bfloat16, 14), make([(40, 33), (100,)], torch.bfloat16, 14)
    one, two = mk.TorchAdamW(a, lr=0.1, state_bits=bits), mk.TorchAdamW(b, lr=0.1, state_bits=bits)
    one.step()
    two.step()
    sd = copy.deepcopy(two.state_dict())
    for name in list(one.state[a[0]]):
        if name != "step":
            new = one.state[a[0]][name].clone()
            new = new // 2 if not new.is_floating_point() else new * 0.5
            one.state[a[0]][name] = new
            sd["state"][0][name] = new.clone()
    one.state[a[1]]["exp_avg"] = torch.zeros_like(one.state[a[1]]["exp_avg"])
    sd["state"][1]["exp_avg"] = torch.zeros_like(sd["state"][1]["exp_avg"])
    two.load_state_dict(sd)
    for x, y in zip(one.flat_state(), two.flat_state()):
        for name in ("exp_avg", "exp_avg_sq", "master"):
            assert torch.equal(x[name], y[name]), name
    one.state[a[1]]["exp_avg_sq"] = one.state[a[1]]["exp_avg_sq"].clone()
    for _ in range(2):
        one.step()
        two.step()
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            for name, s in one.state[p].items():
                assert torch.equal(s, two.state[q][name]) if isinstance(s, torch.Tensor) else s == two.state[q][name]
    one.state[a[0]]["exp_avg"] = one.state[a[0]]["exp_avg"][:3].clone()
    with pytest.raises(ValueError):
        one.step()
    del one.state[a[0]]["exp_avg"]
    with pytest.raises(ValueError):
        one.step()


def test_hooks_of_a_loaded_state(cuda):
    """Hooks before a state dict is loaded may replace it, those behind run when it is there; a refused one runs no more."""
    import metal_kans as mk
    a, b = make([(20,)], torch.float32, 15), make([(20,)], torch.float32, 15)
    one, two = mk.TorchAdamW(a, lr=0.1), mk.TorchAdamW(b)
    one.step()
    seen = []

    def before(opt, sd):
        seen.append(("before", len(opt.state)))
        sd = copy.deepcopy(sd)
        sd["param_groups"][0]["lr"] = 0.25
        return sd
    two.register_load_state_dict_pre_hook(before)
    two.register_load_state_dict_pre_hook(lambda opt, sd: seen.append(("again", sd["param_groups"][0]["lr"])))
    two.register_load_state_dict_post_hook(lambda opt: seen.append(("after", opt.state[b[0]]["step"])))
    sd = one.state_dict()
    two.load_state_dict(sd)
    assert seen == [("before", 0), ("again", 0.25), ("after", 1)]
    assert two.param_groups[0]["lr"] == 0.25 and sd["param_groups"][0]["lr"] == 0.1
    with pytest.raises(ValueError):
        two.load_state_dict(mk.TorchAdamW(a, state_bits=8).state_dict())
    assert seen[3:] == [("before", 1), ("again", 0.25)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_8_bit_alignment_and_strides(cuda, dt):
    """Parameters and gradients at odd addresses and in another order of memory: codes, scales and values as of the same
    elements in a parameter of its own."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(13)
    base = torch.randn(20000, generator=gen, device="cuda").to(DT[dt])
    grads = torch.randn(20000, generator=gen, device="cuda").to(DT[dt])
    pairs = []
    for odd in (1, 2, 3):
        p = torch.nn.Parameter(base[odd:odd + 5003].clone())
        q = base.clone()[odd:odd + 5003].requires_grad_(True)
        p.grad, q.grad = grads[:5003].clone(), torch.cat([grads[:odd], grads])[odd:odd + 5003]
        pairs.append((p, q))
    q = base[:6000].clone().view(60, 100).t().requires_grad_(True)   # strides (1, 100): the order of `flat`
    flat = torch.nn.Parameter(base[:6000].clone())
    q.grad, flat.grad = grads[:6000].view(60, 100).t().contiguous(), grads[:6000].clone()
    opts = [[mk.TorchAdamW([t], lr=0.1, state_bits=8) for t in pair] for pair in (*pairs, (flat, q))]
    for _ in range(3):
        for a, b in opts:
            a.step()
            b.step()
    for (a, b), (x, y) in zip(opts, (*pairs, (flat, q))):
        order = (lambda v: v.t().reshape(-1)) if y.dim() == 2 else (lambda v: v)
        assert torch.equal(x, order(y.detach()))
        for name, s in a.state[x].items():
            if isinstance(s, torch.Tensor):
                other = b.state[y][name]
                assert torch.equal(s, order(other) if other.dim() == 2 else other), name


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_master_follows_a_changed_parameter(cuda, bits, dt):
    """A 16-bit parameter that a program writes between steps (a loaded model, a clamp, other memory) counts where it is not
    its master's rounding any more; elsewhere the master keeps its bits."""
    import metal_kans as mk
    p = make([(30, 70)], DT[dt], 16)
    opt = mk.TorchAdamW(p, lr=0.01, weight_decay=0.0, state_bits=bits)
    opt.step()

    def change_rows():
        with torch.no_grad():
            p[0][:10] = 3.0

    def new_memory():
        new = p[0].detach().clone()
        new[:10] = -2.0
        p[0].data = new

    def load():
        module = torch.nn.Module()
        module.p = p[0]
        module.load_state_dict({"p": torch.full((30, 70), 0.5)})

    def nothing_new():
        with torch.no_grad():
            p[0].copy_(p[0].clone())
    for change, value, rows in ((change_rows, 3.0, 10), (new_memory, -2.0, 10), (nothing_new, None, 0), (load, 0.5, 30)):
        before = opt.state[p[0]]["master"].clone()
        change()
        p[0].grad.zero_()                 # a step of the moments alone: lr an element, or twice that with 8-bit codes
        opt.step()
        master = opt.state[p[0]]["master"]
        assert torch.equal(p[0].detach(), master.to(DT[dt]))
        if rows:
            assert (master[:rows] - value).abs().max() <= 0.05
        assert (master[rows:] - before[rows:]).abs().max() <= 0.05 if rows < 30 else True
        if rows < 30:                     # (the bits below the parameter's own are still there)
            assert not torch.equal(master[rows:], master[rows:].to(DT[dt]).float())


def test_views_of_one_buffer_are_not_taken_for_changed(cuda):
    """Parameters that share a buffer share its version: a step of one is no change of another."""
    import metal_kans as mk
    flat = torch.randn(3000, device="cuda").to(torch.bfloat16)
    params = [flat[i:i + 1000].view(10, 100) for i in (0, 1000, 2000)]
    for p in params:
        p.grad = torch.randn_like(p)
    opt = mk.TorchAdamW([dict(params=params[:2]), dict(params=params[2:], lr=0.1)])
    called = []
    opt.step()
    for arenas in opt._arenas.values():
        for a in arenas:
            a.follow = lambda i, a=a: called.append(i)
    for _ in range(3):
        opt.step()
    assert not called
    flat[1500] = 2.0
    opt.step()
    assert 1 in called
