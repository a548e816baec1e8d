"""The autograd nodes of residual_norm and linear_cross_entropy (run on an MI355X): which gradients are made, on which
stream, and what torch's own machinery around a node does with them."""
import itertools

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cuda(gpu):
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    return torch.device("cuda:0")


def norm_inputs(wants, gate=(2, 1, 40)):
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    t = [rnd(2, 9, 40), rnd(2, 9, 40), rnd(*gate), rnd(40), rnd(40), torch.full((1,), 0.3, device="cuda")]
    for v, want in zip(t, wants):
        v.requires_grad_(want)
    return t, (rnd(2, 9, 40), rnd(2, 9, 40))


def norm_call(t):
    import metal_kans as mk
    x, block, gate, post, pre, scale = t
    return mk.residual_norm(x, block, gate, scale, post, pre)


def xent_inputs(wants=(True, True), n=50, d=24, v=33):
    gen = torch.Generator(device="cuda").manual_seed(4)
    h = torch.randn(n, d, generator=gen, device="cuda").requires_grad_(wants[0])
    w = torch.randn(v, d, generator=gen, device="cuda").requires_grad_(wants[1])
    return h, w, torch.randint(0, v, (n,), generator=gen, device="cuda")


@pytest.mark.parametrize("gate", [(2, 1, 40), (1, 9, 40), (2, 9, 1)])
def test_gradients_of_some_inputs(cuda, gate):
    t, d = norm_inputs([True] * 6, gate)
    want = torch.autograd.grad(norm_call(t), t, d)
    for wants in itertools.product([False, True], repeat=6):
        if not any(wants):
            continue
        t, d = norm_inputs(wants, gate)
        for v, g, w in zip(t, torch.autograd.grad(norm_call(t), [v for v in t if v.requires_grad], d),
                           [w for w, on in zip(want, wants) if on]):
            assert torch.equal(g, w), wants
    h, w, target = xent_inputs()
    import metal_kans as mk
    both = torch.autograd.grad(mk.linear_cross_entropy(h, w, target), (h, w))
    for wants in ((True, False), (False, True)):
        h, w, target = xent_inputs(wants)
        one, = torch.autograd.grad(mk.linear_cross_entropy(h, w, target), [v for v in (h, w) if v.requires_grad])
        assert torch.equal(one, both[wants.index(True)])


def test_absent_inputs_and_unused_outputs(cuda):
    import metal_kans as mk
    t, (dy, dh) = norm_inputs([True] * 6)
    x, block, gate, post, pre, scale = t
    y, h = mk.residual_norm(x, None, pre_weight=pre)
    assert y is x
    assert all(g is not None for g in torch.autograd.grad(h, (x, pre), dh))
    for used, other in ((0, dy), (1, dh)):       # one output's gradient is as if the other's were zeros
        out = norm_call(t)
        got = torch.autograd.grad(out[used], t, other, allow_unused=True)
        zero = [torch.zeros_like(dy), torch.zeros_like(dh)]
        zero[used] = other
        for g, w in zip(got, torch.autograd.grad(norm_call(t), t, zero)):
            assert torch.equal(g, w) if g is not None else not w.any()


def test_no_second_derivative(cuda):
    """Gradients of a kept graph are the same; differentiating them is an error."""
    import metal_kans as mk
    t, d = norm_inputs([True] * 6)
    want = torch.autograd.grad(norm_call(t), t, d)
    got = torch.autograd.grad(norm_call(t), t, d, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="second derivative"):
        got[0].sum().backward()
    h, w, target = xent_inputs()
    dh, dw = torch.autograd.grad(mk.linear_cross_entropy(h, w, target), (h, w), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (dh.sum() + dw.sum()).backward()


def test_streams_and_checkpoints(cuda):
    """On another stream, its own or an external one, and with the forward run again in the backward."""
    import metal_kans as mk
    from torch.utils.checkpoint import checkpoint

    def step(run):
        t, d = norm_inputs([True] * 6)
        h, w, target = xent_inputs()
        torch.cuda.synchronize()
        out = run(lambda *a: norm_call(a), *t)
        grads = torch.autograd.grad(out, t, d)
        loss = run(mk.linear_cross_entropy, h, w, target)
        return [*out, *grads, loss, *torch.autograd.grad(loss, (h, w))]
    want = step(lambda f, *a: f(*a))
    side = torch.cuda.Stream()
    for stream in (side, torch.cuda.ExternalStream(side.cuda_stream)):
        with torch.cuda.stream(stream):
            got = step(lambda f, *a: f(*a))
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = step(lambda f, *a: checkpoint(f, *a, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_tensors_are_guarded(cuda):
    import metal_kans as mk
    h, w, target = xent_inputs()
    loss = mk.linear_cross_entropy(h, w, target)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_no_forward_mode_derivative(cuda):
    """A dual tensor's tangent is never dropped: the calls refuse it, in every input and with or without gradients."""
    import torch.autograd.forward_ad as fwd
    import metal_kans as mk
    for wants in (False, True):
        with fwd.dual_level():
            for i in range(6):
                t, _ = norm_inputs([wants] * 6)
                t[i] = fwd.make_dual(t[i].detach(), torch.ones_like(t[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    norm_call(t)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    norm_call(t)
            for i in range(2):
                h, w, target = xent_inputs((wants, wants))
                a = [h, w]
                a[i] = fwd.make_dual(a[i].detach(), torch.ones_like(a[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    mk.linear_cross_entropy(*a, target)
            t, _ = norm_inputs([wants] * 6)
            norm_call(t)                     # plain tensors inside the level are as outside
    t, (dy, dh) = norm_inputs([True] * 6)
    h, w, target = xent_inputs()
    y, loss = norm_call(t)[0], mk.linear_cross_entropy(h, w, target)
    with fwd.dual_level():                   # forward over backward
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, t[0], fwd.make_dual(dy, dh))
        one = torch.ones((), device="cuda")
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(loss, h, fwd.make_dual(one, one))


def test_tracers_are_refused(cuda):
    """A trace would hold the results' memory and not the call that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    import metal_kans as mk
    t, _ = norm_inputs([False] * 6)
    h, w, target = xent_inputs((False, False))
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    opt = mk.TorchAdamW([p], lr=0.5)

    def step(g):
        p.grad = g
        opt.step()
        return g
    calls = ((lambda *a: norm_call(a)[1], t), (lambda *a: mk.linear_cross_entropy(*a), (h, w, target)),
             (step, (torch.ones(5, device="cuda"),)))
    for call, args in calls:
        for trace in (lambda: torch.jit.trace(call, tuple(args)), lambda: make_fx(call)(*args),
                      lambda: make_fx(call, pre_dispatch=True)(*args)):
            with pytest.raises(RuntimeError, match=None if call is step else "trace"):   # (torch may be the first to refuse)
                trace()
    assert (p == 1).all() and not opt.state.get(p)

    class Watch(TorchDispatchMode):          # other modes see torch's operators pass and change nothing
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    for call, args in calls[:2]:
        want = call(*args)
        with Watch():
            assert torch.equal(call(*args), want)
