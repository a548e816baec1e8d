"""Captured steps of torch operators (run on an MI355X) whose inputs an eager autograd graph on the default stream still holds: refused
with an error, in the forward for the inputs themselves and in the backward for those behind other nodes; without that
graph they are captured and replayed."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cuda(gpu):
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    return torch.device("cuda:0")


def rnd(*shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(7))


def operators():
    """Name: a leaf's shape, and the call on it."""
    import metal_kans as mk
    tokens = torch.arange(30, device="cuda") % 20
    taps, dt, A, B = rnd(24, 4), rnd(2, 9, 24), -rnd(24, 8).abs(), rnd(2, 9, 8)
    scale, table, target = rnd(24), rnd(50, 24), torch.arange(40, device="cuda")
    return {"residual_norm": ((40, 24), lambda x: mk.residual_norm(x, pre_weight=scale)[1]),
            "linear_cross_entropy": ((40, 24), lambda x: mk.linear_cross_entropy(x, table, target)),
            "embedding": ((20, 24), lambda w: mk.embedding(tokens, w)),
            "dropout": ((40, 24), lambda x: mk.dropout(x, 0.3, 5)),
            "causal_conv": ((2, 9, 24), lambda x: mk.causal_conv(x, taps)),
            "selective_scan": ((2, 9, 24), lambda x: mk.selective_scan(x, dt, A, B, B))}


def leaf(shape, order):
    """In order of memory, or with its last two dimensions exchanged there."""
    t = rnd(*shape) if order else rnd(*shape[:-2], shape[-1], shape[-2]).transpose(-1, -2)
    assert t.is_contiguous() == order
    return t.requires_grad_(True)


def captured(step):
    """The outputs of a captured step, warmed up on a stream of its own and replayed."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in out:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
    return [t.clone() for t in out]


def step_of(call, x):
    """A forward and the gradient of x."""
    def step():
        out = call(x)
        return [out.detach(), *torch.autograd.grad(out, x, torch.ones_like(out))]
    return step


@pytest.mark.parametrize("order", [True, False])
@pytest.mark.parametrize("name", ["embedding", "dropout", "causal_conv", "selective_scan"])
def test_inputs_as_they_are_given(cuda, name, order):
    shape, call = operators()[name]
    x = leaf(shape, order)
    want = step_of(call, x)()
    held = call(x)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match=name + " under a graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call(x)
    del held
    assert all(torch.equal(a, b) for a, b in zip(captured(step_of(call, x)), want))


@pytest.mark.parametrize("order", [True, False])
@pytest.mark.parametrize("name", ["embedding", "dropout", "causal_conv", "selective_scan"])
def test_inputs_behind_other_nodes(cuda, name, order):
    shape, call = operators()[name]
    x = leaf(shape, order)

    def through(x):
        return call((x * 2.0).neg())
    want = step_of(through, x)()
    held = through(x)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match=name + "'s backward under a graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            out = through(x)
            torch.autograd.grad(out, x, torch.ones_like(out))
    del held, out
    assert all(torch.equal(a, b) for a, b in zip(captured(step_of(through, x)), want))


def test_gradients_that_are_not_asked_for(cuda):
    """What the backward does not reach may be held."""
    import metal_kans as mk
    x, w = leaf((2, 9, 24), True), leaf((24, 4), True)

    def step():
        out = mk.causal_conv(x * 2.0, w)
        return [out.detach(), *torch.autograd.grad(out, w, torch.ones_like(out))]
    want = step()
    held = x * 3.0
    assert all(torch.equal(a, b) for a, b in zip(captured(step), want))
    del held


@pytest.mark.parametrize("order", [True, False])
@pytest.mark.parametrize("name", ["residual_norm", "linear_cross_entropy"])
def test_norms_and_losses(cuda, name, order):
    """Their forwards may be captured alone; their backwards refuse, whether or not a node stands between."""
    shape, call = operators()[name]
    x = leaf(shape, order)
    for through in (call, lambda x: call((x * 2.0).neg())):
        want = step_of(through, x)()
        held = through(x)
        with torch.no_grad():
            assert torch.equal(captured(lambda: [through(x).detach()])[0], want[0])
        torch.cuda.synchronize()
        alone = torch.cuda.CUDAGraph()
        with torch.cuda.graph(alone):
            out = through(x).detach()
        alone.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0])
        with pytest.raises(RuntimeError, match=name + "'s backward under a graph capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                out = through(x)
                torch.autograd.grad(out, x, torch.ones_like(out))
        del held, out
        assert all(torch.equal(a, b) for a, b in zip(captured(step_of(through, x)), want))


def test_weights_of_norms_and_losses(cuda):
    """The weights' gradients alone."""
    import metal_kans as mk
    x, w, target = rnd(40, 24), leaf((50, 24), True), torch.arange(40, device="cuda")
    scale = leaf((1, 24), True)
    calls = {"linear_cross_entropy": (w, lambda: mk.linear_cross_entropy(x, w, target)),
             "residual_norm": (scale, lambda: mk.residual_norm(x, pre_weight=scale[0])[1])}
    for name, (of, call) in calls.items():
        held = of * 2.0
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=name + "'s backward under a graph capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                out = call()
                torch.autograd.grad(out, of, torch.ones_like(out))
        del held, out
