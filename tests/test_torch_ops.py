"""The torch operators' refusals that need no GPU, and how the compiled module meets the library."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def mk():
    import metal_kans
    metal_kans.device.load_library()
    return metal_kans


def test_module_loads_once(mk):
    from metal_kans import _torch_ops
    assert _torch_ops.load() is _torch_ops.load()


def test_residual_norm_refuses(mk):
    x, v = torch.zeros(3, 4), torch.zeros(4)
    for bad, error in (((x,), ValueError), ((x, x, None, 1.0, v, v, "batch"), ValueError), ((torch.zeros(()),), ValueError),
                       ((torch.zeros(3, 0),), ValueError), ((x, None, v), ValueError), ((x, None, None, 1.0, v), ValueError),
                       ((x, x, None, 1.0, None, None, "rms", -1.0), ValueError),
                       ((x, x, None, 1.0, None, None, "rms", float("nan")), ValueError),
                       ((x.double(),), TypeError), ((x.half(), x), TypeError), ((x, x.half(), v), TypeError),
                       ((x, x, None, torch.zeros(2)), TypeError), ((x, x, None, torch.zeros(1).half()), TypeError),
                       (([1.0],), TypeError), ((x, x, None, "1"), TypeError)):
        with pytest.raises(error):
            mk.residual_norm(*bad)


def test_linear_cross_entropy_refuses(mk):
    h, w, t = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    for bad, error in (((h, w, t), ValueError), ((h, w, t, -100, "max"), ValueError), ((h, w[0], t), ValueError),
                       ((h, w[:, :3], t), ValueError), ((h, w[:0], t), ValueError), ((h, w, t[:2]), ValueError),
                       ((h, w.half(), t), TypeError), ((h.double(), w.double(), t), TypeError), ((h, w, t.int()), TypeError),
                       ((h, None, t), TypeError)):
        with pytest.raises(error):
            mk.linear_cross_entropy(*bad)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_step_checks_where_a_parameter_lies(mk, bits):
    """What the kernel would write beside a parameter is refused before any device is asked for."""
    from metal_kans._torch_ops import load
    from metal_kans.adamw import _Arena
    p = torch.nn.Parameter(torch.zeros(4, 8))
    a = _Arena([p], bits)

    def step(state):
        load().adamw_step(state, a.params, a.numel_q, a.blocks_q, a.flat, 0, bits,
                          lambda i: state.__setitem__(p, a.start(i, state.get(p, {}))), 1e-3, 0.9, 0.99, 1e-8, 0.0)
    for started in (False, True):
        state = {p: a.start(0, {})} if started else {}
        for view in (torch.zeros(4, 16)[:, :8], torch.zeros(4, 16)[:, 5:13], torch.zeros(1, 1).expand(4, 8), torch.zeros(8, 8)[::2],
                     torch.zeros(40).as_strided((4, 8), (8, 1))[:, :8].as_strided((4, 8), (4, 1))):
            p.data, p.grad = view, torch.ones(4, 8)
            with pytest.raises(ValueError, match="dense"):
                step(state)
            with pytest.raises(ValueError, match="dense"):
                a.start(0, {})
        for shape in ((8, 4), (32,), (2, 16), (33,), (5, 8)):
            p.data = torch.zeros(shape)
            p.grad = torch.ones(shape)
            if started or shape in ((33,), (5, 8)):
                with pytest.raises(ValueError):
                    step(state)
        p.data = torch.zeros(2, 8)
        p.grad = torch.ones(2, 8)
        p.data = torch.zeros(4, 8)           # (the gradient's strides are the parameter's)
        with pytest.raises(ValueError, match="shape"):
            step(state)


def test_adamw_states_follow_the_order_of_memory(mk):
    from metal_kans.adamw import _Arena
    p = torch.nn.Parameter(torch.zeros(3, 5))
    values = torch.arange(15.0).view(3, 5)
    a = _Arena([p], 32)
    state = a.start(0, {"step": 2, "exp_avg": values, "exp_avg_sq": values + 1})
    assert torch.equal(a.flat["exp_avg"][:15], values.view(-1))
    p.data = p.data.t().contiguous().t()
    state = a.start(0, state)
    assert state["step"] == 2 and state["exp_avg"].stride() == p.stride()
    assert torch.equal(state["exp_avg"], values) and torch.equal(state["exp_avg_sq"], values + 1)
    assert torch.equal(a.flat["exp_avg"][:15], values.t().reshape(-1)) and not a.flat["exp_avg"][15:].any()
    b = _Arena([torch.nn.Parameter(torch.zeros(3, 5))], 8)
    codes = b.start(0, {})
    assert b.start(0, codes)["exp_avg"].shape == (3, 5)
    b.params[0].data = torch.zeros(5, 3).t()
    with pytest.raises(ValueError, match="order"):
        b.start(0, codes)


def test_adamw_refuses_other_steps(mk):
    """Options of torch's AdamW in a group or a saved state that would be dropped without a word."""
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))
    for option in ("amsgrad", "maximize"):
        with pytest.raises(ValueError, match=option):
            mk.TorchAdamW([dict(params=[p], **{option: True})])
        other = torch.optim.AdamW([q], lr=0.5, **{option: True})
        opt = mk.TorchAdamW([p])
        with pytest.raises(ValueError, match=option):
            opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == 1e-3
    mk.TorchAdamW([dict(params=[p], amsgrad=False, maximize=False)])


def test_embedding_refuses(mk):
    t, w = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    for bad, error in (((t, w), ValueError), ((t, w[0]), ValueError), ((t, w[:0]), ValueError), ((t, w[:, :0]), ValueError),
                       ((t, w, float("nan")), ValueError), ((t, w.double()), TypeError), ((t.int(), w), TypeError),
                       ((None, w), TypeError), ((t, w, "1"), TypeError)):
        with pytest.raises(error):
            mk.embedding(*bad)


def test_dropout_refuses(mk):
    x = torch.zeros(3, 4)
    for bad, error in (((x, 0.1, 1), ValueError), ((x, -0.1, 1), ValueError), ((x, 1.5, 1), ValueError),
                       ((x, float("nan"), 1), ValueError), ((x, 0.1, 1 << 64), ValueError), ((x, 0.1, 1, -(1 << 63) - 1), ValueError),
                       ((x.double(), 0.1, 1), TypeError), ((x, 0.1, torch.zeros(2, dtype=torch.int64)), TypeError),
                       ((x, 0.1, torch.zeros(1)), TypeError), ((x, 0.1, 1.5), TypeError), ((None, 0.1, 1), TypeError)):
        with pytest.raises(error):
            mk.dropout(*bad)


def test_causal_conv_refuses(mk):
    x, w, b = torch.zeros(2, 5, 4), torch.zeros(4, 3), torch.zeros(4)
    n = torch.zeros(2, dtype=torch.int64)
    for bad, error in (((x, w), ValueError), ((x[0], w), ValueError), ((x[..., :0], w[:0]), ValueError), ((x, w[:3]), ValueError),
                       ((x, torch.zeros(4, 9)), ValueError), ((x, w[:, :0]), ValueError), ((x, w, b[:3]), ValueError),
                       ((x, w, b, "relu"), ValueError), ((x, w, b, None, torch.zeros(2, 3, 4)), ValueError),
                       ((x, w, b, None, torch.zeros(2, 4, 2).transpose(1, 2)), ValueError),
                       ((x, w, b, None, torch.zeros(2, 2, 4).half()), TypeError), ((x, w, b, None, None, n[:1]), ValueError),
                       ((x, w, b, None, None, n.int()), TypeError), ((x.double(), w.double()), TypeError), ((x, w.half()), TypeError),
                       ((x, w, b.half()), TypeError), ((None, w), TypeError)):
        with pytest.raises(error):
            mk.causal_conv(*bad)


def test_selective_scan_refuses(mk):
    x, A, B = torch.zeros(2, 5, 4), torch.zeros(4, 16), torch.zeros(2, 5, 16)
    n, state = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 4, 16)
    ok = dict(x=x, dt=x, A=A, B=B, C=B)
    for bad, error in ((dict(), ValueError), (dict(x=x[0]), ValueError), (dict(A=A[:3]), ValueError), (dict(A=A[:, :0]), ValueError),
                       (dict(A=torch.zeros(4, 65), B=torch.zeros(2, 5, 65), C=torch.zeros(2, 5, 65)), ValueError),
                       (dict(dt=x[:, :4]), ValueError), (dict(z=x[:1]), ValueError), (dict(B=B[..., :15]), ValueError),
                       (dict(C=B.half()), TypeError), (dict(dt=x.half()), TypeError), (dict(z=x.half()), TypeError),
                       (dict(A=A.half()), TypeError), (dict(D=torch.zeros(3)), ValueError), (dict(D=torch.zeros(4).half()), TypeError),
                       (dict(dt_bias=torch.zeros(4, 1)), ValueError), (dict(state=state[:1]), ValueError),
                       (dict(state=state.half()), TypeError), (dict(state=torch.zeros(2, 16, 4).transpose(1, 2)), ValueError),
                       (dict(lengths=n[:1]), ValueError), (dict(lengths=n.int()), TypeError),
                       (dict(x=x.double(), dt=x.double(), B=B.double(), C=B.double()), TypeError), (dict(x=None), TypeError)):
        with pytest.raises(error):
            mk.selective_scan(**{**ok, **bad})


def test_embedding_refuses_scales_beyond_fp32(mk):
    t, w = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    for scale in (1e39, -1e39, 1e-39, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            mk.embedding(t, w, scale)
    with pytest.raises(ValueError, match="one GPU"):
        mk.embedding(t, w, 0.0)
