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
