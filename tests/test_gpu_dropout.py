"""dropout (run on an MI355X) against the generator's definition in numpy's 64-bit integers.

Kept elements are one product and one rounding: within (2^-24 + t) of x / (1 - p), where 1 / (1 - p) is itself rounded to
fp32 (2^-24 more) and t is the type's half step; dropped ones are zero.  Numbers below the type's smallest normal one lie a
fixed step apart instead, 2^-24 in fp16 (its smallest normal number 2^-14 has 10 bits behind the leading one), so that
they are up to half of that, 2^-25, off whatever their size: randn in fp16 has such numbers.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


@pytest.fixture(scope="module")
def cuda(gpu):
    if not torch.cuda.is_available():
        pytest.skip("torch sees no GPU")
    return torch.device("cuda:0")


def words(n, seed, offset):
    """The first n random numbers."""
    u, low = np.uint64, np.uint64(0xffffffff)
    c = np.zeros((4, -(-n // 4)), u)
    i = np.arange(c.shape[1], dtype=u)
    c[0], c[1] = i & low, i >> u(32)
    c[2], c[3] = offset % (1 << 32), offset % (1 << 64) >> 32
    k0, k1 = seed % (1 << 32), seed % (1 << 64) >> 32
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = np.stack(((b >> u(32)) ^ c[1] ^ u(k0), b & low, (a >> u(32)) ^ c[3] ^ u(k1), a & low))
        k0, k1 = (k0 + 0x9E3779B9) % (1 << 32), (k1 + 0xBB67AE85) % (1 << 32)
    return c.T.reshape(-1)[:n]


def kept(shape, p, seed, offset):
    n = int(np.prod(shape))
    keep = words(n, seed, offset) >= np.uint64(round(p * 2 ** 32))
    return torch.from_numpy(keep.reshape(shape)).cuda()


def test_known_words():
    """The generator's published answers for counters and keys of all zeros and all ones."""
    assert [hex(int(w)) for w in words(4, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (5, 7), (2047, 10), (3, 129, 65), (1 << 20,), ()])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_against_the_definition(cuda, dt, shape, p):
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(shape, generator=gen, device="cuda").to(dt).requires_grad_(True)
    dy = torch.randn(shape, generator=gen, device="cuda").to(dt)
    y = mk.dropout(x, p, 12345, offset=6)
    dx, = torch.autograd.grad(y, x, dy)
    keep = kept(shape, p, 12345, 6)
    for got, of in ((y.detach(), x.detach()), (dx, dy)):
        want = torch.where(keep, of.double() / (1 - p), torch.zeros((), dtype=torch.float64, device="cuda"))
        assert got.dtype == dt and got.shape == of.shape
        assert ((got.double() - want).abs() <= (HALF[dt] + 2 * 2.0 ** -24) * want.abs() + LEAST[dt]).all()
        assert not got[~keep].any()
    with torch.no_grad():
        assert torch.equal(mk.dropout(x, p, 12345, offset=6), y)


@pytest.mark.parametrize("seed,offset", [(0, 0), (-1, 0), ((1 << 64) - 1, (1 << 64) - 1), (1 << 63, -5), (7, 1 << 33), (1 << 40, 3)])
def test_seeds_and_offsets(cuda, seed, offset):
    import metal_kans as mk
    x = torch.ones(1003, device="cuda")
    keep = kept((1003,), 0.5, seed, offset)
    assert torch.equal(mk.dropout(x, 0.5, seed, offset) != 0, keep)
    if -(1 << 63) <= seed < 1 << 63:
        assert torch.equal(mk.dropout(x, 0.5, torch.tensor([seed], device="cuda"), offset) != 0, keep)
        assert torch.equal(mk.dropout(x, 0.5, torch.tensor(seed, device="cuda"), offset) != 0, keep)


def test_the_ends_of_p(cuda):
    import metal_kans as mk
    x = torch.tensor([1.0, float("inf"), float("nan"), -2.0, 0.0], device="cuda").requires_grad_(True)
    y = mk.dropout(x, 0.0, 3)
    assert torch.equal(y.nan_to_num(7.0), x.nan_to_num(7.0)) and y[2].isnan() and y[1].isinf()
    y = mk.dropout(x, 1.0, 3)
    assert not y.any() and not torch.autograd.grad(y.sum(), x)[0].any()
    assert not mk.dropout(x, 1.0 - 2.0 ** -40, 3).any()      # (rounds to every word)
    assert torch.equal(mk.dropout(x[:1], 2.0 ** -40, 3), x[:1])
    full = torch.full((4096,), float("inf"), device="cuda")
    full[::2] = float("nan")
    keep = kept((4096,), 0.5, 9, 0)
    assert not mk.dropout(full, 0.5, 9)[~keep].any()


def test_orders_of_memory(cuda):
    """Elements are counted in row-major order wherever they lie."""
    import metal_kans as mk
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(33, 70, generator=gen, device="cuda")
    want = mk.dropout(x, 0.3, 5)
    assert torch.equal(mk.dropout(x.t().contiguous().t(), 0.3, 5), want)
    wide = torch.randn(33, 141, generator=gen, device="cuda")
    wide[:, 1::2] = x
    assert torch.equal(mk.dropout(wide[:, 1::2], 0.3, 5), want)
    for dt in (torch.float32, torch.float16):
        at = torch.empty(33 * 70 + 1, device="cuda", dtype=dt)[1:].view(33, 70)
        at.copy_(x)
        assert torch.equal(mk.dropout(at, 0.3, 5), mk.dropout(x.to(dt), 0.3, 5))
    x.requires_grad_(True)
    dx, = torch.autograd.grad(mk.dropout(x, 0.3, 5).sum(), x)   # (an expanded gradient)
    assert torch.equal(dx != 0, kept((33, 70), 0.3, 5, 0))
    assert mk.dropout(x[:0], 0.3, 5).shape == (0, 70)


def test_beyond_32_bits_of_elements(cuda):
    """The last elements of 2^32 + 5: their counters are past 2^30, their addresses past 4 GiB."""
    import metal_kans as mk
    n = (1 << 32) + 5
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = mk.dropout(x, 0.5, 11)
    tail = 4096 + 5
    i = np.arange((n - tail) // 4, -(-n // 4), dtype=np.uint64)
    c = np.zeros((4, i.size), np.uint64)
    c[0] = i
    u, low, k0, k1 = np.uint64, np.uint64(0xffffffff), 11, 0
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = np.stack(((b >> u(32)) ^ c[1] ^ u(k0), b & low, (a >> u(32)) ^ c[3] ^ u(k1), a & low))
        k0, k1 = (k0 + 0x9E3779B9) % (1 << 32), (k1 + 0xBB67AE85) % (1 << 32)
    keep = torch.from_numpy(c.T.reshape(-1)[:tail] >= u(1 << 31)).cuda()
    assert torch.equal(y[n - tail:] != 0, keep)


def test_a_tensor_seed_is_read_when_the_kernel_runs(cuda):
    """Replays of a graph drop what the seed of their time says; a backward what its forward dropped."""
    import metal_kans as mk
    x = torch.ones(5000, device="cuda").requires_grad_(True)
    dy = torch.ones(5000, device="cuda")
    seed = torch.tensor([21], device="cuda")
    y = mk.dropout(x, 0.4, seed, 2)
    seed += 1
    dx, = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, y.detach()) and torch.equal(dx != 0, kept((5000,), 0.4, 21, 2))
    # The eager graph of x still lives, on the default stream: a backward under capture would end the process.
    with pytest.raises(RuntimeError, match="under a graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            mk.dropout(x, 0.4, seed, 2)
    del y
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(mk.dropout(x, 0.4, seed, 2), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mk.dropout(x, 0.4, seed, 2)
        seed.add_(1)
        dx, = torch.autograd.grad(y, x, dy)
    y = y.detach()
    for at in (100, -7, 1 << 50):
        seed.fill_(at)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        keep = kept((5000,), 0.4, at, 2)
        assert torch.equal(y != 0, keep) and torch.equal(dx != 0, keep) and seed.item() == at + 1


def test_share_and_streams(cuda):
    """About p of many elements; other offsets drop others; a second derivative raises."""
    import metal_kans as mk
    x = torch.ones(1 << 22, device="cuda").requires_grad_(True)
    for p in (0.05, 0.3, 0.7):
        share = (mk.dropout(x, p, 77) == 0).double().mean().item()
        assert abs(share - p) <= 6 * (p * (1 - p) / (1 << 22)) ** 0.5
    a, b = mk.dropout(x, 0.5, 1, 0), mk.dropout(x, 0.5, 1, 1)
    assert abs(((a == 0) == (b == 0)).double().mean().item() - 0.5) < 0.002
    dx, = torch.autograd.grad(a, x, torch.ones_like(a), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c = mk.dropout(x, 0.5, 1, 0)
    side.synchronize()
    assert torch.equal(a, c)


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_words_that_all_differ(cuda, p):
    """A seed and an offset of the digits of pi, whose halves are not alike, against the oracle that holds the published answers."""
    import metal_kans as mk
    from philox import words as published
    seed, offset = 0x299f31d0a4093822, 0x0370734413198a2e
    keep = torch.tensor([w >= round(p * 2 ** 32) for w in published(0, 1003, seed, offset)], device="cuda")
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        assert torch.equal(mk.dropout(torch.ones(1003, device="cuda", dtype=dt), p, seed, offset) != 0, keep)
