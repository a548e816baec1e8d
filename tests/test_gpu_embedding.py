"""embedding (run on an MI355X) against its definition in 64 bits.

Tolerances.  u = 2^-24 is one fp32 rounding, t one rounding to the result's type (2^-24 fp32, 2^-11 fp16, 2^-8 bf16 or its
smallest step).  A row of the output is one product: t |result| + u |result|.  A gradient of k rows is a sum of k terms
in some order and one product: at most k roundings of partial sums, each no larger than A, the sum of the terms' magnitudes:
t |result| + (k + 2) u A.
"""
import math

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


def inputs(n, d, v, dt, seed=0, ignored=0.0, hot=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(0, v, (n,), generator=gen, device="cuda")
    if hot:
        tokens[torch.rand(n, generator=gen, device="cuda") < hot] = v // 2
    if ignored:
        tokens[torch.rand(n, generator=gen, device="cuda") < ignored] = -100
    return tokens, torch.randn(v, d, generator=gen, device="cuda").to(dt), torch.randn(n, d, generator=gen, device="cuda").to(dt)


def near(got, want, A, k, dt):
    t, least = STEP[dt]
    assert got.dtype == dt and got.shape == want.shape
    bound = t * want.abs() + (k + 2) * U * A + least
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()


def check(tokens, w, dout, scale):
    import metal_kans as mk
    dt, v = w.dtype, w.shape[0]
    w = w.detach().requires_grad_(True)
    out = mk.embedding(tokens, w, scale=scale)
    dw, = torch.autograd.grad(out, w, dout)
    flat, rows = tokens.reshape(-1), dout.reshape(-1, w.shape[1]).double()
    on = flat != -100
    want = torch.zeros(flat.numel(), w.shape[1], dtype=torch.float64, device="cuda")
    want[on] = w.detach().double()[flat[on]] * scale
    near(out.detach().reshape(want.shape), want, want.abs(), 0, dt)
    sums, mags = torch.zeros_like(w, dtype=torch.float64), torch.zeros_like(w, dtype=torch.float64)
    sums.index_add_(0, flat[on], rows[on] * scale)
    mags.index_add_(0, flat[on], (rows[on] * scale).abs())
    near(dw, sums, mags, torch.bincount(flat[on], minlength=v)[:, None].double(), dt)
    with torch.no_grad():
        assert torch.equal(mk.embedding(tokens, w, scale=scale), out)
    return dw


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,d,v", [(1, 1, 1), (1, 64, 1000), (7, 3, 5), (9, 8, 300), (64, 7, 64), (257, 33, 1025), (1000, 777, 50),
                                   (513, 4100, 7), (3001, 129, 9000), (8193, 16, 70001)])
def test_sizes(cuda, n, d, v, dt):
    check(*inputs(n, d, v, dt, ignored=0.2 if n > 8 else 0.0), math.sqrt(d))


@pytest.mark.parametrize("hot", [0.1, 0.9, 1.0])
@pytest.mark.parametrize("n,d,v", [(500, 40, 100), (20000, 24, 33000)])
def test_frequent_tokens(cuda, n, d, v, hot):
    """Runs over many pieces of the sorted order, and a table of one token."""
    check(*inputs(n, d, v, torch.float32, hot=hot), 0.5)


@pytest.mark.parametrize("n,each", [(12288, 48), (12288, 24), (12000, 25), (20000, 80), (20000, 41), (5000, 16), (5000, 23), (40000, 64), (30000, 57)])
def test_runs_of_every_place(cuda, n, each):
    """Equal tokens in runs that begin and end anywhere in the pieces of the sorted order (of 8 to 64 positions, no powers of two
    among them): whole numbers, exact; the memory that partial rows may come from holds no numbers."""
    import metal_kans as mk
    v = -(-n // each)
    tokens = (torch.arange(n, device="cuda") // each)[torch.randperm(n, generator=torch.Generator("cuda").manual_seed(1), device="cuda")]
    dout = (torch.arange(n * 20, device="cuda").view(n, 20) % 5 - 2).float()
    want = torch.zeros(v, 20, device="cuda").index_add_(0, tokens, dout)
    w = torch.zeros(v, 20, device="cuda", requires_grad=True)
    out = mk.embedding(tokens, w)
    used = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(3)]
    del used
    assert torch.equal(torch.autograd.grad(out, w, dout)[0], want)


def test_large_vocabulary(cuda):
    """Beyond 256 workgroups of 8192 tokens each."""
    check(*inputs(300, 8, (1 << 21) + 77, torch.bfloat16, hot=0.2), 1.0)


@pytest.mark.parametrize("dt", TYPES)
def test_whole_numbers_are_exact(cuda, dt):
    """Sums that every partial sum holds exactly."""
    import metal_kans as mk
    tokens, w, _ = inputs(4000, 100, 37, dt, hot=0.3)
    dout = (torch.arange(4000 * 100, device="cuda").view(4000, 100) % 3 - 1).to(dt)
    want = torch.zeros(37, 100, device="cuda").index_add_(0, tokens, dout.float())
    w.requires_grad_(True)
    dw, = torch.autograd.grad(mk.embedding(tokens, w), w, dout)
    assert torch.equal(dw, want.to(dt))


def test_shapes_and_orders(cuda):
    """Tokens of any shape, a table that is a view, gradients that are views."""
    import metal_kans as mk
    tokens, w, dout = inputs(60, 24, 50, torch.float32)
    want = check(tokens, w, dout, 2.0)
    assert mk.embedding(tokens.view(3, 4, 5), w).shape == (3, 4, 5, 24)
    assert mk.embedding(tokens[0], w).shape == (24,)
    wide = torch.zeros(50, 48, device="cuda")
    wide[:, 1::2] = w
    part = wide[:, 1::2].requires_grad_(True)
    for t, g in ((tokens.view(10, 6).t().contiguous().t(), dout.view(10, 6, 24)), (tokens.view(6, 10), dout.view(6, 10, 24))):
        got, = torch.autograd.grad(mk.embedding(t, part, scale=2.0), part, g.transpose(0, 1).contiguous().transpose(0, 1))
        assert torch.equal(got, want)
    got, = torch.autograd.grad(mk.embedding(tokens, part, scale=2.0).sum(), part)
    assert torch.equal(got, 2.0 * torch.bincount(tokens, minlength=50)[:, None].expand(50, 24).float())
    odd = torch.zeros(50 * 24 + 1, device="cuda", dtype=torch.float16)[1:].view(50, 24)
    odd.copy_(w)
    check(tokens, odd, dout.half(), 1.0)


def test_padding_and_strangers(cuda):
    """Ignored rows are zeros and their gradient is not looked at; tokens from outside give NaN and reach no row."""
    import metal_kans as mk
    tokens, w, dout = inputs(40, 16, 9, torch.float32)
    tokens[5:9], tokens[20] = 3, 9
    tokens[21], tokens[22], tokens[23] = -1, 1 << 40, -(1 << 62)
    w[3] = float("nan")
    dout[5:9] = float("nan")
    dout[20:24] = float("inf")
    w.requires_grad_(True)
    out = mk.embedding(tokens, w, ignore_index=3)
    dw, = torch.autograd.grad(out, w, dout)
    assert not out[tokens == 3].any() and out[20:24].isnan().all()
    rest = (tokens != 3) & (tokens >= 0) & (tokens < 9)
    assert torch.equal(out[rest], w[tokens[rest]])
    assert dw.isfinite().all() and not dw[3].any()
    want = torch.zeros(9, 16, dtype=torch.float64, device="cuda").index_add_(0, tokens[rest], dout[rest].double())
    assert (dw - want).abs().max() < 1e-5
    none = mk.embedding(torch.full((5,), -100, device="cuda"), w)
    assert not none.any() and not torch.autograd.grad(none.sum(), w)[0].any()


def test_no_tokens(cuda):
    import metal_kans as mk
    _, w, _ = inputs(4, 16, 9, torch.bfloat16)
    w.requires_grad_(True)
    out = mk.embedding(torch.zeros(0, 3, dtype=torch.int64, device="cuda"), w)
    assert out.shape == (0, 3, 16)
    dw, = torch.autograd.grad(out, w, torch.zeros_like(out))
    assert dw.shape == w.shape and not dw.any()


def test_same_bits_on_every_run_and_in_a_graph(cuda):
    import metal_kans as mk
    tokens, w, dout = inputs(5000, 72, 400, torch.float32, hot=0.3, ignored=0.1)
    w.requires_grad_(True)

    def step():
        out = mk.embedding(tokens, w, scale=0.3)
        return out.detach(), torch.autograd.grad(out, w, dout)[0]
    want = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (0, 5, 6):
        new = inputs(5000, 72, 400, torch.float32, seed=seed, hot=0.3, ignored=0.1)
        tokens.copy_(new[0])
        dout.copy_(new[2])
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_machinery(cuda):
    """Saved tokens are guarded, a second derivative raises, another stream gives the same."""
    import metal_kans as mk
    tokens, w, dout = inputs(50, 24, 33, torch.float32)
    w.requires_grad_(True)
    out = mk.embedding(tokens, w)
    dw, = torch.autograd.grad(out, w, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dw.sum().backward()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again, = torch.autograd.grad(mk.embedding(tokens, w), w, dout)
    side.synchronize()
    assert torch.equal(again, dw)
    out = mk.embedding(tokens, w)
    tokens += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, w, dout)


def test_gradient_is_the_difference(cuda):
    """dw against differences of the outputs in direction of one element (linear: no remainder but rounding)."""
    import metal_kans as mk
    tokens, w, dout = inputs(30, 8, 6, torch.float32)
    w.requires_grad_(True)
    dw, = torch.autograd.grad(mk.embedding(tokens, w, scale=1.5), w, dout)
    for v, c in ((0, 0), (3, 7), (5, 2)):
        with torch.no_grad():
            up, down = w.clone(), w.clone()
            up[v, c] += 1.0
            down[v, c] -= 1.0
            diff = ((mk.embedding(tokens, up, scale=1.5) - mk.embedding(tokens, down, scale=1.5)).double() * dout).sum() / 2
        assert abs(diff - dw[v, c]) <= 1e-4


@pytest.mark.parametrize("v", [131072, 131073, 200003, 262144, 262145, 500009])
@pytest.mark.parametrize("n,hot", [(3000, 0.3), (20000, 0.5), (20000, 1.0)])
def test_frequent_tokens_of_large_tables(cuda, n, hot, v):
    """Long lists of equal tokens on both sides of the ranges (of up to 512 tokens) that all waves of a workgroup place: whole numbers,
    exact, and the sorted order of the positions through a sum that it changes."""
    import metal_kans as mk
    tokens, _, _ = inputs(n, 1, v, torch.float32, seed=v, hot=hot)
    tokens[:7] = torch.tensor([0, v - 1, v // 2, v // 2 - 1, v // 2 + 1, v - 1, 511], device="cuda")
    dout = (torch.arange(n * 12, device="cuda").view(n, 12) % 7 - 3).float()
    w = torch.zeros(v, 12, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(mk.embedding(tokens, w), w, dout)
    assert torch.equal(dw, torch.zeros(v, 12, device="cuda").index_add_(0, tokens, dout))
    check(*inputs(n, 12, v, torch.float32, seed=v + 1, hot=hot), 0.5)


def test_ends_of_a_large_vocabulary(cuda):
    """Tokens of the 257th sorting workgroup, which has 77 of the table's, and of both ends of those before it."""
    v = (1 << 21) + 77
    tokens, w, dout = inputs(300, 8, v, torch.bfloat16)
    tokens[:10] = torch.tensor([v - 1, v - 77, v - 78, v - 1, 0, 8191, 8192, 1 << 21, (1 << 21) - 8192, v - 40], device="cuda")
    dw = check(tokens, w, dout, 1.0)
    assert dw[v - 1].any() and dw[v - 77].any()
