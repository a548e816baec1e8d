"""Performance cases of the operators that bring tokens into a KAN token model and mix them, on one MI355X.

Four operators that stand before and between a token model's ``TorchMetalKANLinear`` blocks:

* ``embed`` -- ``embedding``: scaled rows of a table for the tokens of a batch (``lookup``), with the
               table's gradient (``train``);
* ``drop``  -- ``dropout``: elements dropped by a counter-based generator, forward (``forward``) or both
               directions (``train``);
* ``conv``  -- ``causal_conv``: the short convolution along the sequence before a scan;
* ``scan``  -- ``selective_scan``: the selective state space scan.

The last two train over whole sequences (``train``) or serve: they carry a state through a prompt
(``prompt``) or through one token of every sequence (``step``), and leave the new state in its place.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what the
program holds before the call, ``run`` is the call, ``work`` its least traffic and arithmetic and
``exact`` the same results in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ESIZE = {"f32": 4, "f16": 2, "bf16": 2}
IGNORE = -100

_LISTED = [
    # one token for each of a few sequences being served, from the largest table: launch latency counts
    {"name": "embed_lookup_bf16_8x4096_of_131072", "op": "embed", "mode": "lookup", "dtype": "bf16", "N": 8, "D": 4096,
     "V": 131072, "ignored": 0.0},
    # half precision, no size a multiple of a tile, a quarter of the tokens padding
    {"name": "embed_train_f16_3001x777_of_50021", "op": "embed", "mode": "train", "dtype": "f16", "N": 3001, "D": 777,
     "V": 50021, "ignored": 0.25},
    # full-precision parameters, as the torch modules hold them by default
    {"name": "embed_train_f32_4096x1024_of_32768", "op": "embed", "mode": "train", "dtype": "f32", "N": 4096, "D": 1024,
     "V": 32768, "ignored": 0.1},
    # a full batch of the wide model
    {"name": "embed_train_bf16_16384x4096_of_65536", "op": "embed", "mode": "train", "dtype": "bf16", "N": 16384,
     "D": 4096, "V": 65536, "ignored": 0.0},
    # odd sizes in full precision
    {"name": "drop_train_f32_2047x1000", "op": "drop", "mode": "train", "dtype": "f32", "N": 2047, "D": 1000, "p": 0.25},
    # a block's output in a full batch of the wide model
    {"name": "drop_train_bf16_16384x4096", "op": "drop", "mode": "train", "dtype": "bf16", "N": 16384, "D": 4096, "p": 0.1},
    # sequences of different lengths in half precision, odd sizes
    {"name": "conv_train_f16_3x777x1300_w3", "op": "conv", "mode": "train", "dtype": "f16", "B": 3, "L": 777, "D": 1300,
     "W": 3, "ragged": True},
    # a full batch of the wide model
    {"name": "conv_train_bf16_8x2048x4096_w4", "op": "conv", "mode": "train", "dtype": "bf16", "B": 8, "L": 2048,
     "D": 4096, "W": 4, "ragged": False},
    # one token for each of 16 sequences being served
    {"name": "scan_step_bf16_16x4096_n16", "op": "scan", "mode": "step", "dtype": "bf16", "B": 16, "L": 1, "D": 4096,
     "N": 16, "gated": True, "ragged": False},
    # one long prompt: few channels, many steps
    {"name": "scan_prompt_f16_1x8192x1024_n16", "op": "scan", "mode": "prompt", "dtype": "f16", "B": 1, "L": 8192,
     "D": 1024, "N": 16, "gated": True, "ragged": False},
    # sequences of different lengths in full precision, odd sizes, a state that is no power of two
    {"name": "scan_train_f32_3x777x1300_n24", "op": "scan", "mode": "train", "dtype": "f32", "B": 3, "L": 777, "D": 1300,
     "N": 24, "gated": False, "ragged": True},
    # a full batch of the wide model: the largest case
    {"name": "scan_train_bf16_8x2048x4096_n16", "op": "scan", "mode": "train", "dtype": "bf16", "B": 8, "L": 2048,
     "D": 4096, "N": 16, "gated": True, "ragged": False},
]

# no drawn case costs more than the largest listed one of its operator
_MOST_ROWS = 16384 * 4096
_MOST_TABLE = 65536 * 4096
_MOST_STATES = 8 * 2048 * 4096 * 16


def listed():
    return [dict(c) for c in _LISTED]


def _size(rng, lo, hi):
    """A size spread over the logarithm of the range: as it comes, or rounded to a multiple of 8 / 64."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    m = rng.choice((1, 8, 64))
    return max(lo, min(hi, v // m * m))


def draw(rng):
    op = rng.choice(("embed", "drop", "conv", "scan", "scan"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    while True:
        if op == "embed":
            c = {"op": op, "mode": rng.choice(("lookup", "train", "train")), "dtype": dtype, "N": _size(rng, 1, 16384),
                 "D": _size(rng, 16, 4096), "V": _size(rng, 10, 131072), "ignored": rng.choice((0.0, 0.1, 0.5))}
            if c["N"] * c["D"] <= _MOST_ROWS and c["V"] * c["D"] <= _MOST_TABLE:
                return c
        elif op == "drop":
            c = {"op": op, "mode": rng.choice(("forward", "train")), "dtype": dtype, "N": _size(rng, 1, 16384),
                 "D": _size(rng, 16, 8192), "p": rng.choice((0.05, 0.1, 0.3, 0.5))}
            if c["N"] * c["D"] <= _MOST_ROWS:
                return c
        else:
            mode = rng.choice(("train", "train", "prompt", "step"))
            c = {"op": op, "mode": mode, "dtype": dtype, "B": _size(rng, 1, 64 if mode == "step" else 16),
                 "L": 1 if mode == "step" else _size(rng, 1, 8192), "D": _size(rng, 16, 4096),
                 "ragged": mode != "step" and rng.random() < 0.5}
            if op == "conv":
                c["W"] = rng.randint(2, 4)
            else:
                c["N"], c["gated"] = rng.choice((4, 8, 16, 16, 16, 24, 32, 64)), rng.random() < 0.7
            if c["B"] * c["L"] * c["D"] <= _MOST_ROWS and c["B"] * c["L"] * c["D"] * c.get("N", 1) <= _MOST_STATES:
                return c


def work(case):
    """Bytes: each input read once and each output written once, in the types that the call hands over.
    Flops: about what a value costs (an exponential counts one)."""
    e = _ESIZE[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "embed":
        n = case["N"] * case["D"]
        # rows of the table (those of a token once: at most the table), rows out; the rows' gradients, the table's
        table = min(case["N"], case["V"]) * case["D"]
        return {"bytes": 8 * case["N"] + e * (table + n) + (e * (n + case["V"] * case["D"]) if train else 0),
                "flops": n * (2 if train else 1)}
    if case["op"] == "drop":
        n = case["N"] * case["D"]
        return {"bytes": e * n * (4 if train else 2), "flops": n * (4 if train else 2)}
    rows = case["B"] * case["L"]
    n = rows * case["D"]
    if case["op"] == "conv":
        state = 0 if train else 2 * e * case["B"] * (case["W"] - 1) * case["D"]
        return {"bytes": e * n * (4 if train else 2) + state, "flops": n * 2 * case["W"] * (3 if train else 1)}
    N, z = case["N"], 1 if case["gated"] else 0
    fwd = e * (n * (3 + z) + 2 * rows * N) + 4 * case["D"] * (N + 2)       # x, dt, z, out; B, C; A, D, dt_bias
    bwd = e * (n * (3 + z) + 2 * rows * N) + 4 * case["D"] * (N + 2)       # dout; dx, ddt, dz; dB, dC; the parameters'
    state = 0 if train else 8 * case["B"] * case["D"] * N
    return {"bytes": fwd + state + (bwd if train else 0), "flops": n * N * (23 if train else 7)}


# ---- inputs --------------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _inputs(case, seed):
    """The inputs of a case, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _DT[case["dtype"]]
    D, train = case["D"], case["mode"] == "train"
    if case["op"] == "embed":
        N, V = case["N"], case["V"]
        # tokens by their rank in a language: the k-th most frequent about 1/k as often as the first
        tokens = (torch.exp(torch.rand(N, generator=gen, device="cuda") * math.log(V)) - 1.0).long().clamp_(0, V - 1)
        tokens = torch.randperm(V, generator=gen, device="cuda")[tokens]
        if case["ignored"]:
            tokens[torch.rand(N, generator=gen, device="cuda") < case["ignored"]] = IGNORE
        weight = torch.empty(V, D, dtype=dt, device="cuda")
        for at in range(0, V, 16384):
            part = weight[at:at + 16384]
            part.copy_(_randn(gen, *part.shape) / math.sqrt(D))
        s = {"tokens": tokens, "weight": weight, "scale": math.sqrt(D)}
        if train:
            s["dout"] = _randn(gen, N, D).to(dt)
        return s
    if case["op"] == "drop":
        s = {"x": _randn(gen, case["N"], D).to(dt), "p": case["p"], "seed": seed * 2654435761 % (1 << 63), "offset": 7 + seed}
        if train:
            s["dout"] = _randn(gen, case["N"], D).to(dt)
        return s
    B, L = case["B"], case["L"]
    s = {"lengths": None, "state": None}
    if case["ragged"]:
        s["lengths"] = torch.randint(L // 4, L + 1, (B,), generator=gen, device="cuda")
    if train:
        s["dout"] = _randn(gen, B, L, D).to(dt)
    if case["op"] == "conv":
        W = case["W"]
        s["xz"] = _randn(gen, B, L, 2 * D).to(dt)        # the input and the gate are one projection's halves
        s["weight"] = (_randn(gen, D, W) / math.sqrt(W)).to(dt)
        s["bias"] = (0.1 * _randn(gen, D)).to(dt)
        s["x"] = s["xz"][..., :D]
        if not train:
            s["state"] = _randn(gen, B, W - 1, D).to(dt)
        return s
    N = case["N"]
    s["x"] = _randn(gen, B, L, D).to(dt)
    s["dt"] = (0.5 * _randn(gen, B, L, D)).to(dt)
    # steps of 0.001 to 0.1 spread over the channels, decays of 1 to N
    step = torch.exp(torch.rand(D, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * torch.exp(0.1 * _randn(gen, D, N))
    s["skip"] = 1.0 + 0.1 * _randn(gen, D)
    s["bc"] = _randn(gen, B, L, 2 * N).to(dt)            # one projection's halves
    s["B"], s["C"] = s["bc"][..., :N], s["bc"][..., N:]
    s["z"] = None
    if case["gated"]:
        s["xz"] = _randn(gen, B, L, 2 * D).to(dt)
        s["z"] = s["xz"][..., D:]
    if not train:
        s["state"] = 0.3 * _randn(gen, B, D, N)
    return s


_GRADS = {"embed": ("weight",), "drop": ("x",), "conv": ("x", "weight", "bias"),
          "scan": ("x", "dt", "A", "B", "C", "skip", "z", "dt_bias")}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["mk"] = _package()
        s["leaves"] = [n for n in _GRADS[case["op"]] if s[n] is not None]
        if case["mode"] == "train":
            for n in s["leaves"]:
                s[n].requires_grad_(True)
    return s


def _package():
    root = os.path.join(os.getcwd(), "metal-kans_amd")
    if root not in sys.path:
        sys.path.insert(1, root)
    import metal_kans
    return metal_kans


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    return {"embed": _plain_embed, "drop": _plain_drop, "conv": _plain_conv, "scan": _plain_scan}[op](state)


def _call(s):
    mk, op = s["mk"], s["case"]["op"]
    if op == "embed":
        return mk.embedding(s["tokens"], s["weight"], scale=s["scale"], ignore_index=IGNORE)
    if op == "drop":
        return mk.dropout(s["x"], s["p"], s["seed"], offset=s["offset"])
    if op == "conv":
        return mk.causal_conv(s["x"], s["weight"], s["bias"], activation="silu", state=s["state"], lengths=s["lengths"])
    return mk.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], dt_bias=s["dt_bias"],
                             softplus=True, state=s["state"], lengths=s["lengths"])


def _own(s):
    if s["case"]["mode"] != "train":
        with torch.no_grad():
            out = {"out": _call(s)}
        if s.get("state") is not None:
            out["state"] = s["state"]
        return out
    out = _call(s)
    grads = torch.autograd.grad(out, [s[n] for n in s["leaves"]], s["dout"])
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(s["leaves"], grads)}}


def _plain_embed(s):
    tokens, w, scale = s["tokens"], s["weight"], s["scale"]
    valid = (tokens != IGNORE)[:, None]
    at = torch.where(valid[:, 0], tokens, torch.zeros_like(tokens))
    out = torch.where(valid, w[at].float() * scale, torch.zeros((), device=w.device))
    result = {"out": out.to(w.dtype)}
    if s["case"]["mode"] == "train":
        g = torch.where(valid, s["dout"].float() * scale, torch.zeros((), device=w.device))
        dw = torch.zeros(w.shape, device=w.device)
        dw.index_add_(0, at, g)
        result["dweight"] = dw.to(w.dtype)
    return result


_LOW = 0xffffffff


def _philox(seed, offset, blocks):
    """Philox 4x32 with ten rounds (Salmon et al., 2011) at the counters (block, offset): int64 [blocks, 4] of 32-bit values."""
    i = torch.arange(blocks, device="cuda")
    c0, c1 = i & _LOW, i >> 32
    c2, c3 = torch.full_like(i, offset & _LOW), torch.full_like(i, (offset >> 32) & _LOW)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57       # the low 64 bits, as a signed number
        c0, c1, c2, c3 = ((q >> 32) & _LOW) ^ c1 ^ k0, q & _LOW, ((p >> 32) & _LOW) ^ c3 ^ k1, p & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack((c0, c1, c2, c3), 1)


def _plain_drop(s):
    x, p = s["x"], s["p"]
    n = x.numel()
    keep = (_philox(s["seed"], s["offset"], (n + 3) // 4).reshape(-1)[:n] >= round(p * 2.0 ** 32)).view(x.shape)
    zero, size = torch.zeros((), device=x.device), 1.0 / (1.0 - p)
    out = {"out": torch.where(keep, x.float() * size, zero).to(x.dtype)}
    if s["case"]["mode"] == "train":
        out["dx"] = torch.where(keep, s["dout"].float() * size, zero).to(x.dtype)
    return out


def _inside(lengths, L, device):
    """[B, L, 1]: which steps belong to their sequence; None: all."""
    return None if lengths is None else (torch.arange(L, device=device) < lengths[:, None])[..., None]


def _plain_conv(s):
    case, x, dt = s["case"], s["x"].float(), s["x"].dtype
    B, L, D, W = case["B"], case["L"], case["D"], case["W"]
    w, bias, inside = s["weight"].float(), s["bias"].float(), _inside(s["lengths"], L, x.device)
    if inside is not None:
        x = x * inside
    before = torch.zeros(B, W - 1, D, device=x.device) if s["state"] is None else s["state"].float()
    long = torch.cat((before, x), 1)
    u = bias + sum(w[:, j] * long[:, j:j + L] for j in range(W))
    sig = 1.0 / (1.0 + torch.exp(-u))
    y = u * sig
    if inside is not None:
        y = y * inside
    out = {"out": y.to(dt)}
    if s["state"] is not None:
        if s["lengths"] is None:
            last = long[:, L:]
        else:
            at = s["lengths"][:, None] + torch.arange(W - 1, device=x.device)
            last = long.gather(1, at[..., None].expand(B, W - 1, D))
        s["state"].copy_(last)
        out["state"] = s["state"]
    if case["mode"] == "train":
        du = s["dout"].float() * (sig * (1.0 + u * (1.0 - sig)))
        if inside is not None:
            du = du * inside
        dlong = torch.zeros_like(long)
        for j in range(W):
            dlong[:, j:j + L] += w[:, j] * du
        dx = dlong[:, W - 1:]
        if inside is not None:
            dx = dx * inside
        out["dx"] = dx.to(dt)
        out["dweight"] = torch.stack([(du * long[:, j:j + L]).sum((0, 1)) for j in range(W)], 1).to(dt)
        out["dbias"] = du.sum((0, 1)).to(dt)
    return out


def _plain_scan(s):
    case, dt = s["case"], s["x"].dtype
    L, train = case["L"], case["mode"] == "train"
    x, Bm, Cm = s["x"].float(), s["B"].float(), s["C"].float()
    A, inside = s["A"], _inside(s["lengths"], L, x.device)
    v = s["dt"].float() + s["dt_bias"]
    step = torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))
    if inside is not None:
        x, step = x * inside, step * inside
    # [L, B, D, N]: time first, so that a step of the recurrence is one piece of memory
    a = torch.exp(step.transpose(0, 1)[..., None] * A)
    h = (step * x).transpose(0, 1)[..., None] * Bm.transpose(0, 1)[:, :, None]
    first = torch.zeros_like(h[0]) if s["state"] is None else s["state"]
    h[0].addcmul_(a[0], first)
    for t in range(1, L):
        h[t].addcmul_(a[t], h[t - 1])
    y = (h * Cm.transpose(0, 1)[:, :, None]).sum(-1).transpose(0, 1) + s["skip"] * x
    if s["z"] is not None:
        z = s["z"].float()
        sig = 1.0 / (1.0 + torch.exp(-z))
        full = y * (z * sig)
    else:
        full = y
    if inside is not None:
        full = full * inside
    out = {"out": full.to(dt)}
    if s["state"] is not None:
        s["state"].copy_(h[L - 1])
        out["state"] = s["state"]
    if not train:
        return out
    dy = s["dout"].float() if inside is None else s["dout"].float() * inside
    if s["z"] is not None:
        dz = dy * y * (sig * (1.0 + z * (1.0 - sig)))
        dy = dy * (z * sig)
    dyt = dy.transpose(0, 1)[..., None]
    out_C = (dyt * h).sum(2).transpose(0, 1)
    g = dyt * Cm.transpose(0, 1)[:, :, None]
    for t in range(L - 2, -1, -1):
        g[t].addcmul_(a[t + 1], g[t + 1])
    gB = (g * Bm.transpose(0, 1)[:, :, None]).sum(-1).transpose(0, 1)
    out_B = (g * (step * x).transpose(0, 1)[..., None]).sum(2).transpose(0, 1)
    k = g[1:] * a[1:] * h[:-1]                           # the derivative by step * A (no state before the first)
    dstep = x * gB
    dstep[:, 1:] += (k * A).sum(-1).transpose(0, 1)
    out["dx"] = step * gB + s["skip"] * dy
    ddt = dstep * (1.0 / (1.0 + torch.exp(-v)))
    if inside is not None:
        out["dx"], ddt = out["dx"] * inside, ddt * inside
    out["dx"], out["ddt"] = out["dx"].to(dt), ddt.to(dt)
    out["dA"] = (k * step.transpose(0, 1)[1:, :, :, None]).sum((0, 1))
    out["dB"], out["dC"] = out_B.to(dt), out_C.to(dt)
    out["dskip"] = (dy * x).sum((0, 1))
    if s["z"] is not None:
        out["dz"] = dz.to(dt)
    out["ddt_bias"] = ddt.sum((0, 1))
    return out


# ---- the same in 64 bits -------------------------------------------------------------------------

def exact(case, seed):
    """What a pass on prepare(case, seed) returns, from the definitions in 64 bits."""
    s = _inputs(case, seed)
    return {"embed": _exact_embed, "drop": _exact_drop, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](case, s)


def _exact_embed(case, s):
    """The tokens sorted, the gradients of equal tokens added up between the ends of their runs."""
    tokens, w = s["tokens"], s["weight"]
    table = torch.cat((w.double() * s["scale"], torch.zeros(1, w.shape[1], dtype=torch.float64, device=w.device)))
    row = torch.where(tokens == IGNORE, torch.full_like(tokens, w.shape[0]), tokens)
    out = {"out": table.index_select(0, row)}
    if case["mode"] == "train":
        order = torch.argsort(row)
        total = torch.cumsum(s["dout"].double()[order], 0) * s["scale"]
        names, count = torch.unique_consecutive(row[order], return_counts=True)
        last = torch.cumsum(count, 0) - 1
        sums = total[last]
        sums[1:] -= total[last[:-1]]
        dw = torch.zeros_like(table)
        dw[names] = sums
        out["dweight"] = dw[:-1]
    return out


def _exact_drop(case, s):
    """The generator in numpy's unsigned 64-bit numbers, counters as arrays of their own."""
    n, low = s["x"].numel(), np.uint64(_LOW)
    c = np.zeros((4, (n + 3) // 4), np.uint64)
    c[0] = np.arange(c.shape[1], dtype=np.uint64) & low
    c[1] = np.arange(c.shape[1], dtype=np.uint64) >> np.uint64(32)
    c[2], c[3] = s["offset"] & _LOW, s["offset"] >> 32
    key = [s["seed"] & _LOW, s["seed"] >> 32]
    for _ in range(10):
        even, odd = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c[0] = (odd >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0])
        c[2] = (even >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1])
        c[1], c[3] = odd & low, even & low
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    keep = c.T.reshape(-1)[:n] >= np.uint64(round(case["p"] * 2 ** 32))
    factor = torch.from_numpy(keep).to(s["x"].device).view(s["x"].shape).double() / (1.0 - case["p"])
    out = {"out": s["x"].double() * factor}
    if case["mode"] == "train":
        out["dx"] = s["dout"].double() * factor
    return out


def _exact_conv(case, s):
    """Every output from its own window of inputs, differentiated by autograd; some channels at a time."""
    B, L, D, W = case["B"], case["L"], case["D"], case["W"]
    device, train = s["x"].device, case["mode"] == "train"
    length = torch.full((B,), L, device=device) if s["lengths"] is None else s["lengths"]
    inside = torch.arange(L, device=device)[None] < length[:, None]
    names = ("x", "weight", "bias")
    pieces = {n: [] for n in ("out", "state", "dx", "dweight", "dbias")}
    per = max(1, (1 << 25) // (B * L))
    for a in range(0, D, per):
        x = s["x"][..., a:a + per].double().requires_grad_(train)
        weight, bias = (s[n][a:a + per].double().requires_grad_(train) for n in names[1:])
        before = torch.zeros(B, W - 1, x.shape[2], dtype=torch.float64, device=device) if s["state"] is None else \
            s["state"][..., a:a + per].double()
        known = torch.cat((before, x), 1)
        u = torch.einsum("bldw,dw->bld", known.unfold(1, W, 1), weight) + bias
        y = torch.where(inside[..., None], u * torch.sigmoid(u), torch.zeros_like(u))
        pieces["out"].append(y.detach())
        if s["state"] is not None:
            pieces["state"].append(torch.stack([known[b, int(n):int(n) + W - 1] for b, n in enumerate(length)]).detach())
        if train:
            for n, g in zip(names, torch.autograd.grad(y, (x, weight, bias), s["dout"][..., a:a + per].double())):
                pieces["d" + n].append(g)
    cat = lambda n: torch.cat(pieces[n], 0 if n in ("dweight", "dbias") else 2)  # noqa: E731
    return {n: cat(n) for n, p in pieces.items() if p}


def _exact_scan(case, s):
    """Pairs (decay, state) joined over distances of 1, 2, 4, ... steps, differentiated by autograd; some channels at a time."""
    B, L, D, N = case["B"], case["L"], case["D"], case["N"]
    device, train = s["x"].device, case["mode"] == "train"
    leaves = [n for n in _GRADS["scan"] if s[n] is not None]
    shared = ("B", "C")
    pieces = {}
    inside = torch.ones(B, L, 1, device=device, dtype=torch.float64)
    if s["lengths"] is not None:
        inside = (torch.arange(L, device=device) < s["lengths"][:, None])[..., None].double()
    per = max(1, (1 << 26) // (B * L * N))
    for at in range(0, D, per):
        own_part = slice(at, at + per)
        v = {n: (s[n] if n in shared else s[n][own_part] if s[n].dim() == 1 or n == "A" else s[n][..., own_part])
             .detach().double().requires_grad_(train) for n in leaves}
        step = torch.logaddexp(v["dt"] + v["dt_bias"], torch.zeros((), dtype=torch.float64, device=device)) * inside
        state = torch.einsum("bld,bln->bldn", step * v["x"], v["B"])
        decay = step[..., None] * v["A"]                 # the logarithm of what is left of the state before
        if s["state"] is not None:
            state = torch.cat((s["state"][:, None, own_part].double(), state), 1)
            decay = torch.cat((torch.zeros_like(decay[:, :1]), decay), 1)
        reach = 1
        while reach < state.shape[1]:
            state = torch.cat((state[:, :reach], state[:, reach:] + decay[:, reach:].exp() * state[:, :-reach]), 1)
            decay = torch.cat((decay[:, :reach], decay[:, reach:] + decay[:, :-reach]), 1)
            reach *= 2
        if s["state"] is not None:
            pieces.setdefault("state", []).append(state[:, -1].detach())
            state = state[:, 1:]
        out = torch.einsum("bldn,bln->bld", state, v["C"]) + v["skip"] * v["x"]
        if "z" in v:
            out = out * v["z"] * torch.sigmoid(v["z"])
        out = out * inside
        pieces.setdefault("out", []).append(out.detach())
        if train:
            for n, g in zip(leaves, torch.autograd.grad(out, [v[n] for n in leaves], s["dout"][..., own_part].double())):
                pieces.setdefault("d" + n, []).append(g)
        del state, decay, out, v
    joined = {}
    for n, p in pieces.items():
        joined[n] = sum(p) if n in ("dB", "dC") else torch.cat(p, 2 if n in ("out", "dx", "ddt", "dz") else 1 if n == "state" else 0)
    order = ["out", "state"] + ["d" + n for n in leaves]
    return {n: joined[n] for n in order if n in joined}
