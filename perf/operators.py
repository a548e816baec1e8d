"""Performance cases of the training-step operators around the KAN layers, on one MI355X.

Three operators that a token model built on ``TorchMetalKANLinear`` blocks calls in every step:

* ``xent``  -- ``linear_cross_entropy``: softmax cross entropy of a linear head over a large
               vocabulary, with the gradients of the hidden rows and of the head (``train``) or the
               loss of every row (``eval``);
* ``norm``  -- ``residual_norm``: the norm behind a block, its gate and residual scale, the residual
               sum and the norm before the next block; forward, or forward and backward;
* ``adamw`` -- ``TorchAdamW.step``: one AdamW step over all tensors of a model, states in 32 or in
               8 bits.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what the
program holds before the call, ``run`` is the call, ``work`` its least traffic and arithmetic and
``exact`` the same results in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ESIZE = {"f32": 4, "f16": 2, "bf16": 2}
IGNORE = -100
EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2
BLOCK = 256          # elements that share a scale of the 8-bit states
TINY = 2.0 ** -126   # least scale
STEP0 = 100          # steps that the optimizer has taken before the pass

_LISTED = [
    # a small classifier head in full precision, one batch of training: launch latency counts
    {"name": "xent_train_f32_256x64x1000", "op": "xent", "mode": "train", "dtype": "f32", "N": 256, "D": 64,
     "V": 1000, "ignored": 0.0, "reduction": "mean"},
    # the losses of a few tokens under a large head (scoring): the head's bytes count
    {"name": "xent_eval_bf16_16x4096x131072", "op": "xent", "mode": "eval", "dtype": "bf16", "N": 16, "D": 4096,
     "V": 131072, "ignored": 0.0, "reduction": "none"},
    # half precision, no size a multiple of a tile, a quarter of the rows padding
    {"name": "xent_train_f16_3001x777x50021", "op": "xent", "mode": "train", "dtype": "f16", "N": 3001, "D": 777,
     "V": 50021, "ignored": 0.25, "reduction": "sum"},
    # full-precision parameters, as the torch modules hold them by default
    {"name": "xent_train_f32_4096x1024x32768", "op": "xent", "mode": "train", "dtype": "f32", "N": 4096, "D": 1024,
     "V": 32768, "ignored": 0.1, "reduction": "mean"},
    # the wide model's head on a full batch of tokens: the largest case
    {"name": "xent_train_bf16_8192x4096x65536", "op": "xent", "mode": "train", "dtype": "bf16", "N": 8192, "D": 4096,
     "V": 65536, "ignored": 0.0, "reduction": "mean"},
    # one token of a wide model between two blocks: launch latency counts
    {"name": "norm_step_bf16_1x4096", "op": "norm", "mode": "forward", "dtype": "bf16", "res": "bf16", "B": 1, "S": 1,
     "D": 4096, "kind": "rms", "gate": "channel", "learned": False},
    # odd sizes in full precision, a gate value for every element (a gating branch's output)
    {"name": "norm_train_f32_2047x1000", "op": "norm", "mode": "train", "dtype": "f32", "res": "f32", "B": 1,
     "S": 2047, "D": 1000, "kind": "layer", "gate": "full", "learned": True},
    # half-precision blocks on a full-precision residual stream, one gate row for each sequence
    {"name": "norm_train_f16_8x512x1024", "op": "norm", "mode": "train", "dtype": "f16", "res": "f32", "B": 8,
     "S": 512, "D": 1024, "kind": "rms", "gate": "group", "learned": True},
    # a full batch of the wide model, one learned gate value a channel
    {"name": "norm_train_bf16_16384x4096", "op": "norm", "mode": "train", "dtype": "bf16", "res": "bf16", "B": 8,
     "S": 2048, "D": 4096, "kind": "rms", "gate": "channel", "learned": True},
    # the digit classifier 784 -> 256 -> 256 -> 10: nine tensors, the smallest of ten elements
    {"name": "adamw32_f32_784_256_256_10", "op": "adamw", "bits": 32, "dtype": "f32", "dims": "784,256,256,10",
     "degree": 9, "repeat": 1},
    # wide layers in bf16 with full-precision masters: the largest step
    {"name": "adamw32_bf16_1024_4096_1024x3", "op": "adamw", "bits": 32, "dtype": "bf16", "dims": "1024,4096,1024",
     "degree": 4, "repeat": 3},
    # ragged layers (no tensor a multiple of the 256 elements of a scale), states in 8 bits
    {"name": "adamw8_f32_777_1300_777x8", "op": "adamw", "bits": 8, "dtype": "f32", "dims": "777,1300,777",
     "degree": 5, "repeat": 8},
]

# no drawn case costs more than the largest listed one of its operator
_MOST_FLOPS = 6 * 8192 * 4096 * 65536
_MOST_LOGITS = 8192 * 65536
_MOST_NORM = 16384 * 4096
_MOST_PARAMS = 126_000_000


def listed():
    return [dict(c) for c in _LISTED]


def _size(rng, lo, hi):
    """A size spread over the logarithm of the range: as it comes, or rounded to a multiple of 8 / 64."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    m = rng.choice((1, 8, 64))
    return max(lo, min(hi, v // m * m))


def draw(rng):
    op = rng.choice(("xent", "norm", "adamw"))
    while True:
        if op == "xent":
            mode = rng.choice(("train", "train", "eval"))
            c = {"op": op, "mode": mode, "dtype": rng.choice(("f32", "f16", "bf16")), "N": _size(rng, 1, 8192),
                 "D": _size(rng, 16, 4096), "V": _size(rng, 10, 131072), "ignored": rng.choice((0.0, 0.1, 0.5)),
                 "reduction": "none" if mode == "eval" else rng.choice(("mean", "sum", "none"))}
            if 6 * c["N"] * c["D"] * c["V"] <= _MOST_FLOPS and c["N"] * c["V"] <= _MOST_LOGITS:
                return c
        elif op == "norm":
            dtype = rng.choice(("f32", "f16", "bf16"))
            c = {"op": op, "mode": rng.choice(("train", "train", "forward")), "dtype": dtype,
                 "res": rng.choice((dtype, "f32")), "B": rng.randint(1, 8), "S": _size(rng, 1, 16384),
                 "D": _size(rng, 16, 8192), "kind": rng.choice(("rms", "layer")),
                 "gate": rng.choice(("none", "channel", "group", "full")), "learned": rng.random() < 0.5}
            if c["B"] * c["S"] * c["D"] <= _MOST_NORM:
                return c
        else:
            dims = [_size(rng, 16, 4096) for _ in range(rng.randint(2, 5))]
            c = {"op": op, "bits": rng.choice((32, 8)), "dtype": rng.choice(("f32", "f16", "bf16")),
                 "dims": ",".join(map(str, dims)), "degree": rng.randint(3, 9), "repeat": rng.randint(1, 12)}
            if sum(_numel(s) for s in _shapes(c)) <= _MOST_PARAMS:
                return c


# ---- sizes ---------------------------------------------------------------------------------------

def _shapes(case):
    """The tensors of the networks: weight, base weight and bias of each layer."""
    dims = [int(v) for v in case["dims"].split(",")]
    one = [s for i, o in zip(dims, dims[1:]) for s in ((o, i * case["degree"]), (o, i), (o,))]
    return one * case["repeat"]


def _numel(shape):
    return math.prod(shape)


def _gate_rows(case):
    return {"none": 0, "channel": 1, "group": case["B"], "full": case["B"] * case["S"]}[case["gate"]]


def work(case):
    """Bytes: each input read once and each output written once, in the types that the call hands over.
    Flops: the products with the head (2 N D V forward, as many again for each gradient); about what a
    value costs for the others."""
    if case["op"] == "xent":
        N, D, V, e = case["N"], case["D"], case["V"], _ESIZE[case["dtype"]]
        train = case["mode"] == "train"
        return {"bytes": (2 if train else 1) * e * (N + V) * D + 8 * N + 4 * N, "flops": (6 if train else 2) * N * D * V}
    if case["op"] == "norm":
        N, D, e, r = case["B"] * case["S"], case["D"], _ESIZE[case["dtype"]], _ESIZE[case["res"]]
        n, g = N * D, _gate_rows(case) * D
        fwd = n * (2 * r + 2 * e) + e * (g + 2 * D)          # x, block, gate, weights; y, h
        bwd = n * (2 * r + 2 * e) + e * (g + 2 * D)          # dy, dh; dx, dblock, dgate, weights' gradients
        train = case["mode"] == "train"
        return {"bytes": fwd + (bwd if train else 0), "flops": n * (36 if train else 12)}
    n, e = sum(_numel(s) for s in _shapes(case)), _ESIZE[case["dtype"]]
    master = 8 if e == 2 else 0
    # the parameter (read as the master where there is one), its gradient, the master; the states as they are
    # held, read and written, and for 8 bits also the values they stand for, written
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
    return {"bytes": n * ((e if master else 2 * e) + e + master + states), "flops": n * 16}


# ---- inputs --------------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _inputs(case, seed):
    """The inputs of a case, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _DT.get(case.get("dtype"))
    if case["op"] == "xent":
        N, D, V = case["N"], case["D"], case["V"]
        # normalized rows and a head whose logits have a spread of about two
        hidden = _randn(gen, N, D).to(dt)
        weight = torch.empty(V, D, dtype=dt, device="cuda")
        for at in range(0, V, 16384):
            part = weight[at:at + 16384]
            part.copy_(_randn(gen, *part.shape) * (2.0 / math.sqrt(D)))
        target = torch.randint(0, V, (N,), generator=gen, device="cuda")
        if case["ignored"]:
            target[torch.rand(N, generator=gen, device="cuda") < case["ignored"]] = IGNORE
            target[0] = 0  # one row at least counts
        grad = None
        if case["mode"] == "train":
            grad = torch.rand(N, generator=gen, device="cuda") + 0.5 if case["reduction"] == "none" else \
                torch.ones((), device="cuda")
        return {"hidden": hidden, "weight": weight, "target": target, "grad": grad}
    if case["op"] == "norm":
        B, S, D, rt = case["B"], case["S"], case["D"], _DT[case["res"]]
        # the residual stream grows over the blocks; a few channels are far larger than the rest
        spread = torch.exp(0.5 * _randn(gen, D))
        s = {"x": (2.0 * spread * _randn(gen, B, S, D)).to(rt), "block": (0.7 * _randn(gen, B, S, D) + 0.1).to(dt)}
        rows = {"none": None, "channel": (D,), "group": (B, 1, D), "full": (B, S, D)}[case["gate"]]
        s["gate"] = None if rows is None else (0.5 + 0.3 * _randn(gen, *rows)).to(dt)
        s["post_weight"] = (1.0 + 0.1 * _randn(gen, D)).to(dt)
        s["pre_weight"] = (1.0 + 0.1 * _randn(gen, D)).to(dt)
        s["scale"] = torch.full((1,), 0.4, device="cuda") if case["learned"] else 0.4
        if case["mode"] == "train":
            s["dy"] = _randn(gen, B, S, D).to(rt)
            s["dh"] = _randn(gen, B, S, D).to(dt)
        return s
    # parameters and states in one buffer each (as for sharding), every tensor at a multiple of BLOCK elements
    shapes = _shapes(case)
    total = sum(_padded(shape) for shape in shapes)
    f32 = lambda: torch.zeros(total, device="cuda")  # noqa: E731
    s = {"flat": torch.zeros(total, dtype=dt, device="cuda"), "grads": [], "exp_avg": f32(), "exp_avg_sq": f32(),
         "master": f32() if dt != torch.float32 else None}
    for part, shape in zip(_parts(shapes), shapes):
        size = math.exp(float(torch.rand((), generator=gen, device="cuda").item()) * 4 - 9)  # of this tensor's gradients
        master = _randn(gen, *shape) / math.sqrt(shape[-1])
        grad = size * _randn(gen, *shape)
        if len(shape) > 1:
            grad[::7] = 0.0      # rows that the batch did not reach
        s["flat"][part].copy_(master.reshape(-1))
        if s["master"] is not None:
            s["master"][part].copy_(master.reshape(-1))
        s["grads"].append(grad.to(dt))
        s["exp_avg"][part].copy_(0.3 * size * _randn(gen, _numel(shape)))
        s["exp_avg_sq"][part].copy_(size * size * (0.02 + torch.rand(_numel(shape), generator=gen, device="cuda")))
    return s


def _padded(shape):
    return -(-_numel(shape) // BLOCK) * BLOCK


def _parts(shapes):
    """Where each tensor lies in a buffer of all of them."""
    at = 0
    for shape in shapes:
        yield slice(at, at + _numel(shape))
        at += _padded(shape)


def _encode_avg(m):
    rows = m.reshape(-1, BLOCK)
    scale = rows.abs().amax(1).clamp_min(TINY)
    code = torch.round(127.0 * torch.sqrt(rows.abs() * (1.0 / scale)[:, None])) * torch.sign(rows)
    return code.clamp(-127, 127).to(torch.int8).reshape(-1), scale


def _decode_avg(code, scale):
    t = code.reshape(-1, BLOCK).to(scale.dtype) * (1.0 / 127.0)
    return (scale[:, None] * (t * t.abs())).reshape(-1)


def _encode_sq(v):
    rows = v.reshape(-1, BLOCK)
    scale = rows.amax(1).clamp_min(TINY)
    code = torch.round(255.0 * torch.sqrt(torch.sqrt(rows * (1.0 / scale)[:, None])))
    code = torch.where(rows > 0, code.clamp(1, 255), torch.zeros_like(code))
    return code.to(torch.uint8).reshape(-1), scale


def _decode_sq(code, scale):
    t = code.reshape(-1, BLOCK).to(scale.dtype) * (1.0 / 255.0)
    t = t * t
    return (scale[:, None] * (t * t)).reshape(-1)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "adamw":
        shapes = _shapes(case)
        s["params"] = [s["flat"][part].view(shape) for part, shape in zip(_parts(shapes), shapes)]
        s["step"] = STEP0
        if case["bits"] == 8:
            s["exp_avg"], s["exp_avg_scale"] = _encode_avg(s["exp_avg"])
            s["exp_avg_sq"], s["exp_avg_sq_scale"] = _encode_sq(s["exp_avg_sq"])
    if not own:
        return s
    s["mk"] = mk = _package()
    if case["op"] == "adamw":
        for p, g in zip(s["params"], s["grads"]):
            p.grad = g
        s["opt"] = opt = mk.TorchAdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY,
                                       state_bits=case["bits"])
        sd = opt.state_dict()
        for i, (part, shape) in enumerate(zip(_parts(shapes), shapes)):
            sd["state"][i] = st = {"step": STEP0}
            for name in ("exp_avg", "exp_avg_sq", "master"):
                if s.get(name) is not None:
                    st[name] = s[name][part].view(shape)
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                if name in s:
                    st[name] = s[name][part.start // BLOCK:(part.stop + BLOCK - 1) // BLOCK]
        opt.load_state_dict(sd)
        for name in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master"):
            s.pop(name, None)    # the optimizer holds them now
    elif case["mode"] == "train":
        for name in ("hidden", "weight", "x", "block", "gate", "post_weight", "pre_weight", "scale"):
            if isinstance(s.get(name), torch.Tensor):
                s[name].requires_grad_(True)
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
        return {"xent": _own_xent, "norm": _own_norm, "adamw": _own_adamw}[op](state)
    return {"xent": _plain_xent, "norm": _plain_norm, "adamw": _plain_adamw}[op](state)


def _own_xent(s):
    case, mk = s["case"], s["mk"]
    if case["mode"] == "eval":
        with torch.no_grad():
            return {"loss": mk.linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE,
                                                    reduction=case["reduction"])}
    loss = mk.linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE,
                                   reduction=case["reduction"])
    dh, dw = torch.autograd.grad(loss, (s["hidden"], s["weight"]), s["grad"])
    return {"loss": loss.detach(), "dhidden": dh, "dweight": dw}


def _own_norm(s):
    case, mk = s["case"], s["mk"]
    call = lambda: mk.residual_norm(s["x"], s["block"], gate=s["gate"], scale=s["scale"],  # noqa: E731
                                    post_weight=s["post_weight"], pre_weight=s["pre_weight"], kind=case["kind"], eps=EPS)
    if case["mode"] == "forward":
        with torch.no_grad():
            y, h = call()
        return {"y": y, "h": h}
    y, h = call()
    names = [n for n in ("x", "block", "gate", "post_weight", "pre_weight", "scale") if isinstance(s[n], torch.Tensor)]
    grads = torch.autograd.grad((y, h), [s[n] for n in names], (s["dy"], s["dh"]))
    return {"y": y.detach(), "h": h.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _own_adamw(s):
    opt = s["opt"]
    opt.step()
    flat = opt.flat_state()[0]   # of the one parameter group
    return {"params": s["flat"], **{n: flat[n] for n in ("exp_avg", "exp_avg_sq", "master") if n in flat}}


def _plain_xent(s):
    case, target, dt = s["case"], s["target"], s["hidden"].dtype
    h, w = s["hidden"].float(), s["weight"].float()
    valid = target != IGNORE
    at = torch.where(valid, target, torch.zeros_like(target))[:, None]
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at)
    prob = logits.sub_(top).exp_()
    total = prob.sum(1, keepdim=True)
    loss = torch.where(valid, (top + torch.log(total) - picked)[:, 0], torch.zeros_like(total[:, 0]))
    count = valid.sum()
    if case["reduction"] == "mean":
        loss = loss.sum() / count
    elif case["reduction"] == "sum":
        loss = loss.sum()
    if case["mode"] == "eval":
        return {"loss": loss}
    row = s["grad"] / count if case["reduction"] == "mean" else s["grad"]
    row = torch.where(valid, row.expand(target.shape), torch.zeros_like(total[:, 0]))[:, None]
    g = prob.div_(total)
    g.scatter_add_(1, at, torch.full_like(total, -1.0))
    g.mul_(row)
    return {"loss": loss, "dhidden": (g @ w).to(dt), "dweight": (g.t() @ h).to(dt)}


def _plain_stats(a, kind):
    """A row's normalized values and the reciprocal of its size."""
    if kind == "layer":
        a = a - a.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((a * a).mean(-1, keepdim=True) + EPS)
    return a * r, r


def _plain_norm_grad(q, n, r, kind):
    """The norm's transposed derivative times q, at normalized values n and reciprocal size r."""
    g = q - n * (q * n).mean(-1, keepdim=True)
    if kind == "layer":
        g = g - q.mean(-1, keepdim=True)
    return r * g


def _plain_norm(s):
    case = s["case"]
    kind, dt, rt = case["kind"], s["block"].dtype, s["x"].dtype
    x, block, gate = s["x"].float(), s["block"].float(), None if s["gate"] is None else s["gate"].float()
    post, pre, scale = s["post_weight"].float(), s["pre_weight"].float(), s["scale"]
    bn, br = _plain_stats(block, kind)
    u = bn * post
    gu = u if gate is None else gate * u
    y = x + scale * gu
    yn, yr = _plain_stats(y, kind)
    out = {"y": y.to(rt), "h": (yn * pre).to(dt)}
    if case["mode"] == "forward":
        return out
    dh = s["dh"].float()
    t = s["dy"].float() + _plain_norm_grad(pre * dh, yn, yr, kind)
    out["dx"] = t.to(rt)
    du = scale * t if gate is None else scale * gate * t
    out["dblock"] = _plain_norm_grad(post * du, bn, br, kind).to(dt)
    if gate is not None:
        dg = scale * t * u
        out["dgate"] = {"channel": lambda: dg.sum((0, 1)), "group": lambda: dg.sum(1, keepdim=True),
                        "full": lambda: dg}[case["gate"]]().to(dt)
    out["dpost_weight"] = (du * bn).sum((0, 1)).to(dt)
    out["dpre_weight"] = (dh * yn).sum((0, 1)).to(dt)
    if case["learned"]:
        out["dscale"] = (t * gu).sum().reshape(1)
    return out


def _plain_adamw(s):
    case = s["case"]
    s["step"] += 1
    size = LR / (1.0 - BETA1 ** s["step"])
    root = 1.0 / math.sqrt(1.0 - BETA2 ** s["step"])
    eight = case["bits"] == 8
    m_all = _decode_avg(s["exp_avg"], s["exp_avg_scale"]) if eight else s["exp_avg"]
    v_all = _decode_sq(s["exp_avg_sq"], s["exp_avg_sq_scale"]) if eight else s["exp_avg_sq"]
    for part, p, g in zip(_parts(_shapes(case)), s["params"], s["grads"]):
        g = g.reshape(-1).float()
        m, v = m_all[part], v_all[part]
        m.copy_(m * BETA1 + g * (1.0 - BETA1))
        v.copy_(v * BETA2 + (g * g) * (1.0 - BETA2))
        p = p.view(-1)
        master = p if s["master"] is None else s["master"][part]
        master.copy_(master * (1.0 - LR * DECAY) - size * (m / (torch.sqrt(v) * root + ADAM_EPS)))
        if master is not p:
            p.copy_(master)
    if eight:
        s["exp_avg"], s["exp_avg_scale"] = _encode_avg(m_all)
        s["exp_avg_sq"], s["exp_avg_sq_scale"] = _encode_sq(v_all)
        m_all, v_all = _decode_avg(s["exp_avg"], s["exp_avg_scale"]), _decode_sq(s["exp_avg_sq"], s["exp_avg_sq_scale"])
    out = {"params": s["flat"], "exp_avg": m_all, "exp_avg_sq": v_all}
    if s["master"] is not None:
        out["master"] = s["master"]
    return out


# ---- the same in 64 bits -------------------------------------------------------------------------

def exact(case, seed):
    """What a pass on prepare(case, seed) returns, from the definitions in 64 bits."""
    s = _inputs(case, seed)
    return {"xent": _exact_xent, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](case, s)


def _exact_xent(case, s):
    """Row by row of the definition, some thousand rows at a time; the gradients from the probabilities."""
    w, target = s["weight"].double(), s["target"]
    N, V = target.numel(), w.shape[0]
    valid = target != IGNORE
    count = int(valid.sum())
    rows = max(1, min(N, (1 << 28) // V))
    loss = torch.zeros(N, dtype=torch.float64, device=w.device)
    train = case["mode"] == "train"
    dh = torch.zeros(s["hidden"].shape, dtype=torch.float64, device=w.device) if train else None
    dw = torch.zeros_like(w) if train else None
    for a in range(0, N, rows):
        ids = torch.nonzero(valid[a:a + rows])[:, 0] + a
        if ids.numel() == 0:
            continue
        h, t = s["hidden"][ids].double(), target[ids]
        logp = torch.log_softmax(h @ w.t(), 1)
        loss[ids] = -logp[torch.arange(t.numel(), device=t.device), t]
        if train:
            g = logp.exp()
            g[torch.arange(t.numel(), device=t.device), t] -= 1.0
            g *= s["grad"].double()[ids][:, None] if case["reduction"] == "none" else \
                s["grad"].double() / (count if case["reduction"] == "mean" else 1)
            dh[ids] = g @ w
            dw += g.t() @ h
    if case["reduction"] == "mean":
        loss = loss.sum() / count
    elif case["reduction"] == "sum":
        loss = loss.sum()
    return {"loss": loss, "dhidden": dh, "dweight": dw} if train else {"loss": loss}


def _exact_norm(case, s):
    """The forward's definition in 64 bits, differentiated by autograd."""
    names = [n for n in ("x", "block", "gate", "post_weight", "pre_weight", "scale") if isinstance(s[n], torch.Tensor)]
    d = dict(s)
    train = case["mode"] == "train"
    for n in names:
        d[n] = s[n].double().requires_grad_(train)

    def normalized(a):
        var, mean = torch.var_mean(a, dim=-1, correction=0, keepdim=True)
        if case["kind"] == "layer":
            return (a - mean) / (var + EPS).sqrt()
        return a / (var + mean.square() + EPS).sqrt()

    branch = normalized(d["block"]) * d["post_weight"] * d["scale"]
    y = d["x"] + (branch if d["gate"] is None else branch * d["gate"])
    h = normalized(y) * d["pre_weight"]
    if not train:
        return {"y": y, "h": h}
    grads = torch.autograd.grad((y, h), [d[n] for n in names], (s["dy"].double(), s["dh"].double()))
    return {"y": y.detach(), "h": h.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _exact_adamw(case, s):
    """The update's definition; 8-bit states are taken up as they are held and come out as the nearest value
    that they can hold."""
    t = STEP0 + 1
    m, v = s["exp_avg"], s["exp_avg_sq"]
    if case["bits"] == 8:
        (mc, ms), (vc, vs) = _encode_avg(m), _encode_sq(v)
        m, v = _decode_avg(mc, ms.double()), _decode_sq(vc, vs.double())
    m, v = m.double(), v.double()
    w = (s["flat"] if s["master"] is None else s["master"]).double()
    g = torch.zeros_like(w)
    for part, one in zip(_parts(_shapes(case)), s["grads"]):
        g[part] = one.reshape(-1).double()
    m = BETA1 * m + (1.0 - BETA1) * g
    v = BETA2 * v + (1.0 - BETA2) * g.square()
    w = w - LR * (m / (1.0 - BETA1 ** t) / ((v / (1.0 - BETA2 ** t)).sqrt() + ADAM_EPS) + DECAY * w)
    if case["bits"] == 8:
        m, v = _decode_avg(*_encode_avg(m)), _decode_sq(*_encode_sq(v))
    out = {"params": w, "exp_avg": m, "exp_avg_sq": v}
    if s["master"] is not None:
        out["master"] = w
    return out
