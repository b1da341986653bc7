"""The operators of a feed-forward block over the rows of a voxel network, as measurable cases.

``norm``     RMS norm of ``[N, C]`` rows with the residual's addition before it; its gradients; or its result in 8 bits with a scale a row;
``dropout``  dropout from a counter-based generator and the residual's addition; its gradients;
``linear``   ``residual + dropout(act(x @ weight.T + bias))``, its gradients; or of operands in 8 bits with scales.

Each runs in a plain form of elementary torch operations in 32 bits, or (``own``) through the framework's entry points.

With a residual the sum ``h = x + residual`` is a result of its own, rounded to the inputs' type, and the norm is that of ``h``.
Eight bits are e4m3: a row's scale is its largest magnitude / 448, 2^-126 at least, and its codes are the row over the scale.

The random bits are Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011) with the seed
as its key and (column / 8, row, row >> 32, 0) as its counter: 128 bits for 8 columns of a row, 16 for each, low halves of words
first.  An element whose 16 bits are below round(65536 p) becomes zero, the others are multiplied by 65536 / (65536 - round(65536 p)).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
DEV = "cuda"
EPS = 1e-6
MOST, LEAST = 448.0, 2.0 ** -126   # the largest e4m3 number, the least scale


def listed():
    return [
        # one scan's summary row after pooling: latency
        {"name": "norm_1x256_f32", "kind": "norm", "rows": 1, "channels": 256, "dtype": "f32", "residual": False, "mode": "infer"},
        # a training batch of four scans
        {"name": "norm_240k_c96_bf16", "kind": "norm", "rows": 240000, "channels": 96, "dtype": "bf16", "residual": True, "mode": "train"},
        # the benchmark's batch of eight rooms on its way into a layer of 8-bit operands
        {"name": "norm_1200k_c96_f16_8bit", "kind": "norm", "rows": 1200000, "channels": 96, "dtype": "f16", "residual": True, "mode": "8bit"},
        # features of one small crop, trained without autocast
        {"name": "dropout_2001_c64_f32", "kind": "dropout", "rows": 2001, "channels": 64, "dtype": "f32", "residual": False, "p": 0.1, "train": True},
        # the hidden rows of a block over a training batch
        {"name": "dropout_240k_c384_bf16", "kind": "dropout", "rows": 240000, "channels": 384, "dtype": "bf16", "residual": True, "p": 0.1, "train": True},
        # one scan's summary row: latency
        {"name": "linear_1x256x1024_bf16", "kind": "linear", "rows": 1, "inputs": 256, "outputs": 1024, "dtype": "bf16", "act": "gelu", "residual": False, "p": 0.0, "train": False},
        # a head of 20 classes over a small crop
        {"name": "linear_2000x96x20_f16", "kind": "linear", "rows": 2000, "inputs": 96, "outputs": 20, "dtype": "f16", "act": "none", "residual": False, "p": 0.0, "train": True},
        # a layer trained without autocast
        {"name": "linear_20k_x64x256_f32", "kind": "linear", "rows": 20000, "inputs": 64, "outputs": 256, "dtype": "f32", "act": "silu", "residual": False, "p": 0.0, "train": True},
        # the two layers of a block over a training batch of four scans
        {"name": "linear_240k_x96x384_bf16", "kind": "linear", "rows": 240000, "inputs": 96, "outputs": 384, "dtype": "bf16", "act": "gelu", "residual": False, "p": 0.0, "train": True},
        {"name": "linear_240k_x384x96_bf16", "kind": "linear", "rows": 240000, "inputs": 384, "outputs": 96, "dtype": "bf16", "act": "none", "residual": True, "p": 0.1, "train": True},
        # the widest level of a network
        {"name": "linear_60k_x256x1024_bf16", "kind": "linear", "rows": 60000, "inputs": 256, "outputs": 1024, "dtype": "bf16", "act": "gelu", "residual": False, "p": 0.1, "train": True},
        # a wide layer in inference, operands in 8 bits
        {"name": "linear_100k_x1024x1024_8bit", "kind": "linear", "rows": 100000, "inputs": 1024, "outputs": 1024, "dtype": "8bit", "act": "silu", "residual": True, "p": 0.0, "train": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "dropout", "linear", "linear"])
    if kind != "linear":
        channels = rng.choice([13, 32, 48, 64, 96, 100, 128, 192, 256, 384, 512, 1024])
        case = {"kind": kind, "rows": _log_int(rng, 1, 9e7 / channels), "channels": channels, "dtype": rng.choice(["f32", "f16", "bf16"]),
                "residual": rng.random() < 0.6}
        if kind == "norm":
            return {**case, "mode": rng.choice(["infer", "train", "train", "8bit"])}
        return {**case, "p": round(rng.uniform(0.02, 0.6), 3), "train": rng.random() < 0.6}
    dtype = rng.choice(["f32", "f16", "bf16", "f16", "bf16", "8bit"])
    train = dtype != "8bit" and rng.random() < 0.7
    inputs, outputs = rng.choice([32, 48, 64, 96, 100, 128, 192, 256, 384, 512, 768, 1024]), rng.choice([13, 20, 32, 64, 96, 128, 200, 256, 384, 512, 1024, 1536])
    # fp32 layers are the small ones; no drawn case costs more than the largest listed ones
    most = (4e9 if dtype == "f32" else 1e11) / (inputs * outputs * (3 if train else 1))
    rows = _log_int(rng, 1, min(240000, most, 9e7 / max(inputs, outputs)))
    return {"kind": kind, "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype, "act": rng.choice(["none", "relu", "silu", "gelu"]),
            "residual": rng.random() < 0.5, "p": rng.choice([0.0, 0.1, 0.25]) if train else 0.0, "train": train}


# --------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _codes(x):
    """(e4m3 codes, scales) of the rows of fp32 x."""
    scale = (x.abs().amax(dim=1) * (1 / MOST)).clamp(min=LEAST)
    return (x * (1 / scale)[:, None]).clamp(-MOST, MOST).to(E4M3), scale


def _features(g, n, c, dtype):
    """Rows of unlike length, channels of unlike size."""
    size = torch.exp(0.5 * torch.randn(n, 1, generator=g, device=DEV)) * (0.5 + torch.rand(c, generator=g, device=DEV))
    return (torch.randn(n, c, generator=g, device=DEV) * size).to(dtype)


def _seed_of(g):
    return int(torch.randint(2 ** 62, (), generator=g, device=DEV))


def _prepare_norm(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    n, c = case["rows"], case["channels"]
    s = {"x": _features(g, n, c, dtype), "weight": torch.rand(c, generator=g, device=DEV) + 0.5,
         "residual": _features(g, n, c, dtype) if case["residual"] else None}
    if case["mode"] == "train":
        s["dy"], s["dh"] = ((torch.randn(n, c, generator=g, device=DEV) * 0.1).to(dtype) for _ in range(2))
    return s


def _prepare_dropout(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    n, c = case["rows"], case["channels"]
    s = {"x": _features(g, n, c, dtype), "residual": _features(g, n, c, dtype) if case["residual"] else None, "seed": _seed_of(g)}
    if case["train"]:
        s["dy"] = (torch.randn(n, c, generator=g, device=DEV) * 0.1).to(dtype)
    return s


def _prepare_linear(case, seed):
    g = _generator(seed)
    n, k, m = case["rows"], case["inputs"], case["outputs"]
    dtype = torch.bfloat16 if case["dtype"] == "8bit" else DTYPES[case["dtype"]]
    x, weight = _features(g, n, k, torch.float32), torch.randn(m, k, generator=g, device=DEV) / math.sqrt(k)
    s = {"bias": (torch.randn(m, generator=g, device=DEV) * 0.2).to(dtype), "seed": _seed_of(g),
         "residual": _features(g, n, m, dtype) if case["residual"] else None}
    if case["dtype"] == "8bit":
        s["x"], s["x_scale"] = _codes(x)
        s["weight"], s["weight_scale"] = _codes(weight)
    else:
        s["x"], s["weight"] = x.to(dtype), weight.to(dtype)
    if case["train"]:
        s["dy"] = (torch.randn(n, m, generator=g, device=DEV) * 0.1).to(dtype)
    return s


def prepare(case, seed):
    s = {"norm": _prepare_norm, "dropout": _prepare_dropout, "linear": _prepare_linear}[case["kind"]](case, seed)
    if "dy" in s:
        for k in ("x", "weight", "bias", "residual"):
            if s.get(k) is not None:
                s[k].requires_grad_(True)
    return {**s, "case": dict(case)}


# --------------------------------------------------------------------------- plain forms

M0, M1, W0, W1, WORD = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _drop_factor(seed, n, c, p):
    """0 or 1 / (1 - p) of every element, and those of rows and columns behind the last left out."""
    least = round(65536 * p)
    a = torch.arange(-(-c // 8), device=DEV).expand(n, -1)
    row = torch.arange(n, device=DEV)[:, None].expand_as(a)
    b, d, e = row & WORD, row >> 32, torch.zeros_like(a)
    k0, k1 = seed & WORD, (seed >> 32) & WORD
    for _ in range(10):
        u, v = a * M0, d * M1
        a, b, d, e = ((v >> 32) & WORD) ^ b ^ k0, v & WORD, ((u >> 32) & WORD) ^ e ^ k1, u & WORD
        k0, k1 = (k0 + W0) & WORD, (k1 + W1) & WORD
    words = torch.stack([a, b, d, e], dim=2)
    bits = torch.stack([words & 0xFFFF, words >> 16], dim=3).view(n, -1)[:, :c]
    return (bits >= least).float() * (65536 / max(1, 65536 - least))


def _activation(z, act):
    """act(z) and its derivative."""
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if act == "gelu":
        p = 0.5 * torch.special.erfc(z * -math.sqrt(0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _plain_norm(s):
    x, dtype, mode = s["x"].detach(), s["x"].dtype, s["case"]["mode"]
    out = {}
    if s["residual"] is not None:
        x = out["h"] = (x.float() + s["residual"].detach().float()).to(dtype)
    h, weight = x.float(), s["weight"].detach()
    r = 1 / torch.sqrt(h.square().mean(dim=1, keepdim=True) + EPS)
    y = h * r * weight
    if mode == "8bit":
        out["q"], out["scale"] = _codes(y)
        return out
    out["y"] = y.to(dtype)
    if mode == "train":
        dy = s["dy"].float()
        u = dy * weight
        dx = r * u - h * (r * r * r) * (u * h).mean(dim=1, keepdim=True)
        out["dx"] = (dx + s["dh"].float() if "h" in out else dx).to(dtype)
        if "h" in out:
            out["dresidual"] = out["dx"]
        out["dweight"] = (dy * h * r).sum(0)
    return out


def _plain_dropout(s):
    x, dtype = s["x"].detach(), s["x"].dtype
    factor = _drop_factor(s["seed"], *x.shape, s["case"]["p"])
    y = x.float() * factor
    out = {"y": (y if s["residual"] is None else y + s["residual"].detach().float()).to(dtype)}
    if s["case"]["train"]:
        out["dx"] = (s["dy"].float() * factor).to(dtype)
        if s["residual"] is not None:
            out["dresidual"] = s["dy"]
    return out


def _plain_linear(s):
    case = s["case"]
    x, w, dtype = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].dtype
    if case["dtype"] == "8bit":
        x, w = x * s["x_scale"][:, None], w * s["weight_scale"][:, None]
    z = x @ w.t() + s["bias"].detach().float()
    y, slope = _activation(z, case["act"])
    factor = _drop_factor(s["seed"], *z.shape, case["p"]) if case["p"] else None
    y = y if factor is None else y * factor
    out = {"y": (y if s["residual"] is None else y + s["residual"].detach().float()).to(dtype)}
    if case["train"]:
        dz = s["dy"].float() * slope
        dz = dz if factor is None else dz * factor
        out.update(dx=(dz @ w).to(dtype), dweight=(dz.t() @ x).to(dtype), dbias=dz.sum(0).to(dtype))
        if s["residual"] is not None:
            out["dresidual"] = s["dy"]
    return out


# --------------------------------------------------------------------------- the framework's operators


def _grads(s, results, names, gradients):
    leaves = [k for k in names if s.get(k) is not None]
    got = torch.autograd.grad(results, [s[k] for k in leaves], gradients)
    return {"d" + k: t for k, t in zip(leaves, got)}


def _own_norm(s):
    from warpconvnet_b200.nn.functional.rms_norm import rms_norm, rms_norm_8bit
    mode = s["case"]["mode"]
    if mode == "8bit":
        with torch.no_grad():
            got = rms_norm_8bit(s["x"], s["weight"], eps=EPS, residual=s["residual"])
        return dict(zip(("q", "scale", "h"), got))
    got = rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"])
    y, h = got if s["residual"] is not None else (got, None)
    out = {"y": y.detach()} if h is None else {"y": y.detach(), "h": h.detach()}
    if mode == "train":
        out.update(_grads(s, [y] if h is None else [y, h], ("x", "residual", "weight"), [s["dy"]] if h is None else [s["dy"], s["dh"]]))
    return out


def _own_dropout(s):
    from warpconvnet_b200.nn.functional.dropout import dropout
    y = dropout(s["x"], s["case"]["p"], seed=s["seed"], residual=s["residual"])
    return {"y": y.detach(), **(_grads(s, [y], ("x", "residual"), [s["dy"]]) if s["case"]["train"] else {})}


def _own_linear(s):
    from warpconvnet_b200.nn.functional.linear import linear, linear_8bit
    case = s["case"]
    act = None if case["act"] == "none" else case["act"]
    if case["dtype"] == "8bit":
        with torch.no_grad():
            return {"y": linear_8bit(s["x"], s["x_scale"], s["weight"], s["weight_scale"], s["bias"], activation=act, residual=s["residual"])}
    y = linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"], dropout_p=case["p"], seed=s["seed"])
    return {"y": y.detach(), **(_grads(s, [y], ("x", "weight", "bias", "residual"), [s["dy"]]) if case["train"] else {})}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "dropout": _own_dropout, "linear": _own_linear}[kind](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "dropout": _plain_dropout, "linear": _plain_linear}[kind](state)


# --------------------------------------------------------------------------- 64 bits


def _exact_norm(case, seed):
    s = prepare(case, seed)
    h, out = s["x"].detach(), {}
    if case["residual"]:
        h = out["h"] = (h.double() + s["residual"].detach().double()).to(h.dtype)
    h, w = h.double(), s["weight"].detach().double()
    if case["residual"]:
        out["h"] = h
    norm = torch.sqrt((h * h).sum(1, keepdim=True) / case["channels"] + EPS)
    unit = h / norm
    y = unit * w
    if case["mode"] == "8bit":
        out["scale"] = (y.abs().max(dim=1).values / 448).clamp(min=2.0 ** -126)
        out["q"] = y / out["scale"][:, None]
        return out
    out["y"] = y
    if case["mode"] == "train":
        dy = s["dy"].double()
        u = dy * w
        out["dx"] = (u - unit * ((u * unit).sum(1, keepdim=True) / case["channels"])) / norm
        if case["residual"]:
            out["dx"] = out["dx"] + s["dh"].double()
            out["dresidual"] = out["dx"]
        out["dweight"] = (dy * unit).sum(0)
    return out


def _exact_kept(seed, n, c, p):
    """Which elements stay, a round at a time over a table of the four words."""
    low, high = torch.meshgrid(torch.arange(n, device=DEV), torch.arange((c + 7) // 8, device=DEV), indexing="ij")
    ctr, key = [high, low % 2 ** 32, low // 2 ** 32, torch.zeros_like(low)], [seed % 2 ** 32, seed // 2 ** 32]
    for _ in range(10):
        p0, p1 = ctr[0] * 0xD2511F53, ctr[2] * 0xCD9E8D57
        hi0, hi1 = (p0 >> 32) % 2 ** 32, (p1 >> 32) % 2 ** 32
        ctr = [hi1 ^ ctr[1] ^ key[0], p1 % 2 ** 32, hi0 ^ ctr[3] ^ key[1], p0 % 2 ** 32]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    pieces = [w // 65536 if half else w % 65536 for w in ctr for half in (0, 1)]
    return torch.stack(pieces, dim=-1).reshape(n, -1)[:, :c] >= round(65536 * p)


def _exact_dropout(case, seed):
    s = prepare(case, seed)
    kept = _exact_kept(s["seed"], case["rows"], case["channels"], case["p"])
    rest = 1 - round(65536 * case["p"]) / 65536
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    y = torch.where(kept, s["x"].detach().double() / rest, zero)
    out = {"y": y + s["residual"].detach().double() if case["residual"] else y}
    if case["train"]:
        out["dx"] = torch.where(kept, s["dy"].double() / rest, zero)
        if case["residual"]:
            out["dresidual"] = s["dy"].double()
    return out


def _exact_linear(case, seed):
    s = prepare(case, seed)
    n, act = case["rows"], case["act"]
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    if case["dtype"] == "8bit":
        w = w * s["weight_scale"].double()[:, None]
    rest = 1 - round(65536 * case["p"]) / 65536
    kept = _exact_kept(s["seed"], n, case["outputs"], case["p"]) if case["p"] else None
    y, dx, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    for lo in range(0, n, 32768):
        rows = slice(lo, lo + 32768)
        x = s["x"].detach()[rows].double()
        if case["dtype"] == "8bit":
            x = x * s["x_scale"][rows].double()[:, None]
        z = torch.addmm(b, x, w.t())
        phi = torch.special.ndtr(z)
        value = {"none": z, "relu": z.clamp(min=0), "silu": z * torch.sigmoid(z), "gelu": z * phi}[act]
        if kept is not None:
            value = torch.where(kept[rows], value / rest, 0.0)
        y.append(value + s["residual"].detach()[rows].double() if case["residual"] else value)
        if case["train"]:
            sg = torch.sigmoid(z)
            slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": sg + z * sg * (1 - sg),
                     "gelu": phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)}[act]
            dz = s["dy"][rows].double() * slope
            if kept is not None:
                dz = torch.where(kept[rows], dz / rest, 0.0)
            dx.append(dz @ w)
            dw += dz.t() @ x
            db += dz.sum(0)
    out = {"y": torch.cat(y)}
    if case["train"]:
        out.update(dx=torch.cat(dx), dweight=dw, dbias=db)
        if case["residual"]:
            out["dresidual"] = s["dy"].double()
    return out


def exact(case, seed):
    with torch.no_grad():
        return {"norm": _exact_norm, "dropout": _exact_dropout, "linear": _exact_linear}[case["kind"]](case, seed)


# --------------------------------------------------------------------------- work


def work(case):
    e = {"f32": 4, "f16": 2, "bf16": 2, "8bit": 2}[case["dtype"]]
    n = float(case["rows"])
    if case["kind"] == "norm":
        c, r = case["channels"], int(case["residual"])
        # x (and the residual) in, y (and their sum) out; in training the gradients of the results in, that of x out
        out = 1.0 + 4.0 / c if case["mode"] == "8bit" else e
        bytes_ = n * c * (e * (1 + 2 * r) + out + (e * (2 + r) if case["mode"] == "train" else 0)) + 4.0 * c
        return {"bytes": bytes_, "flops": n * c * (14 if case["mode"] == "train" else 5)}
    if case["kind"] == "dropout":
        c = case["channels"]
        return {"bytes": n * c * e * (2 + int(case["residual"]) + (2 if case["train"] else 0)), "flops": 2.0 * n * c}
    k, m = case["inputs"], case["outputs"]
    operands = 1 if case["dtype"] == "8bit" else e
    bytes_ = operands * (n * k + k * m) + e * n * m * (1 + int(case["residual"]))
    if case["train"]:
        bytes_ += e * (n * m + n * k + k * m)
    return {"bytes": bytes_, "flops": 2.0 * n * k * m * (3 if case["train"] else 1)}
