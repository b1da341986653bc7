"""The operators of a training step around the network's layers, as measurable cases.

``norm``   segmented group norm with an activation: statistics per scene and channel group of ``[N, C]`` rows;
``loss``   linear cross entropy: the loss of ``x @ weight.T + bias`` against labels, without the logits;
``step``   one AdamW step over many tensors, moments in 32 or in 8 bits.

Each runs in a plain form of elementary torch operations in 32 bits, or (``own``) through the framework's entry points.

Moments in 8 bits are codes of a logarithmic scale, 8 values to an octave, in blocks of 256 elements.  A block has a base; the
code k > 0 stands for the fp32 number whose bits are ``(k + base) << 20``, the code 0 for zero.  The first moment has a sign bit
above 7 bits of magnitude, the second moment 8 bits.  The base puts the block's largest magnitude at the last code but one.  A
number is rounded to one of its two neighbours at random, with probabilities that keep its mean; the random bits are a hash of the
tensor's step and the element's place.  A second moment that is not zero never becomes zero.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
BLOCK = 256
IGNORE = -100
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01
NORM_EPS = 1e-5


def listed():
    return [
        # inference over one small scan in fp32: latency
        {"name": "norm_1x20k_c32_f32", "kind": "norm", "scenes": 1, "rows": 20000, "channels": 32, "groups": 8, "dtype": "f32", "act": "relu", "train": False},
        # a training batch of four scans
        {"name": "norm_4x60k_c64_bf16", "kind": "norm", "scenes": 4, "rows": 240000, "channels": 64, "groups": 16, "dtype": "bf16", "act": "relu", "train": True},
        # crops of objects: many short scenes, odd row counts
        {"name": "norm_300x233_c128_bf16", "kind": "norm", "scenes": 300, "rows": 69901, "channels": 128, "groups": 32, "dtype": "bf16", "act": "gelu", "train": True},
        # the benchmark's batch of eight rooms, the last decoder's width: larger than L2
        {"name": "norm_8x150k_c96_f16", "kind": "norm", "scenes": 8, "rows": 1200000, "channels": 96, "groups": 8, "dtype": "f16", "act": "silu", "train": True},
        # a head of 20 classes over the voxels of one small crop: latency
        {"name": "loss_2k_c96_v20_bf16", "kind": "loss", "rows": 2000, "channels": 96, "classes": 20, "dtype": "bf16", "bias": True, "train": True},
        # a layer trained without autocast
        {"name": "loss_20k_c64_v40_f32", "kind": "loss", "rows": 20000, "channels": 64, "classes": 40, "dtype": "f32", "bias": True, "train": True},
        # segmentation into 200 classes over a batch of four scans
        {"name": "loss_240k_c96_v200_bf16", "kind": "loss", "rows": 240000, "channels": 96, "classes": 200, "dtype": "bf16", "bias": True, "train": True},
        # per-row losses of a validation pass over a codebook of 4096 entries
        {"name": "loss_60k_c128_v4096_f16", "kind": "loss", "rows": 60000, "channels": 128, "classes": 4096, "dtype": "f16", "bias": False, "train": False},
        # prediction of codebook entries for the masked voxels of a batch
        {"name": "loss_30k_c256_v32768_bf16", "kind": "loss", "rows": 30000, "channels": 256, "classes": 32768, "dtype": "bf16", "bias": False, "train": True},
        # a small head and a few norms: latency
        {"name": "step_head_f32", "kind": "step", "shapes": "head", "width": 96, "dtype": "f32", "bits": 32},
        # all parameters of MinkUNet-34
        {"name": "step_unet34_f32", "kind": "step", "shapes": "unet34", "width": 32, "dtype": "f32", "bits": 32},
        {"name": "step_unet34_8bit", "kind": "step", "shapes": "unet34", "width": 32, "dtype": "f32", "bits": 8},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "loss", "step"])
    if kind == "norm":
        groups = rng.choice([1, 4, 8, 16, 32])
        channels = groups * rng.choice([c for c in (1, 2, 3, 4, 6, 8, 12, 16, 32) if 16 <= c * groups <= 256])
        scenes = _log_int(rng, 1, 400)
        rows = max(scenes, _log_int(rng, 300, min(600000, 5.7e7 / channels)))
        return {"kind": kind, "scenes": scenes, "rows": rows, "channels": channels, "groups": groups,
                "dtype": rng.choice(["f32", "f16", "bf16"]), "act": rng.choice(["none", "relu", "silu", "gelu"]), "train": rng.random() < 0.7}
    if kind == "loss":
        dtype = rng.choice(["f32", "f16", "bf16", "f16", "bf16"])
        rows = _log_int(rng, 100, 20000 if dtype == "f32" else 200000)
        channels = rng.choice([32, 48, 64, 96, 100, 128, 192, 256])
        # fp32 heads are the small ones; no drawn case costs more than the largest listed one
        classes = _log_int(rng, 13, min(1000 if dtype == "f32" else 40000, 2.4e11 / (rows * channels)))
        return {"kind": kind, "rows": rows, "channels": channels, "classes": classes, "dtype": dtype, "bias": rng.random() < 0.5,
                "train": rng.random() < 0.75}
    shapes = rng.choice(["head", "unet18", "unet34", "codebook"])
    return {"kind": kind, "shapes": shapes, "width": _log_int(rng, 10, 31 if shapes.startswith("unet") else 200),
            "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "bits": rng.choice([32, 8])}


# --------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _offsets(case):
    """Scene boundaries: unequal scenes, every seventh of them short (of many: empty)."""
    b, n = case["scenes"], case["rows"]
    w = [1.0 + 0.5 * math.sin(1.7 * i) for i in range(b)]
    for i in range(6, b, 7):
        w[i] = 0.01 if b < 50 else 0.0
    at, total, out = 0.0, sum(w), [0]
    for v in w:
        at += v
        out.append(min(n, int(round(n * at / total))))
    out[-1] = n
    return torch.tensor(out, dtype=torch.int64)


def _prepare_norm(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    n, c = case["rows"], case["channels"]
    typical = torch.randn(c, generator=g, device=DEV)
    x = (torch.randn(n, c, generator=g, device=DEV) * 1.5 + typical).to(dtype)
    s = {"kind": "norm", "x": x, "offsets": _offsets(case), "groups": case["groups"], "act": case["act"], "train": case["train"],
         "weight": torch.rand(c, generator=g, device=DEV) + 0.5, "bias": torch.randn(c, generator=g, device=DEV) * 0.2}
    if case["train"]:
        s["dy"] = (torch.randn(n, c, generator=g, device=DEV) * 0.1).to(dtype)
        for k in ("x", "weight", "bias"):
            s[k].requires_grad_(True)
    return s


def _prepare_loss(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    n, c, v = case["rows"], case["channels"], case["classes"]
    weight = torch.randn(v, c, generator=g, device=DEV) / math.sqrt(c)
    # frequent and rare classes; features of a network that has learned something: between the row of its class and noise
    labels = (v * torch.rand(n, generator=g, device=DEV) ** 2).long().clamp_(max=v - 1)
    sure = torch.rand(n, 1, generator=g, device=DEV) * 6
    x = torch.randn(n, c, generator=g, device=DEV) + sure * weight[labels]
    labels = torch.where(torch.rand(n, generator=g, device=DEV) < 0.05, IGNORE, labels)
    s = {"kind": "loss", "x": x.to(dtype), "weight": weight.to(dtype), "labels": labels, "train": case["train"],
         "bias": (torch.randn(v, generator=g, device=DEV) * 0.5).to(dtype) if case["bias"] else None}
    if case["train"]:
        # the gradient that arrives at the loss: training in fp16 scales it up
        s["gradient"] = torch.tensor(65536.0 if case["dtype"] == "f16" else 1.0, device=DEV)
        for k in ("x", "weight", "bias"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _sizes(case):
    """Element counts of the tensors that a step updates, in a network's order."""
    w = case["width"]
    if case["shapes"] == "head":
        return [w * w, w, w, w * w, w, w, w * 20, 20]
    if case["shapes"] == "codebook":
        return [8192 * 8 * w, 8 * w * 96, 96, 13, 1]
    layers = (2, 3, 4, 6, 2, 2, 2, 2) if case["shapes"] == "unet34" else (2,) * 8
    planes = [w * m for m in (1, 2, 4, 8, 8, 4, 3, 3)]
    out = [3 * w, w, w]

    def conv(k, a, b):
        out.extend([k * a * b, b, b])

    def stage(a, b, blocks):
        for i in range(blocks):
            conv(27, a if i == 0 else b, b)
            conv(27, b, b)
            if i == 0 and a != b:
                conv(1, a, b)

    c = w
    for i in range(4):
        conv(8, c, c)
        stage(c, planes[i], layers[i])
        c = planes[i]
    skips = [w] + planes[:3]
    for i in range(4):
        conv(8, c, planes[4 + i])
        stage(planes[4 + i] + skips[3 - i], planes[4 + i], layers[4 + i])
        c = planes[4 + i]
    return out + [c * 20, 20]


def _slots(sizes):
    """First element of each tensor's moments: tensors follow one another, each from a block of its own on."""
    at, out = 0, []
    for n in sizes:
        out.append(at)
        at += -(-n // BLOCK) * BLOCK
    return out, at


def _bits(x):
    return x.contiguous().view(torch.int32).to(torch.int64)


def _number(bits):
    return bits.to(torch.int32).view(torch.float32)


def _decode(codes, base, signed):
    """The numbers that 8-bit codes stand for."""
    k = codes.view(-1, BLOCK).to(torch.int64)
    mag = k & 127 if signed else k
    x = torch.where(mag > 0, _number((mag + base.to(torch.int64)[:, None]) << 20), 0.0)
    return (torch.where(k > 127, -x, x) if signed else x).flatten()


def _encode(x, random, signed):
    """(codes, bases) of numbers, given 20 random bits for each."""
    top = 127 if signed else 255
    bits = _bits(x.abs()).view(-1, BLOCK)
    base = ((bits.max(dim=1).values >> 20) + 1 - top).clamp_(min=0)
    random = random.view(-1, BLOCK)
    code = ((bits + random) >> 20) - base[:, None]
    if signed:  # below the first code: that one or zero, the mean kept
        first = _number((base + 1) << 20)[:, None]
        up = _number(bits) > first * (random.float() * 2.0 ** -20)
        code = torch.where((code < 1) & (base[:, None] > 0), up.to(torch.int64), code)
        code = code + 128 * (x.view(-1, BLOCK) < 0)
    else:
        code = torch.where(bits > 0, code.clamp(min=1), 0)
    return code.to(torch.uint8).flatten(), base.to(torch.int16)


def _mix(h):
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _random(steps, place):
    """20 bits for the first moment and 20 for the second, of a tensor's step and the element's place among the moments."""
    h = _mix(((place * 0x9E3779B9) & 0xFFFFFFFF) ^ _mix(steps))
    return h >> 12, ((h * 0x9E3779B1) & 0xFFFFFFFF) >> 12


def _prepare_step(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    sizes = _sizes(case)
    slots, length = _slots(sizes)
    total = sum(sizes)
    which = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.tensor(sizes, device=DEV), output_size=total)
    shift = torch.tensor(slots, device=DEV) - (torch.tensor(sizes, device=DEV).cumsum(0) - torch.tensor(sizes, device=DEV))
    place = torch.arange(total, device=DEV) + shift[which]
    # gradients of unlike size from channel to channel, moments to match
    scale = torch.zeros(length, device=DEV)
    scale[place] = 1e-3 * torch.exp(torch.randn(total, generator=g, device=DEV))
    m = scale * 0.4 * torch.randn(length, generator=g, device=DEV)
    v = scale.square() * (0.8 + 0.4 * torch.rand(length, generator=g, device=DEV))
    flat = (0.05 * torch.randn(total, generator=g, device=DEV)).to(dtype)
    grad = (scale[place] * torch.randn(total, generator=g, device=DEV)).to(dtype)
    s = {"kind": "step", "bits": case["bits"], "flat": flat, "params": list(flat.split(sizes)), "grad": grad, "grads": list(grad.split(sizes)),
         "steps": torch.full((len(sizes),), 10, dtype=torch.int32, device=DEV), "which": which, "place": place}
    if case["bits"] == 8:
        half = torch.full((length,), 1 << 19, dtype=torch.int64, device=DEV)
        s["m"], s["m_base"] = _encode(m, half, True)
        s["v"], s["v_base"] = _encode(v, half, False)
    else:
        s["m"], s["v"] = m, v
    return s


def prepare(case, seed):
    return {"norm": _prepare_norm, "loss": _prepare_loss, "step": _prepare_step}[case["kind"]](case, seed)


# --------------------------------------------------------------------------- plain forms


def _activation(z, act):
    """act(z) and its derivative."""
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _plain_norm(s):
    x, groups, dtype = s["x"].detach(), s["groups"], s["x"].dtype
    n, c = x.shape
    sizes = (s["offsets"][1:] - s["offsets"][:-1]).to(DEV, non_blocking=True)
    scene = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), sizes, output_size=n)
    count = (sizes * (c // groups)).clamp(min=1).to(torch.float32)[:, None]
    member = (scene == torch.arange(len(sizes), device=DEV)[:, None]).float()

    def per_scene(v):
        """Sums over the rows of a scene, of [N, C] values."""
        return member @ v

    def per_group(v):
        return v.view(len(sizes), groups, -1).sum(2)

    x = x.float()
    mean = per_group(per_scene(x)) / count
    d = x.view(n, groups, -1) - mean[scene][:, :, None]
    rstd = 1 / torch.sqrt(per_group(per_scene(d.square().view(n, c))) / count + NORM_EPS)
    r = rstd[scene][:, :, None]
    xhat = (d * r).view(n, c)
    weight = s["weight"].detach()
    y, slope = _activation(xhat * weight + s["bias"].detach(), s["act"])
    if not s["train"]:
        return [y.to(dtype)]
    dz = s["dy"].float() * slope
    dbeta, dgamma = dz.sum(0), (dz * xhat).sum(0)
    gdz = dz * weight
    s1, s2 = per_group(per_scene(gdz)) / count, per_group(per_scene(gdz * xhat)) / count
    dx = r * (gdz.view(n, groups, -1) - s1[scene][:, :, None] - xhat.view(n, groups, -1) * s2[scene][:, :, None])
    return [y.to(dtype), dx.reshape(n, c).to(dtype), dgamma, dbeta]


def _plain_loss(s):
    x, w, labels, dtype = s["x"].detach().float(), s["weight"].detach().float(), s["labels"], s["x"].dtype
    counts = labels != IGNORE
    label = torch.where(counts, labels, 0)[:, None]
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    row = torch.where(counts, (top + torch.log(total) - z.gather(1, label))[:, 0], 0.0)
    if not s["train"]:
        return [row]
    rows = counts.sum().float()
    g = e / total
    g.scatter_add_(1, label, torch.full_like(total, -1.0))
    g = g * (s["gradient"] * counts / rows)[:, None]
    out = [row.sum() / rows, (g @ w).to(dtype), (g.t() @ x).to(dtype)]
    return out + ([g.sum(0).to(dtype)] if s["bias"] is not None else [])


def _plain_step(s):
    """The moments' updates are written out, each operation rounded once: codes go by the last bit."""
    place, which = s["place"], s["which"]
    steps = s["steps"].add_(1)
    b1, b2 = BETAS
    if s["bits"] == 8:
        m, v = _decode(s["m"], s["m_base"], True), _decode(s["v"], s["v_base"], False)
    else:
        m, v = s["m"], s["v"]
    g = torch.zeros_like(m)
    g[place] = s["grad"].float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    t = steps.double()
    size, root = (LR / (1 - b1 ** t)).float()[which], torch.sqrt(1 - b2 ** t).float()[which]
    p = s["flat"].float() * (1 - LR * DECAY) - size * (m[place] / (torch.sqrt(v[place]) / root + EPS))
    s["flat"].copy_(p)
    if s["bits"] == 8:
        step_of = torch.zeros_like(m, dtype=torch.int64)
        step_of[place] = steps.to(torch.int64)[which]
        for_m, for_v = _random(step_of, torch.arange(m.numel(), device=DEV))
        codes, base = _encode(m, for_m, True)
        s["m"].copy_(codes)
        s["m_base"].copy_(base)
        codes, base = _encode(v, for_v, False)
        s["v"].copy_(codes)
        s["v_base"].copy_(base)
        m, v = _decode(s["m"], s["m_base"], True), _decode(s["v"], s["v_base"], False)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
        m, v = s["m"], s["v"]
    return {"params": s["flat"], "exp_avg": m, "exp_avg_sq": v, "steps": steps}


# --------------------------------------------------------------------------- the framework's operators


def _own_norm(s):
    from warpconvnet_b200.nn.functional.group_norm import segmented_group_norm
    act = None if s["act"] == "none" else s["act"]
    if not s["train"]:
        with torch.no_grad():
            return [segmented_group_norm(s["x"], s["offsets"], s["groups"], s["weight"], s["bias"], eps=NORM_EPS, activation=act)]
    y = segmented_group_norm(s["x"], s["offsets"], s["groups"], s["weight"], s["bias"], eps=NORM_EPS, activation=act)
    return [y.detach(), *torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["dy"])]


def _own_loss(s):
    from warpconvnet_b200.nn.functional.linear_cross_entropy import linear_cross_entropy
    if not s["train"]:
        with torch.no_grad():
            return [linear_cross_entropy(s["x"], s["weight"], s["labels"], s["bias"], ignore_index=IGNORE, reduction="none")]
    loss = linear_cross_entropy(s["x"], s["weight"], s["labels"], s["bias"], ignore_index=IGNORE)
    return [loss.detach(), *torch.autograd.grad(loss, [s[k] for k in ("x", "weight", "bias") if s[k] is not None], s["gradient"])]


def _own_step(s):
    from warpconvnet_b200.optim import adamw_step, decode_moments
    eight = s["bits"] == 8
    adamw_step(s["params"], s["grads"], s["m"], s["v"], s["steps"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
               exp_avg_base=s["m_base"] if eight else None, exp_avg_sq_base=s["v_base"] if eight else None)
    m, v = decode_moments(s["m"], s["m_base"], s["v"], s["v_base"]) if eight else (s["m"], s["v"])
    return {"params": s["flat"], "exp_avg": m, "exp_avg_sq": v, "steps": s["steps"]}


def run(state):
    kind = state["kind"]
    if own:
        return {"norm": _own_norm, "loss": _own_loss, "step": _own_step}[kind](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "loss": _plain_loss, "step": _plain_step}[kind](state)


# --------------------------------------------------------------------------- 64 bits


def _exact_norm(case, seed):
    s = prepare(case, seed)
    n, c, groups = case["rows"], case["channels"], case["groups"]
    x, w, b = s["x"].detach().double(), s["weight"].detach().double(), s["bias"].detach().double()
    y, dx = torch.empty_like(x), torch.empty_like(x)
    dgamma, dbeta = torch.zeros_like(w), torch.zeros_like(b)
    at = s["offsets"].tolist()
    for lo, hi in zip(at, at[1:]):
        if hi == lo:
            continue
        xs = x[lo:hi].view(hi - lo, groups, -1)
        var, mean = torch.var_mean(xs, dim=(0, 2), keepdim=True, correction=0)
        std = torch.sqrt(var + NORM_EPS)
        xhat = ((xs - mean) / std).view(hi - lo, c)
        y[lo:hi], slope = _activation(xhat * w + b, case["act"])
        if case["train"]:
            dz = s["dy"][lo:hi].double() * slope
            dbeta += dz.sum(0)
            dgamma += (dz * xhat).sum(0)
            h = (dz * w).view_as(xs)
            xg = xhat.view_as(xs)
            dx[lo:hi] = ((h - h.mean((0, 2), keepdim=True) - xg * (h * xg).mean((0, 2), keepdim=True)) / std).view(hi - lo, c)
    return [y, dx, dgamma, dbeta] if case["train"] else [y]


def _exact_loss(case, seed):
    s = prepare(case, seed)
    n, piece = case["rows"], max(1, (1 << 28) // case["classes"])
    w = s["weight"].detach().double()
    b = s["bias"].detach().double() if s["bias"] is not None else torch.zeros(case["classes"], dtype=torch.float64, device=DEV)
    used = s["labels"] != IGNORE
    rows = int(used.sum())
    loss, dx = [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for lo in range(0, n, piece):
        x, label, use = s["x"][lo:lo + piece].detach().double(), s["labels"][lo:lo + piece], used[lo:lo + piece]
        logp = torch.log_softmax(torch.addmm(b, x, w.t()), dim=1)
        index = torch.arange(len(x), device=DEV)[use]
        part = torch.zeros(len(x), dtype=torch.float64, device=DEV)
        part[use] = -logp[index, label[use]]
        loss.append(part)
        if case["train"]:
            p = logp.exp_()
            p[index, label[use]] -= 1
            p *= use[:, None].double() * (float(s["gradient"]) / rows)
            dx.append(p @ w)
            dw += p.t() @ x
            db += p.sum(0)
    if not case["train"]:
        return [torch.cat(loss)]
    return [torch.cat(loss).sum() / rows, torch.cat(dx), dw] + ([db] if case["bias"] else [])


def _exact_step(case, seed):
    s = prepare(case, seed)
    t = 11  # (the state is at step 10)
    if case["bits"] == 8:
        m, v = _decode(s["m"], s["m_base"], True).double(), _decode(s["v"], s["v_base"], False).double()
    else:
        m, v = s["m"].double(), s["v"].double()
    g = torch.zeros_like(m)
    g[s["place"]] = s["grad"].double()
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * g * g
    m_hat, v_hat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
    p = s["flat"].double()
    p = p - LR * DECAY * p - LR * (m_hat / (torch.sqrt(v_hat) + EPS))[s["place"]]
    eight = case["bits"] == 8  # codes are rounded at random: only the parameters have a value in 64 bits
    return {"params": p, "exp_avg": None if eight else m, "exp_avg_sq": None if eight else v, "steps": None}


def exact(case, seed):
    with torch.no_grad():
        return {"norm": _exact_norm, "loss": _exact_loss, "step": _exact_step}[case["kind"]](case, seed)


# --------------------------------------------------------------------------- work


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "norm":
        n, c = float(case["rows"]), case["channels"]
        # x in, y out; in training x and its gradients again
        return {"bytes": e * n * c * (4 if case["train"] else 2) + 16.0 * c, "flops": n * c * (30 if case["train"] else 10)}
    if case["kind"] == "loss":
        n, c, v = float(case["rows"]), case["channels"], case["classes"]
        if not case["train"]:
            return {"bytes": e * (n + v) * c + 12.0 * n, "flops": 2.0 * n * c * v}
        return {"bytes": 2 * e * (n + v) * c + 8.0 * n, "flops": 6.0 * n * c * v}
    sizes = _sizes(case)
    n, length = float(sum(sizes)), float(_slots(sizes)[1])
    if case["bits"] == 32:
        return {"bytes": 3 * e * n + 16.0 * length, "flops": 15.0 * n}
    # codes and bases in and out, and the numbers that they stand for
    return {"bytes": 3 * e * n + 4.0 * length * (1 + 2.0 / BLOCK) + 8.0 * length, "flops": 40.0 * n}
