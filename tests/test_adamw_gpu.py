"""AdamW of many tensors in one launch against the formula in 64 bits, and its 8-bit moments against their definition."""
import copy
import io
import pickle

import pytest
import torch

from warpconvnet_b200.optim import AdamW, adamw_step, decode_moments, moment_slots

from conftest import rel_l2

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# one rounding of the stored parameter; a few fp32 roundings of an update that is small beside it
TOL = {torch.float32: 2e-7, torch.float16: 6e-4, torch.bfloat16: 4e-3}
SIZES = [1, 7, 255, 256, 257, 2048, 2049, 5000]


def tensors(sizes, dtype, seed, scale=1.0, shift=0):
    """Views into one buffer, from element ``shift`` on: at any address."""
    g = torch.Generator().manual_seed(seed)
    flat = (torch.randn(sum(sizes) + shift, generator=g) * scale).to(dtype).to(DEV)
    return list(flat[shift:].split(sizes))


def formula(p, g, m, v, t, lr, b1, b2, eps, wd):
    p, g = p.double(), g.double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p, m, v


def close(a, b, tol):
    return rel_l2(a.detach().double().cpu().numpy(), b.detach().double().cpu().numpy()) <= tol


@pytest.mark.parametrize("dtype,grad_dtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                              (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("betas,wd", [((0.9, 0.999), 0.01), ((0.0, 0.5), 0.0)])
def test_steps_follow_the_formula(dtype, grad_dtype, shift, betas, wd):
    params = tensors(SIZES, dtype, 0, 0.1, shift)
    slots, length = moment_slots(SIZES)
    m, v = torch.zeros(length, device=DEV), torch.zeros(length, device=DEV)
    steps = torch.zeros(len(SIZES), dtype=torch.int32, device=DEV)
    ref = [(torch.zeros(n, dtype=torch.float64, device=DEV), torch.zeros(n, dtype=torch.float64, device=DEV)) for n in SIZES]
    for t in range(1, 4):
        grads = tensors(SIZES, grad_dtype, t, 1e-2, shift)
        before = [p.clone() for p in params]
        version = params[0]._version
        adamw_step(params, grads, m, v, steps, lr=1e-2, betas=betas, eps=1e-8, weight_decay=wd)
        assert params[0]._version > version
        for i, n in enumerate(SIZES):
            want, rm, rv = formula(before[i], grads[i], *ref[i], t, 1e-2, *betas, 1e-8, wd)
            ref[i] = rm, rv
            assert close(params[i], want, TOL[dtype])
            assert close(m[slots[i]:slots[i] + n], rm, 1e-6) and close(v[slots[i]:slots[i] + n], rv, 1e-6)
        assert steps.tolist() == [t] * len(SIZES)


# --------------------------------------------------------------------------- codes


def mix(h):
    h ^= h >> 16
    h = (h * 0x85EBCA6B) & 0xFFFFFFFF
    h ^= h >> 13
    h = (h * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def value(k, base):
    return torch.tensor((k + base) << 20, dtype=torch.int32).view(torch.float32).item() if k else 0.0


def encode(x, place, step, signed):
    """Codes and base of one block of 256 fp32 numbers by the definition, one number at a time."""
    top = 127 if signed else 255
    bits = x.abs().view(torch.int32).tolist()
    base = max(0, (max(bits) >> 20) + 1 - top)
    codes = []
    for i, b in enumerate(bits):
        h = mix((((place + i) * 0x9E3779B9) & 0xFFFFFFFF) ^ mix(step))
        r = h >> 12 if signed else ((h * 0x9E3779B1) & 0xFFFFFFFF) >> 12
        q = (b + r) >> 20
        k = q - base
        if signed and q <= base and base > 0:
            first = torch.tensor((base + 1) << 20, dtype=torch.int32).view(torch.float32)
            k = int(x[i].abs() > first * (torch.tensor(float(r)) * 2.0 ** -20))
        elif not signed:
            k = 0 if b == 0 else max(k, 1)
        codes.append(k | (128 if signed and x[i] < 0 else 0))
    return codes, base


@pytest.mark.parametrize("spread", [0.5, 6.0])   # octaves (standard deviation) that the gradients of a block span
def test_codes_follow_their_definition(spread):
    sizes = [300, 256, 1]
    slots, length = moment_slots(sizes)
    g = torch.Generator().manual_seed(1)
    grads = [(torch.randn(n, generator=g) * torch.exp2(torch.randn(n, generator=g) * spread)) for n in sizes]
    grads[0][5] = 0.0
    params = [torch.zeros(n, device=DEV) for n in sizes]
    m, v = (torch.zeros(length, dtype=torch.uint8, device=DEV) for _ in range(2))
    mb, vb = (torch.zeros(length // 256, dtype=torch.int16, device=DEV) for _ in range(2))
    steps = torch.zeros(3, dtype=torch.int32, device=DEV)
    old_m, old_v = torch.zeros(length), torch.zeros(length)
    for t in range(1, 3):
        adamw_step(params, [x.to(DEV) for x in grads], m, v, steps, lr=1e-3, exp_avg_base=mb, exp_avg_sq_base=vb)
        full = torch.zeros(length)
        for s, x in zip(slots, grads):
            full[s:s + len(x)] = x
        b1, b2 = torch.tensor(0.9), torch.tensor(0.999)
        new_m = old_m * b1 + full * torch.tensor(1 - 0.9)
        new_v = old_v * b2 + full * full * torch.tensor(1 - 0.999)
        got_m, got_v = decode_moments(m, mb, v, vb)
        for b in range(length // 256):
            at = slice(b * 256, b * 256 + 256)
            for x, codes, bases, values, signed in ((new_m, m, mb, got_m, True), (new_v, v, vb, got_v, False)):
                want, base = encode(x[at], b * 256, t, signed)
                assert codes[at].tolist() == want and int(bases[b]) == base
                numbers = [(-1 if k > 127 and signed else 1) * value(k & (127 if signed else 255), base) for k in want]
                assert values[at].tolist() == numbers
        assert torch.equal(got_v.cpu() > 0, new_v > 0)   # a second moment that is not zero stays so
        old_m, old_v = got_m.cpu(), got_v.cpu()


def test_codes_keep_the_mean():
    """Of 2^20 equal numbers, most rounded down and some up: the mean within six of its standard deviations."""
    n = 1 << 20
    for x in (1.06, 1.0, 1.1249, -0.37):
        m, v = (torch.zeros(n, dtype=torch.uint8, device=DEV) for _ in range(2))
        mb, vb = (torch.zeros(n // 256, dtype=torch.int16, device=DEV) for _ in range(2))
        adamw_step([torch.zeros(n, device=DEV)], [torch.full((n,), x, device=DEV)], m, v, torch.zeros(1, dtype=torch.int32, device=DEV),
                   lr=0.0, betas=(0.0, 0.0), exp_avg_base=mb, exp_avg_sq_base=vb)
        got_m, got_v = decode_moments(m, mb, v, vb)
        # neighbours are at most 1/8 of the number apart: a standard deviation of at most 1/16 each
        assert abs(float(got_m.double().mean()) - x) <= 6 / 16 / 1024 * abs(x)
        assert abs(float(got_v.double().mean()) - x * x) <= 6 / 16 / 1024 * x * x


def test_training_with_codes_goes_where_training_in_32_bits_goes():
    g = torch.Generator().manual_seed(0)
    a, target = torch.randn(512, 64, generator=g).to(DEV), torch.randn(64, 8, generator=g).to(DEV)
    ends = []
    for bits in (32, 8):
        w = torch.zeros(64, 8, device=DEV, requires_grad=True)
        opt = AdamW([w], lr=2e-2, weight_decay=0.0, state_bits=bits)
        for i in range(400):
            rows = a[(i % 4) * 128:(i % 4 + 1) * 128]
            opt.zero_grad()
            (rows @ w - rows @ target).square().mean().backward()
            opt.step()
        ends.append(float((w.detach() - target).norm() / target.norm()))
    assert ends[0] < 0.05 and ends[1] < 0.05


# --------------------------------------------------------------------------- what a step may meet


def state(n, bits):
    length = moment_slots([n])[1]
    dtype = torch.float32 if bits == 32 else torch.uint8
    base = {} if bits == 32 else {k: torch.zeros(length // 256, dtype=torch.int16, device=DEV) for k in ("exp_avg_base", "exp_avg_sq_base")}
    return torch.zeros(length, dtype=dtype, device=DEV), torch.zeros(length, dtype=dtype, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), base


@pytest.mark.parametrize("bits", [32, 8])
def test_scaled_gradients_and_cancelled_steps(bits):
    p0, g = torch.randn(1000, device=DEV), torch.randn(1000, device=DEV)
    results = []
    for scale in (None, 256.0):
        p = p0.clone()
        m, v, steps, base = state(1000, bits)
        kw = {} if scale is None else {"grad_scale": torch.tensor([scale], device=DEV), "found_inf": torch.zeros(1, device=DEV)}
        adamw_step([p], [g * (scale or 1.0)], m, v, steps, lr=1e-2, **base, **kw)
        results.append((p, m, v))
        kept = [t.clone() for t in (p, m, v, steps, *base.values())]
        adamw_step([p], [g * float("nan")], m, v, steps, lr=1e-2, found_inf=torch.ones(1, device=DEV), **base)
        assert all(torch.equal(a, b) for a, b in zip(kept, (p, m, v, steps, *base.values())))
    assert all(torch.equal(a, b) for a, b in zip(*results))   # (a power of two)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_go_on_counting(bits):
    p0, g = torch.randn(3000, device=DEV), torch.randn(3000, device=DEV)
    runs = []
    for captured in (False, True):
        p, (m, v, steps, base) = p0.clone(), state(3000, bits)
        lr = torch.tensor(1e-2, device=DEV)
        step = lambda: adamw_step([p], [g], m, v, steps, lr=lr, **base)   # noqa: E731
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            step = graph.replay
        for i in range(3):
            lr.fill_(1e-2 / (i + 1))
            step()
        assert int(steps) == 3
        runs.append((p, m, v))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_more_tensors_than_a_launch_takes_and_empty_ones():
    sizes = [3, 0, 700] * 500
    params, grads = tensors(sizes, torch.float32, 0), tensors(sizes, torch.float32, 1)
    before = torch.cat(params)
    length = moment_slots(sizes)[1]
    m, v, steps = torch.zeros(length, device=DEV), torch.zeros(length, device=DEV), torch.zeros(len(sizes), dtype=torch.int32, device=DEV)
    adamw_step(params, grads, m, v, steps, lr=1e-2)
    zero = torch.zeros(before.numel(), dtype=torch.float64, device=DEV)
    want, _, _ = formula(before, torch.cat(grads), zero, zero, 1, 1e-2, 0.9, 0.999, 1e-8, 0.01)
    assert close(torch.cat(params), want, TOL[torch.float32])
    assert steps.tolist() == [1, 0, 1] * 500
    adamw_step([], [], m, v, steps, lr=1e-2)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_that_is_no_number_stays_in_its_place(bits):
    n = 600
    for bad in (float("nan"), float("inf")):
        p, (m, v, steps, base) = torch.ones(n, device=DEV), state(n, bits)
        g = torch.full((n,), 1e-3, device=DEV)
        g[100] = bad
        adamw_step([p], [g], m, v, steps, lr=1e-2, **base)
        assert torch.isnan(p[100]) and torch.isfinite(torch.cat([p[:100], p[101:]])).all()
        got_m, got_v = decode_moments(m, base["exp_avg_base"], v, base["exp_avg_sq_base"]) if bits == 8 else (m, v)
        assert not torch.isfinite(got_m[100]) and not torch.isfinite(got_v[100])
        assert torch.isfinite(got_m[256:]).all() and torch.isfinite(got_v[256:]).all()


# --------------------------------------------------------------------------- the optimizer


def model():
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Linear(65, 7)).to(DEV)


def train(net, opt, steps, seed=0, skip=None):
    g = torch.Generator().manual_seed(seed)
    for i in range(steps):
        opt.zero_grad()
        net(torch.randn(16, 33, generator=g).to(DEV)).square().mean().backward()
        if skip is not None and i % 2:
            net[skip].weight.grad = None
        opt.step()


def same(a, b, tol=0.0):
    return all(close(p, q, tol) for p, q in zip(a.parameters(), b.parameters()))


def test_the_optimizer_is_adamw():
    """Groups with rates of their own and a parameter that is now and then without a gradient, as torch.optim.AdamW."""
    a, b = model(), model()
    groups = lambda n: [{"params": n[0].parameters(), "lr": 3e-3}, {"params": n[1].parameters(), "weight_decay": 0.1}]   # noqa: E731
    mine, ref = AdamW(groups(a), lr=1e-2), torch.optim.AdamW(groups(b), lr=1e-2)
    train(a, mine, 6, skip=1)
    train(b, ref, 6, skip=1)
    assert same(a, b, 1e-5)   # (six steps: gradients differ by the parameters' last bits, an update is at most lr)
    assert int(mine.state[a[1].weight]["step"]) == 3 and int(mine.state[a[0].weight]["step"]) == 6


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["state_dict", "file", "pickle", "deepcopy"])
def test_state_travels(bits, how):
    a = model()
    opt = AdamW(a.parameters(), lr=1e-2, state_bits=bits)
    train(a, opt, 3)
    if how in ("state_dict", "file"):
        b = copy.deepcopy(a)
        other = AdamW(b.parameters(), lr=5.0, state_bits=bits)
        saved = opt.state_dict()
        if how == "file":
            buffer = io.BytesIO()
            torch.save(saved, buffer)
            buffer.seek(0)
            saved = torch.load(buffer, map_location="cpu", weights_only=True)
        other.load_state_dict(saved)
    else:
        b, other = pickle.loads(pickle.dumps((a, opt))) if how == "pickle" else copy.deepcopy((a, opt))
    assert other.param_groups[0]["lr"] == 1e-2
    train(a, opt, 2, seed=1)
    train(b, other, 2, seed=1)
    assert same(a, b) and int(other.state[b[0].weight]["step"]) == 5


def test_state_of_torchs_adamw_is_taken():
    a = model()
    opt = torch.optim.AdamW(a.parameters(), lr=1e-2)
    train(a, opt, 3)
    b = copy.deepcopy(a)
    mine = AdamW(b.parameters())
    mine.load_state_dict(opt.state_dict())
    train(a, opt, 2, seed=1)
    train(b, mine, 2, seed=1)
    assert same(a, b, 1e-5)
    with pytest.raises(ValueError):
        AdamW(b.parameters(), state_bits=8).load_state_dict(opt.state_dict())


def test_gradient_scaler_hands_its_scale_over():
    a, b = model(), model()
    mine, ref = AdamW(a.parameters(), lr=1e-2), AdamW(b.parameters(), lr=1e-2)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0)
    x = torch.randn(16, 33, device=DEV)
    for bad in (False, True, False):
        mine.zero_grad()
        scaler.scale(a(x).square().mean()).backward()
        if bad:
            a[0].bias.grad[3] = float("inf")
        scaler.step(mine)
        scaler.update()
        if not bad:
            ref.zero_grad()
            b(x).square().mean().backward()
            ref.step()
    assert same(a, b, 1e-6) and int(mine.state[a[0].weight]["step"]) == 2


def test_refusals():
    p, g = torch.zeros(512, device=DEV), torch.zeros(512, device=DEV)
    m, v, steps, _ = state(512, 32)
    cases = [([p], [], m, v, steps, {}), ([p], [g[:5]], m, v, steps, {}), ([p], [g], m[:256], v[:256], steps, {}), ([p], [g], m, v, steps[:0], {}),
             ([p], [g], m, v, steps.long(), {}), ([p.view(2, 256).t()], [g.view(2, 256).t()], m, v, steps, {}), ([p.cpu()], [g.cpu()], m, v, steps, {}),
             ([p], [g.cpu()], m, v, steps, {}), ([p], [g], m.double(), v.double(), steps, {}), ([p], [g], m[1:257], v[1:257], steps, {}),
             ([p, p.half()], [g, g], m, v, steps, {}), ([p], [g], m, v, steps, {"slots": [128]}), ([p], [g], m, v, steps, {"slots": [256]}),
             ([p], [g], m, v, steps, {"step_index": [1]}), ([p], [g], m, v, steps, {"exp_avg_base": steps.short()}),
             ([p], [g], m, v, steps, {"grad_scale": torch.ones(1)}), ([p], [g], m, v, steps, {"found_inf": steps})]
    for params, grads, a, b, s, kw in cases:
        with pytest.raises(ValueError):
            adamw_step(params, grads, a, b, s, lr=1e-3, **kw)
    for params, grads in (([p.double()], [g.double()]), ([p], [g.double()]), ([p], [g.to_sparse()])):
        with pytest.raises(TypeError):
            adamw_step(params, grads, m, v, steps, lr=1e-3)
    with pytest.raises(RuntimeError):
        adamw_step([p], [g], m, v, steps, lr=1e-3, betas=(1.0, 0.9))
    assert int(steps) == 0 and not p.any()
