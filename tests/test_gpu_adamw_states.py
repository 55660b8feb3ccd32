"""AdamW with its states in 32 or 8 bits (csrc/adamw.hip) against the formula in 64 bits on the same inputs.

32: p, m and v are a handful of fp32 operations: m within 4 u (|m| + |g|), v within 4 u (v + g^2), p within
8 u (|p| + |update|) and the rounding of its type (u = 2^-24).
8: the codes are compared as codes. One may differ from the 64-bit one by one step only where the 64-bit value lies so near
to the border that an error of 2^-19 of a grid step (the 24 bits of a value of 8 to 16 steps, twice) decides, and a block's
exponent only where its largest value does (never here: the inputs are random, and the test counts)."""
import math

import numpy as np
import pytest
import torch
import torch.nn as nn

from sehip import linear, norm, optim

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
B = 128
HP = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)


def _mix(x):
    x = (x ^ (x >> 15)) * 0x6A09E667 & 0xFFFFFFFF
    x = (x ^ (x >> 13)) * 0xBB67AE85 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _bits(n, seed, step, tensor, start=0):
    key = _mix(_mix(_mix(seed) + step & 0xFFFFFFFF) + tensor & 0xFFFFFFFF)
    i = np.arange(start, start + n, dtype=np.uint64)
    h = (i * np.uint64(0x9E3779B1) + (i >> np.uint64(32)) * np.uint64(0x243F6A89) + np.uint64(key)) & np.uint64(0xFFFFFFFF)
    with np.errstate(over="ignore"):
        h = _np_mix(h)
    return (h & np.uint64(0xFFFF)).astype(np.float64), (h >> np.uint64(16)).astype(np.float64)


def _np_mix(x):
    m = np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x6A09E667)) & m
    x = ((x ^ (x >> np.uint64(13))) * np.uint64(0xBB67AE85)) & m
    return x ^ (x >> np.uint64(16))


def _np(t):
    return t.detach().reshape(-1).double().cpu().numpy()


def _raw(t):
    return t.reshape(-1).view(torch.uint8).cpu().numpy().astype(np.int64)


def _value(code, scale):
    """64-bit values of e4m3 codes and their blocks' exponents."""
    c, n = code & 127, len(code)
    e, f = c >> 3, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    return np.where(code > 127, -v, v) * np.repeat(2.0 ** (scale - 127.0), B)[:n]


def _pack(x, h, floor):
    """(codes, exponents, distance to the border in grid steps)"""
    n = len(x)
    a = np.abs(x)
    top = np.pad(a, (0, -n % B)).reshape(-1, B).max(1)
    f, e = np.frexp(top)
    k = np.maximum(np.where(f <= 0.875, e - 9, e - 8), -126)
    k = np.where(top > 0, k, -126)
    y = a * np.repeat(2.0 ** -k.astype(float), B)[:n]
    ex = np.maximum(np.frexp(y)[1] - 1, -6)
    t = y * 2.0 ** (3.0 - ex) + (h + 0.5) / 65536
    c = (ex + 7) * 8 + np.floor(t).astype(np.int64) - 8
    c = np.where(floor & (a > 0), np.maximum(c, 1), c)
    border = np.abs(t - np.round(t))
    return c | np.where(np.signbit(x), 128, 0), k + 127, border


def _states(ps, bits, gs):
    if bits == 32:
        return [[0.1 * g.float() for g in gs], [0.003 * g.float().square() + 1e-9 for g in gs]]
    m, mk, q, qk = [], [], [], []
    for p in ps:
        n = p.numel()
        gen = torch.Generator().manual_seed(n)
        sign = torch.randint(0, 2, (n,), generator=gen) * 128
        code = lambda lo, hi: torch.randint(lo, hi, (n,), generator=gen)  # noqa: E731
        nb = -(-n // B)
        m.append((code(0, 127) + sign).to(torch.uint8).to(p.device).view(torch.float8_e4m3fn).view(p.shape))
        q.append(code(0, 127).to(torch.uint8).to(p.device).view(torch.float8_e4m3fn).view(p.shape))
        mk.append(torch.randint(105, 110, (nb,), generator=gen).to(torch.uint8).to(p.device).view(torch.float8_e8m0fnu))
        qk.append(torch.randint(110, 114, (nb,), generator=gen).to(torch.uint8).to(p.device).view(torch.float8_e8m0fnu))
    return [m, mk, q, qk]


def _reference(p, g, m, v, step):
    b1, b2 = HP["betas"]
    m = m + (1 - b1) * (g - m)
    v = b2 * v + (1 - b2) * g * g
    up = HP["lr"] / (1 - b1 ** step) * m / (np.sqrt(v) / math.sqrt(1 - b2 ** step) + HP["eps"])
    return p * (1 - HP["lr"] * HP["weight_decay"]) - up, m, v, up


def _check_p(got, ref, old, up, dt):
    e = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 1e-45
    bound = (e if dt != torch.float32 else 0) * np.abs(ref) + 16 * U * (np.abs(old) + np.abs(up)) + tiny
    assert (np.abs(_np(got) - ref) <= bound).all(), (np.abs(_np(got) - ref) / bound).max()


SIZES = [(1,), (2, 3), (127,), (128,), (129,), (8, 16, 3), (2047,), (2048,), (2049,), (0,), (33, 65), (5000,)]


def _tensors(dev, dt, sizes, seed, off=0):
    torch.manual_seed(seed)

    def make(scale):
        out = []
        for s in sizes:   # `off`: each tensor that many elements into its own storage
            n = math.prod(s)
            t = torch.zeros(n + off, device=dev, dtype=dt)[off:].view(s)
            t.copy_(scale * torch.randn(s, device=dev) * torch.exp(torch.randn(s[:1] + (1,) * (len(s) - 1), device=dev)))
            out.append(t)
        return out
    return make(0.05), make(0.01)


@pytest.mark.parametrize("dt", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("off", (0, 1))
def test_32_bits(gpu_device, dt, off):
    ps, gs = _tensors(gpu_device, dt, SIZES * 6, 1, off)     # 72 tensors: two launches
    ms, vs = _states(ps, 32, gs)
    old = [[_np(t) for t in ts] for ts in (ps, gs, ms, vs)]
    optim.adamw32_(ps, gs, ms, vs, step=7, **HP)
    for i, p in enumerate(ps):
        p0, g, m0, v0 = (c[i] for c in old)
        rp, rm, rv, up = _reference(p0, g, m0, v0, 7)
        assert (np.abs(_np(ms[i]) - rm) <= 4 * U * (np.abs(rm) + np.abs(g)) + 1e-45).all()
        assert (np.abs(_np(vs[i]) - rv) <= 4 * U * (rv + g * g) + 1e-45).all()
        _check_p(p, rp, p0, up, dt)
        assert np.array_equal(_np(gs[i]), g)


@pytest.mark.parametrize("dt", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("off", (0, 1))
def test_8_bits(gpu_device, dt, off):
    ps, gs = _tensors(gpu_device, dt, SIZES * 6, 2, off)
    ms, mks, qs, qks = _states(ps, 8, gs)
    if off:   # codes off their alignment too
        move = lambda t: torch.cat([t.reshape(-1).view(torch.uint8)[:0].new_zeros(3), t.reshape(-1).view(torch.uint8)])[3:].view(  # noqa: E731
            torch.float8_e4m3fn).view(t.shape)
        ms, qs = [move(t) for t in ms], [move(t) for t in qs]
    old = [[_np(t) for t in ts] for ts in (ps, gs)] + [[_raw(t) for t in ts] for ts in (ms, mks, qs, qks)]
    near = total = 0
    optim.adamw8_(ps, gs, ms, mks, qs, qks, step=7, seed=12345, **HP)
    for i, p in enumerate(ps):
        p0, g, m0, mk0, q0, qk0 = (c[i] for c in old)
        rp, rm, rv, up = _reference(p0, g, _value(m0, mk0), _value(q0, qk0) ** 2, 7)
        _check_p(p, rp, p0, up, dt)
        lo, hi = _bits(p.numel(), 12345, 7, i)
        for got, gk, x, h, floor in ((ms[i], mks[i], rm, lo, False), (qs[i], qks[i], np.sqrt(rv), hi, True)):
            c, k, border = _pack(x, h, np.full(len(x), floor))
            assert np.array_equal(_raw(gk), k)
            diff = np.abs((_raw(got) & 127) - (c & 127))
            assert ((diff == 0) | ((diff == 1) & (border < 2.0 ** -19))).all(), (i, diff.max())
            nz = (c & 127) > 0
            assert np.array_equal((_raw(got) > 127)[nz], (c > 127)[nz])
            near += int((diff > 0).sum())
            total += len(c)
    assert near <= max(3, total * 2.0 ** -17), (near, total)


def test_stochastic_rounding_is_right_on_average(gpu_device):
    """One fp32 value in all elements of a long tensor: the mean of the stored values is the value itself. n = 2^20, a step
    d: the mean's deviation is at most d / 2 / 1024; six of them, and the hash's resolution of d / 65536."""
    n = 1 << 20
    for x in (0.3, 0.77, 1.003, 13.1):
        p, g = [torch.zeros(n, device=gpu_device)], [torch.full((n,), x, device=gpu_device)]
        ms, mks, qs, qks = (([torch.zeros(k, device=gpu_device, dtype=torch.uint8).view(t)]) for k, t in (
            (n, torch.float8_e4m3fn), (n // B, torch.float8_e8m0fnu), (n, torch.float8_e4m3fn), (n // B, torch.float8_e8m0fnu)))
        optim.adamw8_(p, g, ms, mks, qs, qks, step=1, seed=5, **HP)
        for got, k, want in ((ms, mks, 0.1 * x), (qs, qks, math.sqrt(0.001) * x)):
            v = _value(_raw(got[0]), _raw(k[0]))
            lo, hi = v.min(), v.max()
            assert lo <= want <= hi and hi - lo <= want / 8 * 1.001
            assert abs(v.mean() - want) <= (hi - lo) * (6 / 2048 + 1 / 65536) + 1e-6 * want


def test_a_small_second_moment_keeps_moving(gpu_device):
    """What rounding to the nearest would break: v falls by 0.1 % a step with zero gradients, and after 1000 steps the stored
    values are near exp(-1) of the start (their mean within 3 % of 0.999^1000: the walk of 4096 elements averages out)."""
    n = 4096
    p, g = [torch.zeros(n, device=gpu_device)], [torch.zeros(n, device=gpu_device)]
    ms, qs = ([torch.zeros(n, device=gpu_device, dtype=torch.uint8).view(torch.float8_e4m3fn)] for _ in range(2))
    mks, qks = ([torch.full((n // B,), 127, device=gpu_device, dtype=torch.uint8).view(torch.float8_e8m0fnu)] for _ in range(2))
    qs[0].view(torch.uint8).fill_(0x38)   # 1
    for step in range(1, 1001):
        optim.adamw8_(p, g, ms, mks, qs, qks, step=step, seed=1, **HP)
    q = _value(_raw(qs[0]), _raw(qks[0]))
    # the square of a walk's mean: E q = (0.999^(1/2))^1000, its square exp(-1); a stochastic step is unbiased in q
    assert abs(q.mean() / 0.999 ** 500 - 1) < 0.03


def test_zero_states_and_zero_gradients(gpu_device):
    for bits in (8, 32):
        p = nn.Parameter(torch.ones(300, device=gpu_device))
        p.grad = torch.zeros_like(p)
        o = optim.AdamW([p], state_bits=bits, **HP)
        for _ in range(3):
            o.step()
        assert torch.allclose(p, torch.full_like(p, (1 - 1e-5) ** 3), rtol=1e-6)
        st = o.state[p]
        assert float(st["step"]) == 3 and not st["exp_avg"].view(torch.uint8).any()


def test_extreme_gradients(gpu_device):
    """Gradients from 1e-30 to 1e15 in one block, then a NaN and an infinity: they reach their own elements alone."""
    g0 = torch.logspace(-30, 15, 256, device=gpu_device)
    outs = []
    for bad in (False, True):
        p = nn.Parameter(torch.full((256,), 0.5, device=gpu_device))
        o = optim.AdamW([p], state_bits=8, seed=2, **HP)
        for _ in range(3):
            p.grad = g0.clone()
            if bad:
                p.grad[5], p.grad[200] = float("nan"), float("inf")
            o.step()
        outs.append((p.detach().clone(), o.state[p]))
    clean, dirty = outs
    assert clean[0].isfinite().all()
    # |m| / sqrt(v) cannot be over 10 (three steps of one gradient), so no element moves by more than 3 * 12 lr
    assert (clean[0] - 0.5).abs().max() < 3 * 12e-3
    rest = torch.ones(256, dtype=torch.bool, device=gpu_device)
    rest[[5, 200]] = False
    assert torch.equal(clean[0][rest], dirty[0][rest]) and dirty[0][[5, 200]].isnan().all()
    assert torch.equal(clean[1]["exp_avg"].view(torch.uint8)[rest], dirty[1]["exp_avg"].view(torch.uint8)[rest])


def test_same_call_same_bits_and_seeds_differ(gpu_device):
    def go(seed):
        ps, gs = _tensors(gpu_device, torch.float32, [(3000,), (50, 20)], 3)
        o = optim.AdamW([nn.Parameter(p) for p in ps], state_bits=8, seed=seed, **HP)
        for k in range(4):
            for p, g in zip(o.param_groups[0]["params"], gs):
                p.grad = g * (k + 1)
            o.step()
        return [t.view(torch.uint8).clone() for p in o.param_groups[0]["params"] for t in list(o.state[p].values())[1:]] + \
            [p.detach().clone() for p in o.param_groups[0]["params"]]
    a, b, c = go(1), go(1), go(2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(a[0], c[0])


def test_groups_missing_gradients_and_resume(gpu_device):
    """Two groups, a parameter that joins late, types side by side; and a run that is saved and loaded goes on with the same
    bits."""
    for bits in (8, 32):
        torch.manual_seed(4)
        mk = lambda: [nn.Parameter(torch.randn(700, device=gpu_device)),  # noqa: E731
                      nn.Parameter(torch.randn(40, 9, device=gpu_device).bfloat16()), nn.Parameter(torch.randn(5, device=gpu_device))]
        ps = mk()
        qs = [nn.Parameter(p.detach().clone()) for p in ps]
        make = lambda t: optim.AdamW([{"params": t[:2]}, {"params": t[2:], "lr": 1e-2}], state_bits=bits, **HP)  # noqa: E731
        a = make(ps)
        grads = [[torch.randn_like(p) for p in ps] for _ in range(6)]

        def go(o, params, steps):
            for k in steps:
                for i, p in enumerate(params):
                    p.grad = None if i == 1 and k < 2 else grads[k][i].clone()
                o.step()
        go(a, ps, range(4))
        assert float(a.state[ps[0]]["step"]) == 4 and float(a.state[ps[1]]["step"]) == 2
        sd = a.state_dict()
        b = make(qs)
        with torch.no_grad():
            for p, q in zip(ps, qs):
                q.copy_(p)
        b.load_state_dict(sd)
        go(a, ps, (4, 5))
        go(b, qs, (4, 5))
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
        for p, q in zip(ps, qs):
            for k, t in a.state[p].items():
                assert torch.equal(t.reshape(-1).view(torch.uint8), b.state[q][k].reshape(-1).view(torch.uint8))


def test_32_bit_states_follow_torch(gpu_device):
    """fp32 parameters: the same moments and, over steps, the same parameters as torch.optim.AdamW within its bars elsewhere
    in this suite (1e-6 of the largest)."""
    ps, gs = _tensors(gpu_device, torch.float32, [(3000,), (50, 20), (7,)], 5)
    a, b = ([nn.Parameter(p.clone()) for p in ps] for _ in range(2))
    oa, ob = torch.optim.AdamW(a, **HP), optim.AdamW(b, state_bits=32, **HP)
    for k in range(4):
        for p, q, g in zip(a, b, gs):
            p.grad, q.grad = (g * (k + 1)).clone(), (g * (k + 1)).clone()
        oa.step()
        ob.step()
    for p, q in zip(a, b):
        assert (p - q).abs().max() <= 1e-6 * max(1.0, p.abs().max().item())


def test_offsets_past_32_bits(gpu_device):
    """One tensor of over 2^31 elements: its far end is updated by its own values and its own random bits."""
    n = (1 << 31) + 4096 + 77
    p = [torch.zeros(n, device=gpu_device, dtype=torch.bfloat16)]
    g = [torch.zeros(n, device=gpu_device, dtype=torch.bfloat16)]
    g[0][-5000:].normal_()
    nb = -(-n // B)
    zero = lambda k, t: [torch.zeros(k, device=gpu_device, dtype=torch.uint8).view(t)]  # noqa: E731
    ms, qs = zero(n, torch.float8_e4m3fn), zero(n, torch.float8_e4m3fn)
    mks, qks = zero(nb, torch.float8_e8m0fnu), zero(nb, torch.float8_e8m0fnu)
    optim.adamw8_(p, g, ms, mks, qs, qks, step=1, seed=9, **HP)
    last = n // B * B - 2 * B          # a block's start
    gn = _np(g[0][last:])
    _, rm, rv, _ = _reference(np.zeros(len(gn)), gn, 0 * gn, 0 * gn, 1)
    lo, _ = _bits(len(gn), 9, 1, 0, start=last)
    c, k, border = _pack(rm, lo, np.full(len(gn), False))
    assert np.array_equal(_raw(mks[0][last // B:]), k)
    diff = np.abs((_raw(ms[0][last:]) & 127) - (c & 127))
    assert ((diff == 0) | ((diff == 1) & (border < 2.0 ** -19))).all()
    assert not p[0][:1 << 20].any() and p[0][-5000:].abs().min() > 0


def test_refusals_on_the_gpu(gpu_device):
    f = lambda n=5, dt=torch.float32: torch.zeros(n, device=gpu_device, dtype=dt)  # noqa: E731
    kw = dict(step=1)
    optim.adamw32_([f()], [f()], [f()], [f()], **kw)
    for bad in ([f(6)], [f().cpu()], [f(dt=torch.bfloat16)], [f(10)[::2]]):
        for at in range(1, 4):
            args = [[f()], [f()], [f()], [f()]]
            args[at] = bad
            with pytest.raises(RuntimeError, match="sehip adamw"):
                optim.adamw32_(*args, **kw)
    with pytest.raises(RuntimeError, match="sehip adamw"):
        optim.adamw8_([f()], [f()], [f()], [f(1)], [f()], [f(1)], **kw)
    p, m = f(), f()
    with pytest.raises(RuntimeError, match="twice"):   # two chunks of one launch would update the same memory
        optim.adamw32_([p, p], [f(), f()], [f(), f()], [f(), f()], **kw)
    with pytest.raises(RuntimeError, match="twice"):
        optim.adamw32_([f(), f()], [f(), f()], [m, m], [f(), f()], **kw)
    optim.adamw32_([f(0), f(0), f()], [f(0), f(0), p], [f(0), f(0), f()], [f(0), f(0), f()], **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    t = [[f()], [f()], [f()], [f()]]
    with pytest.raises(RuntimeError, match="captured graph"):
        with torch.cuda.graph(g):
            t[0][0].add_(1)
            optim.adamw32_(*t, **kw)


@pytest.mark.parametrize("bits", (8, 32))
def test_train_step_of_a_model(gpu_device, bits):
    """FRCRN's own training step (sehip.train.train_step) on the 8- and 32-bit states, over its 279 parameter tensors: 32 bits
    gives the default optimizer's parameters (the same fp32 formula: 1e-6 of the largest, as elsewhere in this suite), 8 bits
    the same first step to that bar (its moments start at zero, and the step is taken before they are rounded)."""
    import paramfill
    from sehip import models as M
    from sehip.train import make_optimizer, train_step
    noisy, clean = paramfill.structured_pair(2, 16000, seed=11)
    x, c = torch.from_numpy(noisy).to(gpu_device), torch.from_numpy(clean).to(gpu_device)
    ms = [paramfill.fill_(M.FRCRN(), seed=12).to(gpu_device).train() for _ in range(2)]
    opts = [make_optimizer(ms[0]), make_optimizer(ms[1], state_bits=bits)]
    for m, o in zip(ms, opts):
        assert torch.isfinite(train_step(m, o, x, c))
    for p, q in zip(ms[0].parameters(), ms[1].parameters()):
        assert (p - q).abs().max().item() <= 1e-6 * max(p.abs().max().item(), 1e-2)
    assert torch.isfinite(train_step(ms[1], opts[1], x, c))
    held = sum(t.numel() * t.element_size() for st in opts[1].state.values() for t in st.values() if t.is_cuda)
    total = sum(p.numel() for p in ms[1].parameters())
    assert held == 8 * total if bits == 32 else held < 2.1 * total


@pytest.mark.parametrize("dt,bits", [(torch.float32, 8), (torch.bfloat16, 32), (torch.bfloat16, 8)])
def test_feed_forward_block_in_training(gpu_device, dt, bits):
    """The operators together, as a pre-norm residual block uses them: norm, product + GELU, product + residual, their gradients
    into every parameter against automatic differentiation in 64 bits, and the optimizer's step on them."""
    torch.manual_seed(6)
    C, H, dev = 96, 200, gpu_device
    ln, up, down = nn.LayerNorm(C, device=dev, dtype=dt), nn.Linear(C, H, device=dev, dtype=dt), nn.Linear(H, C, device=dev, dtype=dt)
    params = [p for m in (ln, up, down) for p in m.parameters()]
    opt = optim.AdamW(params, state_bits=bits, **HP)
    x = torch.randn(4, 77, C, device=dev).to(dt)
    target = torch.randn(4, 77, C, device=dev).to(dt)
    for step in range(3):
        opt.zero_grad(set_to_none=True)
        y = linear.linear_act(linear.linear_act(norm.layer_norm(ln, x), up, nn.GELU()), down, None, x)
        dy = (y.detach().float() - target.float()).mul(0.05).to(dt)
        y.backward(dy)
        d = [p.detach().double().requires_grad_(True) for p in params]
        h = torch.nn.functional.layer_norm(x.double(), (C,), d[0], d[1], ln.eps)
        ref = torch.nn.functional.gelu(h @ d[2].t() + d[3]) @ d[4].t() + d[5] + x.double()
        ref.backward(dy.double())
        # norms: each stored intermediate (h, z, act, y and their gradients: at most eight on a path) adds half a step of its type
        bar = 8 * torch.finfo(dt).eps / 2 if dt != torch.float32 else 1e-5
        assert (y.double() - ref).norm() <= bar * ref.norm()
        for p, q in zip(params, d):
            assert (p.grad.double() - q.grad).norm() <= bar * q.grad.norm()
        before = [p.detach().clone() for p in params]
        opt.step()
        # a step moves a weight by about lr = 0.001; bf16's values next to the norm's weights of 1 are 2^-8 below and 2^-7
        # above, and 0.001 is less than half of either: those weights round back to 1
        stuck = [ln.weight] if dt == torch.bfloat16 else []
        assert all(not torch.equal(b, p) for b, p in zip(before, params) if not any(p is t for t in stuck))
        assert all(p.isfinite().all() for p in params)


def test_codes_of_the_exact_states(gpu_device):
    """Of four million random elements every code is that of the 64-bit state, also where 24 bits alone would decide
    otherwise (about one in a million). 32-bit arithmetic puts q within 2.5 and m, where it has not cancelled below half of
    what it was, within 7.5 steps of 2^-20 of a grid step; the kernel takes all within 8 of a border again, with twice
    the bits. The 64-bit reference itself is good to 16 * 2^-50, and a block whose largest value decides its exponent
    is left out."""
    n = 1 << 22
    ps, gs = _tensors(gpu_device, torch.float32, [(n,)], 5)
    ms, mks, qs, qks = _states(ps, 8, gs)
    g = _np(gs[0])
    m0, q0 = _value(_raw(ms[0]), _raw(mks[0])), _value(_raw(qs[0]), _raw(qks[0]))
    optim.adamw8_(ps, gs, ms, mks, qs, qks, step=9, seed=4, **HP)
    b1, b2 = HP["betas"]
    m, q = m0 + (1 - b1) * (g - m0), np.sqrt(b2 * q0 * q0 + (1 - b2) * g * g)
    lo, hi = _bits(n, 4, 9, 0)
    for x, h, floor, code, scale, sure in ((m, lo, False, ms, mks, np.abs(m) >= np.abs(m0) / 2),
                                           (q, hi, True, qs, qks, q == q)):
        want, k, border = _pack(x, h, floor)
        got, kg = _raw(code[0]), _raw(scale[0])
        at = sure & (border > 2.0 ** -44) & np.repeat(k == kg, B)
        assert (k != kg).sum() <= 1
        assert at.mean() > 0.5
        assert np.array_equal(got[at], want[at]), (got[at] != want[at]).sum()


@pytest.mark.parametrize("bits", (8, 32))
def test_one_tensor_in_two_lists(gpu_device, bits):
    """Refused before anything is written: two moments, a parameter and its gradient or moment in the same memory. Tensors of no
    elements may share an address, and two parameters a gradient."""
    def lists():
        f = lambda n, t: torch.ones(n, device=gpu_device, dtype=torch.uint8 if bits == 8 else torch.float32).view(  # noqa: E731
            t if bits == 8 else torch.float32)
        ps, gs = ([torch.ones(n, device=gpu_device) for n in (128, 0, 128)] for _ in range(2))
        cols = [[f(n, t) for n in sizes] for t, sizes in (
            ((torch.float8_e4m3fn, (128, 0, 128)), (torch.float8_e8m0fnu, (1, 0, 1))) * 2 if bits == 8
            else ((None, (128, 0, 128)),) * 2)]
        return [ps, gs, *cols]

    step = optim.adamw8_ if bits == 8 else optim.adamw32_
    step(*lists(), step=1)
    a = lists()
    a[1][2] = a[1][0]
    step(*a, step=1)
    root = 4 if bits == 8 else 3
    for i, j in ((2, root), (0, 1), *(((3, 5),) if bits == 8 else ((0, 2), (1, 3)))):
        for k in (0, 2):
            a = lists()
            a[j][k] = a[i][0]
            with pytest.raises(RuntimeError, match="two of the lists"):
                step(*a, step=1)
            assert all(bool((t == 1).all()) for t in a[0])
    a = lists()
    flat = torch.ones(128, device=gpu_device)     # an empty slice begins where its neighbour does
    a[0][1], a[0][2] = flat[:0], flat
    step(*a, step=1)
