"""The 8-bit states of AdamW (csrc/adamw.hip) as codes of fp32 states: m + (1 - b1) (g - m), b2 v + (1 - b2) g g and its
root, each operation rounded once to fp32 in that order, then one exact stochastic rounding. The reference takes the same
operations in numpy's fp32 and rounds the result in 64 bits, which holds every number that occurs in it: the codes and the
powers of two have to be equal, at any border, after any number of steps."""
import numpy as np
import pytest
import torch

from sehip import optim
from test_gpu_adamw_states import B, HP, U, _bits, _np, _pack, _raw, _states, _value

pytestmark = pytest.mark.gpu
F = np.float32


def _step32(g, m, v):
    b1, b2 = HP["betas"]
    g, m, v = (t.astype(F) for t in (g, m, v))
    m = m + F(1 - b1) * (g - m)
    v = F(b2) * v + F(1 - b2) * g * g
    assert m.dtype == v.dtype == F
    return m, v


def _codes(x, h, floor):
    """_pack of fp32 values; zero has a code of its own (it is in no binade)."""
    c, k, _ = _pack(x.astype(np.float64), h, np.full(len(x), floor))
    return np.where(x == 0, np.signbit(x) * 128, c), k


def _same(ps, gs, ms, mks, qs, qks, seed, step):
    """One step of the kernel on these tensors, its codes against the reference's."""
    old = [[f(t) for t in ts] for f, ts in ((_np, ps), (_np, gs), (_raw, ms), (_raw, mks), (_raw, qs), (_raw, qks))]
    optim.adamw8_(ps, gs, ms, mks, qs, qks, step=step, seed=seed, **HP)
    b1, b2 = HP["betas"]
    for i in range(len(ps)):
        p, g, m, mk, q, qk = (c[i] for c in old)
        m, v = _step32(g, _value(m, mk), _value(q, qk) ** 2)   # a code's square has 8 bits
        r = np.sqrt(v)
        lo, hi = _bits(len(g), seed, step, i)
        for what, got, gk, x, h, floor in (("m", ms[i], mks[i], m, lo, False), ("q", qs[i], qks[i], r, hi, True)):
            c, k = _codes(x, h, floor)
            assert np.array_equal(_raw(gk), k), (what, i, step)
            assert np.array_equal(_raw(got), c), (what, i, step, int((_raw(got) != c).sum()))
        up = HP["lr"] / (1 - b1 ** step) * m.astype(np.float64) / (r.astype(np.float64) / np.sqrt(1 - b2 ** step) + HP["eps"])
        ref = p * (1 - HP["lr"] * HP["weight_decay"]) - up
        if ps[i].dtype == torch.float32:
            assert (np.abs(_np(ps[i]) - ref) <= 16 * U * (np.abs(p) + np.abs(up)) + 1e-45).all()


def _zero_states(n, dev):
    f = lambda k, t: torch.zeros(k, device=dev, dtype=torch.uint8).view(t)  # noqa: E731
    return [[f(k, t)] for k, t in ((n, torch.float8_e4m3fn), (-(-n // B), torch.float8_e8m0fnu)) * 2]


@pytest.mark.parametrize("dt", (torch.float32, torch.bfloat16, torch.float16))
def test_codes_over_steps(gpu_device, dt):
    """Four million elements, of which about one in a million lies where the rounding of an fp32 operation decides its code,
    three steps on from states of every code."""
    n = 1 << 22
    torch.manual_seed(21)
    ps = [(0.05 * torch.randn(n, device=gpu_device)).to(dt)]
    states = _states(ps, 8, ps)
    for step in (9, 10, 11):
        gs = [(0.01 * torch.randn(n, device=gpu_device) * torch.exp(torch.randn(n, device=gpu_device))).to(dt)]
        _same(ps, gs, *states, seed=4, step=step)


def test_largest_values_next_to_a_power_of_two(gpu_device):
    """Blocks whose largest m', or q, lies some fp32 steps on either side of 448 2^k, where the block's power of two changes."""
    n = 4096 * B
    torch.manual_seed(22)
    for share, at in ((0.1, 448.0), (np.sqrt(0.001), 448.0), (0.1, 28.0), (np.sqrt(0.001), 0.875)):
        top = F(at / share)
        tops = (top.view(np.int32) + np.arange(-2048, 2048, dtype=np.int32)).view(F)
        g = 1e-3 * float(top) * torch.randn(4096, B, device=gpu_device)
        g[:, 77] = torch.from_numpy(tops).to(gpu_device)
        _same([torch.zeros(n, device=gpu_device)], [g.view(n)], *_zero_states(n, gpu_device), seed=5, step=1)


def test_moments_that_cancel(gpu_device):
    """g near -9 m: m' is a thousandth to a ten-millionth of m, and what the rounding of g - m left of it."""
    n = 1 << 20
    torch.manual_seed(23)
    p = [torch.zeros(n, device=gpu_device)]
    m, mk, q, qk = _states(p, 8, p)
    m0 = torch.from_numpy(_value(_raw(m[0]), _raw(mk[0]))).to(gpu_device)
    near = 1 + torch.randn(n, device=gpu_device) * 10.0 ** -(3 + 4 * torch.rand(n, device=gpu_device))
    _same(p, [(-9 * m0 * near).float()], m, mk, q, qk, seed=6, step=3)


def test_the_32_bit_states_are_the_same_numbers(gpu_device):
    """What state_bits=32 holds after a step is what state_bits=8 rounds."""
    n = 1 << 20
    torch.manual_seed(24)
    p = [0.05 * torch.randn(n, device=gpu_device)]
    g = [0.01 * torch.randn(n, device=gpu_device)]
    m, mk, q, qk = _states(p, 8, p)
    m32, v32 = ([torch.from_numpy(x).float().to(gpu_device)] for x in (_value(_raw(m[0]), _raw(mk[0])),
                                                                      _value(_raw(q[0]), _raw(qk[0])) ** 2))
    want = _step32(_np(g[0]), _np(m32[0]), _np(v32[0]))
    p32 = [p[0].clone()]
    optim.adamw8_(p, g, m, mk, q, qk, step=3, seed=7, **HP)
    optim.adamw32_(p32, g, m32, v32, step=3, **HP)
    assert np.array_equal(m32[0].cpu().numpy(), want[0]) and np.array_equal(v32[0].cpu().numpy(), want[1])
    assert torch.equal(p[0], p32[0])
