"""The activations of linear_act alone: one feature, weight 1 and no bias, so that z is x itself and y = act(z), dx = dy act'(z)
with dy = 1 carry nothing but the activation's error and one rounding.

Bounds, u = 2^-24, e = eps(type) / 2. The functions come from the hardware's exponential and reciprocal (an ulp each); the
exponent z^2 / 2, or |z| for the sigmoids, is itself rounded, which moves the exponential by its size times a few u: a relative
error of (16 + 4 z^2 + 4 |t|) u, t the sigmoid's argument; in 16 bits the normal distribution adds its approximation's
6e-6. A slope is a sum of two terms, each with that error. Below the smallest normal number 2^-126 an exponential, or a
sigmoid, may be 0: it is multiplied by |z| <= 12 and, in the slope of the tanh form, by |z| 2 sqrt(2 / pi) (1 + 0.134 z^2) <=
12 * 1.6 * 20.4 < 2^9, so 2^-117 may be lost."""
import math

import pytest
import torch
import torch.nn as nn

from sehip import linear

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _terms(name, z):
    """act(z), the two terms of its slope, |t|, in 64 bits."""
    one, c = torch.ones_like(z), math.sqrt(2 / math.pi)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double(), 0 * z, 0 * z
    if name == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * p, p, z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0 * z
    t, d = (z, one) if name == "silu" else (2 * c * (z + 0.044715 * z ** 3), 2 * c * (1 + 3 * 0.044715 * z * z))
    p = torch.sigmoid(t)
    return z * p, p, z * p * torch.sigmoid(-t) * d, t.abs()


ACTS = {"relu": nn.ReLU(), "gelu": nn.GELU(), "gelu_tanh": nn.GELU("tanh"), "silu": nn.SiLU()}


@pytest.mark.parametrize("name", list(ACTS))
@pytest.mark.parametrize("dt", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("rows", (60, 40000))      # the few rows' kernel, the tiles'
def test_activation_and_slope(gpu_device, dt, name, rows):
    z = torch.cat([torch.linspace(-6, 6, rows // 2), torch.linspace(-12, 12, rows // 2)]).to(dt)
    lin = nn.Linear(1, 1, bias=False, device=gpu_device, dtype=dt)
    with torch.no_grad():
        lin.weight.fill_(1)
    x = z.to(gpu_device).view(-1, 1).requires_grad_(True)
    y = linear.linear_act(x, lin, ACTS[name])
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    z = z.double()
    a, s0, s1, t = _terms(name, z)
    e = torch.finfo(dt).eps / 2
    rel = (16 + 4 * z * z + 4 * t) * U + (6e-6 if dt != torch.float32 and name == "gelu" else 0)
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -117
    for what, got, ref, size in (("y", y, a, a.abs()), ("slope", dx, s0 + s1, s0.abs() + s1.abs())):
        err = (got.detach().double().cpu().view(-1) - ref).abs()
        bound = e * ref.abs() + (1 + e) * rel * size + tiny
        bad = err > bound
        assert not bad.any(), (what, int(bad.sum()), z[bad][:4].tolist(), (err / bound).max().item())
