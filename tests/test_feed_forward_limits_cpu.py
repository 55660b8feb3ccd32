"""The feed-forward operators' calls at the edges of what they take: refused or answered on the host, without a GPU."""
import ctypes

import pytest
import torch
import torch.nn as nn

from sehip import _native as N
from sehip import linear, norm, optim


@pytest.mark.parametrize("sizes", [((1 << 32) + 100, 4, 8), (3, (1 << 32) + 4, 8), (3, 4, (1 << 32) + 8), (1 << 31, 4, 8)])
def test_sizes_that_a_c_int_does_not_hold(sizes):
    """ctypes keeps the low 32 bits of a larger number: such a call would compute the first rows alone."""
    with pytest.raises(RuntimeError, match="32-bit"):
        N.LinearDesc(*sizes, 0, 1, 8, 8, 4)
    assert N.LinearDesc((1 << 31) - 1, 4, 8, 0, 1, 8, 8, 4).M == (1 << 31) - 1


def test_a_group_with_its_own_state_bits():
    p = lambda: nn.Parameter(torch.zeros(3))  # noqa: E731
    o = optim.AdamW([{"params": [p()], "state_bits": 8}, {"params": [p()], "state_bits": 32, "seed": 9}, {"params": [p()]}], seed=4)
    assert [(g.get("state_bits"), g.get("seed")) for g in o.param_groups] == [(8, 4), (32, 9), (None, None)]
    o.add_param_group({"params": [p()], "state_bits": 8})
    assert o.param_groups[-1]["seed"] == 4 and "state_bits" not in o.param_groups[2]
    o = optim.AdamW([{"params": [p()]}, {"params": [p()], "state_bits": None}], state_bits=8, seed=2)
    assert [(g["state_bits"], g["seed"]) for g in o.param_groups] == [(8, 2), (None, 2)]
    for bad in (16, "8", 0, -8):
        with pytest.raises(ValueError, match="state_bits"):
            optim.AdamW([{"params": [p()], "state_bits": bad}])
        with pytest.raises(ValueError, match="state_bits"):
            o.add_param_group({"params": [p()], "state_bits": bad})


@pytest.mark.parametrize("to", (None, 32))
def test_a_state_of_8_bits_is_not_taken_for_numbers(to):
    """torch casts what it loads to the parameter's type: codes without their scales. Refused, and nothing is replaced."""
    make = lambda bits: optim.AdamW([nn.Parameter(torch.zeros(7, 40)), nn.Parameter(torch.zeros(3))], lr=0.5, state_bits=bits)  # noqa: E731
    a, b = make(8), make(to)
    p = a.param_groups[0]["params"][0]
    a.state[p] = {"step": torch.tensor(4.0), **optim._state_like(p, 8, torch.zeros)}
    a.param_groups[0]["lr"] = 0.25
    q = b.param_groups[0]["params"][0]
    b.state[q] = {"step": torch.tensor(2.0), "exp_avg": torch.ones(7, 40), "exp_avg_sq": torch.ones(7, 40)}
    with pytest.raises(ValueError, match="exp_avg"):
        b.load_state_dict(a.state_dict())
    assert b.param_groups[0]["lr"] == 0.5 and float(b.state[q]["step"]) == 2 and set(b.state[q]) == {"step", "exp_avg", "exp_avg_sq"}
    t = torch.optim.AdamW([nn.Parameter(torch.zeros(7, 40)), nn.Parameter(torch.zeros(3))], lr=0.125)
    r = t.param_groups[0]["params"][0]
    r.grad = torch.ones_like(r)
    t.step()
    b.load_state_dict(t.state_dict())
    assert b.param_groups[0]["lr"] == 0.125 and torch.equal(b.state[q]["exp_avg"], t.state[r]["exp_avg"])


@pytest.mark.parametrize("base", (nn.Identity, nn.ReLU, nn.GELU, nn.SiLU))
def test_an_activation_with_a_forward_of_its_own(base):
    """Refused; a subclass that only adds something else is its base."""
    class Scaled(base):
        def forward(self, x):
            return 2 * super().forward(x)

    class Named(base):
        name = "named"

    with pytest.raises(NotImplementedError, match="Scaled"):
        linear.linear_act(torch.zeros(3, 8), nn.Linear(8, 4), Scaled())
    assert linear._act_code(Named()) == linear._act_code(base())
    assert linear._act_code(nn.GELU("tanh")) == linear.ACT_GELU_TANH != linear._act_code(nn.GELU())


def test_linear_tile():
    """What multiplies a product is known on the host."""
    def tile(dt, m, k, n, product, act=0):
        splits = ctypes.c_int(-1)
        t = N.lib().se_linear_tile(ctypes.byref(N.LinearDesc(m, n, k, act, dt, k, k, n)), product, ctypes.byref(splits))
        return t, splits.value

    F32, BF16 = 0, 1
    for p in range(3):
        assert tile(BF16, 16384, 4096, 8192, p, 3) == (256, 1)
        assert tile(F32, 100, 64, 72, p)[0] == 64
    assert tile(BF16, 16, 4096, 1024, 0) == (0, 1) and tile(BF16, 16, 4096, 1024, 1)[0] == 128   # few rows: forward alone
    assert tile(BF16, 1000, 64, 72, 0) == (128, 1) and tile(BF16, 20000, 64, 48, 2)[1] > 1
    assert tile(BF16, 100, 64, 72, 3)[0] == tile(BF16, 0, 64, 72, 0)[0] == -1
    assert N.lib().se_linear_tile(ctypes.byref(N.LinearDesc(100, 64, 72, 0, 1, 72, 72, 64)), 0, None) == 128
