"""AdamW(state_bits=8): groups with settings of their own, and the random bits of a group's tensors."""
import pytest
import torch
import torch.nn as nn

from sehip import optim

pytestmark = pytest.mark.gpu
HP = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)


def _codes(o, p):
    return [t.view(torch.uint8).clone() for k, t in o.state[p].items() if k in ("exp_avg", "exp_avg_root")]


def _step(ps, **kw):
    o = optim.AdamW(ps, **kw, **HP)
    for p in (p for g in o.param_groups for p in g["params"]):
        p.grad = torch.full_like(p, 0.3)
    o.step()
    return o


def test_a_group_with_its_own_state_bits(gpu_device):
    f = lambda: nn.Parameter(torch.ones(300, device=gpu_device))  # noqa: E731
    a, b, c = f(), f(), f()
    o = _step([{"params": [a], "state_bits": 8}, {"params": [b], "state_bits": 32}, {"params": [c]}])
    assert set(o.state[a]) == {"step", "exp_avg", "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale"}
    assert o.state[b]["exp_avg"].dtype == torch.float32 and set(o.state[c]) == {"step", "exp_avg", "exp_avg_sq"}
    assert torch.equal(a, b) and (a - c).abs().max() <= 1e-6
    d, e = f(), f()
    o = _step([{"params": [d], "seed": 5}, {"params": [e]}], state_bits=8, seed=5)
    p = _step([f()], state_bits=8, seed=5)
    assert all(torch.equal(x, y) for x, y in zip(_codes(o, d), _codes(p, p.param_groups[0]["params"][0])))
    assert not torch.equal(_codes(o, d)[0], _codes(o, e)[0])


def test_types_side_by_side_have_their_own_random_bits(gpu_device):
    """One group of fp32, bf16 and fp16 tensors of the same values: m' = 0.03 in each, its rounding from bits of its own."""
    n = 1 << 14
    ps = [nn.Parameter(torch.full((n,), 0.5, device=gpu_device, dtype=t)) for t in (torch.float32, torch.bfloat16, torch.float16)]
    o = optim.AdamW(ps, state_bits=8, seed=5, **HP)
    for p in ps:
        p.grad = torch.full_like(p, 0.296875)    # a number of every type
    o.step()
    every = [_codes(o, p) for p in ps]
    for i in range(3):
        for j in range(i):
            for a, b in zip(every[i], every[j]):
                # two values an element: independent bits agree at half to all but a few (share s of the upper one: s^2 + (1-s)^2)
                s = [(t == t.max()).double().mean().item() for t in (a, b)]
                agree, want = (a == b).double().mean().item(), s[0] * s[1] + (1 - s[0]) * (1 - s[1])
                assert abs(agree - want) < 6 * 0.5 / n ** 0.5, (i, j, agree, want)


def test_all_bits_of_the_seed_count(gpu_device):
    out = [_codes(o, o.param_groups[0]["params"][0]) for o in
           (_step([nn.Parameter(torch.ones(3000, device=gpu_device))], state_bits=8, seed=s) for s in (7, 7 + (1 << 32), 7 + (1 << 63)))]
    for i in range(3):
        for j in range(i):
            assert not torch.equal(out[i][0], out[j][0]) and not torch.equal(out[i][1], out[j][1])


@pytest.mark.parametrize("bits", (8, 32))
def test_everything_written_counts_as_changed(gpu_device, bits):
    """Autograd finds a saved tensor changed by its version: parameters, moments and scales each get a new one, gradients none."""
    f = lambda n, t: torch.ones(n, device=gpu_device, dtype=torch.uint8 if t.itemsize == 1 else t).view(t)  # noqa: E731
    kinds = [(5, torch.float32)] * 2 + ([(5, torch.float8_e4m3fn), (1, torch.float8_e8m0fnu)] * 2 if bits == 8 else [(5, torch.float32)] * 2)
    lists = [[f(n, t)] for n, t in kinds]
    before = [ts[0]._version for ts in lists]
    (optim.adamw8_ if bits == 8 else optim.adamw32_)(*lists, step=1)
    assert [ts[0]._version - v for ts, v in zip(lists, before)] == [1, 0] + [1] * (len(lists) - 2)
