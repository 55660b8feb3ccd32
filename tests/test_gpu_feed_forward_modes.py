"""layer_norm and linear_act under forward-mode differentiation and under a trace: with frozen parameters too, a call whose
derivative or graph is asked for has to say that it has none, or be in it."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn as nn

from sehip import linear, norm

pytestmark = pytest.mark.gpu


def _modules(dev, train=False):
    torch.manual_seed(31)
    ln, lin = nn.LayerNorm(24, device=dev), nn.Linear(24, 40, device=dev)
    for p in (*ln.parameters(), *lin.parameters()):
        p.requires_grad_(train)
    return ln, lin


@pytest.mark.parametrize("train", (False, True))
@pytest.mark.parametrize("grad", (False, True))
def test_forward_mode_is_refused(gpu_device, train, grad):
    ln, lin = _modules(gpu_device, train)
    x, t, r = (torch.randn(5, n, device=gpu_device) for n in (24, 24, 40))
    calls = (lambda v: norm.layer_norm(ln, v), lambda v: linear.linear_act(v, lin, nn.GELU()),
             lambda v: linear.linear_act(x, lin, None, torch.cat([v, v], 1)[:, :40]))
    want = [f(x) for f in calls]
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        for f, y in zip(calls, want):
            with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                f(fwAD.make_dual(x, t))
            assert torch.equal(f(x), y)      # no tangent: as ever
    for f in calls:
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (x,), (t,))


def test_a_trace_holds_the_operators(gpu_device):
    ln, lin = _modules(gpu_device)
    down = nn.Linear(40, 24, device=gpu_device)
    for p in down.parameters():
        p.requires_grad_(False)

    def block(x):
        return linear.linear_act(linear.linear_act(norm.layer_norm(ln, x), lin, nn.GELU()), down, None, x)

    x = torch.randn(6, 24, device=gpu_device)
    with torch.no_grad():
        traced = torch.jit.trace(block, x)
        for k in range(3):
            x = torch.randn(6, 24, device=gpu_device)
            torch.full((1 << 16,), float("nan"), device=gpu_device)   # what unwritten memory would show
            assert torch.equal(traced(x), block(x)), k
