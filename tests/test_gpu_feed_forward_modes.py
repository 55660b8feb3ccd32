"""layer_norm and linear_act under forward-mode differentiation and under a trace: with frozen parameters too, a call whose
derivative or graph is asked for has to say that it has none, or be in it."""
import warnings

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
        with warnings.catch_warnings():
            warnings.simplefilter("ignore", torch.jit.TracerWarning)     # sizes that are checked
            traced = torch.jit.trace(block, x)
        for k in range(3):
            x = torch.randn(6, 24, device=gpu_device)
            torch.full((1 << 16,), float("nan"), device=gpu_device)   # what unwritten memory would show
            assert torch.equal(traced(x), block(x)), k


@pytest.mark.parametrize("rows,width", [(7, 24), (1, 24), (1, 1)])
def test_lazily_negated_tensors(gpu_device, rows, width):
    """The imaginary part of a conjugate, and the gradient that comes back through one, carry their sign beside their memory."""
    torch.manual_seed(34)
    dev = gpu_device
    ln, lin, down = nn.LayerNorm(width, device=dev), nn.Linear(width, 2 * width, device=dev), nn.Linear(2 * width, width, device=dev)
    spec = torch.randn(rows, width, device=dev, dtype=torch.complex64)
    g = torch.randn(rows, width, device=dev, dtype=torch.complex64)
    x = spec.conj().imag
    assert x.is_neg()
    ps = [p for m in (ln, lin, down) for p in m.parameters()]
    out = []
    for neg in (True, False):
        v = (x if neg else x.resolve_neg().contiguous()).detach().requires_grad_(True)
        assert v.is_neg() == neg
        y = linear.linear_act(linear.linear_act(norm.layer_norm(ln, v), lin, nn.GELU()), down, None, v)
        if neg:
            torch.autograd.backward(torch.complex(torch.zeros_like(y), y).conj(), g)     # y's gradient: the imaginary part of g's conjugate
        else:
            y.backward(-g.imag.contiguous())
        out.append((y.detach(), v.grad.clone(), *(p.grad.clone() for p in ps)))
        for p in ps:
            p.grad = None
        h = norm.layer_norm(ln, v)
        dh = (torch.autograd.grad(torch.complex(h, h).conj(), (v, ln.weight, ln.bias), g) if neg else
              torch.autograd.grad(h, (v, ln.weight, ln.bias), (g.real - g.imag).contiguous()))
        out[-1] += dh
    assert all(torch.equal(a, b) for a, b in zip(*out)), [torch.equal(a, b) for a, b in zip(*out)]


@pytest.mark.parametrize("bits", (None, 8, 32))
def test_a_parameter_of_one_element_whose_gradient_is_negated(gpu_device, bits):
    from sehip import optim
    ps = [nn.Parameter(torch.ones(1, device=gpu_device)) for _ in range(2)]
    g = torch.tensor([0.5 + 0.25j], device=gpu_device)
    torch.autograd.backward(torch.complex(torch.ones_like(ps[0]), ps[0]).conj(), g)
    assert ps[0].grad.is_neg() and ps[0].grad.item() == -0.25
    ps[1].grad = torch.full_like(ps[1], -0.25)
    for p in ps:
        optim.AdamW([p], lr=0.1, weight_decay=0.0, state_bits=bits).step()
    assert torch.equal(ps[0], ps[1]) and ps[0].item() > 1
