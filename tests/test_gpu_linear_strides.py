"""linear_act on rows that lie further apart than a tile's 32-bit offsets reach (2^21 elements): the last frame of a batch
of sequences, a residual, a gradient or a weight cut out of something large. The result is that of the contiguous copy, bit
for bit: the same kernels on the same numbers, whether they read the rows as they lie or packed ones."""
import pytest
import torch
import torch.nn as nn

from sehip import linear

pytestmark = pytest.mark.gpu
FAR = (1 << 21) + 64     # elements between rows


def _far(dev, dt, m, n, at=0):
    """[m, n] random values, rows FAR apart, `at` elements into theirs."""
    t = torch.empty((m - 1) * FAR + at + n, device=dev, dtype=dt).as_strided((m, n), (FAR, 1), at)
    return t.copy_(torch.randn(m, n, device=dev))


def _run(x, lin, res, dy):
    x = x.detach().requires_grad_(True)
    res = None if res is None else res.detach().requires_grad_(True)
    y = linear.linear_act(x, lin, nn.GELU(), res)
    with torch.no_grad():
        assert torch.equal(linear.linear_act(x, lin, nn.GELU(), res), y)
    return (y, *torch.autograd.grad(y, [t for t in (x, lin.weight, lin.bias) if t is not None], dy))


@pytest.mark.parametrize("dt", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("m,k,n", [(2, 512, 512), (3, 40, 24), (33, 65, 7), (70, 64, 72), (300, 72, 264)])
@pytest.mark.parametrize("at", (0, 1))
def test_rows_far_apart(gpu_device, dt, m, k, n, at):
    torch.manual_seed(32)
    dev = gpu_device
    lin = nn.Linear(k, n, device=dev, dtype=dt)
    x, res, dy = _far(dev, dt, m, k, at), _far(dev, dt, m, n, at), _far(dev, dt, m, n, at)
    want = _run(x.contiguous(), lin, res.contiguous(), dy.contiguous())
    for a, b, c in ((x, res, dy), (x, None, dy.contiguous()), (x.contiguous(), res, dy.contiguous()), (x.contiguous(), res, dy)):
        got = _run(a, lin, b, c)
        ref = want if b is not None else _run(x.contiguous(), lin, None, dy.contiguous())
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
    w = _far(dev, dt, n, k, at).copy_(lin.weight)
    lin.weight = nn.Parameter(w)
    assert lin.weight.stride(0) == FAR or n == 1
    got = _run(x, lin, res, dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_rows_far_apart_without_an_activation(gpu_device):
    """dy goes to dx and dW as it lies where nothing multiplies it, in fp32 in the large form too."""
    torch.manual_seed(33)
    for dt, m, k, n in ((torch.bfloat16, 130, 64, 72), (torch.float32, 130, 64, 72), (torch.float32, 1100, 1030, 1030)):
        lin = nn.Linear(k, n, device=gpu_device, dtype=dt)
        x, dy = _far(gpu_device, dt, m, k), _far(gpu_device, dt, m, n)
        out = []
        for a, b in ((x, dy), (x.contiguous(), dy.contiguous())):
            a = a.detach().requires_grad_(True)
            y = linear.linear_act(a, lin)
            out.append((y, *torch.autograd.grad(y, (a, lin.weight, lin.bias), b)))
        assert all(torch.equal(p, q) for p, q in zip(*out))


def test_the_last_frame_of_each_sequence(gpu_device):
    h = torch.randn(2, 5000, 512, device=gpu_device).bfloat16()
    lin = nn.Linear(512, 96, device=gpu_device, dtype=torch.bfloat16)
    with torch.no_grad():
        assert torch.equal(linear.linear_act(h[:, -1], lin), linear.linear_act(h[:, -1].contiguous(), lin))
