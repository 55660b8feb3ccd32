"""Layer norm on the HIP kernels (sehip.norm.layer_norm, csrc/layernorm.hip) against its formula in 64 bits.

Bounds, u = 2^-24, X = max |x| of the row, s = 1 / sqrt(var + eps), h = (x - mu) s, e = eps(type) / 2:
a row's sums have at most 16 + 6 + 16 = 38 roundings on any path (16 elements a thread, six shuffles, sixteen waves; the wide
form C / 1024 elements a thread, at most 20 here), so mu is off by 40 u X, x - mu by that and its own rounding, and s by
(40 / 2 + 4) u of itself (a shift of the mean enters the variance squared):
  |dy| <= e |y| + u (28 |h w| + 4 |b| + 40 X s |w|)
  dx = s (a - A0 - h A1), a = dy w, A0 = mean a, A1 = mean a h; with E = 28 |h| + 40 X s the error of h in u:
  |d dx| <= e |dx| + u s (28 |dx / s| + 4 |a| + 46 mean |a| + |h| (46 mean |a h| + mean |a| E) + |A1| E)
  the rows' sums: every thread adds rows / (parts * groups) of them, then at most 16 groups, parts / 16 + 16 partials: 160
  roundings cover the cases here; |d dw| <= e |dw| + u (160 sum |dy h| + sum |dy| E), |d db| <= e |db| + 160 u sum |dy|"""
import pytest
import torch
import torch.nn as nn

from sehip import norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _half(dt):
    return torch.finfo(dt).eps / 2


def _module(C, dt, dev, affine=True, bias=True, eps=1e-5):
    m = nn.LayerNorm(C, eps=eps, elementwise_affine=affine, bias=bias, device=dev, dtype=dt)
    with torch.no_grad():
        if m.weight is not None:
            m.weight.copy_(1 + 0.3 * torch.randn(m.weight.shape, device=dev))
        if m.bias is not None:
            m.bias.copy_(0.2 * torch.randn(m.bias.shape, device=dev))
    return m


def _check(x, m, dy, y, dx, dw, db):
    C = m.weight.numel() if m.weight is not None else x.shape[-1]
    x, g = x.detach().double().reshape(-1, C), dy.double().reshape(-1, C)
    w = m.weight.detach().double().view(-1) if m.weight is not None else torch.ones(C, device=x.device).double()
    b = m.bias.detach().double().view(-1) if m.bias is not None else torch.zeros_like(w)
    mu = x.mean(1, keepdim=True)
    s = 1 / ((x - mu).square().mean(1, keepdim=True) + m.eps).sqrt()
    h = (x - mu) * s
    top = x.abs().amax(1, keepdim=True) * s
    E = 28 * h.abs() + 40 * top

    def close(got, ref, bound, what):
        got = got.detach().double().reshape(ref.shape)
        bad = (got - ref).abs() > bound
        assert not bad.any(), (what, int(bad.sum()), ((got - ref).abs() / bound.clamp_min(1e-300)).max().item())

    ref = h * w + b
    close(y, ref, _half(y.dtype) * ref.abs() + U * (28 * (h * w).abs() + 4 * b.abs() + 40 * top * w.abs()) + 1e-45, "y")
    a = g * w
    A0, A1 = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
    mean = lambda t: t.abs().mean(1, keepdim=True)  # noqa: E731
    if dx is not None:
        ref = s * (a - A0 - h * A1)
        # fp16 below 2^-14 keeps steps of 2^-24
        tiny = 2.0 ** -25 if dx.dtype == torch.float16 else 1e-45
        close(dx, ref, _half(dx.dtype) * ref.abs() + tiny + U * s * (28 * (ref / s).abs() + 4 * a.abs() + 46 * mean(a) + h.abs() * (
            46 * mean(a * h) + (a.abs() * E).mean(1, keepdim=True)) + A1.abs() * E), "dx")
    if dw is not None:
        ref = (g * h).sum(0)
        close(dw, ref, _half(dw.dtype) * ref.abs() + U * (160 * (g * h).abs().sum(0) + (g.abs() * E).sum(0)) + 1e-45, "dw")
    if db is not None:
        ref = g.sum(0)
        close(db, ref, _half(db.dtype) * ref.abs() + U * 160 * g.abs().sum(0) + 1e-45, "db")


def _run(x, m, dy):
    x = x.detach().requires_grad_(True)
    y = norm.layer_norm(m, x)
    of = [x] + [p for p in (m.weight, m.bias) if p is not None]
    got = list(torch.autograd.grad(y, of, dy))
    dx = got.pop(0)
    dw = got.pop(0) if m.weight is not None else None
    db = got.pop(0) if m.bias is not None else None
    return y, dx, dw, db


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,C", [
    (1, 1), (1, 1024), (3, 2), (5, 16), (7, 17), (33, 64), (2, 255), (130, 256), (9, 257), (1031, 514), (77, 1000),
    (64, 1024), (5, 1025), (300, 2048), (3, 4096), (40, 4100), (6, 8192), (5, 8193), (3, 16384), (2, 16387), (70, 20000)])
def test_matches_the_formula(gpu_device, dt, rows, C):
    torch.manual_seed(rows * 31 + C)
    x = ((torch.randn(rows, C, device=gpu_device) + torch.randn(C, device=gpu_device))
         * torch.exp(torch.randn(rows, 1, device=gpu_device))).to(dt)
    dy = torch.randn(rows, C, device=gpu_device).to(dt)
    m = _module(C, dt, gpu_device)
    y, dx, dw, db = _run(x, m, dy)
    _check(x, m, dy, y, dx, dw, db)
    with torch.no_grad():   # without gradients: the same values
        assert torch.equal(norm.layer_norm(m, x), y)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("affine,bias", [(False, False), (True, False)])
def test_without_weight_or_bias(gpu_device, dt, affine, bias):
    torch.manual_seed(1)
    x, dy = (torch.randn(37, 96, device=gpu_device).to(dt) for _ in range(2))
    m = _module(96, dt, gpu_device, affine, bias)
    _check(x, m, dy, *_run(x, m, dy))


@pytest.mark.parametrize("dt", TYPES[1:])
@pytest.mark.parametrize("C", [96, 101, 20000])
def test_fp32_weights_beside_16_bit_rows(gpu_device, dt, C):
    torch.manual_seed(2)
    x, dy = (torch.randn(41, C, device=gpu_device).to(dt) for _ in range(2))
    m = _module(C, torch.float32, gpu_device)
    y, dx, dw, db = _run(x, m, dy)
    assert y.dtype == dx.dtype == dt and dw.dtype == db.dtype == torch.float32
    _check(x, m, dy, y, dx, dw, db)


@pytest.mark.parametrize("dt", TYPES)
def test_strides_and_shapes(gpu_device, dt):
    """Rows at a distance, rows off their alignment, copies of what is not rows, several normalised axes."""
    torch.manual_seed(3)
    base = torch.randn(6, 5, 300, device=gpu_device).to(dt)
    m = _module(128, dt, gpu_device)
    for x in (base[:, :, 8:136], base[:, :, 3:131], base[:, 1, 64:192], base[2, 3, :128],
              torch.randn(6, 128, 5, device=gpu_device).to(dt).transpose(1, 2)):
        dy = torch.randn(x.shape, device=gpu_device).to(dt)
        y, dx, dw, db = _run(x, m, dy)
        assert y.is_contiguous() and dx.shape == x.shape
        _check(x, m, dy, y, dx, dw, db)
        for g in (torch.ones((), device=gpu_device, dtype=dt).expand(x.shape), dy.transpose(0, -1).contiguous().transpose(0, -1)):
            _check(x, m, g.contiguous(), *_run(x, m, g))
    m2 = nn.LayerNorm((4, 32), device=gpu_device, dtype=dt)
    with torch.no_grad():
        m2.weight.copy_(torch.randn(4, 32, device=gpu_device))
    x, dy = (torch.randn(7, 4, 32, device=gpu_device).to(dt) for _ in range(2))
    y, dx, dw, db = _run(x, m2, dy)
    assert dw.shape == (4, 32)
    _check(x, m2, dy, y, dx, dw, db)


def test_far_mean_constant_rows_and_tiny_variance(gpu_device):
    """A mean far above the deviation (the squared deviations come from x - mu, not from two large sums), rows of one
    value (variance 0: y = bias), and rows of zeros."""
    torch.manual_seed(4)
    x = 1000 + torch.randn(8, 512, device=gpu_device)
    x[1] = 3.0
    x[2] = 0.0
    m = _module(512, torch.float32, gpu_device)
    dy = torch.randn_like(x)
    y, dx, dw, db = _run(x, m, dy)
    _check(x, m, dy, y, dx, dw, db)
    assert torch.equal(y[1], m.bias) and torch.equal(y[2], m.bias)


@pytest.mark.parametrize("dt", TYPES)
def test_nan_and_infinity_stay_in_their_row(gpu_device, dt):
    torch.manual_seed(5)
    m = _module(200, dt, gpu_device)
    x, dy = (torch.randn(64, 200, device=gpu_device).to(dt) for _ in range(2))
    y0, dx0, _, _ = _run(x, m, dy)
    x[3, 7], x[20, 0], x[41, 199] = float("nan"), float("inf"), float("-inf")
    y, dx, dw, db = _run(x, m, dy)
    bad = torch.tensor([3, 20, 41], device=gpu_device)
    rest = torch.ones(64, dtype=torch.bool, device=gpu_device).index_fill(0, bad, False)
    assert torch.equal(y[rest], y0[rest]) and torch.equal(dx[rest], dx0[rest])
    assert y[bad].isnan().any(1).all() and dx[bad].isnan().any(1).all()


def test_no_rows(gpu_device):
    m = _module(16, torch.float32, gpu_device)
    x = torch.zeros(0, 3, 16, device=gpu_device, requires_grad=True)
    y = norm.layer_norm(m, x)
    dx, dw, db = torch.autograd.grad(y, (x, m.weight, m.bias), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 3, 16) and not dw.any() and not db.any()


def test_only_what_is_asked(gpu_device):
    torch.manual_seed(6)
    x, dy = (torch.randn(50, 96, device=gpu_device) for _ in range(2))
    m = _module(96, torch.float32, gpu_device)
    _, dx, dw, db = _run(x, m, dy)
    for want in range(1, 8):
        xs = x.clone().requires_grad_(bool(want & 1))
        m.weight.requires_grad_(bool(want & 2))
        m.bias.requires_grad_(bool(want & 4))
        y = norm.layer_norm(m, xs)
        of = [(t, r) for t, r in ((xs, dx), (m.weight, dw), (m.bias, db)) if t.requires_grad]
        for got, (_, ref) in zip(torch.autograd.grad(y, [t for t, _ in of], dy), of):
            assert torch.equal(got, ref)


def test_bits_repeat(gpu_device):
    torch.manual_seed(7)
    x, dy = (torch.randn(9002, 514, device=gpu_device) for _ in range(2))
    m = _module(514, torch.float32, gpu_device)
    a, b = _run(x, m, dy), _run(x, m, dy)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradient_against_differences(gpu_device):
    """Directional differences of the forward in fp32: L(x + t v) - L(x - t v) over 2 t. With t = 2^-6 the cubic term is
    t^2 / 6 of the third derivative, of the order of the value itself here, below 1e-3; rounding is u / t, below 1e-4."""
    torch.manual_seed(8)
    x, dy, v = (torch.randn(4, 300, device=gpu_device) for _ in range(3))
    m = _module(300, torch.float32, gpu_device)
    _, dx, dw, db = _run(x, m, dy)
    t = 2.0 ** -6
    with torch.no_grad():
        L = lambda z: (norm.layer_norm(m, z).double() * dy.double()).sum()  # noqa: E731
        num, ana = ((L(x + t * v) - L(x - t * v)) / (2 * t)).item(), (dx.double() * v.double()).sum().item()
    scale = (dx.norm() * v.norm()).item()
    assert abs(num - ana) < 2e-3 * scale


def test_graph_replays_and_other_stream(gpu_device):
    """Forward and backward captured into a graph: every replay on new inputs gives the eager bits; and the same on a
    stream of its own."""
    torch.manual_seed(9)
    m = _module(514, torch.bfloat16, gpu_device)
    x = torch.randn(403, 514, device=gpu_device).bfloat16().requires_grad_(True)
    dy = torch.randn(403, 514, device=gpu_device).bfloat16()

    def step():
        y = norm.layer_norm(m, x)
        return (y, *torch.autograd.grad(y, (x, m.weight, m.bias), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(other, step()))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(403, 514, device=gpu_device))
            dy.copy_(torch.randn(403, 514, device=gpu_device))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step())), k


def test_offsets_past_32_bits(gpu_device):
    """2^31 elements and more: the rows at the far end are as those at the start."""
    C = 4096
    rows = (1 << 31) // C + 100
    m = _module(C, torch.bfloat16, gpu_device)
    x = torch.empty(rows, C, device=gpu_device, dtype=torch.bfloat16)
    x.view(-1)[:1 << 20].normal_()
    x[256:512].copy_(x[:256])
    x[512:] = 0
    x[-100:].copy_(x[:100])
    x.requires_grad_(True)
    y = norm.layer_norm(m, x)
    dy = torch.zeros_like(y)
    dy[:100] = y.detach()[:100]
    dy[-100:] = dy[:100]
    dx, dw = torch.autograd.grad(y, (x, m.weight), dy)
    assert torch.equal(y[-100:], y[:100]) and torch.equal(dx[-100:], dx[:100])
    assert dx[-100:].abs().sum() > 0 and not dx[512:-100].any()


def test_refusals_on_the_gpu(gpu_device):
    x = torch.randn(4, 8, device=gpu_device)
    with pytest.raises(RuntimeError, match="on one GPU"):
        norm.layer_norm(nn.LayerNorm(8), x)
    with pytest.raises(RuntimeError, match="weight and bias"):
        norm.layer_norm(nn.LayerNorm(8, device=gpu_device, dtype=torch.bfloat16), x)
    with pytest.raises(RuntimeError, match="unsupported storage type"):
        norm.layer_norm(nn.LayerNorm(8, device=gpu_device).double(), x.double())
    m = nn.LayerNorm(8, device=gpu_device)
    y = norm.layer_norm(m, x.requires_grad_(True))
    (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):   # once differentiable
        dx.sum().backward()
