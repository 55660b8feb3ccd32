"""The product with bias, activation and residual in its epilogue (sehip.linear.linear_act, csrc/linear.hip) against its
formula in 64 bits on the same inputs.

Bounds, u = 2^-24, e = eps(type) / 2, S = sum_k |x w| (+ |b|):
  16 bits: exact products, at most K + 8 additions of at most 2 u each (the matrix instruction need not round to nearest);
  fp32: x and w are hi + lo of 22 bits (2^-22 each), lo lo is left out (2^-22): 3 2^-22 S, and 3 K + 8 additions.
  z is off by D = S (2 n u + [fp32] 3 2^-22); y by e |y| + 1.13 D + 8 u (|act(z)| + |r|): no slope here is over 1.13, and the
  functions are a few u off.
  g = dy act'(z~), z~ the stored z: off by the slope's range over z (1 +- e) +- D, and rounded once more (e) in 16 bits;
  then dx, dW, db are sums of such terms, each with its own accumulation error, rounded once."""
import ctypes
import math

import pytest
import torch
import torch.nn as nn

from sehip import _native as N
from sehip import linear

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)
ACTS = {"none": nn.Identity(), "relu": nn.ReLU(), "gelu": nn.GELU(), "gelu_tanh": nn.GELU("tanh"), "silu": nn.SiLU()}


def _act(name, z):
    """act(z) and its slope in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _terms(dt, n):
    return (2 * (3 * n + 8) * U + 3 * 2.0 ** -22) if dt == torch.float32 else 2 * (n + 8) * U


def _close(got, ref, bound, what):
    got = got.detach().double().reshape(ref.shape)
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), ((got - ref).abs() / bound).max().item())


def _check(x, w, b, res, name, dy, y, grads):
    dt = x.dtype
    e = torch.finfo(dt).eps / 2
    tiny = {torch.float16: 2.0 ** -25}.get(dt, 1e-40)   # half a step of the type's smallest numbers
    n, k = w.shape
    x, w = x.detach().double().reshape(-1, k), w.detach().double()
    m = x.shape[0]
    b = torch.zeros(n, device=x.device).double() if b is None else b.detach().double()
    r = torch.zeros(m, n, device=x.device).double() if res is None else res.detach().double().reshape(m, n)
    z = x @ w.t() + b
    D = (x.abs() @ w.abs().t() + b.abs()) * _terms(dt, k)
    a, slope = _act(name, z)
    ref = a + r
    _close(y, ref, e * ref.abs() + (1 + e) * (1.13 * D + 8 * U * (a.abs() + r.abs())) + tiny, "y")
    if grads is None:
        return
    dx, dw, db = grads
    g = dy.double().reshape(m, n)
    lo, hi = z - e * z.abs() - D - tiny, z + e * z.abs() + D + tiny
    off = torch.maximum((_act(name, lo)[1] - slope).abs(), (_act(name, hi)[1] - slope).abs())
    G = g * slope
    # the slopes are smooth: their range over the interval is at most twice what its ends show, and 8 u of their own error
    dG = g.abs() * (2 * off + 8 * U * (1 + z.abs())) if name != "none" else torch.zeros_like(g)
    if dt != torch.float32 and name != "none":
        dG = dG + e * (G.abs() + dG) + tiny
    A = G.abs() + dG
    for got, ref, spread, total, cnt, what in (
            (dx, G @ w, dG @ w.abs(), A @ w.abs(), n, "dx"), (dw, G.t() @ x, dG.t() @ x.abs(), A.t() @ x.abs(), m, "dw"),
            (db, G.sum(0), dG.sum(0), A.sum(0), 0, "db")):
        if got is not None:
            acc = total * (_terms(dt, cnt) if cnt else 200 * U)   # db: at most 64 / 4 + 4 + 128 / 16 + 16 additions here
            _close(got, ref, e * ref.abs() + (1 + e) * (spread + acc) + tiny, what)


def _make(dev, dt, m, k, n, bias=True, residual=True, seed=0):
    torch.manual_seed(seed * 1000 + m * 31 + k * 7 + n)
    x = torch.randn(m, k, device=dev).to(dt)
    lin = nn.Linear(k, n, bias=bias, device=dev, dtype=dt)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(n, k, device=dev) / math.sqrt(k))
        if bias:
            lin.bias.copy_(torch.randn(n, device=dev))
    res = torch.randn(m, n, device=dev).to(dt) if residual else None
    return x, lin, res, torch.randn(m, n, device=dev).to(dt)


def _run(x, lin, act, res, dy):
    x = x.detach().requires_grad_(True)
    res = None if res is None else res.detach().requires_grad_(True)
    y = linear.linear_act(x, lin, ACTS[act], res)
    of = [t for t in (x, lin.weight, lin.bias, res) if t is not None]
    got = list(torch.autograd.grad(y, of, dy))
    if res is not None:
        assert torch.equal(got.pop(), dy)
    return y, (got[0], got[1], got[2] if lin.bias is not None else None)


SHAPES = [(1, 1, 1), (1, 64, 8), (1, 1024, 4096), (2, 7, 5), (3, 8, 8), (5, 72, 40), (16, 514, 130), (17, 4096, 64), (33, 65, 257),
          (64, 200, 96), (128, 128, 128), (130, 512, 264), (257, 136, 1030), (403, 514, 512), (1000, 64, 72), (2049, 96, 33)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_matches_the_formula(gpu_device, dt, m, k, n):
    for i, act in enumerate(ACTS):
        if i != (m + k + n) % 5 and i != (m * k + n) % 5:
            continue
        x, lin, res, dy = _make(gpu_device, dt, m, k, n, bias=i != 1, residual=(m + i) % 2 == 0)
        y, grads = _run(x, lin, act, res, dy)
        _check(x, lin.weight, lin.bias, res, act, dy, y, grads)
        with torch.no_grad():
            _check(x, lin.weight, lin.bias, res, act, None, linear.linear_act(x, lin, ACTS[act], res), None)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", list(ACTS))
def test_every_activation(gpu_device, dt, act):
    x, lin, res, dy = _make(gpu_device, dt, 70, 48, 88, seed=1)
    x = x * 3   # into the activations' tails
    y, grads = _run(x, lin, act, res, dy)
    _check(x, lin.weight, lin.bias, res, act, dy, y, grads)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", [(6000, 64, 48), (20000, 40, 264), (300, 9000, 24)])
def test_long_sums(gpu_device, dt, m, k, n):
    """Reductions that are split over workgroups: the batch's rows in dW, a long K in the forward."""
    x, lin, res, dy = _make(gpu_device, dt, m, k, n, seed=2)
    y, (dx, dw, db) = _run(x, lin, "silu", res, dy)
    _check(x, lin.weight, lin.bias, res, "silu", dy, y, (dx, dw, None))
    g = dy.double() * _act("silu", x.double() @ lin.weight.double().t() + lin.bias.double())[1]
    # db: rows / 4 / 128 + 4 + 16 additions, g rounded once
    e = torch.finfo(dt).eps / 2
    _close(db, g.sum(0), e * g.sum(0).abs() + (g.abs().sum(0)) * (200 * U + (3 * e if dt != torch.float32 else 64 * _terms(dt, k))), "db")


@pytest.mark.parametrize("dt", TYPES)
def test_strides(gpu_device, dt):
    """Rows at a distance, on and off 16 bytes, transposed inputs, weights and gradients, an expanded gradient."""
    torch.manual_seed(3)
    dev = gpu_device
    base, wide = torch.randn(3, 50, 200, device=dev).to(dt), torch.randn(3, 50, 160, device=dev).to(dt)
    lin = nn.Linear(64, 72, device=dev, dtype=dt)
    for x in (base[:, :, 8:72], base[:, :, 5:69], base[:, 7, 16:80], base[1, 2, :64],
              torch.randn(3, 64, 50, device=dev).to(dt).transpose(1, 2)):
        full = wide[..., :72] if x.dim() == 3 else wide[:, 7, 1:73] if x.dim() == 2 else wide[0, 0, :72]
        for res, dy in ((full, torch.randn(full.shape, device=dev).to(dt)),
                        (None, torch.randn(full.shape[::-1], device=dev).to(dt).permute(*range(full.dim())[::-1])),
                        (None, torch.full((), 0.5, device=dev, dtype=dt).expand(full.shape))):
            y, grads = _run(x, lin, "gelu", res, dy)
            assert y.is_contiguous() and y.shape == full.shape and grads[0].shape == x.shape
            _check(x, lin.weight, lin.bias, res, "gelu", dy, y, grads)
    lin.weight = nn.Parameter(torch.randn(64, 72, device=dev).to(dt).t())
    x, dy = torch.randn(20, 64, device=dev).to(dt), torch.randn(20, 72, device=dev).to(dt)
    y, grads = _run(x, lin, "none", None, dy)
    _check(x, lin.weight, lin.bias, None, "none", dy, y, grads)


@pytest.mark.parametrize("dt", TYPES)
def test_nan_and_infinity_stay_where_they_belong(gpu_device, dt):
    """A row of x that is not finite makes its row of y so and no other; a row of dy its row of dx."""
    x, lin, res, dy = _make(gpu_device, dt, 140, 96, 136, seed=4)
    y0, (dx0, _, _) = _run(x, lin, "gelu", res, dy)
    x[5, 3], x[77, 95], x[139, 0] = float("nan"), float("inf"), float("-inf")
    dy[9, 1] = float("inf")
    y, (dx, _, _) = _run(x, lin, "gelu", res, dy)
    keep = torch.ones(140, dtype=torch.bool, device=gpu_device)
    keep[[5, 77, 139]] = False
    assert torch.equal(y[keep], y0[keep])
    assert not y[[5, 139]].isfinite().all(1).any() and not y[77].isfinite().all()
    keep[9] = False
    assert torch.equal(dx[keep], dx0[keep]) and not dx[9].isfinite().all()


def test_quiet_rows_keep_their_digits(gpu_device):
    """fp32: frames 2^-30 of the loudest, features 2^-20 of the others: each row of y, row of dx and row and column of dW
    is as exact as the bounds say relative to its own terms."""
    x, lin, res, dy = _make(gpu_device, torch.float32, 200, 160, 96, residual=False, seed=5)
    x[1::2] *= 2.0 ** -30
    with torch.no_grad():
        lin.weight[::3] *= 2.0 ** -20
        lin.bias.zero_()
    dy[:, ::5] *= 2.0 ** -24
    y, grads = _run(x, lin, "none", None, dy)
    _check(x, lin.weight, lin.bias, None, "none", dy, y, grads)


def test_magnitudes_at_the_ends_of_fp32(gpu_device):
    x, lin, _, dy = _make(gpu_device, torch.float32, 40, 64, 48, residual=False, seed=6)
    for sx, sw in ((2.0 ** 120, 2.0 ** -100), (2.0 ** -110, 2.0 ** 100), (2.0 ** 60, 2.0 ** 60)):
        with torch.no_grad():
            w = nn.Linear(64, 48, bias=False, device=gpu_device)
            w.weight.copy_(lin.weight * sw)
            y = linear.linear_act(x * sx, w)
        ref = (x * sx).double() @ w.weight.double().t()
        D = ((x * sx).double().abs() @ w.weight.double().abs().t()) * _terms(torch.float32, 64)
        _close(y, ref, D + U * ref.abs(), (sx, sw))
    y, grads = _run(torch.zeros_like(x), lin, "gelu", None, dy)
    assert torch.equal(grads[1], torch.zeros_like(grads[1]))


def test_no_rows(gpu_device):
    lin = nn.Linear(8, 4, device=gpu_device)
    x = torch.zeros(0, 3, 8, device=gpu_device, requires_grad=True)
    y = linear.linear_act(x, lin, nn.GELU())
    dx, dw, db = torch.autograd.grad(y, (x, lin.weight, lin.bias), torch.zeros_like(y))
    assert y.shape == (0, 3, 4) and dx.shape == x.shape and not dw.any() and not db.any()


@pytest.mark.parametrize("dt", TYPES)
def test_only_what_is_asked(gpu_device, dt):
    x, lin, res, dy = _make(gpu_device, dt, 90, 72, 56, seed=7)
    _, ref = _run(x, lin, "silu", res, dy)
    for want in range(1, 16):
        xs, rs = x.clone().requires_grad_(bool(want & 1)), res.clone().requires_grad_(bool(want & 8))
        lin.weight.requires_grad_(bool(want & 2))
        lin.bias.requires_grad_(bool(want & 4))
        y = linear.linear_act(xs, lin, ACTS["silu"], rs)
        of = [(t, r) for t, r in ((xs, ref[0]), (lin.weight, ref[1]), (lin.bias, ref[2]), (rs, dy)) if t.requires_grad]
        for got, (_, r) in zip(torch.autograd.grad(y, [t for t, _ in of], dy), of):
            assert torch.equal(got, r)


@pytest.mark.parametrize("dt", TYPES)
def test_bits_repeat(gpu_device, dt):
    x, lin, res, dy = _make(gpu_device, dt, 3000, 264, 200, seed=8)
    a, b = _run(x, lin, "gelu", res, dy), _run(x, lin, "gelu", res, dy)
    assert torch.equal(a[0], b[0]) and all(torch.equal(p, q) for p, q in zip(a[1], b[1]))


def test_gradient_against_differences(gpu_device):
    """Directional differences of the fp32 forward, t = 2^-7: t^2 / 6 times a third derivative of order one is below 1e-4 and
    rounding 2^-21 / t below 1e-4 of |gradient| |direction|."""
    x, lin, res, dy = _make(gpu_device, torch.float32, 12, 100, 60, seed=9)
    _, (dx, dw, db) = _run(x, lin, "gelu_tanh", res, dy)
    t = 2.0 ** -7
    for p, g in ((x, dx), (lin.weight, dw), (lin.bias, db)):
        v = torch.randn_like(p)
        L = []
        with torch.no_grad():
            keep = p.clone()
            for s in (t, -t):
                p.copy_(keep + s * v)
                L.append((linear.linear_act(x, lin, ACTS["gelu_tanh"], res).double() * dy.double()).sum().item())
            p.copy_(keep)
        assert abs((L[0] - L[1]) / (2 * t) - (g.double() * v.double()).sum().item()) < 5e-4 * (g.norm() * v.norm()).item()


@pytest.mark.parametrize("dt", TYPES)
def test_graph_replays_and_other_stream(gpu_device, dt):
    """Two graphs with workspaces of their own and the eager call in turn: every replay gives the eager bits."""
    x, lin, res, dy = _make(gpu_device, dt, 403, 514, 130, seed=10)
    x.requires_grad_(True)
    res.requires_grad_(True)

    def step():
        y = linear.linear_act(x, lin, ACTS["gelu"], res)
        return (y, *torch.autograd.grad(y, (x, lin.weight, lin.bias, res), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(other, step()))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device=gpu_device))
            dy.copy_(torch.randn(dy.shape, device=gpu_device))
        for g, _ in graphs:
            g.replay()
        eager = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, eager)), k


def test_offsets_past_32_bits(gpu_device):
    """More than 2^31 outputs: the far rows are as the first ones, dW counts both."""
    n, k = 8192, 16
    m = (1 << 31) // n + 300
    x = torch.zeros(m, k, device=gpu_device, dtype=torch.bfloat16)
    x[:200].normal_()
    x[-200:] = x[:200]
    lin = nn.Linear(k, n, device=gpu_device, dtype=torch.bfloat16)
    x.requires_grad_(True)
    y = linear.linear_act(x, lin, nn.GELU())
    assert torch.equal(y[-200:], y[:200])
    dy = torch.zeros_like(y)
    dy[:200] = y.detach()[:200]
    dy[-200:] = dy[:200]
    del y
    y = linear.linear_act(x, lin, nn.GELU())
    dx, dw = torch.autograd.grad(y, (x, lin.weight), dy)
    assert torch.equal(dx[-200:], dx[:200]) and dx[:200].abs().sum() > 0 and not dx[200:-200].any()
    xs = x.detach()[:200].clone().requires_grad_(True)
    (half,) = torch.autograd.grad(linear.linear_act(xs, lin, nn.GELU()), (lin.weight,), dy[:200].contiguous())
    # the same 200 rows twice, in two other orders of addition: 2^-8 for either rounding, and the sums' 2 * 400 u of sum |g x|
    far = (dw.double() - 2 * half.double()).abs() - 2.0 ** -7 * dw.double().abs()
    assert (far <= 1e-4 * dw.double().abs().max()).all()


def test_refusals_on_the_gpu(gpu_device):
    lin = nn.Linear(8, 4, device=gpu_device)
    x = torch.randn(3, 8, device=gpu_device)
    with pytest.raises(RuntimeError, match="on one GPU"):
        linear.linear_act(x, nn.Linear(8, 4))
    with pytest.raises(RuntimeError, match="throughout"):
        linear.linear_act(x.half(), lin)
    with pytest.raises(RuntimeError, match="throughout"):
        linear.linear_act(x.double(), nn.Linear(8, 4, device=gpu_device).double())
    with pytest.raises(RuntimeError, match="input"):
        linear.linear_act(torch.randn(3, 9, device=gpu_device), lin)
    with pytest.raises(RuntimeError, match="not broadcast"):
        linear.linear_act(x, lin, None, torch.randn(4, device=gpu_device))
    y = linear.linear_act(x.requires_grad_(True), lin, nn.GELU())
    (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):   # once differentiable
        dx.sum().backward()


# ------------------------------------------------------------------ fp32 in both its forms
# Small products multiply fp32 as it lies, large ones the hi and lo halves of a laid-out copy: sizes of either side of the rule.
FORMS = [(2500, 1030, 1030), (1500, 2050, 1026), (700, 1030, 130)]


@pytest.mark.parametrize("m,k,n", FORMS)
@pytest.mark.parametrize("act", ("none", "silu"))
def test_fp32_forms(gpu_device, m, k, n, act):
    x, lin, res, dy = _make(gpu_device, torch.float32, m, k, n, seed=11)
    d = N.LinearDesc(m, n, k, 0, 0, k, k, n)
    need = N.lib().se_linear_fwd_workspace_size(ctypes.byref(d), ctypes.c_void_p(256), ctypes.c_void_p(256))
    # as it lies: no workspace, or a slab of sums for each part of a split K and nothing else
    slabs = {-(-4 * parts * m * n // 256) * 256 for parts in (0, *range(2, 65))}
    assert (need in slabs) == (m < 1000)
    y, grads = _run(x, lin, act, res, dy)
    _check(x, lin.weight, lin.bias, res, act, dy, y, grads)
    again = _run(x, lin, act, res, dy)
    assert torch.equal(y, again[0]) and all(torch.equal(a, b) for a, b in zip(grads, again[1]))


@pytest.mark.parametrize("m,k,n", FORMS)
def test_fp32_forms_keep_rows_apart(gpu_device, m, k, n):
    """As the two tests above it of small sizes: what is not finite stays in its row, quiet rows and columns keep their digits."""
    x, lin, _, dy = _make(gpu_device, torch.float32, m, k, n, residual=False, seed=12)
    x[1::2] *= 2.0 ** -30
    with torch.no_grad():
        lin.weight[::3] *= 2.0 ** -20
        lin.bias.zero_()
    dy[:, ::5] *= 2.0 ** -24
    y, grads = _run(x, lin, "none", None, dy)
    _check(x, lin.weight, lin.bias, None, "none", dy, y, grads)
    x[5, 3], x[77, k - 1], x[m - 1, 0] = float("nan"), float("inf"), float("-inf")
    dy[9, 1] = float("inf")
    z, bad = _run(x, lin, "none", None, dy)
    keep = torch.ones(m, dtype=torch.bool, device=gpu_device)
    keep[[5, 77, m - 1]] = False
    assert torch.equal(z[keep], y[keep]) and not z[[5, m - 1]].isfinite().all(1).any() and not z[77].isfinite().all()
    keep[:] = True
    keep[9] = False
    assert torch.equal(bad[0][keep], grads[0][keep]) and not bad[0][9].isfinite().all()


def test_fp32_as_it_lies_off_16_bytes(gpu_device):
    """Rows, columns and starts off the vector loads' alignment, odd sizes, K in the last eight of a step."""
    torch.manual_seed(13)
    base = torch.randn(90, 140, device=gpu_device)
    for k in (31, 32, 33, 39, 40, 41, 63, 65):
        for off in (0, 1, 4):
            x = base[:, off:off + k]
            lin = nn.Linear(k, 67, device=gpu_device)
            dy = torch.randn(90, 67, device=gpu_device)
            y, grads = _run(x, lin, "gelu", None, dy)
            _check(x, lin.weight, lin.bias, None, "gelu", dy, y, grads)


def test_fp32_halves_in_a_graph(gpu_device):
    """The large form's launches captured and replayed, with eager calls between: every replay gives the eager bits."""
    x, lin, res, dy = _make(gpu_device, torch.float32, *FORMS[1], seed=14)
    x.requires_grad_(True)

    def step():
        y = linear.linear_act(x, lin, ACTS["gelu"], res)
        return (y, *torch.autograd.grad(y, (x, lin.weight, lin.bias), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device=gpu_device) * 2.0 ** (8 * k - 16))
            dy.copy_(torch.randn(dy.shape, device=gpu_device) * 2.0 ** (-6 * k))
        g.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), k
