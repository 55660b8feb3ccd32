"""linear_act where the rule takes the 256 x 256 tile: y, dx and dW in each type against the formula in 64 bits, with sizes
off the tile in every direction, rows of 8, 2 and 1 columns an access, an odd number of k steps, with and without a split of
the reduced length. Which tile a size gets is asked of the library, so that a change of the rule cannot leave these
sizes to another kernel unnoticed."""
import ctypes

import pytest
import torch

from sehip import _native as N
from sehip import linear
from test_gpu_linear_act import ACTS, _check, _make, _run

pytestmark = pytest.mark.gpu
TYPES = (torch.float32, torch.bfloat16, torch.float16)
Y, DX, DW = range(3)


def _tile(dt, m, k, n, product, act="gelu"):
    splits = ctypes.c_int()
    code = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}[act]
    d = N.LinearDesc(m, n, k, code, N.DTYPES[dt], k, k, n)
    tile = N.lib().se_linear_tile(ctypes.byref(d), product, ctypes.byref(splits))
    return tile, splits.value


# (product, m, k, n, whether the reduced length is split): the row length of what is written is n (y) or k (dx, dW)
SIZES = [(Y, 9056, 524, 1288, False), (Y, 11356, 536, 1036, False), (Y, 8297, 514, 1467, False), (Y, 390, 3856, 8536, True),
         (Y, 395, 3814, 8790, True), (Y, 8280, 3760, 435, True),
         (DX, 3336, 3632, 515, False), (DX, 1685, 6990, 568, False), (DX, 10142, 1249, 523, False), (DX, 8526, 392, 3855, True),
         (DX, 520, 6538, 3832, True), (DX, 8298, 385, 3384, True),
         (DW, 520, 11248, 1080, False), (DW, 522, 4070, 3126, False), (DW, 523, 11027, 1040, False), (DW, 4125, 536, 6560, True),
         (DW, 4071, 8346, 400, True), (DW, 3898, 8553, 404, True)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("product,m,k,n,split", SIZES)
def test_large_tiles(gpu_device, dt, product, m, k, n, split):
    act = ("gelu", "silu", "none", "gelu_tanh", "relu")[(m + k + n) % 5]
    tile, splits = _tile(dt, m, k, n, product, act)
    assert tile == 256 and (splits > 1) == split, (tile, splits)
    for residual in ((True, False) if product == Y else (False,)):
        x, lin, res, dy = _make(gpu_device, dt, m, k, n, residual=residual, seed=21)
        y, grads = _run(x, lin, act, res, dy)
        _check(x, lin.weight, lin.bias, res, act, dy, y, grads)
        with torch.no_grad():
            assert torch.equal(linear.linear_act(x, lin, ACTS[act], res), y)


@pytest.mark.parametrize("dt", TYPES)
def test_bits_repeat_and_rows_stay_apart(gpu_device, dt):
    """As of the small tile: the same bits every time; what is not finite stays in its row of y and of dx."""
    m, k, n = 9056, 524, 1288
    assert _tile(dt, m, k, n, Y) == (256, 1)
    x, lin, res, dy = _make(gpu_device, dt, m, k, n, seed=22)
    a, b = _run(x, lin, "gelu", res, dy), _run(x, lin, "gelu", res, dy)
    assert torch.equal(a[0], b[0]) and all(torch.equal(p, q) for p, q in zip(a[1], b[1]))
    x[5, 3], x[777, k - 1], x[m - 1, 0] = float("nan"), float("inf"), float("-inf")
    y, _ = _run(x, lin, "gelu", res, dy)
    keep = torch.ones(m, dtype=torch.bool, device=gpu_device)
    keep[[5, 777, m - 1]] = False
    assert torch.equal(y[keep], a[0][keep])
    assert not y[[5, m - 1]].isfinite().all(1).any() and not y[777].isfinite().all()
