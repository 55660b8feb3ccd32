"""Layer norm, the product with its epilogue and the AdamW step with 8- or 32-bit states: what they refuse, and
the host-side parts, without a GPU."""
import ctypes

import pytest
import torch
import torch.nn as nn

from sehip import _native as N
from sehip import glue, linear, norm, optim


def test_layer_norm_refusals():
    m = nn.LayerNorm(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        norm.layer_norm(m, torch.zeros(3, 8))
    with pytest.raises(RuntimeError, match="does not end in"):
        norm.layer_norm(m, torch.zeros(3, 9))
    with pytest.raises(RuntimeError, match="does not end in"):
        norm.layer_norm(nn.LayerNorm((4, 8)), torch.zeros(8))


def test_layer_norm_c_arguments():
    lib = N.lib()
    p = ctypes.c_void_p(256)   # never read: every call returns before a launch
    f = lib.se_layer_norm_fwd
    assert f(p, 8, 4, 0, None, None, 1e-5, p, None, 0, 0, None) == -1
    assert f(p, 8, 0, 8, None, None, 1e-5, p, None, 0, 0, None) == -1
    assert f(p, 4, 4, 8, None, None, 1e-5, p, None, 0, 0, None) == -1     # rows would overlap
    assert f(None, 8, 4, 8, None, None, 1e-5, p, None, 0, 0, None) == -1
    assert f(p, 8, 4, 8, None, None, 1e-5, p, None, 3, 3, None) == -1     # no such type
    assert f(p, 8, 4, 8, None, None, 1e-5, p, None, 0, 1, None) == -1     # bf16 weights beside fp32
    need = lib.se_layer_norm_workspace_size(4, 8)
    assert need > 0 and lib.se_layer_norm_workspace_size(0, 8) == 0
    b = lib.se_layer_norm_bwd
    assert b(p, 8, p, 8, 4, 8, None, p, p, p, p, 0, 0, p, need - 1, None) == -5
    assert b(p, 8, p, 8, 4, 8, None, p, None, None, None, 0, 0, p, need, None) == -1
    assert b(p, 8, p, 8, 4, 8, None, None, p, None, None, 0, 0, None, 0, None) == -1
    assert b(p, 0, p, 8, 4, 8, None, p, p, None, None, 0, 0, None, 0, None) == -1


def test_linear_act_refusals():
    m = nn.Linear(8, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear.linear_act(torch.zeros(3, 8), m)
    for act in (nn.Tanh(), nn.ReLU6(), nn.PReLU(), "gelu"):
        with pytest.raises(NotImplementedError, match="activation"):
            linear.linear_act(torch.zeros(3, 8), m, act)


def test_linear_c_arguments():
    lib = N.lib()
    p = ctypes.c_void_p(256)
    D = N.LinearDesc

    def fwd(d, ws=0, z=None):
        return lib.se_linear_fwd(ctypes.byref(d), p, p, None, None, p, z, None, ws, None)

    assert fwd(D(0, 4, 8, 0, 0, 8, 8, 4)) == -1
    assert fwd(D(3, 4, 8, 9, 0, 8, 8, 4)) == -1        # no such activation
    assert fwd(D(3, 4, 8, 0, 7, 8, 8, 4)) == -1        # no such type
    assert fwd(D(3, 4, 8, 0, 1, 4, 8, 4)) == -1        # rows of x would overlap
    assert fwd(D(3, 4, 8, 0, 1, 8, 4, 4)) == -1        # rows of W would
    assert fwd(D(3, 4, 1 << 22, 0, 1, 1 << 22, 1 << 22, 4)) == -3
    d = D(2500, 1030, 1030, 0, 0, 1030, 1030, 1030)
    need = lib.se_linear_fwd_workspace_size(ctypes.byref(d), p, p)
    assert need > 0                                     # fp32: the planes
    assert fwd(d, need - 1) == -5
    # a small product multiplies fp32 as it lies
    assert lib.se_linear_fwd_workspace_size(ctypes.byref(D(70, 4, 8, 0, 0, 8, 8, 4)), p, p) == 0
    assert lib.se_linear_fwd_workspace_size(ctypes.byref(D(0, 4, 8, 0, 0, 8, 8, 4)), p, p) == 0
    # bf16 on 16 bytes reads x and W as they lie; a row off 16 bytes is packed
    assert lib.se_linear_fwd_workspace_size(ctypes.byref(D(70, 4, 8, 0, 1, 8, 8, 4)), p, p) == 0
    assert lib.se_linear_fwd_workspace_size(ctypes.byref(D(70, 4, 7, 0, 1, 7, 7, 4)), p, p) > 0
    # few rows never need one
    for dt in range(3):
        assert lib.se_linear_fwd_workspace_size(ctypes.byref(D(64, 4, 7, 0, dt, 7, 7, 4)), p, p) == 0
    d = D(70, 4, 8, 2, 1, 8, 8, 4)
    bwd = lib.se_linear_bwd
    assert bwd(ctypes.byref(d), p, p, p, None, p, None, None, None, 0, None) == -1   # the slope needs z
    assert bwd(ctypes.byref(d), p, p, p, p, None, None, None, None, 0, None) == -1   # nothing wanted
    assert bwd(ctypes.byref(d), p, p, p, p, p, p, p, None, 0, None) == -5


@pytest.mark.parametrize("m,n,k", [((1 << 28) + 1, 4, 8), ((1 << 31) - 1, 1, 1), (1 << 28, 1 << 10, 8),
                                   (1 << 28, 8, 1 << 10), (70, 1 << 21, 1 << 17)])
def test_linear_sizes_behind_32_bits(m, n, k):
    """Refused before anything is launched: row indexes are 32-bit and a launch has less than 2^32 threads."""
    lib = N.lib()
    p = ctypes.c_void_p(256)
    for dt in range(3):
        d = N.LinearDesc(m, n, k, 0, dt, k, k, n)
        assert lib.se_linear_fwd(ctypes.byref(d), p, p, None, None, p, None, None, 0, None) == -3
        assert lib.se_linear_bwd(ctypes.byref(d), p, p, p, None, p, p, p, None, 0, None) == -3
        assert lib.se_linear_fwd_workspace_size(ctypes.byref(d), p, p) == 0
        assert lib.se_linear_bwd_workspace_size(ctypes.byref(d), p, p, p, 1, 1, 1) == 0


def _lists(n=(5,), **over):
    def codes(k, t):
        return torch.zeros(k, dtype=torch.uint8).view(t)
    c = {"params": [torch.zeros(k) for k in n], "grads": [torch.zeros(k) for k in n],
         "exp_avgs": [codes(k, torch.float8_e4m3fn) for k in n],
         "exp_avg_scales": [codes(-(-k // 128), torch.float8_e8m0fnu) for k in n],
         "roots": [codes(k, torch.float8_e4m3fn) for k in n],
         "root_scales": [codes(-(-k // 128), torch.float8_e8m0fnu) for k in n]}
    return {**c, **over}


def test_adamw_refusals():
    with pytest.raises(RuntimeError, match="no CPU path"):
        optim.adamw8_(**_lists(), step=1)
    with pytest.raises(ValueError, match="step 0"):
        optim.adamw8_(**_lists(), step=0)
    with pytest.raises(ValueError, match="betas"):
        optim.adamw8_(**_lists(), step=1, betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="different lengths"):
        optim.adamw8_(**_lists(grads=[]), step=1)
    optim.adamw8_([], [], [], [], [], [], step=1)
    optim.adamw32_([], [], [], [], step=1)
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([nn.Parameter(torch.zeros(3))], state_bits=4)


def test_adamw_c_arguments():
    lib = N.lib()
    row = (ctypes.c_ulonglong * 7)(256, 256, 256, 256, 0, 0, 10)
    kw = (1e-3, 0.9, 0.999, 1e-8, 1e-2)
    f = lib.se_adamw_multi
    assert f(row, 1, 0, 8, *kw, 1, 0, None) == -1      # no scales
    assert f(row, 1, 0, 16, *kw, 1, 0, None) == -1
    assert f(row, 1, 5, 32, *kw, 1, 0, None) == -1
    assert f(row, 1, 0, 32, *kw, 0, 0, None) == -1     # steps count from 1
    assert f(row, 1, 0, 32, 1e-3, 1.0, 0.999, 1e-8, 1e-2, 1, 0, None) == -1
    assert f(row, -1, 0, 32, *kw, 1, 0, None) == -1
    assert f(None, 0, 0, 32, *kw, 1, 0, None) == 0     # nothing to do
    empty = (ctypes.c_ulonglong * 7)(0, 0, 0, 0, 0, 0, 0)
    assert f(empty, 1, 0, 8, *kw, 1, 0, None) == 0


def test_adamw_state_dict_keeps_the_types_of_the_states():
    """torch casts a loaded state to its parameter's type; 8- and 32-bit moments keep their own."""
    for bits in (8, 32):
        ps = [nn.Parameter(torch.zeros(7, 40, dtype=torch.bfloat16)), nn.Parameter(torch.zeros(3, dtype=torch.bfloat16))]
        a = optim.AdamW(ps, state_bits=bits, seed=3)
        for p in ps:
            a.state[p] = {"step": torch.tensor(4.0), **optim._state_like(p, bits, torch.zeros)}
            for t in list(a.state[p].values())[1:]:
                t.view(torch.uint8).random_(1, 100)
        sd = a.state_dict()
        b = optim.AdamW([nn.Parameter(torch.zeros_like(p)) for p in ps], state_bits=bits, seed=9)
        b.load_state_dict(sd)
        assert b.param_groups[0]["state_bits"] == bits and b.param_groups[0]["seed"] == 3
        for p, q in zip(ps, b.param_groups[0]["params"]):
            assert float(b.state[q]["step"]) == 4.0
            for k, t in a.state[p].items():
                assert b.state[q][k].dtype == t.dtype and b.state[q][k].shape == t.shape
                assert torch.equal(b.state[q][k].reshape(-1).view(torch.uint8), t.reshape(-1).view(torch.uint8))
                assert b.state[q][k].data_ptr() != t.data_ptr()
        c = optim.AdamW([nn.Parameter(torch.zeros_like(p)) for p in ps], state_bits=40 - bits)
        with pytest.raises(ValueError, match="the loaded state has no") if bits == 32 else pytest.raises(ValueError):
            c.load_state_dict(sd)
    # the plain optimizer is as it was: no new keys in its groups
    assert "state_bits" not in optim.AdamW([nn.Parameter(torch.zeros(3))]).state_dict()["param_groups"][0]


def test_as_rows_strides():
    """Rows at one distance are used as they lie; every other layout would be copied (refused here: no GPU)."""
    base = torch.arange(4 * 6 * 10.0).view(4, 6, 10)
    assert glue.as_rows(base, 10)[1] == 10
    v = base[:, :, 2:9]
    t, ld = glue.as_rows(v, 7)
    assert ld == 10 and t.data_ptr() == v.data_ptr()
    assert glue.as_rows(base[:, 1, :], 10)[1] == 60
    assert glue.as_rows(base[1:2, :, :3], 3)[1] == 10
    assert glue.as_rows(base[:, 2:3, :5], 5)[1] == 60
    assert glue.as_rows(base[0, 0], 10)[1] == 10
    assert glue.as_rows(base[:, ::2], 10)[1] == 20
    for bad in (base.transpose(1, 2), base[:, :5], base[0, 0, ::2], base[0, :1].expand(5, 10),
                torch.as_strided(base, (3, 1, 5, 8), (80, 80, 8, 1))):
        with pytest.raises(RuntimeError, match="GPU only"):
            glue.as_rows(bad, bad.shape[-1])


def _mix(x):
    x = (x ^ (x >> 15)) * 0x6A09E667 & 0xFFFFFFFF
    x = (x ^ (x >> 13)) * 0xBB67AE85 & 0xFFFFFFFF
    return x ^ (x >> 16)


@pytest.mark.parametrize("seed,step,tensor", [(0, 1, 0), (0, 2, 0), (7, 1000, 55), (65535, 3, 1)])
def test_rounding_hash_is_uniform(seed, step, tensor):
    """Both halves of the counter hash that rounds the 8-bit states: every bit set half of the time, 256 bins of the upper
    byte filled evenly, neighbours and the two halves uncorrelated. n = 2^18 draws: a mean's deviation is sigma / 512;
    six sigma for each."""
    n = 1 << 18
    key = _mix(_mix(_mix(seed) + step & 0xFFFFFFFF) + tensor & 0xFFFFFFFF)
    h = _mix((torch.arange(n) * 0x9E3779B1 + key) & 0xFFFFFFFF)
    for b in range(32):
        assert abs(((h >> b) & 1).double().mean().item() - 0.5) < 6 * 0.5 / 512
    lo, hi = (h & 0xFFFF).double() / 65536, (h >> 16).double() / 65536
    for u in (lo, hi):
        bins = torch.histc(u, 256, 0, 1)
        # chi square of 255 degrees: mean 255, deviation sqrt(510)
        chi = ((bins - n / 256) ** 2 / (n / 256)).sum().item()
        assert abs(chi - 255) < 6 * 510 ** 0.5
        for lag in (1, 2, 8, 128, 2048):
            r = ((u[lag:] - 0.5) * (u[:-lag] - 0.5)).mean().item() * 12
            assert abs(r) < 6 / 512, (lag, r)
    assert abs(((lo - 0.5) * (hi - 0.5)).mean().item() * 12) < 6 / 512
