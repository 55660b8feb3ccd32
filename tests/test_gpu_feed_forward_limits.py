"""The feed-forward operators' calls at the edges of what their documentation allows, each against its formula or refused."""
import pytest
import torch
import torch.nn as nn

from sehip import linear, norm, optim

pytestmark = pytest.mark.gpu


def test_sizes_that_a_c_int_does_not_hold(gpu_device):
    """Refused before anything of that size is made (the inputs are one element, expanded)."""
    one = torch.ones((), device=gpu_device, dtype=torch.bfloat16)
    free = torch.cuda.mem_get_info()[0]
    with pytest.raises(RuntimeError, match="32-bit"):
        linear.linear_act(one.expand((1 << 32) + 100, 8), nn.Linear(8, 4, device=gpu_device, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="32-bit"):
        norm.layer_norm(nn.LayerNorm((1 << 32) + 8, elementwise_affine=False), one.expand(2, (1 << 32) + 8))
    with pytest.raises(RuntimeError, match="32-bit"):
        norm.layer_norm(nn.LayerNorm((1 << 16, (1 << 16) + 1), elementwise_affine=False), one.expand(2, 1 << 16, (1 << 16) + 1))
    assert free - torch.cuda.mem_get_info()[0] < 1 << 28
