"""The feed-forward operators' calls at the edges of what they take: refused or answered on the host, without a GPU."""
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
