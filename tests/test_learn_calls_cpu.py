"""Calls of the operators that learn which have to be refused before any kernel runs, or answered without one."""
import ctypes

import pytest
import torch

from tesm_amd import _lib
from test_learn_ops_cpu import _refused


def _pair(act, z, z_up):
    return _lib.Dense(0, act, 4, 8, 16, 1 << 20, 8, 1 << 21, 8, 1 << 22, 8, None, None, 0, None, 0, z, z_up)


@pytest.mark.parametrize("z,z_up", [(None, None), (1 << 23, 1 << 24)])
def test_a_pair_without_an_activation_has_no_backward_pass(z, z_up):
    """Its kernel reads what the forward call kept, which that refuses to make."""
    b = _lib.DenseGrad(_pair(0, z, z_up), 1 << 25, 16, 1 << 26, None, None, None)
    assert "activation" in _refused("tesm_hip_dense_backward", ctypes.byref(b), None, 0, None)
