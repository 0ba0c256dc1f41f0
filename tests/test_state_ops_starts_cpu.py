"""Starts of packed sequences as the kernels take them."""
import pytest
import torch

from tesm_amd import hip_ops


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_starts_keep_their_order(dtype):
    starts = torch.tensor([0, 3, 3, 70], dtype=dtype)
    got, S = hip_ops._sequences(starts, 1, "op")
    assert got.dtype == torch.int32 and S == 3 and got.tolist() == [0, 3, 3, 70] and got.is_contiguous()
    got, _ = hip_ops._sequences(torch.stack([starts, starts], 1)[:, 0], 1, "op")
    assert got.tolist() == [0, 3, 3, 70] and got.is_contiguous()


def test_starts_past_32_bits_stay_past_the_rows():
    """They count as the rows' end, like every start behind the rows, and as the rows' beginning below zero."""
    got, _ = hip_ops._sequences(torch.tensor([-(1 << 40), -3, 5, (1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 62]), 1, "op")
    assert bool((got[1:] >= got[:-1]).all())
    assert bool((got[:2] < 0).all()) and got[2] == 5 and bool((got[3:] == 2 ** 31 - 1).all())
