"""CPU checks of the cache's whole numbers on their way to the kernels."""

import pytest
import torch

import attnres_ops as ops


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8])
def test_whole_numbers_in_32_bits(dtype):
    """As they are where 32 bits hold them, else the nearest that they hold: what is below zero stays below it for as many
    tokens as it was."""
    i = torch.iinfo(dtype)
    values = [v for v in (-2 ** 63, -2 ** 40, -2 ** 31 - 1, -2 ** 31, -5, -1, 0, 7, 200, 2 ** 31 - 1, 2 ** 31, 2 ** 40) if i.min <= v <= i.max]
    got = ops._int32(torch.tensor(values, dtype=dtype))
    assert got.dtype == torch.int32 and got.tolist() == [max(-2 ** 31, min(2 ** 31 - 1, v)) for v in values]
