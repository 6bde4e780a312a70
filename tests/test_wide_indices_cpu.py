"""Counts and indices that int32 does not hold."""

import torch

from aspire_amd import _lib


def test_indices_beyond_int32_become_its_nearest():
    x = torch.tensor([0, -1, 5, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 3, 2 ** 63 - 1, -2 ** 31, -2 ** 31 - 1, -2 ** 32, -2 ** 63])
    top, low = 2 ** 31 - 1, -2 ** 31
    got = _lib.indices(x)
    assert got.dtype == torch.int32 and got.tolist() == [0, -1, 5, top, top, top, top, top, low, low, low, low]
    assert _lib.indices(x.repeat_interleave(2)[::2]).tolist() == got.tolist()
    same = torch.arange(5, dtype=torch.int32)
    assert _lib.indices(same) is same and _lib.indices(torch.arange(10, dtype=torch.int32)[::2]).is_contiguous()
