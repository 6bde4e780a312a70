"""Outputs of the tree attention that would meet its inputs, or each other, are refused."""

import pytest
import torch

from helpers import say
from test_gpu_tree import BF, Case

pytestmark = pytest.mark.gpu


def test_lse_apart_from_the_rest(gpu):
    say("tree attention lse overlap")
    c = Case(gpu, [20], [4], 8, 2, 128)
    as_lse = lambda t: t.view(torch.float32).flatten()[:32].view(4, 8)
    whole = torch.zeros(4 * 8 * 128 + 64, dtype=BF, device=gpu)
    out = whole[: 4 * 8 * 128].view(4, 8, 128)
    with pytest.raises(ValueError, match="apart"):
        c.run(out=out, lse=as_lse(out))
    with pytest.raises(ValueError, match="apart"):
        c.run(lse=as_lse(c.cache))
    q = c.q
    c.q = c.q.contiguous()
    with pytest.raises(ValueError, match="apart"):
        c.run(lse=as_lse(c.q))
    c.q = q
    want = [t.clone() for t in c.run()]
    got = c.run(out=out, lse=whole[4 * 8 * 128 :].view(torch.float32).view(4, 8))  # right behind each other
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
