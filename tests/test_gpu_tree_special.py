"""Infinities and NaN in V, among the last cached keys and the tree's own, in every layout of the tree attention: they reach the
tokens that see them, in their own dimension, and no others."""

import numpy as np
import pytest
import torch

from helpers import say
from test_gpu_tree import BF, HF, Case
from tree_checks import same_attention

pytestmark = pytest.mark.gpu

# nodes of a row at four query heads a key head: query rows of 16, 32, 64 and 128 to a tile, and several tiles of 128
NODES = [3, 7, 12, 16, 30, 45]


def plant(c, cached, value, last=64):
    """V of the last cached keys and of the row's own: key i's is value in dimension i of every head."""
    for b, (before, n) in enumerate(zip(cached, c.nodes)):
        for key in range(max(0, before - last), before + n):
            c.cache[c.ids[c.kvp[b] + key // c.page], 1, key % c.page, :, key % c.cache.shape[-1]] = value


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("nodes", NODES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_special_values_of_v(gpu, value, nodes, dim, dtype):
    """Trees that begin on both sides of the edges of 32 and of 64 keys."""
    for cached in ([100], [63], [64], [65], [95], [96], [127, 340], [161, 31]):
        say("tree attention special V", value, nodes, dim, dtype, cached)
        c = Case(gpu, cached, [nodes] * len(cached), 8, 2, dim, dtype=dtype, seed=cached[0])
        plant(c, cached, value)
        same_attention(c, *c.run())


@pytest.mark.parametrize("nodes", NODES)
def test_special_values_of_v_in_long_rows(gpu, nodes):
    """Rows whose keys fall to several workgroups, one value in sixty of each kind."""
    say("tree attention special V, long rows", nodes)
    cached = [1500, 700, 2100]
    c = Case(gpu, cached, [nodes, max(1, nodes - 2), nodes], 8, 2, 128, seed=nodes)
    plant(c, cached, float("nan"), last=40)
    r = np.random.default_rng(nodes)
    for b, before in enumerate(cached):  # each in a dimension of its own sign: no infinities of both signs in a sum
        for key in r.integers(0, before, size=20).tolist():
            at = c.cache[c.ids[c.kvp[b] + key // 16], 1, key % 16]
            at[:, key % 64] = float("inf")
            at[:, 64 + key % 64] = float("-inf")
    same_attention(c, *c.run())
