"""A copy of step tables, or of a page pool, writes its own tensors."""

import copy

import pytest
import torch

from aspire_amd.attention.paging import PagePool, StepTables
from helpers import say

pytestmark = pytest.mark.gpu

NAMES = ("qo_indptr", "kv_indptr", "kv_indices", "last_page_len", "positions", "slots", "masks", "totals")


def values(t):
    return [getattr(t, n).tolist() for n in NAMES]


def test_copies_of_tables(gpu):
    say("copies of step tables")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    table = i32([[0, 1], [2, 3]])
    t = StepTables(2, 6, 4, 16, gpu, tree_words=1)
    t.build(table, i32([3, 9]), i32([2, 1]))
    first = values(t)
    other = copy.deepcopy(t)
    other.build(table, i32([20, 0]), i32([3, 3]))
    assert values(t) == first
    fresh = StepTables(2, 6, 4, 16, gpu, tree_words=1)
    fresh.build(table, i32([20, 0]), i32([3, 3]))
    assert values(other) == values(fresh) and values(other) != first


def test_copies_of_pools(gpu):
    say("copies of a page pool")
    pool = PagePool(9, 16, 2, 4, gpu)
    pool.resize(torch.tensor([20, 3], device=gpu))
    other = copy.deepcopy(pool)
    other.resize(torch.tensor([0, 60], device=gpu))
    assert pool.held.tolist() == [2, 1] and other.held.tolist() == [0, 4]
