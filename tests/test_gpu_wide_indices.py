"""int64 counts and indices that int32 does not hold: none of them is taken for its lower half."""

import numpy as np
import pytest
import torch

from aspire_amd.attention.paging import PagePool, StepTables
from aspire_amd.attention.rotary import RotaryConfig, RotaryEmbedding
from aspire_amd.attention.tree import compact_accepted, tree_attention
from aspire_amd.engine.sampling import verify_tree_speculation
from aspire_amd.logits_processor import adjust_logits
from helpers import say
from test_gpu_tree import Case
from tree_cases import Pool, tables
from tree_checks import same_attention

pytestmark = pytest.mark.gpu

FAR = 2 ** 32


def dev(x, gpu, dtype=torch.int64):
    return torch.tensor(x, dtype=dtype, device=gpu)


def test_lengths_of_a_pool(gpu):
    say("wide lengths")
    pool, ref = PagePool(50, 16, 4, 20, gpu), Pool(50, 16, 4, 20)
    for lengths in ([100, 30, 0, 7], [100, FAR, 5, 7], [FAR + 16, 30, 0, 0], [-FAR, -FAR + 40, 64, 1]):
        short = ref.resize([min(max(n, -1), 2 ** 31 - 1) for n in lengths])
        assert pool.resize(dev(lengths, gpu)).tolist() == short
        assert pool.block_table.tolist() == ref.table()


def test_tables(gpu):
    say("wide table counts")
    table = dev(np.arange(12).reshape(3, 4), gpu, torch.int32)
    for cached, fresh in (([FAR, 5, 6], [3, 2, 1]), ([4, 5, 6], [3, FAR + 2, 1]), ([4, -FAR + 5, 6], [3, 2, 1])):
        t = StepTables(3, 20, 12, 16, gpu)
        t.build(table, dev(cached, gpu), dev(fresh, gpu))
        near = lambda x: [min(max(n, -2 ** 31), 2 ** 31 - 1) for n in x]
        ref = tables(table.tolist(), near(cached), near(fresh), None, 16, 3, 20, 12, 0)
        assert t.qo_indptr.tolist() == ref[0] and t.slots.tolist() == ref[5] and t.totals.tolist() == ref[7]
    parents = [-1, 0, FAR, FAR + 1, 1 - FAR] + [0] * 15
    t = StepTables(1, 20, 4, 16, gpu, tree_words=1)
    t.build(table, dev([0], gpu), dev([5], gpu), dev(parents, gpu))
    assert t.positions[:5].tolist() == [0, 1, 0, 0, 0] and t.masks[:5, 0].tolist() == [1, 3, 4, 8, 16]


def test_pages_of_attention(gpu):
    say("wide page ids")
    c = Case(gpu, [70], [5], 4, 2, 128)
    ids = list(c.ids)
    c.ids[1] = 2 ** 31 - 1  # no page of the pool
    ids[1] += FAR
    out, lse = tree_attention(c.q, c.cache, dev(c.qo, gpu), dev(ids, gpu), dev(c.kvp, gpu), dev(c.last, gpu), c.masks, 16, return_lse=True)
    same_attention(c, out, lse)


def test_append_with_rotation(gpu):
    say("wide page ids of an append")
    rotary = RotaryEmbedding(RotaryConfig(head_dim=64, theta=1e4), gpu)
    q, k, v = (torch.randn(3, h, 64, device=gpu).to(torch.bfloat16) for h in (2, 1, 1))
    cache = torch.zeros(4, 2, 16, 1, 64, dtype=torch.bfloat16, device=gpu)
    rotary.append(q, k, v, dev([0, 3], gpu), cache, dev([FAR + 2], gpu), dev([0, 1], gpu), dev([3], gpu), 16)
    assert not cache.any()


def test_paths_moves_and_logits(gpu):
    say("wide parents, counts and lengths")
    out, path, kept = verify_tree_speculation(dev([5, 6, 6], gpu), dev([-1, FAR, 0], gpu), dev([6, 1, 2], gpu), dev([0, 3], gpu), 3)
    assert path.tolist() == [[0, 2, -1]] and kept.tolist() == [2]
    cache = torch.arange(4 * 2 * 16 * 4, device=gpu).view(4, 2, 16, 1, 4).float()
    before = cache.clone()
    compact_accepted(cache, dev([[0, 2]], gpu, torch.int32), dev([2 - FAR], gpu), dev([0, 3], gpu), dev([1, 2, 3], gpu))
    assert torch.equal(cache, before)
    x = torch.zeros(1, 9, device=gpu)
    one = torch.ones(1, device=gpu)
    history = dev([[3, 4, 4]], gpu, torch.int32)
    assert adjust_logits(x, history=history, history_lens=dev([FAR], gpu), presence=one).tolist() == [[0, 0, 0, -1, -1, 0, 0, 0, 0]]
    mask = dev([[0]], gpu, torch.int32)
    assert torch.equal(adjust_logits(x, grammar=mask, grammar_rows=dev([FAR], gpu)), x)
    tree = adjust_logits(x, qo_indptr=dev([0, 1], gpu), tree_tokens=dev([FAR + 3], gpu), tree_masks=dev([[1]], gpu), presence=one)
    assert torch.equal(tree, x)
