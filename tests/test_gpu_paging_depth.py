"""Masks of deep trees: right, and made in one climb of a token's ancestors, whatever the number of words."""

import numpy as np
import pytest
import torch

from aspire_amd.attention.paging import StepTables
from helpers import say
from test_gpu_paging import check_tables
from tree_cases import random_tree

pytestmark = pytest.mark.gpu


def build(gpu, trees, words):
    page = 64
    fresh, cached = [len(t) for t in trees], [(17 * i) % 90 for i in range(len(trees))]
    need = [-(-(c + f) // page) for c, f in zip(cached, fresh)]
    table = torch.arange(len(trees) * max(need), dtype=torch.int32, device=gpu).view(len(trees), -1)
    parents = [p for t in trees for p in t]
    t = StepTables(len(trees), len(parents) + 3, sum(need), page, gpu, tree_words=words)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    args = (table, i32(cached), i32(fresh), i32(parents + [0, 0, 0]))
    if t.masks is not None:
        t.masks.fill_(-1)  # nothing of it may stay
    t.build(*args)
    return t, args, cached, fresh, parents


@pytest.mark.parametrize("words,trees", [
    (64, [list(range(-1, 4095))]),                                       # the longest chain
    (64, [[-1] + [0] * 4000]),                                           # a star
    (3, [list(range(-1, 191)), [-1, 0, 1], list(range(-1, 63))]),
    (5, [[-1] + [max(0, i - 130) for i in range(1, 300)]]),              # every step up passes over two words
    (64, [random_tree(2500, np.random.default_rng(1)), random_tree(70, np.random.default_rng(2))]),
    (2, [[5, -1, 1, 9, 3, 3] + [200] * 90 + [64, 95]]),                  # indices that are no parents
])
def test_masks_of_deep_trees(gpu, words, trees):
    say("deep trees", words, [len(t) for t in trees])
    t, args, cached, fresh, parents = build(gpu, trees, words)
    check_tables(t, args[0], cached, fresh, parents + [0, 0, 0])


def test_words_cost_no_climb_each(gpu):
    """A chain of 4,096 tokens with 64 words takes at most four times as long as without masks (64 climbs took 64 times as long)."""
    say("deep trees, time")
    chain = [list(range(-1, 4095))]

    def ms(words):
        t, args, *_ = build(gpu, chain, words)
        best = float("inf")
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            t.build(*args)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    plain, masked = ms(0), ms(64)
    print(f"{plain:.3f} ms without masks, {masked:.3f} with")
    assert masked < 4 * plain
