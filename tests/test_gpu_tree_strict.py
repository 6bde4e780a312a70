"""The tree attention's and the logits' tests once more, under comparisons that no NaN passes."""

import numpy as np
import pytest
import torch

import test_gpu_adjust_logits as logits_tests
import test_gpu_tree as tree_tests
import test_gpu_tree_step as step_tests
from test_gpu_adjust_logits import (test_biases_and_masks, test_mask_rows, test_odd_histories, test_penalties, test_trees,  # noqa: F401
                                    test_views)
from test_gpu_tree import (test_any_mask, test_bad_pages_are_not_seen, test_batches, test_few_words, test_heads,  # noqa: F401
                           test_large_and_far_scores, test_many_rows, test_matches_the_chain_kernel, test_pages, test_scale, test_strides)
from test_gpu_tree_step import test_steps_of_trees  # noqa: F401
from helpers import say
from tree_checks import same_attention, same_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    loose = tree_tests.Case.check

    def check(case, out, lse, scale=None):
        with np.errstate(invalid="ignore"):
            loose(case, out, lse, scale)
        same_attention(case, out, lse, scale)

    def finite(*args, **kw):
        out = attend(*args, **kw)
        assert torch.isfinite(out).all()
        return out

    attend = step_tests.tree_attention
    monkeypatch.setattr(tree_tests.Case, "check", check)
    monkeypatch.setattr(step_tests, "tree_attention", finite)
    monkeypatch.setattr(logits_tests, "close", same_logits)


def test_tokens_of_no_row_stay_and_the_others_are_right(gpu):
    say("tree attention padding, strict")
    c = tree_tests.Case(gpu, [20, 33], [4, 9], 8, 2, 128, pad=7)
    out = torch.full(c.q.shape, 7.0, dtype=tree_tests.BF, device=gpu)
    lse = torch.full(c.q.shape[:2], 7.0, device=gpu)
    c.run(out=out, lse=lse)
    assert (out[13:] == 7).all() and (lse[13:] == 7).all()
    same_attention(c, out, lse)
