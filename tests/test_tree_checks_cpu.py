"""What the comparisons of the tree and logits tests take and what they do not."""

import numpy as np
import pytest
import torch

from tree_cases import adjusted, ancestors, attention, pack
from tree_checks import same_attention, same_logits, within

NAN, INF = float("nan"), float("inf")


def test_within():
    ref = np.array([1.0, -2.0, 0.0, INF, -INF, NAN])
    limit = np.array([0.5, 0.5, 0.0, NAN, INF, 0.0])
    within(ref, ref, limit)
    within([1.5, -2.5, -0.0, INF, -INF, NAN], ref, limit)
    for i, wrong in ((0, 1.6), (0, NAN), (0, INF), (1, -INF), (2, 1e-300), (2, NAN), (3, 1e308), (3, -INF), (3, NAN), (4, INF), (4, 0.0), (5, 0.0), (5, INF)):
        bad = ref.copy()
        bad[i] = wrong
        with pytest.raises(AssertionError):
            within(bad, ref, limit)
    with pytest.raises(AssertionError):
        within([1.0], [1.0], [NAN])  # a limit that is none
    with pytest.raises(AssertionError):
        within([5.0], [1.0], [INF])


class Small:
    """A row that sees two cached keys and its ancestors, one that sees nothing, and a token of no row."""

    def __init__(self):
        r = np.random.default_rng(0)
        self.page, self.qo, self.kvp, self.ids, self.last = 16, [0, 3, 4], [0, 1, 1], [2], [5, 0]
        self.q = torch.from_numpy(r.normal(size=(5, 2, 8))).to(torch.bfloat16)
        self.cache = torch.from_numpy(r.normal(size=(3, 2, 16, 1, 8))).to(torch.bfloat16)
        self.masks = torch.from_numpy(np.concatenate([pack(ancestors([-1, 0, 0]), 1), np.zeros((2, 1), np.int64)]))
        out, lse, _, _ = attention(self.q, self.cache, self.qo, self.kvp, self.ids, self.last, self.masks)
        self.out, self.lse = torch.from_numpy(np.nan_to_num(out)).to(torch.bfloat16), torch.from_numpy(lse).float()


def test_attention_comparison():
    c = Small()
    same_attention(c, c.out, c.lse)
    for t, row, value in (("out", 1, NAN), ("out", 2, INF), ("out", 0, 3.0), ("out", 3, 1e-3), ("out", 3, NAN), ("lse", 0, NAN), ("lse", 1, -INF),
                          ("lse", 2, INF), ("lse", 3, 0.0), ("lse", 3, NAN), ("lse", 1, 9.0)):
        out, lse = c.out.clone(), c.lse.clone()
        (out if t == "out" else lse)[(row, 1, 5) if t == "out" else (row, 1)] = value
        with pytest.raises(AssertionError):
            same_attention(c, out, lse)
    with pytest.raises(AssertionError):
        same_attention(c, torch.full_like(c.out, NAN), torch.full_like(c.lse, NAN))
    out, lse = c.out.clone(), c.lse.clone()
    out[4], lse[4] = NAN, NAN  # of no row: left to the caller
    same_attention(c, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_logits_comparison(dtype):
    x = torch.randn(3, 20, generator=torch.Generator().manual_seed(0)).to(dtype)
    x[0, 3], x[0, 4], x[0, 5] = INF, -INF, NAN
    p = dict(history=np.array([[1, 1, 7], [2, 3, 3]]), lens=[3, 2], rep=np.float32([1.5, 2.0]), freq=np.float32([0.5, 0.25]), qo=[0, 1, 2])
    ref, touched, size = adjusted(x, **p)
    out = torch.from_numpy(ref).to(dtype)
    same_logits(out, ref, touched, size, x)
    for at, value in (((0, 1), NAN), ((0, 1), INF), ((1, 2), 50.0), ((0, 3), 1.0), ((0, 4), NAN), ((0, 5), 0.0), ((2, 0), NAN), ((2, 0), float(x[2, 0]) + 1)):
        bad = out.clone()
        bad[at] = value
        with pytest.raises(AssertionError):
            same_logits(bad, ref, touched, size, x)
    with pytest.raises(AssertionError):
        same_logits(torch.full_like(out, NAN), ref, touched, size, torch.full_like(out, NAN))
    # past the largest value
    big = torch.finfo(dtype).max
    y = torch.full((1, 2), big).to(dtype)
    ref, touched, size = adjusted(y, history=np.array([[0]]), lens=[1], freq=np.float32([-big]))
    same_logits(torch.tensor([[INF, big]]).to(dtype), ref, touched, size, y)
    for wrong in ([-INF, big], [NAN, big], [0.0, big], [INF, NAN]):
        with pytest.raises(AssertionError):
            same_logits(torch.tensor([wrong]).to(dtype), ref, touched, size, y)
