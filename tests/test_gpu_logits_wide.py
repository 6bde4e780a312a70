"""Logits of so many chunks (512 and more) that a thread takes two vectors of each."""

import numpy as np
import pytest
import torch

from helpers import say
from test_gpu_adjust_logits import TYPES, call, parts
from test_gpu_tree import ancestors, random_tree
from tree_cases import adjusted
from tree_checks import same_logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests,vocab,history", [(513, 61, 30), (260, 8200, 300), (70, 65543, 900)])
@pytest.mark.parametrize("what", ["penalties", "mask", "penalties+mask", "bias", "bias+mask", "all"])
def test_batches(gpu, dtype, requests, vocab, history, what):
    say("logits of many chunks", dtype, requests, vocab, what)
    r = np.random.default_rng(vocab)
    x = torch.randn(requests, vocab, device=gpu, generator=torch.Generator(device=gpu).manual_seed(vocab)).mul_(4).to(dtype)
    p = parts(gpu, requests, vocab, history, vocab) if "pen" in what or what == "all" else {}
    allowed = r.random((requests, vocab)) < r.random(requests)[:, None] if "mask" in what or what == "all" else None
    bias = [{int(i): float(r.normal() * 9) for i in r.choice(vocab, size=b % 7, replace=False)} for b in range(requests)] \
        if "bias" in what or what == "all" else None
    ref = adjusted(x, **p, bias=bias, allowed=allowed)
    same_logits(call(x, p, gpu, bias=bias, allowed=allowed), *ref, x)
    y = x.clone()
    call(y, p, gpu, bias=bias, allowed=allowed, out=y)
    same_logits(y, *ref, x)


@pytest.mark.parametrize("dtype", TYPES)
def test_trees(gpu, dtype):
    say("logits of trees of many chunks", dtype)
    r = np.random.default_rng(3)
    nodes = [int(n) for n in r.integers(0, 4, size=180)]
    vocab, T = 20011, sum(nodes)
    x = torch.randn(T, vocab, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1)).mul_(3).to(dtype)
    p = parts(gpu, len(nodes), vocab, 40, 5)
    tree = (r.integers(0, 5, size=T) * 4999).astype(np.int32)
    see = np.zeros((T, 64), bool)
    at = 0
    for n in nodes:
        see[at : at + n, :n] = ancestors(random_tree(n, r))
        at += n
    qo = [0, *np.cumsum(nodes).tolist()]
    same_logits(call(x, p, gpu, qo=qo, tree=tree, see=see), *adjusted(x, qo=qo, tree=tree, see=see, **p), x)
