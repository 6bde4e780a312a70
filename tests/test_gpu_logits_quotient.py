"""A positive logit of a repeated token is its quotient by the repetition penalty, rounded once."""

import numpy as np
import pytest
import torch

from aspire_amd.logits_processor import adjust_logits
from helpers import say
from tree_checks import within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,times", [(7, 1), (30011, 1), (333, 100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quotients(gpu, dtype, vocab, times):
    """Every token is in the prompt: x / r for positive x, else x * r, to the last bit."""
    say("logits quotients", dtype, vocab)
    r = np.random.default_rng(vocab)
    rep = np.tile(np.float32([1.3, 3.0, 0.7, 1.1, 7.0, 1e-3]), times)
    n = len(rep)
    x = torch.from_numpy(r.normal(scale=4, size=(n, vocab)).astype(np.float32)).to(dtype)
    history = torch.arange(vocab, dtype=torch.int32).repeat(n, 1).to(gpu)
    lens = torch.full((n,), vocab, dtype=torch.int32, device=gpu)
    got = adjust_logits(x.to(gpu), history=history, history_lens=lens, prompt_lens=lens, repetition=torch.from_numpy(rep).to(gpu))
    y = x.float().numpy()
    want = np.where(y > 0, y / rep[:, None], y * rep[:, None]).astype(np.float32)
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype))


@pytest.mark.parametrize("times", [1, 29])  # one vector of logits a thread, and two (512 chunks and more)
def test_far_penalties(gpu, times):
    """Penalties from the least to the largest value, zero and infinity with values of all sizes: the quotient to the last bit, but for one
    below the normal numbers, which is rounded twice (2^-149 there)."""
    say("logits quotients, far")
    inf = float("inf")
    rep = np.float32([2.0 ** -130, 2.0 ** -149, 2.0 ** 127, 3e38, 1.3, 1.0, 1.7 * 2.0 ** -50, 1.3 * 2.0 ** 59, 2.0 ** -126, 1.7 * 2.0 ** -120, 2.0 ** 126,
                      1.3 * 2.0 ** 100, 1.1 * 2.0 ** -60, 1.9 * 2.0 ** -61, 1.1 * 2.0 ** 60, 1.9 * 2.0 ** 59, 1.9 * 2.0 ** -121, 1.3 * 2.0 ** -140, 0.0, inf])
    x = np.float32([2.0 ** -20, 0.0, -1.0, 2.0 ** -126, 2.0 ** -30, -3.0, 2.0 ** -140, 2.0 ** 120, -0.0, -(2.0 ** -10), 3.0, 3e38, 1e30, inf, -inf, 2.0 ** 100, 2.0 ** 10,
                    2.0 ** -100, 7.0, -3e38, 1e-3, 1.1e-30, 1.3e20, 0.7])
    rep = np.tile(rep, times)
    n, k = len(rep), len(x)
    history = torch.arange(k, dtype=torch.int32).repeat(n, 1).to(gpu)
    lens = torch.full((n,), k, dtype=torch.int32, device=gpu)
    got = adjust_logits(torch.from_numpy(np.tile(x, (n, 1))).to(gpu), history=history, history_lens=lens, prompt_lens=lens, repetition=torch.from_numpy(rep).to(gpu))
    with np.errstate(over="ignore", under="ignore", divide="ignore", invalid="ignore"):
        want = np.where(x > 0, x / rep[:, None], x * rep[:, None])
    assert want.dtype == np.float32
    low = (x > 0) & (np.abs(want) < 2.0 ** -126)
    within(got.cpu().numpy(), want, np.where(low, 2.0 ** -149, 0.0), "quotient")
