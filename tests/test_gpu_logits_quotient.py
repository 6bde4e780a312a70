"""A positive logit of a repeated token is its quotient by the repetition penalty, rounded once."""

import numpy as np
import pytest
import torch

from aspire_amd.logits_processor import adjust_logits
from helpers import say
from tree_checks import within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [7, 30011])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quotients(gpu, dtype, vocab):
    """Every token is in the prompt: x / r for positive x, else x * r, to the last bit."""
    say("logits quotients", dtype, vocab)
    r = np.random.default_rng(vocab)
    rep = np.float32([1.3, 3.0, 0.7, 1.1, 7.0, 1e-3])
    x = torch.from_numpy(r.normal(scale=4, size=(6, vocab)).astype(np.float32)).to(dtype)
    history = torch.arange(vocab, dtype=torch.int32).repeat(6, 1).to(gpu)
    lens = torch.full((6,), vocab, dtype=torch.int32, device=gpu)
    got = adjust_logits(x.to(gpu), history=history, history_lens=lens, prompt_lens=lens, repetition=torch.from_numpy(rep).to(gpu))
    y = x.float().numpy()
    want = np.where(y > 0, y / rep[:, None], y * rep[:, None]).astype(np.float32)
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype))


def test_far_penalties(gpu):
    """Infinite and far values; penalties past 2^60 and below 2^-60, where the quotient may be off by a step."""
    say("logits quotients, far")
    inf = float("inf")
    rep = np.float32([1.3, 1.0, 1.7 * 2.0 ** -50, 1.3 * 2.0 ** 59, 2.0 ** -126, 1.7 * 2.0 ** -120, 2.0 ** 126, 1.3 * 2.0 ** 100, 0.0, inf])
    x = np.float32([[2.0 ** -20, 0.0, -1.0, inf, -inf, 1e30, 3.0], [3e38, inf, -inf, 2.0 ** -100, 7.0, -3e38, 1e-3]]).reshape(1, 14).repeat(10, 0)
    history = torch.arange(14, dtype=torch.int32).repeat(10, 1).to(gpu)
    lens = torch.full((10,), 14, dtype=torch.int32, device=gpu)
    got = adjust_logits(torch.from_numpy(x).to(gpu), history=history, history_lens=lens, prompt_lens=lens, repetition=torch.from_numpy(rep).to(gpu))
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        want = np.where(x > 0, x / rep[:, None], x * rep[:, None])
    got = got.cpu().numpy()
    assert np.array_equal(got[:4], want[:4])
    within(got[4:], want[4:], np.abs(want[4:].astype(np.float64)) * 2.0 ** -22 + 2.0 ** -149, "quotient")
