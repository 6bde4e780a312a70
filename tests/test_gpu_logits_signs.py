"""A logit without an entry in its request's biases keeps its bits, the sign of a zero among them."""

import pytest
import torch

from aspire_amd.logits_processor import LogitBias, adjust_logits
from helpers import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 64, 9003])
def test_zeros_keep_their_sign(gpu, dtype, vocab):
    say("logits signs", dtype, vocab)
    x = torch.zeros(2, vocab, device=gpu).to(dtype)
    x[:, ::2] = -0.0
    x[0, 1], x[0, 2], x[1, 3] = float("inf"), float("-inf"), 1.0
    want = x.clone()
    want[0, 4], want[1, 4] = 1.5, 0.0  # -0 + 0 is 0
    raw = lambda t: t.view(torch.int32 if dtype == torch.float32 else torch.int16)
    out = adjust_logits(x, bias=LogitBias([{4: 1.5}, {4: 0.0}], gpu))
    assert torch.equal(raw(out), raw(want))
    one = torch.ones(2, device=gpu)
    history, lens = torch.full((2, 1), vocab, dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    out = adjust_logits(x, bias=LogitBias([{4: 1.5}, {4: 0.0}], gpu), history=history, history_lens=lens, presence=one)
    assert torch.equal(raw(out), raw(want))
