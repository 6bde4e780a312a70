"""Tree attention, the moves and the logits are not differentiable: whatever of a call asks for a derivative, or carries one, is
refused, so that none is dropped."""

import pytest
import torch
from torch.autograd import forward_ad

from aspire_amd.attention.tree import compact_accepted, tree_attention
from aspire_amd.logits_processor import LogitBias, adjust_logits
from helpers import say
from test_gpu_tree import Case

pytestmark = pytest.mark.gpu


def each_is_refused(call, floats):
    """call with one of its floating tensors after the other asking for a gradient, then carrying a tangent; not under no_grad."""
    call(**floats)
    for name, t in floats.items():
        leaf = t.detach().clone().requires_grad_()
        with pytest.raises(ValueError, match="not differentiable"):
            call(**{**floats, name: leaf})
        with torch.no_grad():
            call(**{**floats, name: leaf})
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t.detach().clone(), torch.ones_like(t))
            with pytest.raises(ValueError, match="not differentiable"):
                call(**{**floats, name: dual})


def test_tree_attention(gpu):
    say("tree attention derivatives")
    c = Case(gpu, [20], [4], 8, 2, 128)
    lists = (c.dev(c.qo), c.dev(c.ids), c.dev(c.kvp), c.dev(c.last), c.masks, 16)
    each_is_refused(lambda q, kv_cache, out, lse: tree_attention(q, kv_cache, *lists, out=out, lse=lse),
                    dict(q=c.q, kv_cache=c.cache, out=torch.empty(c.q.shape, dtype=c.q.dtype, device=gpu), lse=torch.empty(4, 8, device=gpu)))


def test_logits(gpu):
    say("logits derivatives")
    x = torch.randn(3, 50, device=gpu)
    history, lens = torch.zeros(3, 4, dtype=torch.int32, device=gpu), torch.full((3,), 4, dtype=torch.int32, device=gpu)
    bias = LogitBias([{1: 2.0}, {}, {3: 1.0}], gpu)

    def call(values, **kw):
        bias.values = values
        adjust_logits(history=history, history_lens=lens, bias=bias, **kw)

    one = torch.ones(3, device=gpu)
    each_is_refused(call, dict(logits=x, out=torch.empty_like(x), repetition=one, presence=one, frequency=one, values=bias.values))


def test_moves(gpu):
    say("compact derivatives")
    i = lambda n: torch.zeros(n, dtype=torch.int32, device=gpu)
    where = (i(4).view(2, 2), i(2), i(3), torch.zeros(4, dtype=torch.int64, device=gpu))
    cache = torch.zeros(3, 2, 16, 2, 8, device=gpu)
    each_is_refused(lambda a: compact_accepted(a, *where), dict(a=cache))
    each_is_refused(lambda a, b: compact_accepted([a, b], *where), dict(a=cache, b=cache.clone()))
