"""Calls at the edges of what the drafted trees' operators take: tables with more rows than requests, tokens in front of the first
row, masks without words."""

import numpy as np
import pytest
import torch

from aspire_amd.attention.paging import PagePool, StepTables
from aspire_amd.attention.tree import compact_accepted, tree_attention
from aspire_amd.engine.sampling import verify_tree_speculation
from aspire_amd.logits_processor import adjust_logits
from helpers import say
from test_gpu_tree import BF, Case
from tree_cases import ancestors, pack, random_tree
from tree_checks import same_attention

pytestmark = pytest.mark.gpu


def i32(x, gpu):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("nodes", [[3, 9], [12, 14], [40, 33]])
def test_tables_with_more_rows_than_requests(gpu, nodes):
    """Attention from tables for 64 requests, most of them empty, with the whole last_page_len and with a slice of it."""
    say("padded tables", nodes)
    cached = [100, 63]
    c = Case(gpu, cached, nodes, 8, 2, 128)
    t = StepTables(64, 128, 64, 16, gpu, tree_words=1)
    table = torch.full((64, 12), -1, dtype=torch.int32)
    for b in range(2):
        table[b, : c.kvp[b + 1] - c.kvp[b]] = torch.tensor(c.ids[c.kvp[b] : c.kvp[b + 1]])
    parents = [p for tree in c.trees for p in tree]
    t.build(table.to(gpu), i32(cached + [0] * 62, gpu), i32(nodes + [0] * 62, gpu), i32(parents + [0] * (128 - len(parents)), gpu))
    T = sum(nodes)
    q = torch.randn(128, 8, 128, device=gpu).to(BF)  # as many rows as the tables have
    q[:T] = c.q
    for last in (t.last_page_len, t.last_page_len[:2]):
        out, lse = torch.full_like(q, 7.0), torch.full((128, 8), 7.0, device=gpu)
        tree_attention(q, c.cache, t.qo_indptr, t.kv_indices, t.kv_indptr, last, t.masks, 16, out=out, lse=lse)
        same_attention(c, out, lse)
        assert (out[T:] == 7).all() and (lse[T:] == 7).all()


@pytest.mark.parametrize("front", [1, 5, 70])
def test_tokens_in_front_of_the_first_row(gpu, front):
    say("tokens in front", front)
    c = Case(gpu, [50, 20], [7, 4], 8, 2, 64)
    shift = lambda t, fill: torch.cat([torch.full((front, *t.shape[1:]), fill, dtype=t.dtype, device=gpu), t])
    want = c.run()
    q, masks = shift(c.q, 3.0), shift(c.masks, -1)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=gpu)
    qo = c.dev([x + front for x in c.qo])
    tree_attention(q, c.cache, qo, c.dev(c.ids), c.dev(c.kvp), c.dev(c.last), masks, 16, out=out, lse=lse)
    assert torch.equal(out[front:], want[0]) and torch.equal(lse[front:], want[1])
    assert (out[:front] == 7).all() and (lse[:front] == 7).all()
    # the path, the moves and the logits of the same rows
    parents = [0] * front + [p for t in c.trees for p in t]
    tokens = torch.zeros(front + 11, dtype=torch.int32, device=gpu)
    got = verify_tree_speculation(tokens, i32(parents, gpu), tokens, qo, 5)
    plain = verify_tree_speculation(tokens[front:], i32(parents[front:], gpu), tokens[front:], c.dev(c.qo), 5)
    assert all(torch.equal(a, b) for a, b in zip(got, plain))
    slots = torch.arange(front + 11, device=gpu)
    caches = [torch.randn(8, 2, 16, 2, 8, device=gpu)] * 2
    caches[1] = caches[0].clone()
    compact_accepted(caches[0], got[1], got[2], qo, slots)
    compact_accepted(caches[1], got[1], got[2], c.dev(c.qo), slots[front:])
    assert torch.equal(caches[0], caches[1])
    x, one = torch.randn(front + 11, 40, device=gpu), torch.ones(2, device=gpu)
    out = adjust_logits(x, qo_indptr=qo, tree_tokens=tokens, tree_masks=masks, presence=one, out=torch.full_like(x, 7.0))
    assert (out[:front] == 7).all()
    assert torch.equal(out[front:], adjust_logits(x[front:], qo_indptr=c.dev(c.qo), tree_tokens=tokens[front:], tree_masks=masks[front:], presence=one))


def test_masks_without_words(gpu):
    """No drafted token is on a row's path: the history's penalties alone, or none."""
    say("masks without words")
    x = torch.randn(3, 20, device=gpu)
    qo, tokens, one = i32([0, 2, 3], gpu), i32([1, 2, 3], gpu), torch.ones(2, device=gpu)
    none = torch.zeros(3, 0, dtype=torch.int64, device=gpu)
    assert torch.equal(adjust_logits(x, qo_indptr=qo, tree_tokens=tokens, tree_masks=none, presence=one), x)
    history = dict(history=i32([[4, 5], [6, 7]], gpu), history_lens=i32([2, 1], gpu))
    assert torch.equal(adjust_logits(x, qo_indptr=qo, tree_tokens=tokens, tree_masks=none, presence=one, **history),
                       adjust_logits(x, qo_indptr=qo, presence=one, **history))
    empty = dict(history=torch.zeros(2, 0, dtype=torch.int32, device=gpu), history_lens=i32([0, 0], gpu))
    assert torch.equal(adjust_logits(x, qo_indptr=qo, presence=one, **empty), x)


def test_a_captured_step_of_changing_requests(gpu):
    """Resize, tables, attention, path and moves in one graph, replayed as requests come and go, against the same calls made eagerly."""
    say("captured step")
    rows, most, page, layers = 6, 60, 16, 2
    g = torch.Generator(device=gpu).manual_seed(0)
    r = np.random.default_rng(0)
    state = {}

    def fresh():
        pool = PagePool(40, page, rows, 8, gpu)
        t = StepTables(rows, most, 40, page, gpu, tree_words=1)
        return pool, t

    inputs = {k: torch.zeros(n, dtype=torch.int32, device=gpu) for k, n in (("cached", rows), ("new", rows), ("length", rows), ("parents", most),
                                                                             ("tokens", most), ("targets", most))}
    q = torch.randn(most, 8, 64, device=gpu, generator=g).to(BF)
    first = torch.randn(layers, 40, 2, page, 2, 64, device=gpu, generator=g).to(BF)

    def step(pool, t, cache, out):
        pool.resize(inputs["length"])
        t.build(pool.block_table, inputs["cached"], inputs["new"], inputs["parents"])
        for layer in range(layers):
            tree_attention(q, cache[layer], t.qo_indptr, t.kv_indices, t.kv_indptr, t.last_page_len, t.masks, page, out=out[layer])
        found = verify_tree_speculation(inputs["tokens"], inputs["parents"], inputs["targets"], t.qo_indptr, 5)
        compact_accepted(cache, found[1], found[2], t.qo_indptr, t.slots)
        return found

    pool, t = fresh()
    cache, out = first.clone(), torch.zeros(layers, most, 8, 64, dtype=BF, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        found = step(pool, t, cache, out)
    other_pool, other_t = fresh()
    other_cache, other_out = first.clone(), torch.zeros_like(out)
    for replay in range(6):
        new = r.integers(0, 11, size=rows) * (r.random(rows) < 0.7)
        cached = np.where(new > 0, r.integers(0, 100, size=rows), 0)
        parents = [p for n in new for p in random_tree(int(n), r)]
        for k, v in (("cached", cached), ("new", new), ("length", cached + new), ("parents", parents + [0] * (most - len(parents))),
                     ("tokens", r.integers(0, 2, size=most)), ("targets", r.integers(0, 2, size=most))):
            inputs[k].copy_(i32(v, gpu))
        graph.replay()
        torch.cuda.synchronize()
        want = step(other_pool, other_t, other_cache, other_out)
        for a, b in zip((pool.block_table, t.positions, t.masks, t.totals, out, cache, *found),
                        (other_pool.block_table, other_t.positions, other_t.masks, other_t.totals, other_out, other_cache, *want)):
            assert torch.equal(a, b)
