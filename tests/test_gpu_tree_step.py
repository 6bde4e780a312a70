"""A step that drafts and verifies trees, as a program runs it: pages and tables from lengths, the append at the positions of
the tokens' depths, tree attention, adjusted logits, the accepted paths and the moves; each stage against its plain form on
the stage's own inputs, and the caches after several steps against ones that only ever appended the accepted tokens."""

import numpy as np
import pytest
import torch

from aspire_amd.attention.paging import PagePool, StepTables
from aspire_amd.attention.rotary import RotaryConfig, RotaryEmbedding
from aspire_amd.attention.tree import compact_accepted, tree_attention
from aspire_amd.engine.sampling import verify_tree_speculation
from aspire_amd.logits_processor import LogitBias, adjust_logits
from helpers import say
from tree_cases import Pool, accept, adjusted, ancestors, attention, attention_limit, random_tree, tables

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
PAGE, HQ, HKV, D, LAYERS, VOCAB, ROWS, WIDTH, MOST = 16, 8, 2, 64, 3, 61, 4, 12, 9


def test_steps_of_trees(gpu):
    r = np.random.default_rng(0)
    g = torch.Generator(device=gpu).manual_seed(0)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=g)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=gpu)
    # what a token is to the layers: q, k and v by its id
    table = randn(LAYERS, VOCAB, (HQ + 2 * HKV) * D).to(BF)
    head = randn(HQ * D, VOCAB)
    rotary = RotaryEmbedding(RotaryConfig(head_dim=D, theta=1e4), gpu)
    pool, plain_pool = PagePool(60, PAGE, ROWS, WIDTH, gpu), Pool(60, PAGE, ROWS, WIDTH)
    cache = randn(LAYERS, 60, 2, PAGE, HKV, D).to(BF)
    t = StepTables(ROWS, ROWS * MOST, 60, PAGE, gpu, tree_words=1)
    text = [r.integers(0, VOCAB, size=n).tolist() for n in (20, 3, 47, 15)]  # tokens that are in the cache, but the last
    # the prompts: chains
    cached, fresh = [0] * ROWS, [len(x) - 1 for x in text]
    prompt = StepTables(ROWS, sum(fresh), 60, PAGE, gpu)
    pool.resize(i32(fresh))
    plain_pool.resize(fresh)
    prompt.build(pool.block_table, i32(cached), i32(fresh))

    def append(tab, ids, into, layer):
        qkv = table[layer][ids].view(len(ids), HQ + 2 * HKV, D)
        q, k, v = (x.contiguous() for x in qkv.split([HQ, HKV, HKV], 1))
        return rotary.append(q, k, v, tab.qo_indptr, into[layer], tab.kv_indices, tab.kv_indptr, tab.last_page_len, PAGE, positions=tab.positions[: len(ids)])

    ids = torch.tensor([x for row in text for x in row[:-1]], device=gpu)
    for layer in range(LAYERS):
        append(prompt, ids, cache, layer)
    moves = 0
    for step in range(4):
        say("tree step", step)
        cached = [len(x) - 1 for x in text]
        trees = [random_tree(int(n), r) for n in r.integers(1, MOST + 1, size=ROWS)]
        fresh = [len(x) for x in trees]
        drafted = [[row[-1], *r.integers(0, VOCAB, size=n - 1).tolist()] for row, n in zip(text, fresh)]
        tokens = sum(fresh)
        parents = [p for x in trees for p in x]
        lengths = [c + f for c, f in zip(cached, fresh)]
        assert pool.resize(i32(lengths)).tolist() == plain_pool.resize(lengths)
        assert pool.block_table.tolist() == plain_pool.table()
        t.build(pool.block_table, i32(cached), i32(fresh), i32(parents + [0] * (t.max_tokens - tokens)))
        ref = tables(plain_pool.table(), cached, fresh, parents, PAGE, ROWS, t.max_tokens, 60, 1)
        assert t.positions.tolist() == ref[4] and t.slots.tolist() == ref[5] and np.array_equal(t.masks.cpu().numpy(), ref[6])
        flat = torch.tensor([x for row in drafted for x in row], device=gpu)
        for layer in range(LAYERS):
            q = append(t, flat, cache, layer)
            out = tree_attention(q, cache[layer], t.qo_indptr, t.kv_indices, t.kv_indptr, t.last_page_len, t.masks, PAGE)
            want, _, size, most = attention(q, cache[layer], ref[0], ref[1], ref[2], ref[3], t.masks[:tokens])
            off = np.abs(out.cpu().double().numpy() - want) - attention_limit(want, size, most, BF, max(lengths), D)
            assert not (off > 0).any()
        # greedy targets of the last layer; one tree out of two is steered along its first chain, so that paths have moves
        logits = (out.float().view(tokens, -1) @ head)
        see = np.zeros((tokens, 64), bool)
        at = 0
        for tree, own in zip(trees, drafted):
            n = len(tree)
            see[at : at + n, :n] = ancestors(tree)
            if (at + step) % 2 == 0:
                for i in range(1, n):
                    logits[at + tree[i], own[i]] += 1000.0
            at += n
        history = torch.zeros(ROWS, 128, dtype=torch.int32, device=gpu)
        for b, row in enumerate(text):
            history[b, : len(row) - 1] = i32(row[:-1])
        lens, freq = [len(x) - 1 for x in text], np.float32([0.1, 0.0, 0.3, 0.2])
        bias = [{int(i): float(r.normal()) for i in r.integers(0, VOCAB, size=3)} for _ in range(ROWS)]
        got = adjust_logits(logits, qo_indptr=t.qo_indptr, history=history, history_lens=i32(lens), frequency=torch.from_numpy(freq).to(gpu),
                            tree_tokens=flat.int(), tree_masks=t.masks, bias=LogitBias(bias, gpu))
        want, _, size = adjusted(logits, qo=ref[0], history=history.cpu().numpy(), lens=lens, freq=freq, tree=flat.cpu().numpy(), see=see, bias=bias)
        assert (np.abs(got.cpu().double().numpy() - want) <= 2.0 ** -24 * np.abs(want) + 8 * 2.0 ** -24 * size).all()
        targets = got.argmax(1)
        output, path, kept = verify_tree_speculation(flat, i32(parents), targets, t.qo_indptr, MOST)
        answer = accept(flat.tolist(), parents, targets.tolist(), ref[0], MOST)
        assert [output.tolist(), path.tolist(), kept.tolist()] == list(answer)
        compact_accepted(cache, path, kept, t.qo_indptr, t.slots)
        moves += sum(node > j for row in answer[1] for j, node in enumerate(row))
        for b in range(ROWS):
            text[b] += answer[0][b][: answer[2][b]]
    assert moves > 0  # some path left tokens out, so that its later ones went to other places
    # the caches hold what chains of the kept tokens would have put there
    cached = [len(x) - 1 for x in text]
    ids = torch.tensor([x for row in text for x in row[:-1]], device=gpu)
    again = torch.zeros_like(cache)
    chain = StepTables(ROWS, sum(cached), 60, PAGE, gpu)
    chain.build(pool.block_table, i32([0] * ROWS), i32(cached))
    for layer in range(LAYERS):
        append(chain, ids, again, layer)
    slots = chain.slots
    for kv in (0, 1):
        assert torch.equal(cache[:, slots // PAGE, kv, slots % PAGE], again[:, slots // PAGE, kv, slots % PAGE])


def test_two_streams_at_once(gpu):
    """Calls on two streams share nothing."""
    say("tree step on two streams")
    from test_gpu_tree import Case

    a, b = Case(gpu, [900, 30], [9, 20], 8, 2, 128, seed=1), Case(gpu, [400, 1200], [30, 4], 8, 2, 128, seed=2)
    want = [[x.clone() for x in c.run()] for c in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        got = []
        for c, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                got.append(c.run())
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for w, g in zip(want, got) for x, y in zip(w, g))
