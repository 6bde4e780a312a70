"""The page pool and a step's tables against plain Python: whole numbers, every one equal."""

import numpy as np
import pytest
import torch

from aspire_amd.attention.paging import PagePool, StepTables
from helpers import say
from tree_cases import Pool, random_tree, tables

pytestmark = pytest.mark.gpu


def dev(x, gpu, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=gpu)


def same_pool(pool, ref, short):
    assert pool.block_table.tolist() == ref.table()
    assert pool.held.tolist() == [len(r) for r in ref.rows]
    n = int(pool.free_count)
    assert n == len(ref.stack) and pool.free[:n].tolist() == ref.stack
    assert (pool.free[n:] == -1).all()
    assert pool.shortage.tolist() == short
    held = sorted(p for r in ref.rows for p in r) + sorted(ref.stack)
    assert sorted(held) == list(range(ref.pages))


@pytest.mark.parametrize("rows,width,pages,page", [(1, 1, 1, 16), (3, 4, 9, 16), (64, 40, 1500, 16), (7, 300, 1000, 1), (300, 9, 1200, 64),
                                                   (1025, 6, 3000, 32), (4096, 3, 9000, 16)])
def test_resize(gpu, rows, width, pages, page):
    say("resize", rows, width, pages, page)
    r = np.random.default_rng(rows)
    pool, ref = PagePool(pages, page, rows, width, gpu), Pool(pages, page, rows, width)
    for step in range(8):
        lengths = r.integers(-1, width * page + (3 if step % 3 == 2 else 1), size=rows)
        lengths[r.random(rows) < 0.3] = 0
        if step == 4:
            lengths[:] = 0
        if step == 5:
            lengths[:] = -1
        short = ref.resize(lengths.tolist())
        got = pool.resize(dev(lengths, gpu))
        assert got is pool.shortage
        same_pool(pool, ref, short)


def test_resize_gives_the_same_pages_back(gpu):
    """What was taken for a step and given back is taken again by the next step of the same lengths."""
    say("resize there and back")
    pool = PagePool(100, 16, 5, 20, gpu)
    a, b = dev([100, 3, 0, 64, 17], gpu), dev([200, 30, 1, 64, 300], gpu)
    pool.resize(a)
    pool.resize(b)
    table, free = pool.block_table.clone(), pool.free.clone()
    pool.resize(a)
    pool.resize(b)
    assert torch.equal(table, pool.block_table) and torch.equal(free, pool.free)


def test_resize_far_lengths(gpu):
    say("resize far lengths")
    pool, ref = PagePool(50, 1, 4, 20, gpu), Pool(50, 1, 4, 20)
    for lengths in ([5, 2 ** 31 - 1, 2, 0], [20, 20, 11, 1], [-2 ** 31, 3, 3, 3]):
        short = ref.resize(lengths)
        pool.resize(dev(lengths, gpu))
        same_pool(pool, ref, short)


def check_tables(t, table, cached, fresh, parents):
    ref = tables(table.tolist(), cached, fresh, parents, t.page_size, t.max_rows, t.max_tokens, t.max_entries, t.tree_words)
    qo, kvp, ids, last, positions, slots, masks, totals = ref
    assert t.totals.tolist() == totals
    assert t.qo_indptr.tolist() == qo and t.kv_indptr.tolist() == kvp
    assert t.kv_indices[: len(ids)].tolist() == ids
    assert t.last_page_len.tolist() == last
    assert t.positions.tolist() == positions and t.slots.tolist() == slots
    if t.tree_words:
        assert np.array_equal(t.masks.cpu().numpy(), masks)


def build(gpu, cached, fresh, page=16, words=0, tree=False, slack=(0, 0, 0), seed=0, width=None):
    r = np.random.default_rng(seed)
    need = [-(-(c + f) // page) for c, f in zip(cached, fresh)]
    width = max([1, *need]) if width is None else width
    table = torch.from_numpy(r.permutation(len(cached) * width + 5)[: len(cached) * width].astype(np.int32)).view(len(cached), width).to(gpu)
    entries = sum(n for n, f in zip(need, fresh) if f > 0)
    t = StepTables(len(cached) + slack[0], sum(fresh) + slack[1], entries + slack[2], page, gpu, tree_words=words)
    parents = None
    if tree:
        parents = [p for f in fresh for p in random_tree(f, r)]
        parents += [0] * (t.max_tokens - len(parents))
    got = t.build(table, dev(cached, gpu), dev(fresh, gpu), None if parents is None else dev(parents, gpu))
    assert got is t
    check_tables(t, table, cached, fresh, parents)
    return t, table


@pytest.mark.parametrize("tree,words", [(False, 0), (False, 2), (True, 0), (True, 1), (True, 3)])
@pytest.mark.parametrize("cached,fresh", [([0], [1]), ([15, 16, 17], [1, 1, 2]), ([5, 0, 100, 7], [0, 3, 0, 9]), ([0, 0], [0, 0]),
                                          ([1000, 3, 64], [64, 1, 33]), ([31], [17])])
def test_tables(gpu, tree, words, cached, fresh):
    say("tables", tree, words, cached, fresh)
    build(gpu, cached, fresh, words=words, tree=tree)
    build(gpu, cached, fresh, words=words, tree=tree, slack=(3, 9, 5), page=64)


@pytest.mark.parametrize("rows,page", [(257, 16), (1000, 1), (4096, 32)])
def test_many_rows(gpu, rows, page):
    say("tables of many rows", rows)
    r = np.random.default_rng(rows)
    build(gpu, r.integers(0, 90, size=rows).tolist(), r.integers(0, 4, size=rows).tolist(), page=page, words=1, tree=True, slack=(0, 40, 7))


def test_large_trees_and_prompts(gpu):
    say("tables of large trees")
    build(gpu, [10, 0, 5], [190, 256, 100], words=4, tree=True)
    build(gpu, [7, 3], [4096, 1500], words=64, tree=True)   # more ancestors before a workgroup's tokens than it holds
    build(gpu, [100, 9], [3000, 20], tree=False)
    build(gpu, [100, 9], [2000, 20], tree=True)


def test_rows_that_do_not_fit(gpu):
    say("tables that are too small")
    cached, fresh, page = [20, 3, 50, 8], [5, 9, 4, 6], 16
    table = dev(np.arange(4 * 6).reshape(4, 6), gpu)
    for tokens, entries, words in ((24, 99, 0), (14, 99, 0), (13, 99, 0), (4, 99, 0), (0, 99, 0), (99, 7, 0), (99, 2, 0), (99, 0, 0), (24, 8, 1)):
        t = StepTables(5, tokens, entries, page, gpu, tree_words=words)
        t.build(table, dev(cached, gpu), dev(fresh, gpu))
        check_tables(t, table, cached, fresh, None)
    t = StepTables(3, 300, 300, page, gpu, tree_words=1)
    t.build(table[:3], dev([0, 0, 0], gpu), dev([64, 65, 3], gpu))
    check_tables(t, table[:3], [0, 0, 0], [64, 65, 3], None)


def test_longest_trees(gpu):
    """A tree without masks has 4,096 tokens at most, a chain any number."""
    say("tables of the longest trees")
    table = dev(np.arange(2 * 600).reshape(2, 600), gpu)
    for first, chain in ((4096, False), (4097, False), (4097, True)):
        t = StepTables(2, 4400, 1200, 16, gpu)
        parents = None if chain else np.r_[np.arange(-1, first - 1), [-1, 0, 0], np.zeros(4400 - first - 3, int)].astype(np.int32)
        t.build(table, dev([5, 9], gpu), dev([first, 3], gpu), None if chain else dev(parents, gpu))
        check_tables(t, table, [5, 9], [first, 3], parents)
        assert int(t.totals[2]) == (0 if first > 4096 and not chain else 2)


def test_odd_inputs(gpu):
    """Negative counts, sums past 2^31, tables that are too narrow or have holes, parents that are none."""
    say("tables of odd inputs")
    table = dev([[3, -1, 4], [5, 6, 7], [8, 9, 1], [2, 0, 10]], gpu)
    for cached, fresh in (([10, -1, 4, 5], [30, 5, -3, 2]), ([2 ** 31 - 5, 40, 0, 3], [9, 30, 1, 0]), ([10, 10, 10, 10], [60, 1, 1, 60])):
        t = StepTables(4, 200, 60, 16, gpu, tree_words=1)
        t.build(table, dev(cached, gpu), dev(fresh, gpu))
        check_tables(t, table, cached, fresh, None)
    parents = [5, 0, 1, 3, -7, 2, 2 ** 31 - 1, 6, 7, 8]
    t = StepTables(1, 10, 5, 16, gpu, tree_words=1)
    t.build(table[1:2], dev([4], gpu), dev([10], gpu), dev(parents, gpu))
    check_tables(t, table[1:2], [4], [10], parents)


def test_wide_table_as_a_view(gpu):
    say("tables from a view")
    whole = dev(np.arange(6 * 40).reshape(6, 40), gpu)
    t = StepTables(3, 12, 40, 16, gpu)
    t.build(whole[2:5, 4:30], dev([100, 20, 33], gpu), dev([4, 4, 4], gpu))
    check_tables(t, whole[2:5, 4:30], [100, 20, 33], [4, 4, 4], None)


def test_graph_of_a_step(gpu):
    """Resize and build, captured once, replayed as lengths change."""
    say("paging graph")
    pool, ref = PagePool(400, 16, 6, 30, gpu), Pool(400, 16, 6, 30)
    t = StepTables(6, 40, 180, 16, gpu, tree_words=1)
    cached, fresh, wanted = (torch.zeros(6, dtype=torch.int32, device=gpu) for _ in range(3))
    parents = torch.zeros(40, dtype=torch.int32, device=gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.resize(wanted)
        t.build(pool.block_table, cached, fresh, parents)
    r = np.random.default_rng(0)
    for _ in range(5):
        c, f = r.integers(0, 400, size=6), r.integers(0, 7, size=6)
        p = [x for n in f for x in random_tree(int(n), r)]
        p += [0] * (40 - len(p))
        cached.copy_(dev(c, gpu)), fresh.copy_(dev(f, gpu)), wanted.copy_(dev(c + f, gpu)), parents.copy_(dev(p, gpu))
        g.replay()
        torch.cuda.synchronize()
        short = ref.resize((c + f).tolist())
        same_pool(pool, ref, short)
        check_tables(t, pool.block_table, c.tolist(), f.tolist(), p)


def test_refusals(gpu):
    say("paging refusals")
    for args in ((0, 16, 4, 4), (10, 0, 4, 4), (10, 16, 0, 4), (10, 16, 4097, 4), (10, 16, 4, 0), (10, 16, 4096, 1 << 20)):
        with pytest.raises(ValueError):
            PagePool(*args, gpu)
    pool = PagePool(10, 16, 4, 4, gpu)
    for bad in (dev([1, 2, 3], gpu), dev([[1, 2, 3, 4]], gpu), torch.ones(4, device=gpu)):
        with pytest.raises(ValueError):
            pool.resize(bad)
    with pytest.raises(RuntimeError):
        pool.resize(torch.ones(4, dtype=torch.int32))
    for args in ((4097, 1, 1, 16), (4, -1, 1, 16), (4, 1, 1, 0)):
        with pytest.raises(ValueError):
            StepTables(*args, gpu)
    with pytest.raises(ValueError):
        StepTables(4, 4, 4, 16, gpu, tree_words=65)
    t = StepTables(2, 8, 8, 16, gpu)
    table, two = dev([[0, 1], [2, 3]], gpu), dev([1, 1], gpu)
    for args in ((table[:1], two, two), (table.long(), two, two), (table, two, two[:1]), (table, dev([1, 1, 1], gpu), dev([1, 1, 1], gpu)),
                 (table.t(), two, two), (table, two.float(), two), (table, two, two, dev([0] * 7, gpu)), (table[0], two, two)):
        with pytest.raises(ValueError):
            t.build(*args)
