"""The accepted path of drafted trees and the move of its rows, against plain Python: every value equal."""

import numpy as np
import pytest
import torch

from aspire_amd.attention.tree import compact_accepted
from aspire_amd.engine.sampling import verify_tree_speculation
from helpers import say
from tree_cases import accept, random_tree

pytestmark = pytest.mark.gpu


def dev(x, gpu, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=gpu)


def forest(nodes, r, vocab=3):
    """Parents, tokens and targets with many matches (few tokens in all)."""
    parents = [p for n in nodes for p in random_tree(n, r)]
    T = len(parents)
    return parents, r.integers(0, vocab, size=T).tolist(), r.integers(0, vocab, size=T).tolist(), [0, *np.cumsum(nodes).tolist()]


@pytest.mark.parametrize("nodes", [[1], [2], [0, 5, 0], [64, 65, 7], [200, 1, 33], [2048, 3], [2049, 2], [5000]])
@pytest.mark.parametrize("max_path", [1, 3, 64, 65, 200])
def test_paths(gpu, nodes, max_path):
    say("tree path", nodes, max_path)
    r = np.random.default_rng(sum(nodes) + max_path)
    for vocab in (1, 3):
        parents, tokens, targets, qo = forest(nodes, r, vocab)
        got = verify_tree_speculation(dev(tokens, gpu), dev(parents, gpu), dev(targets, gpu), dev(qo, gpu), max_path)
        for t, ref in zip(got, accept(tokens, parents, targets, qo, max_path)):
            assert t.dtype == torch.int32 and t.tolist() == ref


def test_chain_and_odd_parents(gpu):
    say("tree path of a chain")
    n = 300
    parents, tokens = list(range(-1, n - 1)), list(range(n))
    targets = tokens[1:] + [7]
    for stop in (n, 130):
        t = list(targets)
        if stop < n:
            t[stop] = -5
        got = verify_tree_speculation(dev(tokens, gpu), dev(parents, gpu), dev(t, gpu), dev([0, n], gpu), n + 3)
        for x, ref in zip(got, accept(tokens, parents, t, [0, n], n + 3)):
            assert x.tolist() == ref
    # indices that are no parents: itself, later ones, negative ones, far ones
    parents = [0, 1, 5, 0, -9, 3, 2 ** 31 - 1, -2 ** 31]
    got = verify_tree_speculation(dev([4] * 8, gpu), dev(parents, gpu), dev([4] * 8, gpu), dev([0, 8], gpu), 8)
    assert got[1].tolist() == [[0, 3, 5, -1, -1, -1, -1, -1]] and got[2].tolist() == [3]
    for x, ref in zip(got, accept([4] * 8, parents, [4] * 8, [0, 8], 8)):
        assert x.tolist() == ref


def test_int64_and_padding(gpu):
    say("tree path int64")
    parents, tokens, targets, qo = forest([5, 9], np.random.default_rng(0))
    pad = lambda x: dev(x + [0] * 4, gpu, torch.int64)
    got = verify_tree_speculation(pad(tokens), pad(parents), pad(targets), dev(qo, gpu, torch.int64), 6)
    for x, ref in zip(got, accept(tokens, parents, targets, qo, 6)):
        assert x.tolist() == ref


def moved(caches, path, kept, qo, slots, page):
    """The caches after the moves, on the CPU."""
    out = [c.clone() for c in caches]
    for b in range(len(kept)):
        n = qo[b + 1] - qo[b]
        for j in range(1, min(kept[b], len(path[b]))):
            a = path[b][j]
            if not j < a < n:
                continue
            s, d = slots[qo[b] + a], slots[qo[b] + j]
            if s < 0 or d < 0 or s // page >= caches[0].shape[0] or d // page >= caches[0].shape[0]:
                continue
            for c in out:
                c[d // page, :, d % page] = c[s // page, :, s % page]
    return out


@pytest.mark.parametrize("layers,heads,dim,page,dtype", [(1, 8, 128, 16, torch.bfloat16), (3, 2, 64, 32, torch.float16), (2, 1, 80, 16, torch.bfloat16),
                                                         (2, 3, 7, 4, torch.float32), (1, 5, 9, 16, torch.uint8), (70, 1, 16, 16, torch.bfloat16),
                                                         (2, 64, 128, 16, torch.bfloat16)])
def test_moves(gpu, layers, heads, dim, page, dtype):
    say("tree moves", layers, heads, dim, page, dtype)
    r = np.random.default_rng(layers + dim)
    nodes = [9, 0, 40, 1, 17]
    parents, tokens, targets, qo = forest(nodes, r, 1)  # every token matches: long paths
    T, pages = sum(nodes), 12 * 64 // page
    slots = r.permutation(pages * page)[:T].tolist()
    shape = (pages, 2, page, heads, dim)
    make = (lambda: torch.randint(0, 255, shape, dtype=torch.uint8)) if dtype == torch.uint8 else (lambda: torch.randn(shape).to(dtype))
    caches = [make() for _ in range(layers)]
    out, path, kept = verify_tree_speculation(dev(tokens, gpu), dev(parents, gpu), dev(targets, gpu), dev(qo, gpu), 30)
    assert max(kept.tolist()) > 4
    want = moved(caches, path.tolist(), kept.tolist(), qo, slots, page)
    where = (path, kept, dev(qo, gpu), dev(slots, gpu, torch.int64))
    lists = [c.to(gpu) for c in caches]
    compact_accepted(lists, *where)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(lists, want))
    stacked = torch.stack([c.to(gpu) for c in caches])
    compact_accepted(stacked, *where)
    assert torch.equal(stacked.cpu(), torch.stack(want))
    single = caches[0].to(gpu)
    compact_accepted(single, *where)
    assert torch.equal(single.cpu(), want[0])
    # every second byte row of a larger cache: other strides, narrower vectors
    big = torch.zeros(pages, 2, page + 1, heads, dim + 1, dtype=dtype, device=gpu)
    view = big[:, :, 1:, :, 1:]
    view.copy_(caches[0])
    compact_accepted(view, *where)
    assert torch.equal(view.cpu(), want[0]) and (big[:, :, 0] == 0).all() and (big[..., 0] == 0).all()


def test_moves_of_long_paths(gpu):
    """More moves than a workgroup lists at once, each source one above its place: a chain of reads before writes."""
    say("tree moves of long paths")
    n, page = 700, 16
    caches = torch.arange(45 * 2 * page * 4, dtype=torch.int32).view(45, 2, page, 1, 4)
    path = [[0, *range(2, n)]]
    slots = list(range(5, 5 + n))
    want = moved([caches], path, [n - 1], [0, n], slots, page)[0]
    got = caches.to(gpu)
    compact_accepted(got, dev(path, gpu), dev([n - 1], gpu), dev([0, n], gpu), dev(slots, gpu, torch.int64))
    assert torch.equal(got.cpu(), want)


def test_passed_over(gpu):
    """Entries that are not above their place or not of the row, slots of none and outside, counts past the path."""
    say("tree moves passed over")
    page = 16
    caches = torch.randn(4, 2, page, 2, 8)
    path, kept, qo = [[0, 3, 1, 9, 4, -1], [0, 2, 5, 5, 5, 5], [0, 1, 2, 3, 4, 5]], [5, 99, -3], [0, 6, 12, 18]
    slots = [3, 9, -1, 12, 64, 20, 30, 31, 32, 33, 34, 2 ** 40, 40, 41, 42, 43, 44, 45]
    want = moved([caches], path, [5, 6, 0], qo, slots, page)[0]
    got = caches.to(gpu)
    compact_accepted(got, dev(path, gpu), dev(kept, gpu), dev(qo, gpu), dev(slots, gpu, torch.int64))
    assert torch.equal(got.cpu(), want)
    before = got.clone()
    compact_accepted(got, dev([[0, 2]], gpu), dev([2], gpu), dev([-5, 3], gpu), dev([1, 2, 3], gpu, torch.int64))
    assert torch.equal(got, before)


def test_far_pages(gpu):
    """A cache past 2^32 bytes."""
    say("tree moves far pages")
    pages = 2 ** 32 // (2 * 16 * 8 * 128 * 2) + 40
    cache = torch.zeros(pages, 2, 16, 8, 128, dtype=torch.bfloat16, device=gpu)
    cache[-1, :, 3] = 5
    slots = [16 * (pages - 30), 16 * (pages - 20) + 1, 16 * pages - 13]
    compact_accepted(cache, dev([[0, 2]], gpu), dev([2], gpu), dev([0, 3], gpu), dev(slots, gpu, torch.int64))
    assert (cache[pages - 20, :, 1] == 5).all() and int((cache[-64:] != 0).sum()) == 2 * 2 * 8 * 128


def test_graph(gpu):
    say("tree accept graph")
    r = np.random.default_rng(0)
    nodes = [8, 20, 3]
    parents, tokens, targets, qo = forest(nodes, r, 2)
    t = [dev(x, gpu) for x in (tokens, parents, targets, qo)]
    slots = dev(r.permutation(10 * 16)[: sum(nodes)].tolist(), gpu, torch.int64)
    cache = torch.randn(2, 10, 2, 16, 2, 64, device=gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        output, path, kept = verify_tree_speculation(*t, 10)
        compact_accepted(cache, path, kept, t[3], slots)
    for _ in range(4):
        new = r.integers(0, 2, size=sum(nodes)).tolist()
        t[2].copy_(dev(new, gpu))
        before = [c.cpu() for c in cache.clone()]
        g.replay()
        torch.cuda.synchronize()
        ref = accept(tokens, parents, new, qo, 10)
        assert [output.tolist(), path.tolist(), kept.tolist()] == list(ref)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(cache, moved(before, ref[1], ref[2], qo, slots.tolist(), 16)))


def test_refusals(gpu):
    say("tree accept refusals")
    i = lambda n: torch.zeros(n, dtype=torch.int32, device=gpu)
    ok = (i(4), i(4), i(4), i(3), 5)
    verify_tree_speculation(*ok)
    for k, bad in ((0, i(4).float()), (0, i(4).view(2, 2)), (1, i(3)), (2, i(3)), (3, i(0)), (4, 0), (4, 2 ** 31), (2, i(4).bool())):
        args = list(ok)
        args[k] = bad
        with pytest.raises(ValueError):
            verify_tree_speculation(*args)
    with pytest.raises(RuntimeError):
        verify_tree_speculation(i(4), i(4).cpu(), i(4), i(3), 5)
    c = torch.zeros(3, 2, 16, 2, 8, device=gpu)
    path, slots = i(4).view(2, 2), torch.zeros(4, dtype=torch.int64, device=gpu)
    compact_accepted(c, path, i(2), i(3), slots)
    compact_accepted([], path, i(2), i(3), slots)
    for args in ((c[0], path, i(2), i(3), slots), (c[:, :1], path, i(2), i(3), slots), ([c, c], path, i(2), i(3), slots),
                 ([c, c.half()], path, i(2), i(3), slots), ([c, c[:2].clone()], path, i(2), i(3), slots), (c, path.long(), i(2), i(3), slots),
                 (c, path.t(), i(2), i(3), slots), (c, path, i(1), i(3), slots), (c, path, i(2), i(2), slots), (c, path, i(2), i(3), slots.int()),
                 (c.clone().requires_grad_(), path, i(2), i(3), slots), (c.transpose(3, 4), path, i(2), i(3), slots)):
        with pytest.raises(ValueError):
            compact_accepted(*args)


def test_shared_memory_is_refused(gpu):
    say("compact shared memory")
    path, kept = torch.zeros(1, 2, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    qo, slots = torch.zeros(2, dtype=torch.int32, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    c = torch.zeros(2, 4, 2, 16, 2, 8, device=gpu)
    for caches in ([c[0, :3], c[0, 1:]], [c[0], c[0]], c[:1].expand(2, -1, -1, -1, -1, -1), c[0, :, :, :, :1].expand(-1, -1, -1, 2, -1)):
        with pytest.raises(ValueError, match="share memory"):
            compact_accepted(caches, path, kept, qo, slots)
    compact_accepted([c[0], c[1]], path, kept, qo, slots)
    compact_accepted(list(torch.zeros(4, 2, 2, 16, 2, 8, device=gpu).unbind(1)), path, kept, qo, slots)
