"""Attention of drafted trees over a paged cache against the definition in 64 bits."""

import numpy as np
import pytest
import torch

from aspire_amd.attention.tree import tree_attention
from helpers import say
from tree_cases import ancestors, attention, attention_limit, lse_limit, pack, random_tree

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


class Case:
    """A batch of trees: lengths before the trees, nodes a row, as tensors on the device; ``pad`` tokens of no row behind."""

    def __init__(self, gpu, cached, nodes, hq, hkv, dim, page=16, dtype=BF, words=None, pad=0, seed=0, extra_pages=3):
        r = np.random.default_rng(seed + 1)
        g = torch.Generator(device=gpu).manual_seed(seed)
        self.page, self.nodes = page, nodes
        length = [c + n for c, n in zip(cached, nodes)]
        pages = [-(-x // page) for x in length]
        self.qo, self.kvp = [0, *np.cumsum(nodes).tolist()], [0, *np.cumsum(pages).tolist()]
        self.last = [(x - 1) % page + 1 if x else 0 for x in length]
        self.ids = r.permutation(sum(pages) + extra_pages)[: sum(pages)].tolist()
        self.trees = [random_tree(n, r) for n in nodes]
        self.words = max([1, *((n + 63) // 64 for n in nodes)]) if words is None else words
        rows = [pack(ancestors(t), self.words) for t in self.trees if t]
        T = sum(nodes) + pad
        m = np.concatenate([*rows, np.zeros((pad, self.words), np.int64)]) if rows or pad else np.zeros((0, self.words), np.int64)
        self.masks = torch.from_numpy(m).to(gpu)
        randn = lambda *s: torch.randn(*s, device=gpu, generator=g).to(dtype)
        qkv = randn(T, (hq + 2 * hkv) * dim)
        self.q = qkv[:, : hq * dim].view(T, hq, dim)
        self.cache = randn(sum(pages) + extra_pages, 2, page, hkv, dim)
        self.gpu = gpu

    def dev(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.gpu)

    def run(self, **kw):
        return tree_attention(self.q, self.cache, self.dev(self.qo), self.dev(self.ids), self.dev(self.kvp), self.dev(self.last),
                              self.masks, self.page, return_lse=True, **kw)

    def check(self, out, lse, scale=None):
        ref, ref_lse, size, most = attention(self.q, self.cache, self.qo, self.kvp, self.ids, self.last, self.masks, scale)
        keys = max([1, *(b - a for a, b in zip(self.kvp[:-1], self.kvp[1:]))]) * self.page
        got, got_lse = out.detach().cpu().double().numpy(), lse.cpu().double().numpy()
        there = ~np.isnan(ref_lse)
        assert np.array_equal(np.isneginf(got_lse[there]), np.isneginf(ref_lse[there]))
        seen = there & ~np.isneginf(ref_lse)
        assert (got[there & ~seen] == 0).all()
        off = np.abs(got - ref) - attention_limit(ref, size, most, out.dtype, keys, ref.shape[2])
        assert not (off[seen] > 0).any(), f"{int((off[seen] > 0).sum())} of {off[seen].size} off, worst by {off[seen].max()}"
        off = np.abs(got_lse - ref_lse) - lse_limit(ref_lse, most, keys, ref.shape[2])
        assert not (off[seen] > 0).any(), f"lse off by {off[seen].max()} more than it may"


BATCHES = {
    # cached tokens, nodes of each row
    "one token, nothing before it": ([0], [1]),
    "one token behind one": ([1], [1]),
    "a tile's edge": ([31], [1]),
    "a tile and a token": ([32], [2]),
    "pages that end inside a tile": ([15, 16, 17, 47], [1, 2, 3, 4]),
    "empty rows between": ([0, 40, 0, 100, 7], [0, 3, 0, 5, 0]),
    "rows with keys and no tokens": ([50, 60], [0, 4]),
    "trees past a word": ([10, 200], [65, 130]),
    "a tree at a word's end": ([100], [64]),
    "uneven": ([700, 5, 300, 64], [9, 33, 1, 17]),
    "long": ([2500], [6]),
}
HEADS = [(8, 8, 128), (16, 8, 128), (32, 8, 128), (5, 1, 128), (14, 2, 64), (7, 1, 64), (64, 4, 128), (24, 2, 64), (40, 1, 128)]


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("heads", [(8, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_batches(gpu, name, heads, dtype):
    say("tree attention", name, heads, dtype)
    c = Case(gpu, *BATCHES[name], *heads, dtype=dtype)
    c.check(*c.run())


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("nodes", [1, 3, 8, 21, 70])
def test_heads(gpu, heads, nodes):
    say("tree attention heads", heads, nodes)
    c = Case(gpu, [130, 37], [nodes, max(1, nodes // 2)], *heads, seed=nodes)
    c.check(*c.run())


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_pages(gpu, page, dim):
    say("tree attention pages", page, dim)
    c = Case(gpu, [3, 255, 513], [2, 7, 30], 8, 2, dim, page=page, seed=page)
    c.check(*c.run())


def test_any_mask(gpu):
    """Bits need not be a tree's: rows without any, bits of later tokens, bits beyond the row's tokens (not seen)."""
    say("tree attention any mask")
    c = Case(gpu, [0, 0, 45], [9, 70, 20], 8, 2, 128)
    g = torch.Generator(device=gpu).manual_seed(5)
    c.masks = torch.randint(-2 ** 62, 2 ** 62, c.masks.shape, device=gpu, generator=g) * 2 + 1
    c.masks[3] = 0     # sees nothing: no cached tokens either
    c.masks[40] = 0
    c.masks[85] = 0    # sees the cached tokens alone
    c.masks[10] = -1
    c.masks[80] = -1
    c.check(*c.run())


def test_few_words(gpu):
    """Nodes past the words that a mask has are not seen."""
    say("tree attention few words")
    c = Case(gpu, [20, 0], [100, 80], 4, 2, 64, words=1)
    c.check(*c.run())
    c.masks = c.masks[:, :0]
    c.check(*c.run())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("nodes", [6, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_unseen_keys_hold_anything(gpu, value, nodes, dtype):
    """What a token does not see does not touch it: stale slots of the last page, pages of no row, other branches' K and V."""
    say("tree attention unseen", value, nodes, dtype)
    c = Case(gpu, [37, 90], [nodes, 3], 8, 2, 128, dtype=dtype)
    clean = c.run()
    c.check(*clean)
    used = torch.zeros(c.cache.shape[0], dtype=torch.bool, device=gpu)
    used[torch.tensor(c.ids, device=gpu)] = True
    c.cache[~used] = value
    for b, (n, cached) in enumerate(zip(c.nodes, (37, 90))):  # stale slots behind the row's last key
        page = c.ids[c.kvp[b + 1] - 1]
        c.cache[page, :, c.last[b]:] = value
    again = c.run()
    assert torch.equal(again[0].view(torch.int16), clean[0].view(torch.int16)) and torch.equal(again[1], clean[1])
    # one node that few see
    see = ancestors(c.trees[0])
    bad = int(see.sum(0).argmin())
    key = 37 + bad
    for which in (0, 1):
        c.cache[c.ids[key // 16], which, key % 16, :, ::3] = value
    out, lse = c.run()
    blind = torch.tensor(np.concatenate([~see[:, bad], np.ones(3, bool)]), device=gpu)
    assert torch.equal(out[blind].view(torch.int16), clean[0][blind].view(torch.int16)) and torch.equal(lse[blind], clean[1][blind])
    sees = ~blind
    c.cache[c.ids[key // 16], 0, key % 16] = 0  # with a score of 0 its V alone is not finite
    out, lse = c.run()
    assert torch.isfinite(lse).all()
    assert torch.equal(torch.isnan(out[sees][..., ::3]) if value != value else out[sees][..., ::3] == value,
                       torch.ones_like(out[sees][..., ::3], dtype=torch.bool))
    rest = [d for d in range(128) if d % 3]
    assert torch.isfinite(out[sees][..., rest]).all() and torch.isfinite(out[blind]).all()


def test_visible_nan_reaches_its_rows(gpu):
    say("tree attention visible NaN")
    c = Case(gpu, [70], [5], 4, 2, 128)
    c.cache[c.ids[1], 1, 3, 0] = float("nan")
    out, _ = c.run()
    assert torch.isnan(out[:, :2]).all() and torch.isfinite(out[:, 2:]).all()


def test_large_and_far_scores(gpu):
    """Scores of some hundreds, rising and falling along the keys, and rows whose first keys lie far below the others."""
    say("tree attention far scores")
    c = Case(gpu, [600, 300], [12, 7], 8, 2, 128, dtype=BF)
    for b in range(2):
        pages = c.ids[c.kvp[b] : c.kvp[b + 1]]
        for i, p in enumerate(pages):
            c.cache[p, 0] *= [0.01, 30.0, 1.0, 8.0, 0.1][i % 5]
    c.check(*c.run())
    c.q.mul_(-4)
    c.check(*c.run())


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_scale(gpu, scale):
    say("tree attention scale", scale)
    c = Case(gpu, [100], [10], 4, 1, 64)
    c.check(*c.run(sm_scale=scale), scale)


def test_tokens_of_no_row_stay(gpu):
    say("tree attention padding")
    c = Case(gpu, [20, 33], [4, 9], 8, 2, 128, pad=7)
    out = torch.full(c.q.shape, 7.0, dtype=BF, device=gpu)
    lse = torch.full(c.q.shape[:2], 7.0, device=gpu)
    res = c.run(out=out, lse=lse)
    assert res[0] is out and res[1] is lse
    assert (out[13:] == 7).all() and (lse[13:] == 7).all()
    ref, ref_lse, size, most = attention(c.q, c.cache, c.qo, c.kvp, c.ids, c.last, c.masks)
    off = np.abs(out.cpu().double().numpy() - ref) - attention_limit(ref, size, most, BF, 48, 128)
    assert not (off[:13] > 0).any()


def test_strides(gpu):
    """A cache whose pages are a slice of larger ones, K and V apart, masks with longer rows, out as a view."""
    say("tree attention strides")
    c = Case(gpu, [90, 20], [11, 5], 8, 2, 128)
    big = torch.randn(c.cache.shape[0], 3, 20, 4, 136, device=gpu).to(BF)
    view = big[:, 1:, 2:18, 1:3, 8:]
    view.copy_(c.cache)
    c.cache = view
    wide = torch.zeros(c.masks.shape[0], 5, dtype=torch.int64, device=gpu)
    wide[:, : c.words] = c.masks
    c.masks = wide[:, : c.words]
    out = torch.zeros(16, 12, 136, dtype=BF, device=gpu)[:, 2:10, :128]
    c.check(*c.run(out=out))
    c.cache = torch.empty(2, 16, 2, c.cache.shape[0], 128, dtype=BF, device=gpu).permute(3, 0, 1, 2, 4).copy_(c.cache)
    c.check(*c.run())


def test_bad_pages_are_not_seen(gpu):
    """Page ids and list entries outside the pool and the list: no access, no key."""
    say("tree attention bad pages")
    c = Case(gpu, [200, 60], [5, 3], 8, 2, 128)
    c.ids[2], c.ids[5] = -1, c.cache.shape[0]
    c.ids[7] = 2 ** 31 - 1
    c.check(*c.run())
    c.ids = c.ids[:-2]  # the last row's entries pass the list's end
    c.check(*c.run())
    c.ids = [-1] * len(c.ids)
    out, lse = c.run()
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_far_pages(gpu):
    """Offsets past 2^31 elements into the cache."""
    say("tree attention far pages")
    c = Case(gpu, [100], [6], 8, 8, 128)
    per = 2 * 16 * 8 * 128
    pages = (2 ** 31 + 2 ** 28) // per
    far = torch.zeros(pages, 2, 16, 8, 128, dtype=BF, device=gpu)
    ids = [pages - 1 - i * 5 for i in range(len(c.ids))]
    far[torch.tensor(ids, device=gpu)] = c.cache[torch.tensor(c.ids, device=gpu)]
    want = c.run()
    got = tree_attention(c.q, far, c.dev(c.qo), c.dev(ids), c.dev(c.kvp), c.dev(c.last), c.masks, 16, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_repeats_and_streams(gpu):
    """The same call gives the same bits, on another stream and from a graph whose lengths changed since its capture."""
    say("tree attention graph")
    c = Case(gpu, [1500, 900, 40], [12, 30, 3], 16, 4, 128, seed=3)
    want = [t.clone() for t in c.run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = c.run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    qo, ids, kvp, last = (c.dev(x) for x in (c.qo, c.ids, c.kvp, c.last))
    out, lse = torch.zeros_like(c.q, memory_format=torch.contiguous_format), torch.zeros(c.q.shape[:2], device=gpu)
    call = lambda: tree_attention(c.q, c.cache, qo, ids, kvp, last, c.masks, 16, out=out, lse=lse)
    graphs = []
    for _ in range(2):  # two graphs of one call: each has a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    last_before = c.last[1]
    for step in range(6):
        c.last[1] = 1 + (last_before + step) % 16
        last.copy_(c.dev(c.last))
        eager = [t.clone() for t in c.run()]
        out.zero_()
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])


def test_matches_the_chain_kernel(gpu):
    """A chain of drafted tokens is what the mixed kernel verifies."""
    say("tree attention chain")
    from aspire_amd.attention.holistic_wrapper import HolisticAttentionWrapper

    c = Case(gpu, [333, 70], [5, 8], 32, 8, 128)
    c.trees = [[i - 1 for i in range(n)] for n in c.nodes]
    c.masks = torch.from_numpy(np.concatenate([pack(ancestors(t), 1) for t in c.trees])).to(gpu)
    out, lse = c.run()
    w = HolisticAttentionWrapper(torch.empty(1, device=gpu), "NHD")
    w.plan(c.dev(c.qo), c.dev(c.kvp), c.dev(c.ids), c.dev(c.last), 32, 8, 128, 16, causal=True)
    ref, ref_lse = w.run(c.q.contiguous(), c.cache, return_lse=True)
    assert (out.float() - ref.float()).abs().max() <= 2e-2
    assert (lse - ref_lse).abs().max() <= 2e-3
    c.check(out, lse)


def test_refusals(gpu):
    say("tree attention refusals")
    c = Case(gpu, [20], [4], 8, 2, 128)
    base = dict(q=c.q, kv_cache=c.cache, qo_indptr=c.dev(c.qo), kv_page_indices=c.dev(c.ids), kv_page_indptr=c.dev(c.kvp),
                kv_last_page_len=c.dev(c.last), tree_masks=c.masks, page_size=16)
    call = lambda **kw: tree_attention(**{**base, **kw})
    call()
    odd = torch.zeros(4, 8, 132, dtype=BF, device=gpu)[..., 3:131]
    for kw in (dict(q=c.q.float()), dict(q=c.q[0]), dict(q=c.q[..., :96]), dict(q=odd), dict(q=c.q[:, :7]),
               dict(q=c.q.half()), dict(kv_cache=c.cache.float()), dict(kv_cache=c.cache[:, :1]), dict(kv_cache=c.cache[..., :64]),
               dict(page_size=32), dict(tree_masks=c.masks.int()), dict(tree_masks=c.masks[:2]), dict(tree_masks=c.masks[:, 0]),
               dict(qo_indptr=c.dev(c.qo)[:1]), dict(kv_page_indptr=c.dev(c.kvp)[:1]), dict(qo_indptr=c.dev(c.qo).float()),
               dict(out=torch.empty(4, 8, 64, dtype=BF, device=gpu)), dict(out=torch.empty(4, 8, 128, dtype=HF, device=gpu)),
               dict(out=c.q), dict(lse=torch.empty(4, 7, device=gpu)), dict(lse=torch.empty(4, 8, device=gpu).double()),
               dict(sm_scale=float("nan")), dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(sm_scale=float("inf")),
               dict(q=c.q.detach().clone().requires_grad_()),
               dict(kv_cache=c.cache[:, :, :12].contiguous(), page_size=12)):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(RuntimeError):
        call(q=c.q.cpu())
    with torch.no_grad():
        call(q=c.q.detach().clone().requires_grad_())
    empty = call(q=c.q[:0], tree_masks=c.masks[:0], qo_indptr=c.dev([0]), kv_page_indptr=c.dev([0]), kv_last_page_len=c.dev([]),
                 kv_page_indices=c.dev([]))
    assert empty.shape == (0, 8, 128)


def test_no_pages_at_all(gpu):
    say("tree attention no pages")
    c = Case(gpu, [20], [4], 8, 2, 128)
    for cache, ids in ((c.cache[:0], c.dev(c.ids)), (c.cache, c.dev([]))):
        out, lse = tree_attention(c.q, cache, c.dev(c.qo), ids, c.dev(c.kvp), c.dev(c.last), c.masks, 16, return_lse=True)
        assert (out == 0).all() and torch.isneginf(lse).all()


def test_many_rows(gpu):
    """More rows than a wave reads at once, most of them empty, and more than the chip has workgroups."""
    say("tree attention many rows")
    r = np.random.default_rng(0)
    nodes = [int(n) for n in r.integers(0, 3, size=700)]
    c = Case(gpu, [int(x) if n else 0 for x, n in zip(r.integers(0, 60, size=700), nodes)], nodes, 4, 1, 64)
    c.check(*c.run())


def test_out_whose_rows_share_memory(gpu):
    say("tree attention out shared")
    c = Case(gpu, [20], [4], 8, 2, 128)
    for bad in (torch.zeros(1, 8, 128, dtype=BF, device=gpu).expand(4, -1, -1), torch.zeros(4, 1, 128, dtype=BF, device=gpu).expand(-1, 8, -1)):
        with pytest.raises(ValueError, match="share memory"):
            c.run(out=bad)
