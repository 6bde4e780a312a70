"""Refusals of the tree, paging and logits entries before anything reaches a GPU, and the plain forms that the GPU tests use."""

import ctypes

import numpy as np
import pytest
import torch

from aspire_amd import _lib
from aspire_amd.attention import paging, tree
from aspire_amd.logits_processor import _ADJUST, LogitBias
from tree_cases import Pool, accept, adjusted, ancestors, attention, pack, random_tree, tables

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libaspire_hip.so not built")

TREE = dict(q=4096, qt=1024, qh=128, cache=4096, sp=32768, skv=16384, st=1024, sh=128, pages=4, entries=4, qo=4096, ids=4096, ptr=4096, last=4096,
            masks=4096, mst=1, out=4096, ot=1024, oh=128, lse=0, tokens=4, rows=1, words=1, hq=8, hkv=8, dim=128, page=16, dtype=0, scale=0.1,
            zero=0, ws=4096, floats=1 << 40)


def message():
    return _lib.lib().aspire_last_error().decode()


@pytest.mark.parametrize("change,word", [
    (dict(dim=96), "head_dim"), (dict(page=12), "page_size"), (dict(page=24), "page_size"), (dict(page=2048), "page_size"), (dict(hq=7), "q heads"),
    (dict(hq=2048, hkv=1024), "q heads"), (dict(dtype=2), "dtype"), (dict(scale=float("nan")), "sm_scale"), (dict(scale=0.0), "sm_scale"),
    (dict(scale=float("inf")), "sm_scale"), (dict(tokens=-1), "sizes"), (dict(tokens=(1 << 20) + 1), "2^20"), (dict(rows=(1 << 20) + 1), "2^20"),
    (dict(q=0), "null"), (dict(masks=0), "null"), (dict(cache=0), "null"), (dict(q=4104), "16 bytes"), (dict(qt=1020), "16 bytes"),
    (dict(sp=32764), "16 bytes"), (dict(oh=4), "16 bytes"), (dict(st=64), "head_dim"), (dict(st=1 << 20), "2^20"), (dict(sp=1 << 31), "2^31"),
    (dict(ws=0), "workspace"), (dict(floats=100), "workspace"), (dict(ws=4100), "workspace")])
def test_attention_refuses_on_the_host(change, word):
    args = tree._ARGS.pack(*{**TREE, **change}.values())
    assert _lib.lib().aspire_tree_attention(args, None) == _lib.ASPIRE_ERR_INVALID
    assert word in message()


def test_nothing_to_do_is_no_launch():
    for change in (dict(tokens=0), dict(rows=0)):
        assert _lib.lib().aspire_tree_attention(tree._ARGS.pack(*{**TREE, **change}.values()), None) == _lib.ASPIRE_OK
    assert _lib.lib().aspire_tree_attention_workspace(0, 4, 8, 8, 128) == 0
    assert _lib.lib().aspire_verify_tree(None, None, None, None, 0, 0, 4, None, None, None, None) == _lib.ASPIRE_OK
    assert _lib.lib().aspire_page_resize(paging._RESIZE.pack(0, 0, 0, 0, 0, 0, 0, 4, 4, 16), None) == _lib.ASPIRE_OK


def test_other_entries_refuse_on_the_host():
    L, bad = _lib.lib(), _lib.ASPIRE_ERR_INVALID
    for rows, width, pages, page in ((4097, 4, 4, 16), (-1, 4, 4, 16), (4, -1, 4, 16), (4, 4, 4, 0), (4096, 1 << 20, 4, 16), (4, 4, 4, 16)):
        assert L.aspire_page_resize(paging._RESIZE.pack(0, 0, 0, 0, 0, 0, rows, width, pages, page), None) == bad
    table = lambda *n: paging._TABLES.pack(4096, 4, 4096, 4096, 0, *n, 0, 4096, 4096, 4096, 4096, 4096, 4096, 0, 4096)
    for n in ((5, 4, 4, 9, 9, 16, 0), (4097, 4, 4097, 9, 9, 16, 0), (4, 4, 4, -1, 9, 16, 0), (4, 4, 4, 9, 9, 0, 0), (4, 4, 4, 9, 9, 16, 65),
              (4, 4, 4, (1 << 30) + 1, 9, 16, 0), (4, 4, 4, 9, 9, 16, 1)):
        assert L.aspire_step_tables(table(*n), None) == bad
    assert L.aspire_verify_tree(4096, 4096, 4096, 4096, 4, 2, 0, 4096, 4096, 4096, None) == bad
    assert L.aspire_verify_tree(0, 4096, 4096, 4096, 4, 2, 3, 4096, 4096, 4096, None) == bad
    move = lambda first, heads, size, page: tree._MOVE.pack(0, first, 0, 1, 1, 1, 1, 4, 4096, 4096, 4096, 4096, 1, heads, size, page, 2, 9, 4, 0)
    for n in ((0, 2, 16, 16), (4096, 2, 16, 0), (4096, -1, 16, 16), (4096, 1 << 20, 1 << 10, 16)):
        assert L.aspire_compact_accepted(move(*n), None) == bad
    base = dict(logits=4096, st=100, out=4096, ost=100, qo=0, hist=0, hst=0, lens=0, told=0, rep=0, pres=0, freq=0, tt=0, tm=0, mst=0, bi=0, bv=0, bp=0,
                g=0, gst=0, gr=0, start=0, tokens=3, vocab=100, requests=3, dtype=2, hl=0, words=0, gn=0, be=0)
    for change in (dict(requests=65536, tokens=70000), dict(requests=4), dict(dtype=3), dict(logits=0), dict(hist=4096), dict(tt=4096), dict(tt=4096, tm=4096),
                   dict(bp=4096, be=3), dict(vocab=(1 << 30) + 1), dict(start=-1), dict(start=(1 << 31) - 50)):
        assert L.aspire_adjust_logits(_ADJUST.pack(*{**base, **change}.values()), None) == bad


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError):
        tree.tree_attention(torch.zeros(1, 1, 64).bfloat16(), torch.zeros(1, 2, 16, 1, 64).bfloat16(), *[torch.zeros(2, dtype=torch.int32)] * 4,
                            torch.zeros(1, 1, dtype=torch.int64), 16)
    pool = paging.PagePool(4, 16, 2, 2, "cpu")
    with pytest.raises(RuntimeError):
        pool.resize(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        paging.StepTables(2, 4, 4, 16, "cpu").build(pool.block_table, torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_biases_are_sorted_by_request():
    b = LogitBias([{7: 1.0, 2: -2.0}, None, {}, {5: float("-inf")}], "cpu")
    assert b.ids.tolist() == [2, 7, 5] and b.values.tolist() == [-2.0, 1.0, float("-inf")] and b.indptr.tolist() == [0, 2, 2, 2, 3]
    for bad in ({-1: 1.0}, {1 << 31: 1.0}, {1: float("nan")}):
        with pytest.raises(ValueError):
            LogitBias([bad], "cpu")


def test_packed_structures_match_the_header():
    # four-byte counts and eight-byte addresses as the C compiler lays them out
    assert (paging._RESIZE.size, paging._TABLES.size, tree._ARGS.size, tree._MOVE.size, _ADJUST.size) == (64, 136, 216, 128, 208)
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_plain_attention_of_a_chain():
    """The plain form with a chain's masks is causal attention."""
    r = np.random.default_rng(0)
    q, cache = torch.from_numpy(r.normal(size=(3, 2, 8))), torch.from_numpy(r.normal(size=(2, 2, 16, 1, 8)))
    masks = torch.from_numpy(pack(ancestors([-1, 0, 1]), 1))
    out, lse, _, _ = attention(q, cache, [0, 3], [0, 2], [1, 0], [4], masks)
    k, v = cache[[1, 0], 0].reshape(32, 8)[:20], cache[[1, 0], 1].reshape(32, 8)[:20]
    x = torch.einsum("thd,kd->htk", q, k) * 8 ** -0.5
    x = x.masked_fill(torch.arange(20) > torch.arange(17, 20)[:, None], float("-inf"))
    assert np.allclose(out, torch.einsum("htk,kd->thd", x.softmax(-1), v)) and np.allclose(lse, torch.logsumexp(x, -1).T / np.log(2))


def test_plain_pool_and_tables():
    pool = Pool(6, 16, 3, 4)
    assert pool.resize([20, 0, 33]) == [0, 0, 0] and pool.rows == [[0, 1], [], [2, 3, 4]]
    assert pool.resize([1, 40, 33]) == [0, 3, 0] and pool.rows == [[0], [], [2, 3, 4]] and pool.stack == [5, 1]
    qo, kvp, ids, last, pos, slots, masks, totals = tables([[4, 9], [7, 5]], [15, 3], [2, 3], [-1, 0, -1, 0, 0], 16, 3, 6, 9, 1)
    assert (qo, kvp, ids, last) == ([0, 2, 5, 5], [0, 2, 3, 3], [4, 9, 7], [1, 6, 0])
    assert pos == [15, 16, 3, 4, 4, -1] and slots == [79, 144, 115, 116, 117, -1] and masks[:, 0].tolist() == [1, 3, 1, 3, 5, 0]
    assert totals == [5, 3, 2]


def test_plain_acceptance_and_logits():
    assert accept([5, 6, 7, 6, 8], [-1, 0, 0, 0, 3], [6, 0, 0, 8, 9], [0, 5], 4) == ([[6, 0, -1, -1]], [[0, 1, -1, -1]], [2])
    r = np.random.default_rng(1)
    assert all(p < i for i, p in enumerate(random_tree(40, r)))
    y, touched, _ = adjusted(torch.tensor([[1.0, -1.0, 2.0]]), history=np.array([[1, 0, 0]]), lens=[3], prompts=[1], rep=[2.0], freq=[0.5], pres=[0.25])
    assert y.tolist() == [[0.5 - 1.25, -2.0, 2.0]] and touched.all()


def test_longest_paths_are_bounded():
    assert _lib.lib().aspire_verify_tree(4096, 4096, 4096, 4096, 4, 2, (1 << 30) + 1, 4096, 4096, 4096, None) == _lib.ASPIRE_ERR_INVALID
    move = tree._MOVE.pack(0, 4096, 0, 1, 1, 1, 1, 4, 4096, 4096, 4096, 4096, 1, 2, 16, 16, 2, 9, (1 << 30) + 1, 0)
    assert _lib.lib().aspire_compact_accepted(move, None) == _lib.ASPIRE_ERR_INVALID


def test_shared_memory_is_found():
    c = torch.zeros(3, 4, 2, 16, 2, 8)
    apart = lambda ts: tree._starts_apart([t.data_ptr() for t in ts], ts[0].shape, ts[0].stride(), 4)
    assert apart([c[0], c[1], c[2]]) and apart([c[2], c[0]])
    assert not apart([c[0], c[0]]) and not apart([c[0, 0:3], c[0, 1:4]]) and not apart([c[0], c[1], c[1]])
    inner = torch.zeros(4, 3, 2, 16, 2, 8)  # layers inside of pages
    assert apart(list(inner.unbind(1))) and not apart([inner[:, 0], inner[:, 0]]) and not apart([inner[:3, 0], inner[1:, 0]])
    assert tree._apart(c.shape, c.stride()) and not tree._apart((3, 4), (0, 1)) and not tree._apart((3, 4), (2, 1)) and tree._apart((1, 4), (0, 1))
