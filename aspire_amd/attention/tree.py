"""Attention of drafted trees over the paged cache, and the move of what is kept of them (HIP).

The mixed attention kernel verifies chains of drafted tokens (aspire/models/sparse_draft_runner.py:595-612: causal among a
row's new tokens). A step that drafts a tree for each request appends its tokens in any order that puts parents first,
turned to the position of their depth (``StepTables.positions`` with ``RotaryEmbedding.append``), and

* ``tree_attention`` lets each of them see the request's cached tokens and its own ancestors;
* ``aspire_amd.engine.sampling.verify_tree_speculation`` finds the path that the target model agrees with;
* ``compact_accepted`` moves that path's K and V rows to where a chain of them would stand, in every layer.

All three read lengths on the device and can be captured.
"""

from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd import forward_ad

from aspire_amd import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
HEAD_DIMS = (64, 128)
_ARGS = struct.Struct("PqqPqqqqqqPPPPPqPqqP8ifiPq")  # aspire_tree_attention_args
_MOVE = struct.Struct("PPqqqqqqPPPP8i")              # aspire_compact_args


def _list(t: torch.Tensor, index: int, what: str, name: str) -> torch.Tensor:
    """An index array as int32 in one piece."""
    if t.dtype is torch.int32 and t.get_device() == index and t.dim() == 1 and t.is_contiguous():
        return t
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64) or t.get_device() != index:
        raise ValueError(f"{what}: {name} must be 1-D int32 on cuda:{index}")
    return _lib.indices(t)


def _rows16(t: torch.Tensor):
    """The strides of a 16-bit tensor if every row of its last dimension is in one piece that starts on 16 bytes (0 for
    dimensions of one), else None."""
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0:
        for s in st[:-1]:
            if s % 8:
                break
        else:
            return st
    if (st[-1] != 1 and t.shape[-1] > 1) or t.data_ptr() % 16:
        return None
    st = tuple(0 if n <= 1 else s for n, s in zip(t.shape, st))
    return None if any(s % 8 for s in st[:-1]) else st


def tree_attention(q: torch.Tensor, kv_cache: torch.Tensor, qo_indptr: torch.Tensor, kv_page_indices: torch.Tensor,
                   kv_page_indptr: torch.Tensor, kv_last_page_len: torch.Tensor, tree_masks: torch.Tensor, page_size: int,
                   *, sm_scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                   return_lse: bool = False):
    """Attention of the trees' tokens ``q`` ``[T, H_q, D]`` over ``kv_cache`` ``[P, 2, page, H_kv, D]`` (bf16 or fp16, D 64 or
    128, pages of 16 to 1,024 tokens by powers of two; up to 2^20 tokens and rows), which holds them already: row ``b`` has
    tokens ``qo_indptr[b]`` to ``qo_indptr[b + 1]`` and the pages ``kv_page_indices[kv_page_indptr[b] : kv_page_indptr[b + 1]]``,
    the last one filled to ``kv_last_page_len[b]``; its last keys are its tokens'. ``tree_masks`` int64 ``[T, W]`` has bit ``j % 64`` of word ``j // 64``
    set where a token sees its row's token ``j`` (itself among them); all cached keys before the tree are seen.

    Returns ``out``, with ``return_lse`` and the base-2 ``lse`` fp32 ``[T, H_q]``: new ones, or the tensors given, whose memory from
    first to last value must lie apart from that of q, of the cache and of each other. A token that sees no key gets zeros and
    ``-inf``. Keys that a token does not see do not touch it, whatever they hold. Tokens of no row are left as they were. Sums and
    softmax are fp32; weights of keys, up to 2^8 of the row's largest, are rounded to q's type for the product with v (values of v of
    2^100 and more may overflow on the way). The launch goes by the mean tokens of a row: rows without tokens are better left out,
    ``kv_last_page_len[:requests]``, where their number is known (32 requests of 16 tokens over 32,768 take twice as long with 32
    empty rows behind them). Not differentiable."""
    what = "tree_attention"
    index, dtype, shape, cs = q.get_device(), q.dtype, q.shape, kv_cache.shape
    if index < 0:
        _lib.require_cuda(q, what=what)
    if torch.is_grad_enabled() and (q.requires_grad or kv_cache.requires_grad or out is not None and out.requires_grad
                                    or lse is not None and lse.requires_grad) \
            or forward_ad._current_level >= 0 and _lib.has_tangent(q, kv_cache, out, lse):
        raise ValueError(f"{what}: not differentiable")
    code = _DTYPES.get(dtype)
    if code is None or len(shape) != 3 or shape[2] not in HEAD_DIMS or (qs := _rows16(q)) is None:
        raise ValueError(f"{what}: q must be bf16 or fp16 [T, H_q, 64 or 128] with 16-byte aligned heads")
    tokens, hq, dim = shape
    if kv_cache.dtype is not dtype or kv_cache.get_device() != index or len(cs) != 5 or cs[1] != 2 or cs[2] != page_size \
            or cs[4] != dim or (c := _rows16(kv_cache)) is None:
        raise ValueError(f"{what}: kv_cache must be {dtype} [P, 2, {page_size}, H_kv, {dim}] on {q.device} with 16-byte aligned heads")
    if cs[3] < 1 or hq % cs[3]:
        raise ValueError(f"{what}: q heads must be a multiple of the kv heads")
    ms, mst = tree_masks.shape, tree_masks.stride()
    if tree_masks.dtype is not torch.int64 or len(ms) != 2 or ms[0] < tokens or tree_masks.get_device() != index \
            or (ms[1] > 1 and mst[1] != 1):
        raise ValueError(f"{what}: tree_masks must be int64 [T, words] on {q.device} with contiguous rows")
    qo, ind = _list(qo_indptr, index, what, "qo_indptr"), _list(kv_page_indices, index, what, "kv_page_indices")
    ptr, last = _list(kv_page_indptr, index, what, "kv_page_indptr"), _list(kv_last_page_len, index, what, "kv_last_page_len")
    rows = last.shape[0]
    if qo.shape[0] <= rows or ptr.shape[0] <= rows:
        raise ValueError(f"{what}: qo_indptr and kv_page_indptr need len(kv_last_page_len) + 1 entries")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=q.device)
        os = out.stride()
    elif out.shape != shape or out.dtype is not dtype or out.get_device() != index or (os := _rows16(out)) is None:
        raise ValueError(f"{what}: out must be {dtype} of q's shape on {q.device} with 16-byte aligned heads")
    else:
        if tokens > 1 and os[0] == 0 or hq > 1 and os[1] == 0 or not (out.is_contiguous() or _apart(shape, os)):
            raise ValueError(f"{what}: the rows of out share memory")
        o0, o1 = _lib.extent(out, os)
        for t, st in ((q, qs), (kv_cache, c)):
            t0, t1 = _lib.extent(t, st)
            if o0 < t1 and t0 < o1:
                raise ValueError(f"{what}: out must lie apart from q and the cache")
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.shape != (tokens, hq) or lse.get_device() != index or not lse.is_contiguous():
            raise ValueError(f"{what}: lse must be a contiguous fp32 [T, H_q] tensor on {q.device}")
        l0, l1 = _lib.extent(lse, lse.stride())
        for t, st in ((q, qs), (kv_cache, c), (out, os)):
            t0, t1 = _lib.extent(t, st)
            if l0 < t1 and t0 < l1:
                raise ValueError(f"{what}: lse must lie apart from q, the cache and out")
    elif return_lse:
        lse = torch.empty(tokens, hq, dtype=torch.float32, device=q.device)
    L, ws, at = _lib.lib(), None, 0
    floats = L.aspire_tree_attention_workspace(tokens, rows, hq, cs[3], dim)
    if floats:  # the call's own, from torch's pool: calls on several streams or in several graphs share none
        ws = torch.empty(floats, dtype=torch.float32, device=q.device)
        at = ws.data_ptr()
    args = _ARGS.pack(q.data_ptr(), qs[0], qs[1], kv_cache.data_ptr(), c[0], c[1], c[2], c[3], cs[0], ind.shape[0], qo.data_ptr(),
                      ind.data_ptr(), ptr.data_ptr(), last.data_ptr(), tree_masks.data_ptr(), mst[0], out.data_ptr(), os[0], os[1],
                      0 if lse is None else lse.data_ptr(), tokens, rows, ms[1], hq, cs[3], dim, page_size, code,
                      dim ** -0.5 if sm_scale is None else float(sm_scale), 0, at, floats)
    _lib.launch(L.aspire_tree_attention, index, what, args)
    return (out, lse) if return_lse else out


def compact_accepted(kv_caches, path: torch.Tensor, kept: torch.Tensor, qo_indptr: torch.Tensor, slots: torch.Tensor) -> None:
    """Move each kept token's K and V rows from its slot to that of its place in the path, in place: the row at
    ``slots[qo_indptr[b] + path[b, j]]`` goes to ``slots[qo_indptr[b] + j]`` for ``j < kept[b]``, in every layer.

    ``kv_caches``: one cache ``[P, 2, page, H, D]``, all layers' as ``[L, P, 2, page, H, D]``, or a list of caches of one layout
    (any element type; no two may share memory). ``path`` int32 ``[B, M]`` and ``kept`` int32 ``[B]`` are what
    ``verify_tree_speculation`` returns, ``slots`` int64 ``[T]`` what the step's tables hold. A path rises: entries that are not
    above their place, or not of the row, are passed over, and so are slots outside the cache."""
    what = "compact_accepted"
    index = path.get_device()
    if index < 0:
        _lib.require_cuda(path, what=what)
    stacked = isinstance(kv_caches, torch.Tensor)
    layers = [kv_caches] if stacked else list(kv_caches)
    if not layers:
        return
    c = layers[0]
    cs, st, es, dtype = c.shape, c.stride(), c.element_size(), c.dtype
    if len(cs) == 6 and stacked:
        count, step, cs, st = cs[0], st[0] * es, cs[1:], st[1:]
    else:
        count, step = len(layers), 0
    if len(cs) != 5 or cs[1] != 2 or (cs[4] > 1 and st[4] != 1) or cs[2] < 1:
        raise ValueError(f"{what}: the caches must be [P, 2, page, H, D], or stacked as [L, P, 2, page, H, D], with contiguous head dims")
    table = None
    for t in layers:
        if t.get_device() != index:
            _lib.require_cuda(t, what=what)
            raise ValueError(f"{what}: a cache is on {t.device}, path on {path.device}")
        if t.requires_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0 and _lib.has_tangent(t):
            raise ValueError(f"{what}: not differentiable")
    if not stacked:
        if any(t.shape != cs or t.stride() != st or t.dtype is not dtype for t in layers):
            raise ValueError(f"{what}: the caches must be of one layout and type")
        starts = [t.data_ptr() for t in layers]
        table = (ctypes.c_uint64 * count)(*starts)
        if count > 1 and c.numel() and not _starts_apart(starts, cs, st, es):
            raise ValueError(f"{what}: the caches share memory")
    if not (c.is_contiguous() or _apart(c.shape, c.stride())):
        raise ValueError(f"{what}: parts of a cache share memory")
    if path.dim() != 2 or path.dtype is not torch.int32 or not path.is_contiguous():
        raise ValueError(f"{what}: path must be a contiguous int32 [B, M] tensor")
    kept, qo = _list(kept, index, what, "kept"), _list(qo_indptr, index, what, "qo_indptr")
    rows, most = path.shape
    if kept.shape[0] != rows or qo.shape[0] <= rows:
        raise ValueError(f"{what}: kept needs {rows} entries and qo_indptr {rows + 1}")
    if slots.dim() != 1 or slots.dtype is not torch.int64 or slots.get_device() != index:
        raise ValueError(f"{what}: slots must be int64 [T] on {path.device}")
    slots = slots.contiguous()
    args = _MOVE.pack(0 if table is None else ctypes.addressof(table), c.data_ptr(), step, st[0] * es, st[1] * es, st[2] * es, st[3] * es,
                      cs[0], path.data_ptr(), kept.data_ptr(), qo.data_ptr(), slots.data_ptr(), count, cs[3], cs[4] * es, cs[2], rows,
                      slots.shape[0], most, 0)
    _lib.launch(_lib.lib().aspire_compact_accepted, index, what, args)


def _apart(shape, strides) -> bool:
    """Whether no two elements share memory, by the dimensions in the order of their strides."""
    reach = 0
    for s, n in sorted((s, n) for n, s in zip(shape, strides) if n > 1):
        if s <= reach:
            return False
        reach += (n - 1) * s
    return True


def _starts_apart(starts, shape, strides, es: int) -> bool:
    """Whether tensors of one layout at these addresses share no memory: they lie behind each other, or interleaved at equal
    distances (layers inside of pages)."""
    starts = sorted(starts)
    gaps = [b - a for a, b in zip(starts, starts[1:])]
    least = min(gaps)
    if least >= (1 + sum((n - 1) * s for n, s in zip(shape, strides))) * es:
        return True
    return max(gaps) == least and least > 0 and least % es == 0 and _apart((len(starts), *shape), (least // es, *strides))


__all__ = ["HEAD_DIMS", "tree_attention", "compact_accepted"]
