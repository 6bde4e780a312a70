"""Drafted trees, page pools and logits in plain Python and 64-bit numpy: what the kernels are compared with."""

import numpy as np
import torch


def ancestors(parents):
    """[n, n] truth: a node's ancestors and itself; an index that is not below its node's is no parent."""
    n = len(parents)
    see = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            see[i] = see[p]
        see[i, i] = True
    return see


def pack(see, words):
    """Bits of [n, m] truth as int64 [n, words]."""
    bits = np.zeros((see.shape[0], words * 64), dtype=np.uint8)
    m = min(see.shape[1], words * 64)
    bits[:, :m] = see[:, :m]
    return np.packbits(bits, axis=1, bitorder="little").view(np.int64).reshape(see.shape[0], words)


def random_tree(n, r, branch=0.6):
    """Parents of a tree of n nodes, parents first."""
    return [-1] + [i - 1 if r.random() > branch else int(r.integers(0, i)) for i in range(1, n)] if n else []


def attention(q, cache, qo, kvp, ids, last, masks, scale=None):
    """(out, lse base 2, weighted |v|, largest sum of |q k| of a seen key) in 64 bits, on the CPU; rows of no request are NaN.
    Bits beyond a row's tokens are not seen, nor are keys on pages or entries outside."""
    q, cache = q.detach().cpu().double().numpy(), cache.detach().cpu().double().numpy()
    masks = masks.cpu().numpy().view(np.uint64)
    T, hq, d = q.shape
    pages, _, page, hkv, _ = cache.shape
    group, scale = hq // hkv, d ** -0.5 if scale is None else scale
    out, size = np.full((T, hq, d), np.nan), np.full((T, hq, d), np.nan)
    lse, most = np.full((T, hq), np.nan), np.zeros((T, hq))
    for b in range(len(last)):
        n, first = qo[b + 1] - qo[b], kvp[b]
        np_ = kvp[b + 1] - first
        length = (np_ - 1) * page + last[b] if np_ > 0 else 0
        key = np.arange(length)
        entry = first + key // page
        inside = (entry >= 0) & (entry < len(ids))
        pid = np.where(inside, np.asarray(ids)[np.clip(entry, 0, max(len(ids) - 1, 0))] if len(ids) else -1, -1)
        there = (pid >= 0) & (pid < pages)
        pid = np.where(there, pid, 0)
        k = cache[pid, 0, key % page] if length else np.zeros((0, hkv, d))
        v = cache[pid, 1, key % page] if length else np.zeros((0, hkv, d))
        for i in range(n):
            t, see = qo[b] + i, there.copy()
            for j in range(max(0, length - n), length):
                node = j - (length - n)
                word = masks[t, node // 64] if node // 64 < masks.shape[1] else np.uint64(0)
                see[j] &= bool((int(word) >> (node % 64)) & 1)
            for h in range(hq):
                g = h // group
                ks, vs = k[see, g], v[see, g]
                if not see.any():
                    out[t, h], size[t, h], lse[t, h] = 0, 0, -np.inf
                    continue
                x = scale * (ks @ q[t, h])
                most[t, h] = np.nanmax(scale * (np.abs(ks) @ np.abs(q[t, h])))
                w = np.exp(x - x.max())
                out[t, h], size[t, h] = w @ vs / w.sum(), w @ np.abs(vs) / w.sum()
                lse[t, h] = (x.max() + np.log(w.sum())) / np.log(2)
    return out, lse, size, most


def attention_limit(out, size, most, dtype, keys, dim):
    """How far an output may be off. A weight is off by half a step of its type for the product with v, by twice the error of its score (a
    sum of dim products, each and each partial sum rounded to 2^-24 of what it adds up to, and some roundings of the scaled
    score), and by the sum's (keys + 64 additions of positive numbers and some joins of parts); the output is rounded once. Weights that
    fp16 cannot hold as normal numbers are off by 2^-25 of 2^-7 of the largest at most, each."""
    half = torch.finfo(dtype).eps / 2
    weight = half + 2 * (dim + 8) * 2.0 ** -24 * most[..., None] + 2 * (keys + 64) * 2.0 ** -24
    bound = size * weight * 1.01 + (keys * 2.0 ** -30 * 8 if dtype == torch.float16 else 0)
    return bound + half * (np.abs(out) + bound) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133)


def lse_limit(lse, most, keys, dim):
    """Base-2 logarithm of the sum: the errors above without the weights' rounding, one rounding of the result and three of the
    largest score."""
    return 1.45 * ((dim + 8) * 2.0 ** -24 * most + (keys + 64) * 2.0 ** -24) + 2.0 ** -22 * (np.abs(lse) + 8)


class Pool:
    """The page pool in plain Python."""

    def __init__(self, num_pages, page, rows, width):
        self.page, self.width = page, width
        self.rows = [[] for _ in range(rows)]
        self.stack = list(range(num_pages - 1, -1, -1))
        self.pages = num_pages

    def resize(self, lengths):
        want = [len(r) if n < 0 else -(-n // self.page) for n, r in zip(lengths, self.rows)]
        back = []
        for r, w in zip(self.rows, want):
            back += r[w:]
            del r[w:]
        self.stack += back[::-1]
        short, stop = [0] * len(want), False
        for b, (r, w) in enumerate(zip(self.rows, want)):
            lack = max(0, w - len(r))
            if lack and (w > self.width or lack > len(self.stack)):
                stop = True
            if stop:
                short[b] = lack
                continue
            r += [self.stack.pop() for _ in range(lack)]
        return short

    def table(self):
        return [r + [-1] * (self.width - len(r)) for r in self.rows]


def tables(table, cached, fresh, parents, page, max_rows, max_tokens, max_entries, words):
    """(qo_indptr, kv_indptr, kv_indices, last_page_len, positions, slots, masks, totals) in plain Python."""
    ok = [c >= 0 and f >= 0 and c + f < 2 ** 31 for c, f in zip(cached, fresh)]
    fresh = [f if good else 0 for f, good in zip(fresh, ok)]
    need = [-(-(c + f) // page) if f else 0 for c, f in zip(cached, fresh)]
    qo, kvp, ids, last = [0], [0], [], [0] * max_rows
    positions, slots, masks = [-1] * max_tokens, [-1] * max_tokens, np.zeros((max_tokens, words), np.int64)
    left, most = len(fresh), 64 * words if words else 2 ** 31 if parents is None else 4096
    for b, (c, f, p) in enumerate(zip(cached, fresh, need)):
        if left < b or qo[-1] + f > max_tokens or kvp[-1] + p > max_entries or f > most:
            left = min(left, b)
            f = p = 0
        row = [table[b][i] if i < len(table[b]) else -1 for i in range(p)]
        ids += row
        last[b] = c + f - (p - 1) * page if p else 0
        at = qo[-1]
        up = [i - 1 for i in range(f)] if parents is None else [int(x) for x in parents[at : at + f]]
        see = ancestors(up)
        for i in range(f):
            page_id = row[(c + i) // page]
            positions[at + i] = c + int(see[i].sum()) - 1
            slots[at + i] = page_id * page + (c + i) % page if page_id >= 0 else -1
        if words and f:
            masks[at : at + f] = pack(see, words)
        qo.append(at + f)
        kvp.append(kvp[-1] + p)
    qo += [qo[-1]] * (max_rows + 1 - len(qo))
    kvp += [kvp[-1]] * (max_rows + 1 - len(kvp))
    return qo, kvp, ids, last, positions, slots, masks, [sum(fresh), sum(need), left]


def accept(tokens, parents, targets, qo, max_path):
    """(output, path, kept) in plain Python."""
    outs, paths, kept = [], [], []
    for a, e in zip(qo[:-1], qo[1:]):
        a, e = max(a, 0), min(e, len(tokens))
        path, cur = [], 0 if e > a else None
        while cur is not None and len(path) < max_path:
            path.append(cur)
            cur = next((i for i in range(cur + 1, e - a) if parents[a + i] == cur and tokens[a + i] == targets[a + cur]), None)
        pad = [-1] * (max_path - len(path))
        paths.append(path + pad)
        outs.append([targets[a + i] for i in path] + pad)
        kept.append(len(path))
    return outs, paths, kept


def adjusted(logits, qo=None, history=None, lens=None, prompts=None, rep=None, pres=None, freq=None, tree=None, see=None,
             bias=None, allowed=None, start=0):
    """The definition in 64 bits (float32 parameters as they are); see [T, n] truth over a row's own tokens, allowed [T, V] truth."""
    y = logits.detach().cpu().double().numpy().copy()
    T, V = y.shape
    touched = np.zeros((T, V), dtype=bool)
    size = np.abs(np.where(np.isfinite(y), y, 0))
    qo = list(range(T + 1)) if qo is None else qo
    for b in range(len(qo) - 1):
        for t in range(max(qo[b], 0), min(qo[b + 1], T)):
            touched[t] = True
            out, prompt = np.zeros(V), np.zeros(V, bool)
            def at(ids):
                ids = np.asarray(ids, dtype=np.int64) - start
                return ids[(ids >= 0) & (ids < V)]
            if history is not None:
                n, told = min(int(lens[b]), history.shape[1]), 0 if prompts is None else int(prompts[b])
                h = np.asarray(history[b])[: max(n, 0)]
                prompt[at(h[: max(told, 0)])] = True
                np.add.at(out, at(h[max(told, 0):]), 1)
            if tree is not None:
                mine = np.asarray(tree)[max(qo[b], 0) : min(qo[b + 1], T)]
                on = see[t][: len(mine)]
                np.add.at(out, at(mine[: len(on)][on]), 1)
            known = prompt | (out > 0)
            if history is not None or tree is not None:
                r = 1.0 if rep is None else float(rep[b])
                with np.errstate(invalid="ignore"):
                    y[t] = np.where(known, np.where(y[t] > 0, y[t] / r, y[t] * r), y[t])
                size[t] = np.maximum(size[t], np.abs(np.where(np.isfinite(y[t]), y[t], 0)))
                f, p = (0.0 if x is None else float(x[b]) for x in (freq, pres))
                y[t] -= f * out + p * (out > 0)
                size[t] += np.abs(f) * out + np.abs(p) * (out > 0)
            if bias is not None:
                for token, value in (bias[b] or {}).items():
                    if 0 <= token - start < V:
                        y[t, token - start] += float(np.float32(value))
                        size[t, token - start] += abs(value) if np.isfinite(value) else 0
            if allowed is not None:
                y[t] = np.where(allowed[t], y[t], -np.inf)
    return y, touched, size
