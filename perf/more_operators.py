"""Operators of a step that drafts and verifies a tree of tokens for each request, as cases that can be timed and
compared:

* ``tree``    attention of the trees' tokens over the paged cache: a token sees its request's cached tokens and its own
              ancestors;
* ``logits``  penalties for repeated tokens, biases and grammar masks on the logits of requests' tokens, or of trees',
              whose ancestors count as output;
* ``tables``  the pages of requests that grew, and a step's page lists, slots, positions and masks, from lengths;
* ``accept``  the accepted path of each tree, and its rows of every layer's cache moved to where they stay.

Sizes are the benchmark's and the tests' (heads 32/8 and 16/8 of 128, 36 layers, contexts to 32,768, batches to 64 and
steps of 208 tokens, 151,936 vocabulary entries, 16-token pages), or generic ones of other models.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one request with a small tree behind a short conversation: latency
        {"name": "tree_chat", "kind": "tree", "rows": 1, "nodes": 8, "even": True, "ctx": 2048, "hq": 16, "hkv": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "rows_seed": 0},
        # a batch of uneven trees over uneven contexts, the benchmark's heads
        {"name": "tree_batch", "kind": "tree", "rows": 16, "nodes": 40, "even": False, "ctx": 8192, "hq": 32, "hkv": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "rows_seed": 1},
        # the benchmark's 32 requests of 32,768 tokens: a stream of keys and values
        {"name": "tree_long", "kind": "tree", "rows": 32, "nodes": 16, "even": True, "ctx": 32768, "hq": 32, "hkv": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "rows_seed": 2},
        # few requests with large trees, five query heads to a key head: products
        {"name": "tree_wide", "kind": "tree", "rows": 5, "nodes": 190, "even": False, "ctx": 12001, "hq": 40, "hkv": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "rows_seed": 3},
        # half as wide heads in fp16 on larger pages
        {"name": "tree_narrow", "kind": "tree", "rows": 24, "nodes": 33, "even": False, "ctx": 5000, "hq": 14, "hkv": 2,
         "dim": 64, "page": 32, "dtype": "fp16", "rows_seed": 4},
        # one request's next token: penalties and a few biases, latency
        {"name": "logits_token", "kind": "logits", "rows": 1, "nodes": 0, "vocab": 32000, "history": 700,
         "penalties": True, "bias": 12, "grammar": False, "dtype": "fp32", "rows_seed": 5},
        # 64 requests that write structured text after long prompts, one token each
        {"name": "logits_batch", "kind": "logits", "rows": 64, "nodes": 0, "vocab": 151936, "history": 8192,
         "penalties": True, "bias": 0, "grammar": True, "dtype": "bf16", "rows_seed": 6},
        # 16 trees of up to 24 tokens, every path with its own repetitions, an odd vocabulary
        {"name": "logits_tree", "kind": "logits", "rows": 16, "nodes": 24, "vocab": 128257, "history": 20000,
         "penalties": True, "bias": 100, "grammar": True, "dtype": "bf16", "rows_seed": 7},
        # four requests, one token each
        {"name": "tables_decode", "kind": "tables", "rows": 4, "nodes": 1, "tree": False, "ctx": 4096, "page": 16,
         "rows_seed": 8},
        # the benchmark's 64 rows of long contexts with trees of up to 16 tokens
        {"name": "tables_step", "kind": "tables", "rows": 64, "nodes": 16, "tree": True, "ctx": 32768, "page": 16,
         "rows_seed": 9},
        # four requests on a model of 28 layers, small trees
        {"name": "accept_small", "kind": "accept", "rows": 4, "nodes": 12, "layers": 28, "hkv": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "rows_seed": 10},
        # 64 requests on the benchmark's 36 layers
        {"name": "accept_step", "kind": "accept", "rows": 64, "nodes": 48, "layers": 36, "hkv": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "rows_seed": 11},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "logits", "logits", "tables", "accept"])
    c = {"kind": kind, "rows_seed": rng.randrange(1 << 20)}
    if kind == "tree":
        hq, hkv = rng.choice([(32, 8), (16, 8), (40, 8), (64, 8), (8, 8), (14, 2), (7, 1)])
        dim = rng.choice([64, 128, 128])
        ctx = _log(rng, 1, 32768)
        rows = _log(rng, 1, max(1, min(64, 32 * 32768 * 8 * 128 // (ctx * hkv * dim))))
        nodes = _log(rng, 1, max(1, min(256, 700_000_000_000 // (4 * rows * ctx * hq * dim))))
        c.update(rows=rows, nodes=nodes, even=rng.random() < 0.4, ctx=ctx, hq=hq, hkv=hkv, dim=dim,
                 page=rng.choice([16, 16, 16, 32, 64]), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    elif kind == "logits":
        vocab = _log(rng, 1000, 160000)
        rows = rng.randint(1, 64)
        nodes = rng.choice([0, 0, _log(rng, 1, 64)])
        while rows * max(1, nodes) * vocab > 48_000_000:
            rows = max(1, rows // 2)
            nodes = nodes // 2
        penalties, grammar = rng.random() < 0.8, rng.random() < 0.5
        c.update(rows=rows, nodes=nodes, vocab=vocab, history=_log(rng, 1, 32768), penalties=penalties,
                 bias=rng.choice([0, 1, _log(rng, 2, 300)]) if penalties or grammar else 17, grammar=grammar,
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    elif kind == "tables":
        c.update(rows=rng.randint(1, 128), nodes=_log(rng, 1, 64), tree=rng.random() < 0.5, ctx=_log(rng, 1, 32768),
                 page=rng.choice([16, 16, 32, 64]))
    else:
        rows, layers = rng.randint(1, 64), rng.randint(1, 48)
        hkv, dim = rng.choice([(8, 128), (2, 64), (1, 128), (4, 80)])
        while rows * layers > 36 * 64:
            rows //= 2
        c.update(rows=rows, nodes=_log(rng, 1, 48), layers=layers, hkv=hkv, dim=dim, page=rng.choice([16, 16, 32]),
                 dtype=rng.choice(["bf16", "fp16"]))
    return c


# ------------------------------------------------------------------------- what a case's trees are
def _trees(c):
    """Parents (numpy, -1 for the root, each before its children) of each request's tree: the likeliest chain first,
    then branches off it that are no longer than it."""
    r = np.random.default_rng(c["rows_seed"])
    trees = []
    for b in range(c["rows"]):
        n = c["nodes"] if c.get("even") else int(r.integers(1, c["nodes"] + 1))
        chain = min(n, max(1, int(round(n ** 0.6))))
        parents, depth = list(range(-1, chain - 1)), list(range(chain))
        while len(parents) < n:
            inner = [i for i in range(len(parents)) if depth[i] + 1 < chain] or [0]
            p = inner[int(r.integers(0, len(inner)))]
            parents.append(p)
            depth.append(depth[p] + 1)
        trees.append(np.array(parents, dtype=np.int64))
    return trees


def _contexts(c):
    """Cached tokens of each request, before its tree."""
    r = np.random.default_rng(c["rows_seed"] + 1)
    if c.get("even"):
        return np.full(c["rows"], max(0, c["ctx"] - c["nodes"]), dtype=np.int64)
    return r.integers(c["ctx"] // 4, c["ctx"] + 1, size=c["rows"]).astype(np.int64)


def _sees(parents):
    """[n, n] truth: a node's ancestors and itself."""
    n = len(parents)
    see = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see


def _words(trees):
    return max(1, max((len(t) + 63) // 64 for t in trees))


def _packed(trees):
    """The nodes' ancestors as bits: int64 [T, W], bit j of a row for its request's node j."""
    words = _words(trees)
    out = []
    for t in trees:
        bits = np.zeros((len(t), words * 64), dtype=np.uint8)
        bits[:, : len(t)] = _sees(t)
        out.append(np.packbits(bits, axis=1, bitorder="little").view(np.int64))
    return np.concatenate(out)


def _ptr(a):
    return np.concatenate([[0], np.cumsum(a)]).astype(np.int64)


# ---------------------------------------------------------------------------------- the inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, gen, dtype, std=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        piece = flat[at : at + (1 << 28)]
        piece.copy_(torch.empty(piece.numel(), dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen))
    return out


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def _tree_inputs(c, seed):
    gen, dtype = _gen(seed), TYPES[c["dtype"]]
    trees, cached = _trees(c), _contexts(c)
    new = np.array([len(t) for t in trees])
    length = cached + new
    pages = (length + c["page"] - 1) // c["page"]
    order = np.random.default_rng(seed + 77).permutation(int(pages.sum()))
    tokens, hq, hkv, d = int(new.sum()), c["hq"], c["hkv"], c["dim"]
    qkv = _normal((tokens, (hq + 2 * hkv) * d), gen, dtype)  # q as a view of the fused projection
    cache = _normal((int(pages.sum()), 2, c["page"], hkv, d), gen, dtype)
    return {"q": qkv[:, : hq * d].view(tokens, hq, d), "cache": cache, "qo_indptr": _dev(_ptr(new)),
            "page_indices": _dev(order), "page_indptr": _dev(_ptr(pages)),
            "last_page_len": _dev((length - 1) % c["page"] + 1), "masks": _dev(_packed(trees), torch.int64),
            "lengths": length.tolist(), "new": new.tolist()}


def _logits_inputs(c, seed):
    """Logits as a model has them; histories in which few tokens are frequent; a mask that leaves some hundred tokens or
    most of the vocabulary."""
    gen, dtype, r = _gen(seed), TYPES[c["dtype"]], np.random.default_rng(seed + 5)
    rows, vocab = c["rows"], c["vocab"]
    trees = _trees(c) if c["nodes"] else [np.array([-1])] * rows
    tokens = sum(len(t) for t in trees)
    frequent = lambda *shape: (torch.rand(*shape, device="cuda", generator=gen) ** 6 * vocab).to(torch.int32).clamp_(max=vocab - 1)
    s = {"logits": _normal((tokens, vocab), gen, dtype, 3.0)}
    if c["nodes"]:
        s["qo_indptr"] = _dev(_ptr([len(t) for t in trees]))
        s["tree_tokens"], s["masks"] = frequent(tokens), _dev(_packed(trees), torch.int64)
    if c["penalties"]:
        s["history"] = frequent(rows, c["history"])
        lens = np.random.default_rng(c["rows_seed"] + 2).integers(c["history"] // 2, c["history"] + 1, size=rows)
        s["history_lens"] = _dev(lens)
        s["prompt_lens"] = _dev(r.integers(0, lens + 1))
        s["repetition"] = torch.rand(rows, device="cuda", generator=gen) * 0.5 + 1.0
        s["presence"] = torch.rand(rows, device="cuda", generator=gen)
        s["frequency"] = torch.rand(rows, device="cuda", generator=gen) * 0.5
    if c["bias"]:
        s["bias"] = [{int(i): float(v) for i, v in zip(r.choice(vocab, size=min(c["bias"], vocab), replace=False),
                                                       r.normal(0.0, 5.0, size=c["bias"]))} for _ in range(rows)]
    if c["grammar"]:
        words = (vocab + 31) // 32
        full = torch.randint(-2 ** 31, 2 ** 31, (tokens, words), device="cuda", generator=gen)
        sparse = full & torch.randint(-2 ** 31, 2 ** 31, (tokens, words), device="cuda", generator=gen)
        for _ in range(6):
            sparse &= torch.randint(-2 ** 31, 2 ** 31, (tokens, words), device="cuda", generator=gen)
        narrow = torch.rand(tokens, 1, device="cuda", generator=gen) < 0.5
        s["grammar"] = torch.where(narrow, sparse, ~sparse).to(torch.int32)
    return s


def _tables_inputs(c, seed):
    """Requests that hold the pages of their cached tokens, the others on the stack of free pages."""
    r = np.random.default_rng(seed)
    trees, cached = _trees(c), _contexts(c)
    new = np.array([len(t) for t in trees])
    page, rows = c["page"], c["rows"]
    held, need = -(-cached // page), -(-(cached + new) // page)
    width, total = int(need.max()) + 3, int(need.sum()) + 5
    order = r.permutation(total).astype(np.int32)
    table, at = np.full((rows, width), -1, dtype=np.int32), 0
    for b in range(rows):
        table[b, : held[b]] = order[at : at + held[b]]
        at += int(held[b])
    free = np.full(total, -1, dtype=np.int32)
    free[: total - at] = order[at:]
    parents = np.concatenate(trees) if c["tree"] else None
    return {"table": _dev(table), "held": _dev(held), "free": _dev(free), "free_count": total - at,
            "cached": _dev(cached), "new": _dev(new), "wanted": _dev(cached + new),
            "parents": None if parents is None else _dev(parents), "tokens": int(new.sum()), "entries": int(need.sum()),
            "words": _words(trees), "levels": 1 + max(int(_sees(t).sum(1).max()) for t in trees)}


def _accept_inputs(c, seed):
    """Trees behind a few cached tokens in every layer's pages; targets that follow the tree for a while."""
    gen, dtype, r = _gen(seed), TYPES[c["dtype"]], np.random.default_rng(seed)
    trees = _trees(c)
    page, most = c["page"], max(len(t) for t in trees)
    pages = (most + 2 * page - 1) // page
    order = r.permutation(c["rows"] * pages)
    parents, tokens, targets, slots = [], [], [], []
    for b, t in enumerate(trees):
        n, start = len(t), int(r.integers(0, page))
        tok = r.integers(0, 151936, size=n)
        for i in range(n):  # siblings differ
            while i and any(tok[j] == tok[i] and t[j] == t[i] for j in range(1, i)):
                tok[i] = int(r.integers(0, 151936))
        tgt = r.integers(151936, 152000, size=n)  # no drafted token
        for i in range(n):
            children = np.flatnonzero(t == i)
            if len(children) and r.random() < 0.8:
                tgt[i] = tok[children[int(r.integers(0, len(children)))]]
        place = start + np.arange(n)
        slots.append(order[b * pages + place // page] * page + place % page)
        parents.append(t), tokens.append(tok), targets.append(tgt)
    count = [len(t) for t in trees]
    return {"parents": _dev(np.concatenate(parents)), "tokens": _dev(np.concatenate(tokens)),
            "targets": _dev(np.concatenate(targets)), "qo_indptr": _dev(_ptr(count)),
            "slots": _dev(np.concatenate(slots), torch.int64), "most": most, "count": count,
            "cache": _normal((c["layers"], c["rows"] * pages, 2, page, c["hkv"], c["dim"]), gen, dtype)}


def prepare(case, seed):
    c = case
    s = {"tree": _tree_inputs, "logits": _logits_inputs, "tables": _tables_inputs, "accept": _accept_inputs}[c["kind"]](c, seed)
    s["case"] = c
    if c["kind"] == "tree":
        s["out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    if c["kind"] == "logits":
        s["out"] = torch.empty_like(s["logits"])
        if c["bias"]:
            if own:
                from aspire_amd.logits_processor import LogitBias

                s["bias"] = LogitBias(s["bias"], "cuda")
            else:
                s["bias_row"] = _dev(np.repeat(np.arange(c["rows"]), [len(m) for m in s["bias"]]), torch.int64)
                s["bias_ids"] = _dev(np.array([i for m in s["bias"] for i in m]), torch.int64)
                s["bias_values"] = _dev(np.array([v for m in s["bias"] for v in m.values()]), torch.float32)
    if c["kind"] == "tables":
        if own:
            from aspire_amd.attention.paging import PagePool, StepTables

            s["pool"] = PagePool(s["free"].shape[0], c["page"], c["rows"], s["table"].shape[1], "cuda")
            s["pool"].block_table.copy_(s["table"])
            s["pool"].held.copy_(s["held"])
            s["pool"].free.copy_(s["free"])
            s["pool"].free_count.fill_(s["free_count"])
            s["tables"] = StepTables(c["rows"], s["tokens"], s["entries"], c["page"], "cuda",
                                     tree_words=s["words"] if c["tree"] else 0)
        else:
            s["free_count"] = torch.full((1,), s["free_count"], dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------------------- the plain forms
def _seen_nodes(masks, n):
    """[n, n] truth from a request's packed rows."""
    bit = torch.arange(n, device="cuda")
    return ((masks[:, bit // 64] >> (bit % 64)) & 1).bool()


def _plain_tree(s):
    c = s["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["dim"], c["page"]
    at = first = 0
    for n, length in zip(s["new"], s["lengths"]):
        pages = -(-length // page)
        ids = s["page_indices"][first : first + pages].long()
        kv = s["cache"][ids].float()  # [pages, 2, page, hkv, d]
        k = kv[:, 0].reshape(-1, hkv, d)[:length].permute(1, 2, 0).contiguous()
        v = kv[:, 1].reshape(-1, hkv, d)[:length].permute(1, 0, 2).contiguous()
        q = s["q"][at : at + n].float().view(n, hkv, hq // hkv, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)
        x = torch.bmm(q, k).mul_(d ** -0.5).view(hkv, n, hq // hkv, length)
        hidden = ~_seen_nodes(s["masks"][at : at + n], n)
        x[..., length - n :].masked_fill_(hidden[None, :, None, :], float("-inf"))
        top = x.amax(dim=-1, keepdim=True)
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        p = torch.exp_(x.sub_(top))
        total = p.sum(dim=-1, keepdim=True)
        o = torch.bmm(p.view(hkv, -1, length), v).view(hkv, n, hq // hkv, d)
        o = torch.where(total > 0, o / total, torch.zeros_like(o))
        s["out"][at : at + n] = o.permute(1, 0, 2, 3).reshape(n, hq, d).to(s["out"].dtype)
        at += n
        first += pages
    return s["out"]


def _plain_logits(s):
    c, logits = s["case"], s["logits"]
    tokens, vocab = logits.shape
    x = logits.float()
    if "qo_indptr" in s:
        row = torch.searchsorted(s["qo_indptr"].long(), torch.arange(tokens, device="cuda"), right=True) - 1
    else:
        row = torch.arange(tokens, device="cuda")
    if c["penalties"]:
        place = torch.arange(s["history"].shape[1], device="cuda")[None, :]
        live = place < s["history_lens"][:, None]
        prompt = live & (place < s["prompt_lens"][:, None])
        ids = s["history"].long()
        counts = torch.zeros(c["rows"], vocab, dtype=torch.int32, device="cuda").scatter_add_(1, ids, (live & ~prompt).int())
        known = torch.zeros(c["rows"], vocab, dtype=torch.int32, device="cuda").scatter_add_(1, ids, prompt.int())[row] > 0
        counts = counts[row]
        if c["nodes"]:
            bit = torch.arange(c["nodes"], device="cuda")
            on = ((s["masks"][:, bit // 64] >> (bit % 64)) & 1).int()
            node = (s["qo_indptr"].long()[row][:, None] + bit).clamp_(max=tokens - 1)
            counts.scatter_add_(1, s["tree_tokens"].long()[node], on)
        rep, pres, freq = (s[k][row][:, None] for k in ("repetition", "presence", "frequency"))
        x = torch.where(known | (counts > 0), torch.where(x > 0, x / rep, x * rep), x)
        x = x - freq * counts - pres * (counts > 0)
    if c["bias"]:
        extra = torch.zeros(c["rows"], vocab, device="cuda")
        extra[s["bias_row"], s["bias_ids"]] = s["bias_values"]
        x = x + extra[row]
    if c["grammar"]:
        bit = torch.arange(32, device="cuda", dtype=torch.int32)
        allowed = ((s["grammar"][:, :, None] >> bit) & 1).view(tokens, -1)[:, :vocab] > 0
        x = torch.where(allowed, x, torch.full_like(x, float("-inf")))
    s["out"].copy_(x)
    return s["out"]


def _plain_resize(s, lengths):
    """Rows give back the pages that they no longer need, then take what they lack, in row order; the pages that went
    last come first."""
    page, table, held, free = s["case"]["page"], s["table"], s["held"], s["free"]
    want = (lengths + page - 1) // page
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    back = (held - want).clamp_(min=0)
    first = torch.cumsum(back, 0) - back
    total = back.sum()
    going = (col >= want[:, None]) & (col < held[:, None])
    spare = free.shape[0]  # what is not moved goes to a place behind the end
    stack = torch.cat([free, free.new_zeros(1)])
    to = s["free_count"] + total - 1 - (first[:, None] + col - want[:, None])
    stack.scatter_(0, torch.where(going, to, spare).long().view(-1), table.view(-1))
    table = torch.where(going, -1, table)
    held, count = torch.minimum(held, want), s["free_count"] + total
    lack = want - held
    after = torch.cumsum(lack, 0)
    short = (after > count) | (want > table.shape[1])
    short = torch.cumsum(short & (lack > 0), 0) > 0  # from the first row that cannot be served
    lack = torch.where(short, 0, lack)
    first = torch.cumsum(lack, 0) - lack
    taken = (col >= held[:, None]) & (col < (held + lack)[:, None])
    at = torch.where(taken, count - 1 - (first[:, None] + col - held[:, None]), spare).long()
    table = torch.where(taken, stack[at], table)
    stack.scatter_(0, at.view(-1), -1)
    s["table"].copy_(table)
    s["held"].copy_(held + lack)
    s["free"].copy_(stack[:spare])
    s["free_count"].copy_(count - lack.sum())


def _plain_build(s):
    c, page, tokens, entries = s["case"], s["case"]["page"], s["tokens"], s["entries"]
    new, cached = s["new"].long(), s["cached"].long()
    zero = new.new_zeros(1)
    qo = torch.cat([zero, torch.cumsum(new, 0)])
    length = cached + new
    pages = (length + page - 1) // page
    ptr = torch.cat([zero, torch.cumsum(pages, 0)])
    e = torch.arange(entries, device="cuda")
    owner = torch.searchsorted(ptr, e, right=True) - 1
    indices = s["table"][owner, e - ptr[owner]]
    t = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(qo, t, right=True) - 1
    node = t - qo[row]
    place = cached[row] + node
    slots = s["table"][row, place // page].long() * page + place % page
    outs = [qo.int(), ptr.int(), indices, (length - (pages - 1) * page).int()]
    if not c["tree"]:
        return outs + [place.int(), slots]
    masks = torch.zeros(tokens, s["words"], dtype=torch.int64, device="cuda")
    depth, up = torch.full_like(node, -1), node.clone()
    for _ in range(s["levels"]):  # one level of every token's ancestors at a time
        live = up >= 0
        at = up.clamp(min=0)
        masks.scatter_(1, (at // 64)[:, None], (masks.gather(1, (at // 64)[:, None])[:, 0]
                                               | torch.where(live, 1 << (at % 64), 0))[:, None])
        depth += live
        up = torch.where(live, s["parents"].long()[qo[row] + at], up)
    return outs + [(cached[row] + depth).int(), slots, masks]


def _plain_tables(s):
    _plain_resize(s, s["cached"])  # what the last step drafted for nothing
    _plain_resize(s, s["wanted"])
    return [s["table"], s["held"], s["free"], s["free_count"], *_plain_build(s)]


def _plain_accept(s):
    rows, most, qo = s["case"]["rows"], s["most"], s["qo_indptr"].long()
    tokens = s["parents"].shape[0]
    at = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(qo, at, right=True) - 1
    node = at - qo[row]
    cur, live = torch.zeros(rows, dtype=torch.int64, device="cuda"), qo[1:] > qo[:-1]
    path = torch.full((rows, most), -1, dtype=torch.int32, device="cuda")
    output = torch.full((rows, most), -1, dtype=torch.int32, device="cuda")
    for j in range(most):
        target = s["targets"][(qo[:-1] + cur).clamp(max=tokens - 1)]
        path[:, j] = torch.where(live, cur, -1)
        output[:, j] = torch.where(live, target, -1)
        fits = (s["parents"] == cur[row]) & (s["tokens"] == target[row]) & (node > 0)
        best = torch.full((rows,), tokens, dtype=torch.int64, device="cuda")
        best.scatter_reduce_(0, row, torch.where(fits, node, tokens), "amin")
        live = live & (best < tokens)
        cur = torch.where(live, best, cur)
    kept = (path >= 0).sum(1).int()
    page = s["case"]["page"]
    moved = path > torch.arange(most, device="cuda")
    src = s["slots"][(qo[:-1, None] + path.clamp(min=0)).clamp_(max=tokens - 1)]
    dst = s["slots"][(qo[:-1, None] + torch.arange(most, device="cuda")).clamp_(max=tokens - 1)]
    src, dst = torch.where(moved, src, dst).view(-1), dst.view(-1)
    # places that are not moved write nothing new: those behind a short tree's end would, and stay out
    inside = (torch.arange(most, device="cuda")[None, :] < (qo[1:] - qo[:-1])[:, None]).view(-1)
    src, dst = torch.where(inside, src, s["slots"][0]), torch.where(inside, dst, s["slots"][0])
    flat = s["cache"]
    flat[:, dst // page, :, dst % page] = flat[:, src // page, :, src % page]
    return [output, path, kept, s["cache"]]


# --------------------------------------------------------------------------------------- one pass
def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        return _run_own(s, s["case"])
    return {"tree": _plain_tree, "logits": _plain_logits, "tables": _plain_tables, "accept": _plain_accept}[kind](s)


def _run_own(s, c):
    if c["kind"] == "tree":
        from aspire_amd.attention.tree import tree_attention

        return tree_attention(s["q"], s["cache"], s["qo_indptr"], s["page_indices"], s["page_indptr"], s["last_page_len"],
                              s["masks"], c["page"], out=s["out"])
    if c["kind"] == "logits":
        from aspire_amd.logits_processor import adjust_logits

        return adjust_logits(s["logits"], qo_indptr=s.get("qo_indptr"), history=s.get("history"),
                             history_lens=s.get("history_lens"), prompt_lens=s.get("prompt_lens"),
                             repetition=s.get("repetition"), presence=s.get("presence"), frequency=s.get("frequency"),
                             tree_tokens=s.get("tree_tokens"), tree_masks=s.get("masks"), bias=s.get("bias"),
                             grammar=s.get("grammar"), out=s["out"])
    if c["kind"] == "tables":
        pool, t = s["pool"], s["tables"]
        pool.resize(s["cached"])
        pool.resize(s["wanted"])
        t.build(pool.block_table, s["cached"], s["new"], s["parents"])
        outs = [pool.block_table, pool.held, pool.free, pool.free_count, t.qo_indptr, t.kv_indptr, t.kv_indices,
                t.last_page_len, t.positions, t.slots]
        return outs + [t.masks] if c["tree"] else outs
    from aspire_amd.attention.tree import compact_accepted
    from aspire_amd.engine.sampling import verify_tree_speculation

    output, path, kept = verify_tree_speculation(s["tokens"], s["parents"], s["targets"], s["qo_indptr"], s["most"])
    compact_accepted(s["cache"], path, kept, s["qo_indptr"], s["slots"])
    return [output, path, kept, s["cache"]]


# ------------------------------------------------------------------------------------ what it takes
def _accepted(c, seed=0):
    """Accepted nodes that are not in place, as the targets follow the tree 0.8 of the time (the mean of a few draws)."""
    r, total = np.random.default_rng(seed), 0
    for t in _trees(c):
        for _ in range(8):
            node, j = 0, 0
            while True:
                children = np.flatnonzero(t == node)
                if not len(children) or r.random() >= 0.8:
                    break
                node, j = int(children[int(r.integers(0, len(children)))]), j + 1
                total += node > j
    return total / 8


def work(case):
    c = case
    trees = _trees(c) if c["nodes"] else [np.array([-1])] * c["rows"]
    tokens = sum(len(t) for t in trees)
    if c["kind"] == "tree":
        cached = _contexts(c)
        keys = int(cached.sum()) + tokens
        pairs = sum(int(n) * len(t) + int(_sees(t).sum()) for n, t in zip(cached, trees))
        return {"bytes": keys * 2 * c["hkv"] * c["dim"] * 2 + 4 * tokens * c["hq"] * c["dim"] + 8 * tokens * _words(trees)
                + 4 * (keys // c["page"]), "flops": 4 * pairs * c["hq"] * c["dim"]}
    if c["kind"] == "logits":
        size = 4 if c["dtype"] == "fp32" else 2
        total = 2 * tokens * c["vocab"] * size + (tokens * c["vocab"] // 8 if c["grammar"] else 0) + 8 * c["rows"] * c["bias"]
        if c["penalties"]:
            total += 4 * int(np.random.default_rng(c["rows_seed"] + 2).integers(c["history"] // 2, c["history"] + 1,
                                                                                size=c["rows"]).sum())
        return {"bytes": total, "flops": 6 * tokens * c["vocab"]}
    if c["kind"] == "tables":
        entries = int((-(-(_contexts(c) + np.array([len(t) for t in trees])) // c["page"])).sum())
        return {"bytes": 8 * entries + tokens * (12 + (4 + 8 * _words(trees) if c["tree"] else 0)) + 40 * c["rows"],
                "flops": 0}
    size = 2 * c["hkv"] * c["dim"] * 2
    return {"bytes": int(2 * _accepted(c) * c["layers"] * size) + 20 * tokens, "flops": 0}


# -------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    c = case
    if c["kind"] == "tree":
        return _exact_tree(c, seed)
    if c["kind"] == "logits":
        return _exact_logits(c, seed)
    if c["kind"] == "accept":
        return _exact_accept(c, seed)
    return None  # whole numbers


def _exact_tree(c, seed):
    s = _tree_inputs(c, seed)
    group, d, page = c["hq"] // c["hkv"], c["dim"], c["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = first = 0
    for tree, cached in zip(_trees(c), _contexts(c).tolist()):
        n = len(tree)
        length = cached + n
        where = torch.arange(length, device="cuda")
        ids = s["page_indices"].long()[first + where // page]
        see = torch.ones(n, length, dtype=torch.bool, device="cuda")
        see[:, cached:] = torch.from_numpy(_sees(tree)).to("cuda")
        for g in range(c["hkv"]):
            k, v = (s["cache"][ids, i, where % page, g].double() for i in (0, 1))
            for h in range(g * group, (g + 1) * group):
                x = s["q"][at : at + n, h].double() @ k.t() / math.sqrt(d)
                out[at : at + n, h] = torch.softmax(x.masked_fill(~see, float("-inf")), dim=-1) @ v
        at += n
        first += -(-length // page)
    return out


def _exact_logits(c, seed):
    s = _logits_inputs(c, seed)
    vocab, out, at = c["vocab"], [], 0
    for b, tree in enumerate(_trees(c) if c["nodes"] else [np.array([-1])] * c["rows"]):
        see = _sees(tree)
        if c["bias"]:
            ids = _dev(np.array(list(s["bias"][b])), torch.int64)
            extra = torch.tensor(list(s["bias"][b].values()), dtype=torch.float32, device="cuda").double()
        if c["penalties"]:
            told, end = int(s["prompt_lens"][b]), int(s["history_lens"][b])
            prompt = torch.bincount(s["history"][b, :told], minlength=vocab)
            written = torch.bincount(s["history"][b, told:end], minlength=vocab)
        for i in range(len(tree)):
            y = s["logits"][at + i].double()
            if c["penalties"]:
                count = written
                if c["nodes"]:
                    path = s["tree_tokens"][at : at + len(tree)][torch.from_numpy(see[i]).to("cuda")]
                    count = written + torch.bincount(path, minlength=vocab)
                rep, pres, freq = (s[k][b].double() for k in ("repetition", "presence", "frequency"))
                factor = torch.where(y > 0, 1 / rep, rep)
                y = y * torch.where((prompt + count) > 0, factor, torch.ones_like(y))
                y = y - (freq * count.double() + torch.where(count > 0, pres, torch.zeros_like(y)))
            if c["bias"]:
                y.index_add_(0, ids, extra)
            if c["grammar"]:
                words = s["grammar"][at + i].cpu().numpy().view(np.uint8)
                allowed = np.unpackbits(words, bitorder="little")[:vocab].astype(bool)
                y[torch.from_numpy(~allowed).to("cuda")] = float("-inf")
            out.append(y)
        at += len(tree)
    return torch.stack(out)


def _exact_accept(c, seed):
    """Each tree walked on the host; the moved rows of the cache (the other outputs are whole numbers)."""
    s = _accept_inputs(c, seed)
    tokens, targets, slots = (s[k].tolist() for k in ("tokens", "targets", "slots"))
    cache, at, src, dst = s["cache"].double(), 0, [], []
    for tree in _trees(c):
        child = {(int(p), tokens[at + i]): i for i, p in reversed(list(enumerate(tree))) if p >= 0}
        node, place = 0, 0
        while (node, targets[at + node]) in child:
            node, place = child[node, targets[at + node]], place + 1
            src.append(slots[at + node]), dst.append(slots[at + place])
        at += len(tree)
    src, dst = _dev(np.array(src), torch.int64), _dev(np.array(dst), torch.int64)
    cache[:, dst // c["page"], :, dst % c["page"]] = cache[:, src // c["page"], :, src % c["page"]]
    return [None, None, None, cache]
