"""Operators of a decode step for checkpoints in other forms than the benchmark model's, as cases that
can be timed and compared:

* ``rotary``   rotary positions of q and k: half or interleaved pairs, a part of the head, frequencies scaled for
               long contexts; ``train`` adds the gradient;
* ``append``   a layer's new tokens: q rotated, the rotated k and v written into the paged cache;
* ``int4``     products with 4-bit weights in groups with a scale (and a zero point) each, for a few token rows up to
               a prompt chunk's; ``swiglu`` joins the gate and up halves.

Sizes are the benchmark's and the tests' (heads 32/8 and 16/8 of 128, widths 2,048 and 4,096 with 6,144 and 12,288
inner columns, 151,936 vocabulary entries, 16-token pages), or generic ones of other models.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ROTARY = {
    # plain frequencies, and the three ways in which checkpoints stretch them
    "none": {},
    "linear": {"factor": 4.0},
    "llama3": {"factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position": 8192},
    "yarn": {"factor": 4.0, "beta_fast": 32.0, "beta_slow": 1.0, "original_max_position": 32768},
}
THETA = {"none": 1e6, "linear": 1e4, "llama3": 5e5, "yarn": 1e6}


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of a small batch of requests, one token each, far into their contexts: launches count
        {"name": "rotary_decode", "kind": "rotary", "tokens": 4, "hq": 16, "hkv": 8, "dim": 128, "rot": 128,
         "layout": "half", "scaling": "llama3", "dtype": "bf16", "far": 131072, "train": False},
        # a prompt chunk of the benchmark's layer, in the half layout that most checkpoints are stored in
        {"name": "rotary_chunk", "kind": "rotary", "tokens": 8192, "hq": 32, "hkv": 8, "dim": 128, "rot": 128,
         "layout": "half", "scaling": "none", "dtype": "bf16", "far": 40960, "train": False},
        # fine-tuning on an odd number of packed tokens, a quarter of each head rotated, 80 values a head
        {"name": "rotary_train", "kind": "rotary", "tokens": 4001, "hq": 32, "hkv": 32, "dim": 80, "rot": 20,
         "layout": "half", "scaling": "linear", "dtype": "fp32", "far": 8192, "train": True},
        # the same for interleaved pairs over half of the head, in the type that training runs in
        {"name": "rotary_train_pairs", "kind": "rotary", "tokens": 2047, "hq": 32, "hkv": 8, "dim": 128, "rot": 64,
         "layout": "interleaved", "scaling": "yarn", "dtype": "bf16", "far": 131072, "train": True},
        # the smallest decode step: four requests, one token each, and four tokens of padding behind them
        {"name": "append_decode", "kind": "append", "rows": 4, "tokens": 4, "pad": 4, "prefix": 4096, "hq": 16,
         "hkv": 8, "dim": 128, "rot": 128, "layout": "half", "scaling": "none", "dtype": "bf16", "rows_seed": 0},
        # the benchmark's decode step: 64 rows with 208 tokens over long contexts
        {"name": "append_step", "kind": "append", "rows": 64, "tokens": 208, "pad": 0, "prefix": 2048, "hq": 32,
         "hkv": 8, "dim": 128, "rot": 128, "layout": "half", "scaling": "llama3", "dtype": "bf16", "rows_seed": 1},
        # prompt chunks of three requests: ragged lengths behind odd prefixes, half of the head rotated
        {"name": "append_chunk", "kind": "append", "rows": 3, "tokens": 8191, "pad": 1, "prefix": 5000, "hq": 32,
         "hkv": 8, "dim": 128, "rot": 64, "layout": "interleaved", "scaling": "yarn", "dtype": "fp16", "rows_seed": 2},
        # one token against an output projection: latency
        {"name": "int4_token", "kind": "int4", "rows": 1, "n": 4096, "k": 4096, "group": 128, "zeros": False,
         "dtype": "bf16", "swiglu": False},
        # a small decode batch against the gate and up projections
        {"name": "int4_swiglu", "kind": "int4", "rows": 12, "n": 24576, "k": 4096, "group": 128, "zeros": True,
         "dtype": "bf16", "swiglu": True},
        # a down projection in groups of 32, rows and columns that fill no tile
        {"name": "int4_ragged", "kind": "int4", "rows": 33, "n": 4001, "k": 12288, "group": 32, "zeros": True,
         "dtype": "fp16", "swiglu": False},
        # the benchmark's decode step of 208 tokens against the vocabulary
        {"name": "int4_vocab", "kind": "int4", "rows": 208, "n": 151936, "k": 4096, "group": 64, "zeros": False,
         "dtype": "bf16", "swiglu": False},
        # a prompt chunk through the fused q, k and v projection
        {"name": "int4_chunk", "kind": "int4", "rows": 2048, "n": 6144, "k": 4096, "group": 128, "zeros": True,
         "dtype": "bf16", "swiglu": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "int4", "int4"])
    if kind == "int4":
        group = rng.choice([32, 64, 128])
        swiglu = rng.random() < 0.3
        k = group * max(1, _log(rng, 256, 14336) // group)
        n = _log(rng, 256, 32768)
        if swiglu:
            n = 32 * max(1, n // 32)
        rows = min(_log(rng, 1, 2048), max(1, 100_000_000_000 // (n * k)))
        return {"kind": kind, "rows": rows, "n": n, "k": k, "group": group, "zeros": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "swiglu": swiglu}
    dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    hq, hkv = rng.choice([(32, 8), (16, 8), (32, 32), (64, 8), (40, 8), (12, 2), (7, 1)])
    c = {"kind": kind, "hq": hq, "hkv": hkv, "dim": dim,
         "rot": rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
         "layout": rng.choice(["half", "half", "interleaved"]), "scaling": rng.choice(list(ROTARY))}
    most = max(1, 8192 * 48 * 128 // ((hq + 2 * hkv) * dim))
    if kind == "rotary":
        c.update(dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), far=_log(rng, 64, 1 << 20),
                 train=rng.random() < 0.4)
        c["tokens"] = _log(rng, 1, max(1, most // (4 if c["train"] else 2)))
        return c
    rows = rng.randint(1, 64)
    c.update(dtype=rng.choice(["bf16", "bf16", "fp16"]), rows=rows, tokens=max(rows, _log(rng, 1, min(most, 8192))),
             pad=rng.choice([0, 0, 1, 7]), prefix=_log(rng, 16, 4096), rows_seed=rng.randrange(1 << 20))
    return c


# ---------------------------------------------------------------------------------- the inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, gen, dtype, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen).to(dtype)


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def _rotary_inputs(c, seed):
    """q and k as views of one fused projection, positions of tokens of several packed sequences."""
    gen, dtype = _gen(seed), TYPES[c["dtype"]]
    T, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["dim"]
    qkv = _normal((T, (hq + 2 * hkv) * d), gen, dtype)
    start = torch.randint(0, max(1, c["far"] - T), (), device="cuda", generator=gen)
    positions = (torch.arange(T, device="cuda") + start) % c["far"]
    if T <= 64:  # a decode step: every token in a context of its own
        positions = torch.randint(0, c["far"], (T,), device="cuda", generator=gen)
    s = {"q": qkv[:, : hq * d].view(T, hq, d), "k": qkv[:, hq * d : (hq + hkv) * d].view(T, hkv, d),
         "positions": positions.to(torch.int32)}
    if c["train"]:
        s["dq"], s["dk"] = _normal((T, hq, d), gen, dtype), _normal((T, hkv, d), gen, dtype)
    return s


def _append_rows(c):
    """(length after the append, new tokens) of each row, from the case alone."""
    r = np.random.default_rng(c["rows_seed"])
    cuts = np.sort(r.choice(np.arange(1, c["tokens"]), size=c["rows"] - 1, replace=False)) if c["rows"] > 1 \
        else np.zeros(0, np.int64)
    new = np.diff(np.concatenate([[0], cuts, [c["tokens"]]])).astype(np.int64)
    return r.integers(0, c["prefix"] + 1, size=c["rows"]).astype(np.int64) + new, new


def _append_inputs(c, seed):
    gen, dtype = _gen(seed), TYPES[c["dtype"]]
    ctx, new = _append_rows(c)
    pages = (ctx + PAGE - 1) // PAGE
    order = np.random.default_rng(seed + 77).permutation(int(pages.sum())).astype(np.int32)
    T, hq, hkv, d = c["tokens"] + c["pad"], c["hq"], c["hkv"], c["dim"]
    qkv = _normal((T, (hq + 2 * hkv) * d), gen, dtype)
    q, k, v = (qkv[:, a * d : b * d].view(T, b - a, d) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    ptr = lambda a: np.concatenate([[0], np.cumsum(a)])
    return {"q": q, "k": k, "v": v, "cache": _normal((int(pages.sum()), 2, PAGE, hkv, d), gen, dtype),
            "indptr": _dev(ptr(new)), "page_indices": _dev(order), "page_indptr": _dev(ptr(pages)),
            "last_page_len": _dev((ctx - 1) % PAGE + 1)}


def _int4_inputs(c, seed):
    """Activations with a few loud channels; weights as a checkpoint holds them: codes [N, K] two to a byte (the even
    column in the low half), a scale and a zero point for each group of a row."""
    gen, dtype = _gen(seed), TYPES[c["dtype"]]
    rows, n, k, group = c["rows"], c["n"], c["k"], c["group"]
    x = _normal((rows, k), gen, dtype)
    loud = torch.randint(0, k, (max(1, k // 512),), device="cuda", generator=gen)
    x[:, loud] *= 8
    packed = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    for at in range(0, n, 16384):
        m = min(16384, n - at)
        codes = torch.empty(m, k, device="cuda").normal_(7.5, 2.6, generator=gen).round_().clamp_(0, 15).to(torch.uint8)
        packed[at : at + m] = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scales = (torch.rand(n, k // group, device="cuda", generator=gen) + 0.5) * (k ** -0.5 / 2.6)
    zeros = None
    if c["zeros"]:
        zeros = torch.randint(5, 11, (n, k // group), device="cuda", generator=gen, dtype=torch.uint8)
    return {"x": x, "packed": packed, "scales": scales.to(dtype), "zeros": zeros}


def prepare(case, seed):
    c = case
    s = {"rotary": _rotary_inputs, "append": _append_inputs, "int4": _int4_inputs}[c["kind"]](c, seed)
    s["case"] = c
    if c["kind"] == "int4":
        s["out"] = torch.empty(c["rows"], c["n"] // 2 if c["swiglu"] else c["n"], dtype=s["x"].dtype, device="cuda")
        if own:  # laid out once, as a program does when it loads the weights
            from aspire_amd.linear_int4 import Int4Weight

            s["weight"] = Int4Weight.from_packed(s["packed"], s["scales"], s["zeros"], group=c["group"])
        return s
    if c["kind"] == "append":
        s["q_out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    if c["kind"] == "rotary" and c["train"]:
        s["q"], s["k"] = s["q"].contiguous().requires_grad_(), s["k"].contiguous().requires_grad_()
    if own:
        from aspire_amd.attention.rotary import RotaryConfig, RotaryEmbedding

        s["rotary"] = RotaryEmbedding(RotaryConfig(head_dim=c["dim"], rotary_dim=c["rot"], layout=c["layout"],
                                                   theta=THETA[c["scaling"]], scaling=c["scaling"],
                                                   **ROTARY[c["scaling"]]), "cuda")
    else:
        f, amplitude = _frequencies(c)
        s["frequencies"], s["amplitude"] = torch.from_numpy(f).to("cuda"), amplitude
    return s


# ------------------------------------------------------------------------------- the plain forms
def _frequencies(c):
    """Radians a position of each rotated pair (float64), and the factor on cos and sin."""
    rot, scaling, p = c["rot"], c["scaling"], ROTARY[c["scaling"]]
    theta = THETA[scaling]
    i = np.arange(rot // 2, dtype=np.float64)
    f = theta ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / p["factor"], 1.0
    if scaling == "llama3":
        turns = p["original_max_position"] * f / (2 * math.pi)  # of the trained context
        keep = np.clip((turns - p["low_freq_factor"]) / (p["high_freq_factor"] - p["low_freq_factor"]), 0.0, 1.0)
        return keep * f + (1 - keep) * f / p["factor"], 1.0
    if scaling == "yarn":
        pair = lambda turns: rot * math.log(p["original_max_position"] / (2 * math.pi * turns)) / (2 * math.log(theta))
        low, high = max(math.floor(pair(p["beta_fast"])), 0), min(math.ceil(pair(p["beta_slow"])), rot - 1)
        keep = 1 - np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
        return keep * f + (1 - keep) * f / p["factor"], 0.1 * math.log(p["factor"]) + 1.0
    return f, 1.0


def _turn(x, cos, sin, c, inverse=False):
    """x [T, H, D] with its pairs turned; cos and sin [T, rot / 2] fp32."""
    rot = c["rot"]
    xf = x.float()
    cos, sin = cos[:, None, :], (-sin if inverse else sin)[:, None, :]
    if c["layout"] == "half":
        a, b = xf[..., : rot // 2], xf[..., rot // 2 : rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([y, xf[..., rot:]], dim=-1).to(x.dtype)


def _cos_sin(s, positions):
    angle = positions.double()[:, None] * s["frequencies"]  # far positions need more than 32 bits
    return (torch.cos(angle) * s["amplitude"]).float(), (torch.sin(angle) * s["amplitude"]).float()


def _owners(s, tokens):
    """Row, place in the row's sequence and truth of having one, of every token."""
    at = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(s["indptr"].long(), at, right=True) - 1
    last = s["indptr"].shape[0] - 2
    live = row <= last
    row = row.clamp(max=last)
    pages = (s["page_indptr"][1:] - s["page_indptr"][:-1]).long()
    length = (pages - 1) * PAGE + s["last_page_len"].long()
    return row, length[row] - s["indptr"].long()[row + 1] + at, live


def _plain_append(s):
    c, q = s["case"], s["q"]
    row, place, live = _owners(s, q.shape[0])
    cos, sin = _cos_sin(s, place)
    s["q_out"].copy_(torch.where(live[:, None, None], _turn(q, cos, sin, c), q))
    k = _turn(s["k"], cos, sin, c)
    n = c["tokens"]  # the padding stands behind the last row
    page = s["page_indices"].long()[s["page_indptr"].long()[row[:n]] + place[:n] // PAGE]
    s["cache"][page, 0, place[:n] % PAGE] = k[:n]
    s["cache"][page, 1, place[:n] % PAGE] = s["v"][:n]
    return [s["q_out"], s["cache"]]


def _plain_int4(s):
    c, packed = s["case"], s["packed"]
    n, group = packed.shape[0], c["group"]
    w = torch.stack([packed & 15, packed >> 4], dim=-1).view(n, -1, group).float()
    w -= 8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None]
    w *= s["scales"].float()[:, :, None]
    y = s["x"].float() @ w.view(n, -1).t()
    if c["swiglu"]:
        gate, up = y[:, : n // 2], y[:, n // 2 :]
        y = gate / (1 + torch.exp(-gate)) * up
    s["out"].copy_(y)
    return s["out"]


# --------------------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "int4":
        return _plain_int4(s)
    if c["kind"] == "append":
        return _plain_append(s)
    cos, sin = _cos_sin(s, s["positions"])
    with torch.no_grad():
        outs = [_turn(s["q"], cos, sin, c), _turn(s["k"], cos, sin, c)]
        if c["train"]:
            outs += [_turn(s["dq"], cos, sin, c, inverse=True), _turn(s["dk"], cos, sin, c, inverse=True)]
    return outs


def _run_own(s, c):
    if c["kind"] == "int4":
        from aspire_amd.linear_int4 import linear_int4

        return linear_int4(s["x"], s["weight"], s["out"], swiglu=c["swiglu"])
    if c["kind"] == "append":
        q = s["rotary"].append(s["q"], s["k"], s["v"], s["indptr"], s["cache"], s["page_indices"], s["page_indptr"],
                               s["last_page_len"], PAGE, q_out=s["q_out"])
        return [q, s["cache"]]
    q, k = s["rotary"].apply(s["q"], s["k"], s["positions"])
    if not c["train"]:
        return [q, k]
    return [q, k, *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])]


# ------------------------------------------------------------------------------------ what it takes
def work(case):
    c = case
    if c["kind"] == "int4":
        rows, n, k = c["rows"], c["n"], c["k"]
        groups = n * (k // c["group"])
        out = n // 2 if c["swiglu"] else n
        return {"bytes": n * k // 2 + groups * (3 if c["zeros"] else 2) + 2 * rows * (k + out),
                "flops": 2 * rows * n * k}
    size = 4 if c["dtype"] == "fp32" else 2
    tokens = c["tokens"]
    pairs = tokens * (c["hq"] + c["hkv"]) * (c["rot"] // 2)
    if c["kind"] == "append":
        values = tokens * (c["hq"] + 2 * c["hkv"]) * c["dim"] + c["pad"] * c["hq"] * c["dim"]
        return {"bytes": 2 * values * size + 4 * (c["rows"] * 3 + tokens // PAGE + 1), "flops": 6 * pairs}
    ways = 2 if c["train"] else 1
    values = tokens * (c["hq"] + c["hkv"]) * c["dim"]
    return {"bytes": ways * 2 * values * size + 4 * tokens, "flops": ways * 6 * pairs}


# -------------------------------------------------------------------------- the definition in 64 bits
def _exact_angles(c):
    """Angle of a position as a function of the pair, written from the definitions."""
    scaling, p, half = c["scaling"], ROTARY[c["scaling"]], c["rot"] // 2
    out, amplitude = [], 1.0
    for j in range(half):
        f = math.exp(-math.log(THETA[scaling]) * (2 * j) / c["rot"])
        if scaling == "linear":
            f /= p["factor"]
        elif scaling == "llama3":
            wave = 2 * math.pi / f
            long, short = p["original_max_position"] / p["low_freq_factor"], p["original_max_position"] / p["high_freq_factor"]
            if wave > long:
                f /= p["factor"]
            elif wave >= short:
                t = (p["original_max_position"] / wave - p["low_freq_factor"]) / (p["high_freq_factor"] - p["low_freq_factor"])
                f = (1 - t) * f / p["factor"] + t * f
        elif scaling == "yarn":
            # the pairs that turn beta_fast and beta_slow times over the trained context, whole numbers
            ends = [c["rot"] * math.log(p["original_max_position"] / (b * 2 * math.pi)) / (2 * math.log(THETA[scaling]))
                    for b in (p["beta_fast"], p["beta_slow"])]
            lo, hi = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), c["rot"] - 1)
            ramp = min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = ramp * f / p["factor"] + (1 - ramp) * f
            amplitude = 0.1 * math.log(p["factor"]) + 1.0
        out.append(f)
    return torch.tensor(out, dtype=torch.float64, device="cuda"), amplitude


def _exact_turn(x, positions, c, sign=1.0):
    """Each pair as a complex number, multiplied by amplitude * exp(i * sign * position * f)."""
    f, amplitude = _exact_angles(c)
    rot = c["rot"]
    turn = torch.polar(torch.full((), amplitude, dtype=torch.float64, device="cuda").expand(positions.shape[0], f.shape[0]).contiguous(),
                       sign * positions.double()[:, None] * f)[:, None, :]
    y = x.detach().double().clone()
    if c["layout"] == "half":
        first, second = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        first, second = slice(0, rot, 2), slice(1, rot, 2)
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    c = case
    if c["kind"] == "rotary":
        s = _rotary_inputs(c, seed)
        outs = [_exact_turn(s["q"], s["positions"], c), _exact_turn(s["k"], s["positions"], c)]
        if c["train"]:  # the transpose of a rotation is the rotation back
            outs += [_exact_turn(s["dq"], s["positions"], c, -1.0), _exact_turn(s["dk"], s["positions"], c, -1.0)]
        return outs
    if c["kind"] == "append":
        s = _append_inputs(c, seed)
        ctx, new = _append_rows(c)
        q, k, cache = s["q"].double(), s["k"].double(), s["cache"].double()
        ids, first, at = s["page_indices"].cpu().numpy(), 0, 0
        for length, count in zip(ctx.tolist(), new.tolist()):
            place = np.arange(length - count, length)
            rows = slice(at, at + count)
            where = torch.from_numpy(place).to("cuda")
            q[rows] = _exact_turn(q[rows], where, c)
            pages = _dev(ids[first + place // PAGE], torch.int64)
            cache[pages, 0, where % PAGE] = _exact_turn(k[rows], where, c)
            cache[pages, 1, where % PAGE] = s["v"][rows].double()
            first += (length + PAGE - 1) // PAGE
            at += count
        return [q, cache]
    s = _int4_inputs(c, seed)
    x, n = s["x"].double(), c["n"]

    def product(lo, hi):
        packed = s["packed"][lo:hi].to(torch.int64)
        w = torch.empty(hi - lo, c["k"], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (packed % 16).double(), torch.div(packed, 16, rounding_mode="floor").double()
        spread = lambda t: t[lo:hi].double().repeat_interleave(c["group"], dim=1)
        w = (w - (spread(s["zeros"]) if c["zeros"] else 8.0)) * spread(s["scales"])
        return x @ w.t()

    y = torch.cat([product(lo, min(lo + 8192, n)) for lo in range(0, n, 8192)], dim=1)
    if c["swiglu"]:
        y = y[:, : n // 2] * torch.sigmoid(y[:, : n // 2]) * y[:, n // 2 :]
    return y
