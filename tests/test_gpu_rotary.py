"""Rotary positions and the append with rotation against the definition in 64 bits."""

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwad

from aspire_amd.attention.rotary import RotaryConfig, RotaryEmbedding
from helpers import bits, say
from oracle.append import paged_kv_append
from test_rotary_cpu import PI, true_frequencies

pytestmark = pytest.mark.gpu

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
CONFIGS = {
    "none": dict(theta=1e6),
    "linear": dict(theta=1e4, scaling="linear", factor=4.0),
    "llama3": dict(theta=5e5, scaling="llama3", factor=8.0, original_max_position=8192),
    "yarn": dict(theta=1e6, scaling="yarn", factor=4.0, original_max_position=32768),
}


def turned(x, positions, config, inverse=False):
    """The definition in 64 bits on the CPU: each pair as a complex number."""
    y = x.detach().double().cpu().clone()
    r = config.rotated
    first, second = (slice(0, r // 2), slice(r // 2, r)) if config.layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    f = torch.tensor(config.frequencies(), dtype=torch.float64)
    p = positions.cpu()
    angle = p.double()[:, None, None] * f * (-1 if inverse else 1)
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous())
    z = torch.where((p >= 0)[:, None, None], z * config.scale * torch.exp(1j * angle), z)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def close(got, ref, x, config):
    """Half a step of the output's type, and 10 * 2^-24 of a pair's two values times the amplitude: the reduced angle
    (at most 0.785) carries 3 roundings (2.4), each series 2, the amplitude 2, the two products and their sum 2, sum 8.4.
    fp16 values below its normal range step by 2^-24."""
    g = got.detach().double().cpu()
    r = config.rotated
    size = x.detach().double().cpu().abs()
    pair = size[..., :r]
    pair = pair.unflatten(-1, (2, r // 2) if config.layout == "half" else (r // 2, 2)).sum(-2 if config.layout == "half" else -1)
    pair = torch.cat([pair, pair], -1) if config.layout == "half" else pair.repeat_interleave(2, -1)
    bound = torch.zeros_like(size)
    bound[..., :r] = 10 * 2.0 ** -24 * max(config.scale, 1.0) * pair
    limit = bound + torch.finfo(got.dtype).eps / 2 * (ref.abs() + bound) + (2.0 ** -25 if got.dtype == HF else 0)
    off = (g - ref).abs()
    assert not (off > limit).any(), f"{int((off > limit).sum())} of {off.numel()} off, worst {float((off - limit).max())}"
    assert torch.equal(g[..., r:], x.detach().double().cpu()[..., r:])


def tensors(T, hq, hkv, d, dtype, gpu, pad=0, seed=0):
    """q and k as views of one projection whose rows are ``pad`` values longer than the heads, and v."""
    g = torch.Generator(device=gpu).manual_seed(seed + T * 7 + hq + d)
    qkv = torch.randn(T, (hq + 2 * hkv) * d + pad, device=gpu, generator=g).to(dtype)
    cut = lambda a, b: qkv[:, a * d : b * d].view(T, b - a, d) if pad == 0 else qkv[:, a * d : b * d].unflatten(1, (b - a, d))
    return cut(0, hq), cut(hq, hq + hkv), cut(hq + hkv, hq + 2 * hkv)


FORMS = [
    # T, hq, hkv, D, R, layout, dtype, scaling, pad
    (1, 16, 8, 128, 128, "half", BF, "llama3", 0),
    (1, 1, 1, 2, 2, "half", SF, "none", 0),            # one pair, one head
    (1, 3, 1, 8, 8, "half", BF, "none", 0),            # heads of a few tasks
    (3, 32, 8, 128, 128, "half", BF, "none", 0),
    (67, 32, 8, 128, 64, "interleaved", BF, "yarn", 0),
    (130, 40, 8, 96, 96, "half", HF, "linear", 8),
    (33, 7, 1, 80, 20, "half", SF, "none", 0),         # pairs of 10, two values an access
    (33, 7, 1, 80, 20, "half", BF, "none", 2),
    (5, 12, 2, 64, 64, "interleaved", HF, "none", 1),  # rows that are not aligned: single values
    (5, 12, 2, 64, 30, "half", BF, "yarn", 1),
    (29, 8, 8, 256, 256, "half", BF, "llama3", 0),     # 128 pairs: two angles a lane
    (29, 8, 8, 256, 200, "interleaved", SF, "linear", 4),
    (11, 64, 8, 192, 134, "interleaved", BF, "none", 0),
    (9, 5, 5, 75, 50, "half", BF, "none", 0),          # an odd head width
    (2100, 32, 8, 128, 128, "half", BF, "yarn", 0),    # one wave a token
    (4100, 2, 1, 64, 32, "interleaved", HF, "llama3", 0),
]


@pytest.mark.parametrize("T,hq,hkv,d,r,layout,dtype,scaling,pad", FORMS)
def test_apply(gpu, T, hq, hkv, d, r, layout, dtype, scaling, pad):
    """New tensors and in place; positions near and far (past 2^31 too), in both integer types, some negative."""
    say("rotary apply", T, hq, hkv, d, r, layout, dtype, scaling, pad)
    config = RotaryConfig(head_dim=d, rotary_dim=r, layout=layout, **CONFIGS[scaling])
    rot = RotaryEmbedding(config, gpu)
    q, k, _ = tensors(T, hq, hkv, d, dtype, gpu, pad)
    g = torch.Generator().manual_seed(T)
    pos = torch.randint(0, 1 << 20, (T,), generator=g)
    pos[0] = 0 if T > 1 else 131071
    if T > 4:
        pos[1], pos[2], pos[3], pos[4] = 1, -1, 1 << 33, (1 << 31) - 1
    before = q.clone(), k.clone()
    qo, ko = rot.apply(q, k, pos.to(gpu))
    assert torch.equal(q, before[0]) and torch.equal(k, before[1]) and qo.is_contiguous()
    refs = turned(q, pos, config), turned(k, pos, config)
    # a 64-bit angle has 53 bits: past 2^33 * f it is off by 2^-20, more than fp32's steps allow
    near = pos < 1 << 31
    for got, ref, x in ((qo, refs[0], q), (ko, refs[1], k)):
        close(got[near.to(gpu)], ref[near], x[near.to(gpu)], config)
    pos32 = torch.where(near, pos, 5).to(torch.int32).to(gpu)
    q1, none = rot.apply(q, None, pos32)
    assert none is None and torch.equal(bits16(q1[near.to(gpu)]), bits16(qo[near.to(gpu)]))
    rot.apply_inplace(q, k, pos32)
    assert torch.equal(bits16(q), bits16(q1)) and torch.equal(bits16(k[near.to(gpu)]), bits16(ko[near.to(gpu)]))


def bits16(t):
    return t.contiguous().view(torch.int32 if t.dtype == SF else torch.int16).cpu()


def test_far_positions_are_exact(gpu):
    """Positions whose angle has no 24 or 53 bits, against whole-number arithmetic on the host."""
    say("rotary far")
    config = RotaryConfig(head_dim=64, theta=1e4)
    rot = RotaryEmbedding(config, gpu)
    pos = [(1 << 40) + 12345, (1 << 62) + 99, (1 << 31) + 7]
    x = torch.zeros(3, 1, 64, device=gpu)
    x[..., :32] = 1
    y, _ = rot.apply(x, None, torch.tensor(pos, device=gpu))
    turns = [int(t) % (1 << 64) for t in rot.turns.cpu().tolist()]
    for i, p in enumerate(pos):
        angle = np.array([(p * t % (1 << 64)) / 2.0 ** 64 * 2 * np.pi for t in turns])
        ref = np.concatenate([np.cos(angle), np.sin(angle)])
        assert np.abs(y[i, 0].cpu().double().numpy() - ref).max() <= 10 * 2.0 ** -24


def test_special_values_stay_in_their_pairs(gpu):
    """NaN and infinities reach the two values of their pair only."""
    say("rotary special values")
    for layout in ("half", "interleaved"):
        config = RotaryConfig(head_dim=128, rotary_dim=64, layout=layout)
        rot = RotaryEmbedding(config, gpu)
        x = torch.randn(2, 3, 128, device=gpu).to(BF)
        x[0, 0, 1], x[0, 1, 3], x[1, 2, 100] = float("nan"), float("inf"), float("nan")
        y, _ = rot.apply(x, None, torch.tensor([5, 9], device=gpu))
        bad = torch.zeros(2, 3, 128, dtype=torch.bool)
        mates = {"half": ((1, 33), (3, 35)), "interleaved": ((0, 1), (2, 3))}[layout]
        for d in mates[0]:
            bad[0, 0, d] = True
        for d in mates[1]:
            bad[0, 1, d] = True
        bad[1, 2, 100] = True
        assert torch.equal(~torch.isfinite(y).cpu(), bad)


def test_pair_factors_and_amplitude(gpu):
    say("rotary pair factors")
    factors = tuple(1.0 + 0.5 * i for i in range(16))
    config = RotaryConfig(head_dim=48, rotary_dim=32, theta=1e4, pair_factors=factors, amplitude=1.25)
    rot = RotaryEmbedding(config, gpu)
    q, k, _ = tensors(9, 4, 2, 48, SF, gpu)
    pos = torch.arange(9) * 1001
    qo, ko = rot.apply(q, k, pos.to(gpu))
    close(qo, turned(q, pos, config), q, config)
    close(ko, turned(k, pos, config), k, config)


@pytest.mark.parametrize("T,hq,hkv,d,r,layout,dtype,scaling,pad", [FORMS[i] for i in (0, 4, 6, 8, 11)])
def test_gradients(gpu, T, hq, hkv, d, r, layout, dtype, scaling, pad):
    """The formula's gradient (the turn back), differences (the operator is linear), gradients that are expanded or
    strided, of one output only, and the second derivative."""
    say("rotary gradients", T, hq, hkv, d, r, layout, dtype, scaling)
    config = RotaryConfig(head_dim=d, rotary_dim=r, layout=layout, **CONFIGS[scaling])
    rot = RotaryEmbedding(config, gpu)
    q, k, _ = (t.detach().clone() for t in tensors(T, hq, hkv, d, dtype, gpu, pad))
    pos = torch.arange(T) * 37
    pos[-1] = -1 if T > 1 else 77
    q.requires_grad_(), k.requires_grad_()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    qo, ko = rot.apply(q, k, pos.to(gpu))
    gq, gk = torch.autograd.grad([qo, ko], [q, k], [dq, dk])
    close(gq, turned(dq, pos, config, inverse=True), dq, config)
    close(gk, turned(dk, pos, config, inverse=True), dk, config)
    # <dk, y(k + h) - y(k)> = <gradient, h> in 64 bits: the operator is linear
    h = torch.randn_like(k)
    with torch.no_grad():
        step = turned(k.double() + h.double(), pos, config) - turned(k, pos, config)
    lhs, rhs = (dk.double().cpu() * step).sum(), (gk.double().cpu() * h.double().cpu()).sum()
    # each of the gradient's values is within half a step and 20 * 2^-24 of its pair, both below eps of |gradient| + |dk|
    slack = torch.finfo(dtype).eps * ((gk.double().cpu().abs() + 2 * dk.double().cpu().abs()) * h.double().cpu().abs()).sum()
    assert abs(lhs - rhs) <= slack
    # only k, and a gradient that is one number expanded
    qo, ko = rot.apply(q, k, pos.to(gpu))
    (only,) = torch.autograd.grad(ko.sum(), [k])
    ones = torch.ones_like(k)
    close(only, turned(ones, pos, config, inverse=True), ones, config)
    # the gradient's own gradient turns forward again
    qo, _ = rot.apply(q, None, pos.to(gpu))
    seed = torch.randn_like(q).requires_grad_()
    (first,) = torch.autograd.grad(qo, [q], seed, create_graph=True)
    (again,) = torch.autograd.grad(first, [seed], dq)
    close(again, turned(dq, pos, config), dq, config)


# ------------------------------------------------------------------------------------- the append
def pages_of(ctx, new, page, gpu, seed, spare=3, pad=0):
    ctx, new = np.asarray(ctx), np.asarray(new)
    n = (ctx + page - 1) // page
    ids = np.random.default_rng(seed).permutation(int(n.sum()) + spare)[: int(n.sum())]
    ptr = lambda a: np.concatenate([[0], np.cumsum(a)])
    last = np.where(ctx > 0, (ctx - 1) % page + 1, 0)
    host = dict(indptr=ptr(new), ids=ids, page_indptr=ptr(n), last=last)
    dev = [torch.from_numpy(np.ascontiguousarray(host[x])).to(torch.int32).to(gpu) for x in ("indptr", "ids", "page_indptr", "last")]
    places = np.full(int(new.sum()) + pad, -1)
    at = 0
    for c, t in zip(ctx, new):
        places[at : at + t] = np.arange(c - t, c)
        at += t
    return host, dev, torch.from_numpy(places), int(n.sum()) + spare


@pytest.mark.parametrize("hq,hkv,d,r,layout,dtype,scaling,ctx,new,pad,page,view", [
    (16, 8, 128, 128, "half", BF, "none", [4097], [1], 0, 16, "nhd"),           # the smallest call
    (32, 8, 128, 128, "half", BF, "llama3", [33, 16, 0, 17, 5], [1, 4, 0, 17, 5], 4, 16, "nhd"),
    (32, 8, 128, 64, "interleaved", HF, "yarn", [700, 45], [300, 45], 1, 16, "hnd"),
    (7, 1, 80, 20, "half", BF, "linear", [40, 41, 42], [3, 2, 1], 0, 8, "nhd"),
    (12, 2, 75, 50, "half", HF, "none", [40, 9], [3, 9], 2, 5, "nhd"),          # odd widths and pages
    (6, 3, 64, 64, "interleaved", BF, "none", [1] * 70, [1] * 70, 0, 16, "hnd"),  # more rows than a wave has lanes
    (8, 2, 256, 256, "half", BF, "yarn", [100, 1000], [100, 900], 3, 64, "nhd"),
])
def test_append(gpu, hq, hkv, d, r, layout, dtype, scaling, ctx, new, pad, page, view):
    """q beside its input and in place, turned k and copied v in their pages, everything else left alone."""
    say("rotary append", hq, hkv, d, r, layout, dtype, scaling, ctx[:4], new[:4], pad, page, view)
    config = RotaryConfig(head_dim=d, rotary_dim=r, layout=layout, **CONFIGS[scaling])
    rot = RotaryEmbedding(config, gpu)
    T = sum(new) + pad
    q, k, v = tensors(T, hq, hkv, d, dtype, gpu)
    host, dev, places, pool = pages_of(ctx, new, page, gpu, seed=T, pad=pad)
    if view == "nhd":
        cache = torch.randn(pool, 2, page, hkv, d, device=gpu).to(dtype)
    else:
        cache = torch.randn(pool, 2, hkv, page, d, device=gpu).to(dtype).transpose(2, 3)
    before = cache.cpu().contiguous()
    kb, vb = k.clone(), v.clone()
    q_out = torch.full((T, hq, d), 7.0, dtype=dtype, device=gpu)
    assert rot.append(q, k, v, dev[0], cache, dev[1], dev[2], dev[3], page, q_out=q_out) is q_out
    assert torch.equal(k, kb) and torch.equal(v, vb)
    close(q_out, turned(q, places, config), q, config)
    if pad:
        assert torch.equal(q_out[-pad:], q[-pad:])
    ref_k = turned(k, places, config)
    where = paged_kv_append(bits(torch.ones_like(k)), bits(v.contiguous()), host["indptr"], np.zeros_like(bits(before)),
                            host["ids"], host["page_indptr"], host["last"], page)
    written = torch.from_numpy(where.view(np.int16)).view(dtype)[:, 0, :, :1, :1] == 1  # [pool, 1, page]: K slots
    got = cache.cpu().contiguous()
    slots = written.view(pool, page)
    assert int(slots.sum()) == sum(new)
    assert torch.equal(got[:, 0][~slots], before[:, 0][~slots]) and torch.equal(got[:, 1][~slots], before[:, 1][~slots])
    at = 0
    for b, (c, t) in enumerate(zip(ctx, new)):
        ids = host["ids"][host["page_indptr"][b] : host["page_indptr"][b + 1]]
        place = np.arange(c - t, c)
        if t:
            rows = torch.from_numpy(ids[place // page].astype(np.int64)), torch.from_numpy(place % page)
            close(got[rows[0], 0, rows[1]], ref_k[at : at + t], k[at : at + t], config)
            assert torch.equal(got[rows[0], 1, rows[1]], v[at : at + t].cpu())
        at += t
    first = got.clone()
    cache.copy_(before.to(gpu))
    rot.append(q, k, v, dev[0], cache, dev[1], dev[2], dev[3], page)
    assert torch.equal(bits16(q), bits16(q_out)) and torch.equal(bits16(cache), bits16(first))


def test_append_at_given_positions(gpu):
    """Positions that are not the places in the cache (a shifted prompt, an evicted prefix)."""
    say("rotary append positions")
    config = RotaryConfig(head_dim=64, theta=1e4)
    rot = RotaryEmbedding(config, gpu)
    host, dev, places, pool = pages_of([20, 9], [5, 9], 16, gpu, 3)
    q, k, v = tensors(14, 4, 2, 64, BF, gpu)
    cache = torch.zeros(pool, 2, 16, 2, 64, dtype=BF, device=gpu)
    for dt in (torch.int32, torch.int64):
        pos = torch.arange(14, dtype=dt) * 1000 + 3
        out = rot.append(q, k, v, dev[0], cache, dev[1], dev[2], dev[3], 16, positions=pos.to(gpu),
                         q_out=torch.empty_like(q))
        close(out, turned(q, pos, config), q, config)
        page = host["ids"][host["page_indptr"][0] + 15 // 16]
        close(cache[page, 0, 15][None], turned(k, pos, config)[:1], k[:1], config)


def test_append_skips_what_lies_outside(gpu):
    """Page ids and list entries outside the pool and the list: those tokens are not written, the others are."""
    say("rotary append bad pages")
    config = RotaryConfig(head_dim=64)
    rot = RotaryEmbedding(config, gpu)
    host, dev, places, pool = pages_of([30, 18, 40], [4, 18, 3], 16, gpu, 5)
    q, k, v = tensors(25, 4, 2, 64, BF, gpu)
    good = torch.zeros(pool, 2, 16, 2, 64, dtype=BF, device=gpu)
    rot.append(q.clone(), k, v, dev[0], good, dev[1], dev[2], dev[3], 16)
    for bad in (-1, pool, 1 << 30):
        ids = dev[1].clone()
        ids[1] = bad                       # row 0's second page: its four new tokens
        cache = torch.zeros_like(good)
        out = rot.append(q, k, v, dev[0], cache, ids, dev[2], dev[3], 16, q_out=torch.empty_like(q))
        want = good.clone()
        want[host["ids"][1]] = 0
        assert torch.equal(cache, want)
        close(out, turned(q, places, config), q, config)
    short = dev[1][: host["page_indptr"][2]].contiguous()   # row 2's entries are past the list
    cache = torch.zeros_like(good)
    rot.append(q.clone(), k, v, dev[0], cache, short, dev[2], dev[3], 16)
    want = good.clone()
    want[host["ids"][host["page_indptr"][2] :]] = 0
    assert torch.equal(cache, want)


def test_append_past_32_bit_offsets(gpu):
    """A pool of more than 2^31 values: pages at its end."""
    say("rotary append long cache")
    config = RotaryConfig(head_dim=128)
    rot = RotaryEmbedding(config, gpu)
    pool = 70000                                 # x 32,768 values = 2.3e9
    cache = torch.zeros(pool, 2, 16, 8, 128, dtype=BF, device=gpu)
    q, k, v = tensors(2, 16, 8, 128, BF, gpu)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    rot.append(q, k, v, i32(0, 1, 2), cache, i32(pool - 1, 5), i32(0, 1, 2), i32(16, 1), 16)
    close(cache[pool - 1, 0, 15][None], turned(k, torch.tensor([15, 0]), config)[:1], k[:1], config)
    assert torch.equal(cache[pool - 1, 1, 15], v[0]) and torch.equal(cache[5, :, 0], torch.stack([k[1], v[1]]))
    assert int(torch.count_nonzero(cache[: pool - 1]).item()) == int(torch.count_nonzero(cache[5]).item())


def test_graph_and_streams(gpu):
    """Captured once, replayed on new contents of the same tensors; on a side stream; two calls on two streams."""
    say("rotary graph")
    config = RotaryConfig(head_dim=128, rotary_dim=96)
    rot = RotaryEmbedding(config, gpu)
    host, dev, places, pool = pages_of([50, 20], [3, 20], 16, gpu, 9)
    q, k, v = tensors(23, 8, 2, 128, BF, gpu)
    pos = places.to(gpu)
    cache = torch.zeros(pool, 2, 16, 2, 128, dtype=BF, device=gpu)
    q_out = torch.empty(23, 8, 128, dtype=BF, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rot.append(q, k, v, *dev[:1], cache, *dev[1:], 16, q_out=q_out)
        other, _ = rot.apply(q, k, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rot.append(q, k, v, *dev[:1], cache, *dev[1:], 16, q_out=q_out)
        qa, ka = rot.apply(q, k, pos)
    for i in range(4):
        q.copy_(torch.randn_like(q)), k.copy_(torch.randn_like(k)), v.copy_(torch.randn_like(v))
        graph.replay()
        torch.cuda.synchronize()
        eq, ek = rot.apply(q, k, pos)
        fresh = torch.zeros_like(cache)
        rot.append(q, k, v, *dev[:1], fresh, *dev[1:], 16, q_out=torch.empty_like(q_out))
        assert torch.equal(q_out, eq) and torch.equal(qa, eq) and torch.equal(ka, ek) and torch.equal(cache, fresh)


def test_refusals(gpu):
    say("rotary refusals")
    rot = RotaryEmbedding(RotaryConfig(head_dim=64), gpu)
    q, k, v = tensors(4, 4, 2, 64, BF, gpu)
    pos = torch.arange(4, device=gpu)
    bad = pytest.raises(ValueError)
    for args in ((q.half(), k, pos), (q.double(), None, pos), (q[..., :32], None, pos), (q[:, 0], None, pos),
                 (q, k[:3], pos), (q, k, pos[:3]), (q, k, pos.float()), (q, k, pos.cpu()), (q.transpose(1, 2), None, pos),
                 (q, k, pos[None])):
        with bad:
            rot.apply(*args)
    with pytest.raises(RuntimeError):
        rot.apply(q.cpu(), None, pos)
    with bad:
        RotaryEmbedding(RotaryConfig(head_dim=64), "cpu").apply(q, k, pos)
    with bad:
        rot.apply_inplace(q.clone().requires_grad_(), None, pos)
    host, dev, places, pool = pages_of([20], [4], 16, gpu, 1)
    cache = torch.zeros(pool, 2, 16, 2, 64, dtype=BF, device=gpu)
    args = lambda **kw: [kw.get(n, x) for n, x in zip("q k v indptr cache ids ptr last page".split(),
                                                      (q, k, v, dev[0], cache, dev[1], dev[2], dev[3], 16))]
    for kw in (dict(v=v[:, :1]), dict(k=k[:2]), dict(cache=cache.half()), dict(page=8), dict(cache=cache[..., :32]),
               dict(indptr=dev[0][:1]), dict(ptr=dev[2][:1]), dict(ids=dev[1].float()), dict(last=dev[3].cpu()),
               dict(q=q.float(), k=k.float(), v=v.float(), cache=cache.float())):
        with bad:
            rot.append(*args(**kw))
    with bad:
        rot.append(*args(), q_out=torch.empty(4, 4, 32, dtype=BF, device=gpu))
    with bad:
        rot.append(*args(), positions=pos[:2])
    square = torch.zeros(4, 4, 64, dtype=BF, device=gpu)
    with bad:
        rot.append(*args(q=square), q_out=square.transpose(0, 1))
    empty = rot.apply(q[:0], k[:0], pos[:0])
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 2, 64)
    rot.append(q[:0], k[:0], v[:0], dev[0], cache, dev[1], dev[2], dev[3], 16)
    assert not cache.any()


@pytest.mark.parametrize("dtype", [BF, SF])
def test_forward_mode(gpu, dtype):
    """Tangents of a dual q and k, one alone, and the tangent of a gradient."""
    say("rotary forward mode", dtype)
    config = RotaryConfig(head_dim=80, rotary_dim=20, layout="interleaved", **CONFIGS["yarn"])
    rot = RotaryEmbedding(config, gpu)
    q, k, _ = (t.contiguous() for t in tensors(9, 4, 2, 80, dtype, gpu))
    tq, tk, dq = torch.randn_like(q), torch.randn_like(k), torch.randn_like(q)
    pos = torch.arange(9) * 1001 - 1
    with fwad.dual_level():
        a, b = rot.apply(fwad.make_dual(q, tq), fwad.make_dual(k, tk), pos.to(gpu))
        close(a, turned(q, pos, config), q, config)
        close(fwad.unpack_dual(a).tangent, turned(tq, pos, config), tq, config)
        close(fwad.unpack_dual(b).tangent, turned(tk, pos, config), tk, config)
        a, b = rot.apply(q, fwad.make_dual(k, tk), pos.to(gpu))
        assert not fwad.unpack_dual(a).tangent.any()
        close(fwad.unpack_dual(b).tangent, turned(tk, pos, config), tk, config)
        leaf = q.clone().requires_grad_()
        a, _ = rot.apply(leaf, None, pos.to(gpu))
        (grad,) = torch.autograd.grad(a, [leaf], fwad.make_dual(dq, tq))
        close(grad, turned(dq, pos, config, inverse=True), dq, config)
        close(fwad.unpack_dual(grad).tangent, turned(tq, pos, config, inverse=True), tq, config)


@pytest.mark.parametrize("kw", [dict(head_dim=128, theta=1e6), dict(head_dim=64, **CONFIGS["llama3"])])
def test_far_positions_against_the_true_frequencies(gpu, kw):
    """cos and sin themselves, against frequencies to 200 bits. The table's entries are off by half a step of 2^-64 turns,
    which the position multiplies; the rest is the kernel's own (see close)."""
    say("rotary far, true", kw)
    config = RotaryConfig(**kw)
    rot = RotaryEmbedding(config, gpu)
    pos = [131071, (1 << 31) - 1, (1 << 33) + 5, 1 << 38]
    x = torch.zeros(len(pos), 1, config.head_dim, device=gpu)
    x[..., : config.head_dim // 2] = 1
    y, _ = rot.apply(x, None, torch.tensor(pos, device=gpu))
    true = true_frequencies(config)
    for i, p in enumerate(pos):
        angle = np.array([float(p * f / (2 * PI) % 1) * 2 * np.pi for f in true])
        ref = np.concatenate([np.cos(angle), np.sin(angle)])
        assert np.abs(y[i, 0].cpu().double().numpy() - ref).max() <= 10 * 2.0 ** -24 + p * 2.0 ** -65 * 2 * np.pi
