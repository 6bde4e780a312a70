"""Penalties, biases and masks on logits against the definition in 64 bits."""

import numpy as np
import pytest
import torch

from aspire_amd.logits_processor import LogitBias, adjust_logits
from helpers import say
from tree_cases import adjusted, ancestors, pack, random_tree

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def close(out, ref, touched, size, before):
    """Half a step of the output's type of the value, and 8 * 2^-24 of the largest magnitude on the way: a quotient or product, the
    product and sum of the frequency, the presence and the bias round once each, all within that size, and their parameters are fp32."""
    got = out.detach().cpu().double().numpy()
    assert np.array_equal(got[~touched], before.cpu().double().numpy()[~touched])
    ref = np.where(touched, ref, got)
    finite = np.isfinite(ref)
    assert np.array_equal(got[~finite], ref[~finite], equal_nan=True)
    big = float(torch.finfo(out.dtype).max)
    half = torch.finfo(out.dtype).eps / 2
    inside = finite & (np.abs(ref) < big * (1 - half))
    limit = half * np.abs(ref) + 8 * 2.0 ** -24 * size * (1 + half) + (2.0 ** -25 if out.dtype == torch.float16 else 0)
    off = np.abs(np.where(inside, got - ref, 0)) - limit
    assert not (off > 0).any(), f"{int((off > 0).sum())} of {off.size} off, worst by {off.max()}"


def mask_bits(allowed):
    T, V = allowed.shape
    wide = np.zeros((T, (V + 31) // 32 * 32), np.uint8)
    wide[:, :V] = allowed
    return np.packbits(wide, axis=1, bitorder="little").view(np.int32)


def parts(gpu, requests, vocab, history, seed):
    r = np.random.default_rng(seed)
    ids = (r.random((requests, history)) ** 4 * vocab).astype(np.int32)
    lens = r.integers(0, history + 1, size=requests)
    return dict(history=ids, lens=lens, prompts=r.integers(0, lens + 1), rep=(r.random(requests) + 0.6).astype(np.float32),
                pres=r.normal(size=requests).astype(np.float32), freq=r.normal(size=requests).astype(np.float32))


def call(logits, p, gpu, out=None, bias=None, allowed=None, qo=None, tree=None, see=None, words=1, start=0, grammar_rows=None):
    t = lambda x, d=None: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(gpu) if d is None else torch.tensor(x, dtype=d, device=gpu)
    kw = {}
    if p:
        names = dict(history="history", lens="history_lens", prompts="prompt_lens", rep="repetition", pres="presence", freq="frequency")
        for k, n in names.items():
            if p.get(k) is not None:
                kw[n] = t(p[k] if k not in ("lens", "prompts") else np.asarray(p[k], np.int32))
    return adjust_logits(logits, qo_indptr=t(qo, torch.int32) if qo is not None else None, tree_tokens=t(tree),
                         tree_masks=None if see is None else t(pack(see, words)),
                         bias=None if bias is None else LogitBias(bias, gpu), grammar=None if allowed is None else t(mask_bits(allowed)),
                         grammar_rows=t(grammar_rows), vocab_start=start, out=out, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests,vocab,history", [(1, 1, 1), (1, 7, 5), (3, 31, 40), (2, 4096, 600), (5, 4097, 1), (2, 20011, 4001),
                                                    (64, 1000, 100), (1, 151936, 9000)])
def test_penalties(gpu, dtype, requests, vocab, history):
    say("penalties", dtype, requests, vocab, history)
    g = torch.Generator(device=gpu).manual_seed(vocab)
    x = torch.randn(requests, vocab, device=gpu, generator=g).mul_(4).to(dtype)
    p = parts(gpu, requests, vocab, history, vocab)
    out = call(x, p, gpu)
    close(out, *adjusted(x, **p), x)
    for drop in (("rep",), ("pres", "freq"), ("prompts",), ("freq", "rep")):
        q = {k: v for k, v in p.items() if k not in drop}
        close(call(x, q, gpu), *adjusted(x, **q), x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 30, 32, 33, 4099, 12345])
@pytest.mark.parametrize("what", ["bias", "mask", "bias+mask", "all", "nothing"])
def test_biases_and_masks(gpu, dtype, vocab, what):
    say("biases and masks", dtype, vocab, what)
    r = np.random.default_rng(vocab)
    T = 6
    x = torch.randn(T, vocab, device=gpu, generator=torch.Generator(device=gpu).manual_seed(vocab)).mul_(3).to(dtype)
    bias = [{int(i): float(r.normal() * 9) for i in r.choice(vocab, size=min(vocab, n), replace=False)} for n in (0, 1, 5, 50, 3, 7)]
    bias[0] = None
    bias[2][int(r.integers(0, vocab))] = float("-inf")
    bias[3][vocab + 4] = 3.0  # beyond the vocabulary: no column
    allowed = r.random((T, vocab)) < np.array([0.5, 0.0, 1.0, 0.01, 0.99, 0.5])[:, None]
    p = parts(gpu, T, vocab, 50, 1) if what == "all" else None
    bias, allowed = (b if what in (n, "bias+mask", "all") else None for b, n in ((bias, "bias"), (allowed, "mask")))
    out = call(x, p, gpu, bias=bias, allowed=allowed)
    ref = adjusted(x, **(p or {}), bias=bias, allowed=allowed)
    close(out, *ref, x)
    if what == "nothing":
        assert torch.equal(out, x)
    if allowed is not None:
        assert torch.isneginf(out[1]).all()  # a mask that leaves nothing
    same = call(x.clone(), p, gpu, bias=bias, allowed=allowed, out=None)
    assert torch.equal(same.view(torch.uint8), out.view(torch.uint8))
    y = x.clone()
    assert call(y, p, gpu, bias=bias, allowed=allowed, out=y) is y
    assert torch.equal(y.view(torch.uint8), out.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nodes", [[1], [4, 0, 9], [70, 3], [64, 1, 130]])
def test_trees(gpu, dtype, nodes):
    """Each drafted token's own path counts as output, the same token on it several times too; rows behind the last request stay."""
    say("logits of trees", dtype, nodes)
    r = np.random.default_rng(sum(nodes))
    vocab, T, pad, words = 5003, sum(nodes), 3, 3
    x = torch.randn(T + pad, vocab, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1)).mul_(3).to(dtype)
    p = parts(gpu, len(nodes), vocab, 300, 5)
    tree = np.concatenate([r.integers(0, 6, size=T) * 911, np.zeros(pad)]).astype(np.int32)
    tree[0] = -1                                # of no column
    tree[T - 1] = vocab
    see = np.zeros((T + pad, words * 64), bool)
    at = 0
    for n in nodes:
        see[at : at + n, :n] = ancestors(random_tree(n, r))
        at += n
    see[T:] = True
    qo = [0, *np.cumsum(nodes).tolist()]
    bias = [{911: 2.5, 4999: -1.0} for _ in nodes]
    out = torch.full_like(x, 5.0)
    call(x, p, gpu, qo=qo, tree=tree, see=see, words=words, bias=bias, out=out)
    ref, touched, size = adjusted(x, qo=qo, tree=tree, see=see, bias=bias, **p)
    close(out, ref, touched, size, torch.full_like(x, 5.0))
    # the path alone, without a history
    q = {k: p[k] for k in ("rep", "pres", "freq")}
    out = call(x[:T], q, gpu, qo=qo, tree=tree[:T], see=see[:T], words=words)
    close(out, *adjusted(x[:T], qo=qo, tree=tree[:T], see=see[:T], **q), x[:T])


def test_shards_add_up(gpu):
    say("logits shards")
    vocab, T = 9001, 4
    x = torch.randn(T, vocab, device=gpu)
    p = parts(gpu, T, vocab, 500, 3)
    bias = [{5: 1.0, 8999: 2.0}] * T
    whole = call(x, p, gpu, bias=bias)
    cut = 4511
    left = call(x[:, :cut], p, gpu, bias=bias)
    right = call(x[:, cut:], p, gpu, bias=bias, start=cut)
    assert torch.equal(torch.cat([left, right], 1), whole)


def test_mask_rows(gpu):
    """Several rows share a mask; an index outside means none."""
    say("mask rows")
    r = np.random.default_rng(0)
    x = torch.randn(6, 777, device=gpu).to(torch.bfloat16)
    allowed = r.random((3, 777)) < 0.3
    which = np.array([2, 0, -1, 0, 3, 1], np.int32)
    full = np.stack([allowed[w] if 0 <= w < 3 else np.ones(777, bool) for w in which])
    out = call(x, None, gpu, allowed=allowed, grammar_rows=which)
    close(out, *adjusted(x, allowed=full), x)


def test_values(gpu):
    """Infinities, NaN, zeros and the type's lowest value; a masked place is -inf whatever it holds."""
    say("logits values")
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        x = torch.tensor([[float("-inf"), float("inf"), 0.0, -0.0, low, -low, float("nan"), 1.0]] * 2, device=gpu).to(dtype)
        p = dict(history=np.array([list(range(8))] * 2, np.int32), lens=[8, 8], rep=np.float32([1.5, 2.0]), freq=np.float32([0.5, 0.25]))
        out = call(x, p, gpu)
        ref, touched, size = adjusted(x, **p)
        got = out.cpu().double().numpy()
        nan = np.isnan(ref)
        assert np.array_equal(np.isnan(got), nan)
        keep = ~nan & np.isfinite(ref) & (np.abs(ref) < abs(low))
        assert np.allclose(got[keep], ref[keep], rtol=torch.finfo(dtype).eps, atol=1e-7)
        assert got[0, 0] == -np.inf and got[0, 1] == np.inf
        allowed = np.zeros((2, 8), bool)
        allowed[:, 7] = True
        out = call(x, p, gpu, allowed=allowed)
        assert torch.isneginf(out[:, :7]).all() and torch.isfinite(out[:, 7]).all()


def test_odd_histories(gpu):
    """Lengths of none and past the buffer, tokens outside the vocabulary, prompts longer than the history."""
    say("odd histories")
    x = torch.randn(5, 300, device=gpu)
    p = parts(gpu, 5, 300, 64, 0)
    p["history"][:, ::5] = -1
    p["history"][:, 1::7] = 300
    p["history"][:, 2::9] = 2 ** 31 - 1
    p["lens"], p["prompts"] = np.array([0, -4, 1000, 64, 3]), np.array([0, 2, 1000, 10, 64])
    close(call(x, p, gpu), *adjusted(x, **p), x)
    one = dict(history=np.full((1, 40000), 17, np.int32), lens=[40000], prompts=[1], freq=np.float32([0.125]))
    y = torch.zeros(1, 20, device=gpu)
    out = call(y, one, gpu)
    assert float(out[0, 17]) == -0.125 * 39999 and float(out.sum()) == -0.125 * 39999


def test_views(gpu):
    """Rows of logits, masks and histories inside larger ones, at every alignment."""
    say("logits views")
    for dtype in TYPES:
        big = torch.randn(4, 1300, device=gpu).to(dtype)
        for a in (0, 1, 3, 8):
            x = big[:, a : a + 1201]
            p = parts(gpu, 4, 1201, 64, a)
            allowed = np.random.default_rng(a).random((4, 1201)) < 0.7
            wide = torch.full((4, 1210), 9.0, device=gpu).to(dtype)
            out = wide[:, 5 : 5 + 1201]
            call(x, p, gpu, allowed=allowed, out=out)
            close(out, *adjusted(x, **p, allowed=allowed), x)
            assert (wide[:, :5] == 9).all() and (wide[:, 1206:] == 9).all()


def test_graph_and_stream(gpu):
    say("logits graph")
    x = torch.randn(8, 3000, device=gpu).to(torch.bfloat16)
    p = parts(gpu, 8, 3000, 200, 0)
    t = {k: torch.from_numpy(np.ascontiguousarray(v if k not in ("lens", "prompts") else v.astype(np.int32))).to(gpu) for k, v in p.items()}
    out = torch.empty_like(x)
    run = lambda o: adjust_logits(x, history=t["history"], history_lens=t["lens"], prompt_lens=t["prompts"], repetition=t["rep"],
                                  presence=t["pres"], frequency=t["freq"], out=o)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(out)
    for step in range(4):
        t["lens"].copy_(torch.randint(0, 200, (8,), device=gpu))
        x.normal_()
        want = run(None)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(gpu):
    say("logits refusals")
    x = torch.randn(3, 100, device=gpu)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)
    f = torch.ones(3, device=gpu)
    h = dict(history=i32(3, 5), history_lens=i32(3), repetition=f)
    adjust_logits(x, **h)
    for kw in (dict(history=i32(3, 5)), dict(history=i32(3, 5), history_lens=i32(3)), dict(history_lens=i32(3)), dict(repetition=f),
               {**h, "history": i32(2, 5)}, {**h, "history": i32(3, 5).long()}, {**h, "repetition": f[:2]}, {**h, "repetition": f.double()},
               {**h, "prompt_lens": i32(2)}, dict(prompt_lens=i32(3)), dict(bias=LogitBias([{}, {}], gpu)), dict(grammar=i32(3, 3)),
               dict(grammar=i32(2, 4)), dict(grammar=i32(3, 4).long()), dict(grammar_rows=i32(3)), dict(grammar=i32(1, 4), grammar_rows=i32(2)),
               dict(tree_tokens=i32(3), tree_masks=torch.zeros(3, 1, dtype=torch.int64, device=gpu), presence=f),
               dict(tree_tokens=i32(3), qo_indptr=i32(2)), dict(qo_indptr=i32(0)), dict(vocab_start=-1),
               dict(out=torch.empty(3, 99, device=gpu)), dict(out=torch.empty(3, 100, device=gpu).half()), dict(out=x.t()),
               dict(out=torch.empty(1, 100, device=gpu).expand(3, 100))):
        with pytest.raises(ValueError):
            adjust_logits(x, **kw)
    buf = torch.randn(4, 100, device=gpu)
    with pytest.raises(ValueError):
        adjust_logits(buf[:3], out=buf[1:])  # a part of it
    with pytest.raises(ValueError):
        adjust_logits(x.double())
    with pytest.raises(ValueError):
        adjust_logits(x[0])
    with pytest.raises(ValueError):
        adjust_logits(x.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        adjust_logits(x.cpu())
    for bad in ({-1: 1.0}, {2 ** 31: 1.0}, {3: float("nan")}):
        with pytest.raises(ValueError):
            LogitBias([bad], gpu)
    assert adjust_logits(x[:0]).shape == (0, 100) and adjust_logits(x[:, :0]).shape == (3, 0)
