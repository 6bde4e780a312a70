"""Rotary configurations and the host-side checks of the rotary entry points (no GPU)."""

import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwad

from aspire_amd import _lib
from aspire_amd.attention import rotary
from aspire_amd.attention.rope import RopeConfig, rope_frequencies
from aspire_amd.attention.rotary import RotaryConfig, RotaryEmbedding


def test_frequencies_equal_the_fused_kernels_where_both_exist():
    """Plain, divided and llama3 frequencies against aspire_rope_frequencies, whose fp32 values are the 64-bit ones rounded."""
    for mine, theirs in ((RotaryConfig(theta=1e6), RopeConfig(1e6)),
                         (RotaryConfig(theta=1e4, scaling="linear", factor=2.0), RopeConfig(1e4, 2.0)),
                         (RotaryConfig(theta=5e5, scaling="llama3", factor=8.0, original_max_position=8192),
                          RopeConfig(5e5, 8.0, 1.0, 4.0, 8192))):
        f, g = np.array(mine.frequencies()), rope_frequencies(128, theirs).double().numpy()
        assert np.all(np.abs(f - g) <= 2.0 ** -23 * g)


def test_yarn_regions():
    """Pairs that turn more than beta_fast times over the trained context keep their frequency, those below beta_slow
    are divided, the ones between lie between and never rise back."""
    c = RotaryConfig(theta=1e6, scaling="yarn", factor=4.0, original_max_position=32768)
    base = np.array(RotaryConfig(theta=1e6).frequencies())
    f, turns = np.array(c.frequencies()), 32768 * base / (2 * math.pi)
    keep = (f / base - 0.25) / 0.75
    assert np.allclose(keep[turns > 32 * 1.3], 1) and np.allclose(keep[turns < 1 / 1.3], 0, atol=1e-12)
    assert np.all(np.diff(keep) <= 1e-12) and ((keep > 0.01) & (keep < 0.99)).any()
    assert c.scale == 0.1 * math.log(4.0) + 1 and RotaryConfig().scale == 1
    assert RotaryConfig(scaling="yarn", original_max_position=4096).scale == 1     # nothing stretched
    assert RotaryConfig(amplitude=0.5).scale == 0.5


def test_partial_heads_use_the_rotated_width():
    whole, part = RotaryConfig(head_dim=64, theta=1e4), RotaryConfig(head_dim=256, rotary_dim=64, theta=1e4)
    assert whole.frequencies() == part.frequencies() and len(part.frequencies()) == 32


def test_turns_are_fractions_of_a_turn():
    c = RotaryConfig(head_dim=64, pair_factors=(0.01,) + (1.0,) * 31)  # 100 radians a position: many whole turns
    t = [x % (1 << 64) for x in RotaryEmbedding(c, "cpu").turns.tolist()]
    for x, f in zip(t, c.frequencies()):
        want = f / (2 * math.pi) % 1.0
        assert abs(x / 2.0 ** 64 - want) < 1e-13


@pytest.mark.parametrize("kw", [
    dict(head_dim=0), dict(head_dim=257), dict(rotary_dim=0), dict(rotary_dim=33), dict(rotary_dim=130), dict(head_dim=75),
    dict(layout="neox"), dict(scaling="dynamic"), dict(theta=0.0), dict(theta=float("nan")), dict(factor=-1.0),
    dict(scaling="yarn"), dict(scaling="llama3"), dict(scaling="yarn", original_max_position=4096, theta=1.0),
    dict(scaling="llama3", original_max_position=8192, high_freq_factor=1.0), dict(amplitude=float("inf")),
    dict(pair_factors=(1.0,)), dict(pair_factors=(1.0,) * 64, scaling="linear"),
])
def test_refused_configurations(kw):
    with pytest.raises(ValueError):
        RotaryConfig(**kw)


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libaspire_hip.so not built")
def test_entry_points_refuse_on_the_host():
    """Everything that the C entries can see to be wrong is refused before a launch (so this runs without a GPU)."""
    L = _lib.lib()

    def args(**kw):
        a = _lib.RotaryArgs(q=4096, q_out=8192, k=12288, k_out=16384, v=20480, num_qo_heads=4, num_kv_heads=2,
                            total_tokens=3, head_dim=64, rotary_dim=32, turns=4096, amplitude=1.0, positions=4096,
                            kv_cache=4096, num_pages=4, num_page_indices=4, page_size=16, num_seq=1, append_indptr=4096,
                            kv_page_indices=4096, kv_page_indptr=4096, kv_last_page_len=4096)
        for name, value in kw.items():
            setattr(a, name, value)
        return ctypes.byref(a)

    both = [dict(dtype=3), dict(dtype=-1), dict(head_dim=257), dict(rotary_dim=31), dict(rotary_dim=66), dict(rotary_dim=0),
            dict(total_tokens=-1), dict(total_tokens=1 << 26), dict(num_qo_heads=-1), dict(num_kv_heads=1025), dict(turns=None), dict(q=None), dict(q_out=None),
            dict(k=None)]
    for kw in both:
        for entry in (L.aspire_rotary, L.aspire_rotary_append):
            assert entry(args(**kw), None) == _lib.ASPIRE_ERR_INVALID, kw
    for kw in (dict(positions=None), dict(k_out=None)):
        assert L.aspire_rotary(args(**kw), None) == _lib.ASPIRE_ERR_INVALID, kw
    for kw in (dict(dtype=2), dict(v=None), dict(kv_cache=None), dict(page_size=0), dict(num_pages=-1), dict(num_seq=-1),
               dict(append_indptr=None), dict(kv_page_indptr=None), dict(kv_last_page_len=None), dict(kv_page_indices=None)):
        assert L.aspire_rotary_append(args(**kw), None) == _lib.ASPIRE_ERR_INVALID, kw
    assert "aspire_rotary_append" in _lib.lib().aspire_last_error().decode()
    assert L.aspire_rotary(args(total_tokens=0), None) == _lib.ASPIRE_OK
    assert L.aspire_rotary(None, None) == _lib.ASPIRE_ERR_INVALID


def test_packed_arguments_match_the_structure():
    """The string that the entry points get in place of the structure: every field at its place."""
    values = [float(i) if i == 25 else i for i in range(1, 41)]
    a = _lib.RotaryArgs.from_buffer_copy(rotary._ARGS.pack(*values))
    assert ctypes.sizeof(_lib.RotaryArgs) == rotary._ARGS.size
    assert [getattr(a, f[0]) for f in a._fields_] == values


def test_cpu_tensors_are_refused():
    rot = RotaryEmbedding(RotaryConfig(head_dim=64), "cpu")
    x, pos, i = torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    calls = (lambda: rot.apply(x, None, pos), lambda: rot.apply_inplace(x, x.clone(), pos),
             lambda: rot.append(x.half(), x.half(), x.half(), i, torch.zeros(1, 2, 16, 1, 64).half(), i, i, i[:1], 16))
    for call in calls:
        with pytest.raises(RuntimeError, match="GPU"):
            call()


class PlainTurn(RotaryEmbedding):
    """The turn in elementary operations, for what autograd does around it (half layout, whole heads)."""

    def _turn(self, q, k, positions, inverse, in_place, what):
        f = torch.tensor(self.config.frequencies(), dtype=torch.float64)
        angle = positions.double()[:, None, None] * f * (-1 if inverse else 1)
        outs = []
        for x in (q, k):
            a, b = (None, None) if x is None else x.detach().double().chunk(2, dim=-1)
            y = None if x is None else torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)
            outs.append(None if x is None else y.to(x.dtype))
        return tuple(outs)


def test_apply_carries_forward_mode_tangents():
    """A dual tensor's tangent turns as the values do (with grad mode on and off, of q or k alone, beside a gradient), and a
    gradient's tangent turns back."""
    rot = PlainTurn(RotaryConfig(head_dim=8), "cpu")
    pos = torch.tensor([3, 5, 11])
    g = torch.Generator().manual_seed(0)
    q, k, tq, tk = (torch.randn(3, h, 8, generator=g, dtype=torch.float64) for h in (4, 2, 4, 2))
    wq, wk = rot._turn(tq, tk, pos, False, False, "")
    back, _ = rot._turn(tq, None, pos, True, False, "")
    with fwad.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                a, b = rot.apply(fwad.make_dual(q, tq), fwad.make_dual(k, tk), pos)
                assert torch.equal(fwad.unpack_dual(a).tangent, wq) and torch.equal(fwad.unpack_dual(b).tangent, wk)
                a, b = rot.apply(q, fwad.make_dual(k, tk), pos)
                assert torch.equal(fwad.unpack_dual(b).tangent, wk) and torch.equal(a, rot.apply(q, None, pos)[0])
                assert not fwad.unpack_dual(a).tangent.any()
                a, none = rot.apply(fwad.make_dual(q, tq), None, pos)
                assert torch.equal(fwad.unpack_dual(a).tangent, wq) and none is None
                a, _ = rot.apply(fwad.make_dual(q, tq.transpose(0, 2).contiguous().transpose(0, 2)), None, pos)
                assert torch.equal(fwad.unpack_dual(a).tangent, wq)
        leaf = q.clone().requires_grad_()
        a, _ = rot.apply(fwad.make_dual(leaf, tq), None, pos)
        assert torch.equal(fwad.unpack_dual(a).tangent, wq)
        (grad,) = torch.autograd.grad(a, [leaf], fwad.make_dual(torch.ones_like(q), tq))
        assert torch.equal(fwad.unpack_dual(grad).tangent, back)
        a, b = rot.apply(leaf, k.clone().requires_grad_(), pos)
        (grad,) = torch.autograd.grad([a, b], [leaf], [fwad.make_dual(torch.ones_like(q), tq), torch.ones_like(k)])
        assert torch.equal(fwad.unpack_dual(grad).tangent, back)


def test_dual_tensors_are_refused_where_there_is_no_derivative():
    rot = RotaryEmbedding(RotaryConfig(head_dim=64), "cpu")
    x, i, pos = torch.zeros(1, 1, 64).half(), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    cache = torch.zeros(1, 2, 16, 1, 64).half()
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))
        calls = [lambda: rot.apply_inplace(dual(x), None, pos), lambda: rot.apply_inplace(x, dual(x.clone()), pos)]
        for at in range(5):
            given = [dual(t) if n == at else t for n, t in enumerate((x, x, x, cache, x.clone()))]
            calls.append(lambda a=given: rot.append(*a[:3], i, a[3], i, i, i[:1], 16, q_out=a[4]))
        for call in calls:
            with pytest.raises(ValueError, match="not differentiable"):
                call()


def arctan_inverse(n, one):
    """one * arctan(1 / n), its series in whole numbers."""
    total, power, k = 0, one // n, 1
    while power:
        total += power // k if k % 4 == 1 else -(power // k)
        power, k = power // (n * n), k + 2
    return total


BITS = 260
PI = Fraction(4 * (4 * arctan_inverse(5, 1 << BITS) - arctan_inverse(239, 1 << BITS)), 1 << BITS)  # Machin


def root(x, r):
    """floor(x ** (1 / r)) by bisection, all whole numbers."""
    lo, hi = 0, 1 << (x.bit_length() // r + 1)
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if mid ** r <= x else (lo, mid)
    return lo


def true_frequencies(config):
    """theta ** (-2 i / R) and what the scalings make of it, to some 200 bits: the R-th root of theta ** (-2 i)."""
    r, theta = config.rotated, Fraction(config.theta)
    base = [Fraction(root(int((1 << (220 * r)) / theta ** (2 * i)), r), 1 << 220) for i in range(r // 2)]
    factor = Fraction(config.factor)
    if config.pair_factors is not None:
        return [f / Fraction(s) for f, s in zip(base, config.pair_factors)]
    if config.scaling == "linear":
        return [f / factor for f in base]
    if config.scaling == "llama3":
        lo, hi = Fraction(config.low_freq_factor), Fraction(config.high_freq_factor)
        keep = [min(max((config.original_max_position * f / (2 * PI) - lo) / (hi - lo), Fraction(0)), Fraction(1)) for f in base]
    elif config.scaling == "yarn":
        # the pairs that turn beta_fast and beta_slow times over the trained context, out to whole numbers
        ends = [r * math.log(config.original_max_position / (b * 2 * math.pi)) / (2 * math.log(config.theta))
                for b in (config.beta_fast, config.beta_slow)]
        first, last = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), r - 1)
        keep = [1 - min(max(Fraction(i - first, last - first), Fraction(0)), Fraction(1)) for i in range(r // 2)]
    else:
        return base
    return [t * f + (1 - t) * f / factor for t, f in zip(keep, base)]


TABLES = [dict(theta=1e6), dict(theta=1e4, head_dim=80, rotary_dim=20), dict(theta=1e4, scaling="linear", factor=4.0),
          dict(theta=5e5, scaling="llama3", factor=8.0, original_max_position=8192),
          dict(theta=1e6, scaling="yarn", factor=4.0, original_max_position=32768, head_dim=64),
          dict(theta=10000.5, head_dim=2), dict(theta=0.125, head_dim=8, pair_factors=(3.0, 0.001, 1.0, 2.0 ** -40))]


@pytest.mark.parametrize("kw", TABLES)
def test_the_table_of_turns_has_all_its_bits(kw):
    """Every entry is the nearest 64-bit fraction of a turn (an entry that was made in a double has 53 bits, and a position
    multiplies what is missing), and frequencies() the nearest doubles."""
    config = RotaryConfig(**kw)
    true = true_frequencies(config)
    for got, f in zip(RotaryEmbedding(config, "cpu").turns.tolist(), true):
        off = (got - f / (2 * PI) * 2 ** 64) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + Fraction(1, 2 ** 20)
    assert config.frequencies() == [float(f) for f in true]


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libaspire_hip.so not built")
@pytest.mark.parametrize("tokens", [(1 << 26) - 3, (1 << 26) - 2, (1 << 26) - 1, (1 << 31) - 1])
def test_launches_of_2_to_the_32_threads_are_refused(tokens):
    """Workgroups of 4 tokens and 256 threads: past 2^26 - 4 tokens the last, partly filled one makes 2^32 threads."""
    L = _lib.lib()
    a = _lib.RotaryArgs(q=4096, q_out=8192, num_qo_heads=1, total_tokens=tokens, head_dim=64, rotary_dim=64, turns=4096,
                        amplitude=1.0, positions=4096, kv_cache=4096, num_pages=4, page_size=16)
    for entry in (L.aspire_rotary, L.aspire_rotary_append):
        assert entry(ctypes.byref(a), None) == _lib.ASPIRE_ERR_INVALID
