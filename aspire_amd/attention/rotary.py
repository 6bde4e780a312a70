"""Rotary positions in the forms that checkpoints have, alone and with the paged append (HIP).

``rope`` serves one form (interleaved pairs of whole 128-wide bf16 heads, in place, behind the q/k norm). Here a
``RotaryConfig`` says how a model turns its heads, and a ``RotaryEmbedding`` holds its frequencies on a device:

* pairs ``(i, i + R/2)`` (``layout="half"``) or ``(2i, 2i + 1)`` (``"interleaved"``) of the first ``R = rotary_dim``
  values of a head of up to 256; the others pass unchanged;
* frequencies ``f_i = theta^(-2i/R)``, or scaled for long contexts: ``"linear"`` (``f / factor``), ``"llama3"``
  (the smoothing of ``RopeConfig``), ``"yarn"`` (between the pairs that turn ``beta_fast`` and ``beta_slow`` times
  over the trained context ``f`` becomes ``f / factor`` linearly; cos and sin times ``0.1 ln(factor) + 1``), or
  divided by given ``pair_factors``;
* a frequency is the nearest 64-bit fraction of a turn, made from some 45 digits, and its product with the position drops
  whole turns only: angles ``position * f_i`` are within ``position * 2^-65`` turns (2^-24 radians at 2^38); cos and sin
  and the products fp32, one rounding to the output's type.

``apply`` is differentiable (the gradient turns back by the same angles); ``append`` is
``mylib::update_kv_padded`` (aspire/attention/kv_ops.py:63-187) with the turn on the way, one launch.
"""

from __future__ import annotations

import math
import struct
from dataclasses import dataclass
from decimal import Context, Decimal, localcontext

import torch
from torch.autograd import forward_ad

from aspire_amd import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
SCALINGS = ("none", "linear", "llama3", "yarn")
MAX_HEAD_DIM = 256
_PI = Decimal("3.1415926535897932384626433832795028841971693993751058209749445923078164062862089986")


@dataclass(frozen=True)
class RotaryConfig:
    head_dim: int = 128
    rotary_dim: int | None = None            # None: the whole head
    layout: str = "half"                     # or "interleaved"
    theta: float = 10000.0
    scaling: str = "none"
    factor: float = 1.0
    low_freq_factor: float = 1.0             # llama3
    high_freq_factor: float = 4.0
    original_max_position: int | None = None  # llama3, yarn: the trained context
    beta_fast: float = 32.0                  # yarn
    beta_slow: float = 1.0
    amplitude: float | None = None           # on cos and sin; None: yarn's 0.1 ln(factor) + 1, else 1
    pair_factors: tuple | None = None        # f_i / pair_factors[i], with scaling "none"

    def __post_init__(self):
        if not 0 < self.head_dim <= MAX_HEAD_DIM:
            raise ValueError(f"RotaryConfig: head_dim must be 1 to {MAX_HEAD_DIM}")
        r = self.rotated
        if r <= 0 or r % 2 or r > self.head_dim:
            raise ValueError("RotaryConfig: rotary_dim must be even, positive and within head_dim")
        if self.layout not in ("half", "interleaved"):
            raise ValueError("RotaryConfig: layout must be 'half' or 'interleaved'")
        if self.scaling not in SCALINGS:
            raise ValueError(f"RotaryConfig: scaling must be one of {SCALINGS}")
        finite = [self.theta, self.factor, self.low_freq_factor, self.high_freq_factor, self.beta_fast, self.beta_slow,
                  *(self.pair_factors or ()), *(() if self.amplitude is None else (self.amplitude,))]
        if not all(math.isfinite(x) and x > 0 for x in finite):
            raise ValueError("RotaryConfig: theta, factors, betas and amplitude must be positive and finite")
        if self.scaling in ("llama3", "yarn") and not (self.original_max_position or 0) > 0:
            raise ValueError(f"RotaryConfig: scaling {self.scaling!r} needs original_max_position")
        if self.scaling == "llama3" and self.high_freq_factor <= self.low_freq_factor:
            raise ValueError("RotaryConfig: high_freq_factor must be above low_freq_factor")
        if self.scaling == "yarn" and (self.beta_fast < self.beta_slow or self.theta <= 1):
            raise ValueError("RotaryConfig: yarn needs beta_fast >= beta_slow and theta > 1")
        if self.pair_factors is not None and (self.scaling != "none" or len(self.pair_factors) != r // 2):
            raise ValueError("RotaryConfig: pair_factors go with scaling 'none', one for each pair")

    @property
    def rotated(self) -> int:
        return self.head_dim if self.rotary_dim is None else int(self.rotary_dim)

    @property
    def scale(self) -> float:
        """The factor on cos and sin."""
        if self.amplitude is not None:
            return float(self.amplitude)
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "yarn" and self.factor > 1 else 1.0

    def _exact_frequencies(self) -> list[Decimal]:
        """Radians a position of each pair, to more digits than 64 bits of a turn need (whole turns of a small theta or
        divisor are dropped later, so their digits come on top)."""
        r, divisors = self.rotated, (self.factor, *(self.pair_factors or ()))
        whole = max(0.0, -math.log10(self.theta)) + max(0.0, -math.log10(min(divisors)))
        with localcontext(Context(prec=45 + math.ceil(whole))):
            exact = lambda x: Decimal(float(x))
            ratio, base = (exact(self.theta).ln() * -2 / r).exp(), [Decimal(1)]
            while len(base) < r // 2:
                base.append(base[-1] * ratio)
            if self.pair_factors is not None:
                return [f / exact(s) for f, s in zip(base, self.pair_factors)]
            factor = exact(self.factor)
            if self.scaling == "linear":
                return [f / factor for f in base]
            if self.scaling == "llama3":
                lo, hi, old = exact(self.low_freq_factor), exact(self.high_freq_factor), exact(self.original_max_position)
                slope, start = old / (2 * _PI) / (hi - lo), lo / (hi - lo)
                keep = [f * slope - start for f in base]
            elif self.scaling == "yarn":
                def at(turns):  # the pair that turns so often over the trained context
                    return r * math.log(self.original_max_position / (2 * math.pi * turns)) / (2 * math.log(self.theta))
                first, last = max(math.floor(at(self.beta_fast)), 0), min(math.ceil(at(self.beta_slow)), r - 1)
                width = Decimal(max(last - first, 0.001))
                keep = [1 - (i - first) / width for i in range(r // 2)]
            else:
                return base
            return [f if t >= 1 else f / factor if t <= 0 else t * f + (1 - t) * f / factor for t, f in zip(keep, base)]

    def frequencies(self) -> list[float]:
        """Radians a position of each pair, as the nearest doubles."""
        return [float(f) for f in self._exact_frequencies()]

    def _turns(self) -> torch.Tensor:
        """The frequencies as 64-bit fixed-point fractions of a turn a position, to the nearest (int64 holding the bits)."""
        frequencies = self._exact_frequencies()
        with localcontext(Context(prec=45 + max(0, *(f.adjusted() for f in frequencies)))):
            scale, half = 2 ** 63 / _PI, Decimal("0.5")
            turns = [int(f * scale + half) % (1 << 64) for f in frequencies]
        return torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64)


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether ``b`` of ``a``'s shape can stand for it: no shared start, or the same layout."""
    return a.data_ptr() != b.data_ptr() or all(n == 1 or x == y for n, x, y in zip(a.shape, a.stride(), b.stride()))


# aspire_rotary_args as one packed string: filling a ctypes structure field by field takes longer than the launch.
# q .. v (pointer and strides), eight counts, turns, amplitude, positions; then the cache, its strides and lists.
_HEAD = struct.Struct("PqqPqqPqqPqqPqq8iPfiP")
_ARGS = struct.Struct(_HEAD.format + "P4q2q2i4P")
_NO_CACHE = bytes(_ARGS.size - _HEAD.size)
_NONE = (0, 0, 0)
_INTS = (torch.int32, torch.int64)


class RotaryEmbedding:
    """A model's rotary positions on one device, for up to 1,024 q and 1,024 k heads and 2^26 - 4 tokens a call."""

    def __init__(self, config: RotaryConfig, device="cuda"):
        self.config = config
        self.turns = config._turns().to(device)
        self.device = self.turns.device
        self._index = self.turns.get_device() if self.turns.is_cuda else -2  # (-2: no tensor's)
        self._dims = (config.head_dim, config.rotated, int(config.layout == "interleaved"))

    # ------------------------------------------------------------------ checks
    def _heads(self, t: torch.Tensor, dtype: torch.dtype, what: str, name: str):
        """A head tensor's shape, its address and strides, after its checks."""
        shape, strides = t.shape, t.stride()
        if t.get_device() == self._index and t.dtype is dtype and len(shape) == 3 and shape[2] == self._dims[0] \
                and (strides[2] == 1 or not t.numel()):
            return shape, (t.data_ptr(), strides[0], strides[1])
        _lib.require_cuda(t, what=what)
        if t.get_device() != self._index:
            raise ValueError(f"{what}: {name} is on {t.device}, the frequencies on {self.device}")
        raise ValueError(f"{what}: {name} must be {dtype} [T, H, {self._dims[0]}] with contiguous head dims")

    def _list(self, t: torch.Tensor, what: str):
        """An index array as int32 in one piece, and its length."""
        if t.dim() != 1 or t.get_device() != self._index or t.dtype not in _INTS:
            raise ValueError(f"{what}: the index arrays must be 1-D int32 on {self.device}")
        t = _lib.indices(t)
        return t, t.shape[0]

    def _dtype(self, t: torch.Tensor, what: str) -> int:
        code = _DTYPES.get(t.dtype)
        if code is None:
            raise ValueError(f"{what}: bf16, fp16 or fp32 tensors")
        return code

    def _positions(self, positions: torch.Tensor, tokens: int, what: str) -> torch.Tensor:
        if positions.dtype not in _INTS or positions.shape != (tokens,):
            raise ValueError(f"{what}: positions must be int32 or int64 [T]")
        if positions.get_device() != self._index:
            raise ValueError(f"{what}: positions are on {positions.device}, the frequencies on {self.device}")
        return positions if positions.stride(0) == 1 else positions.contiguous()

    def _launch(self, entry, args: bytes, what: str) -> None:
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        if torch._C._cuda_getDevice() == self._index:
            rc = entry(args, stream)
        else:
            with torch.cuda.device(self._index):
                rc = entry(args, stream)
        if rc:
            _lib.check(rc, what)

    def _turn(self, q, k, positions, inverse, in_place, what):
        """q and k (either may be None) turned, in place or into new tensors, which it returns."""
        first = q if q is not None else k
        code, dtype = self._dtype(first, what), first.dtype
        tokens, hq, hkv, qa, ka, qo, ko = first.shape[0], 0, 0, _NONE, _NONE, _NONE, _NONE
        q_out, k_out = q, k
        if q is not None:
            shape, qa = self._heads(q, dtype, what, "q")
            hq, qo = shape[1], qa
            if not in_place:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
                qo = (q_out.data_ptr(), hq * shape[2], shape[2])
        if k is not None:
            shape, ka = self._heads(k, dtype, what, "k")
            if shape[0] != tokens:
                raise ValueError(f"{what}: q and k must have the same number of tokens")
            hkv, ko = shape[1], ka
            if not in_place:
                k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
                ko = (k_out.data_ptr(), hkv * shape[2], shape[2])
        positions = self._positions(positions, tokens, what)
        args = _HEAD.pack(*qa, *qo, *ka, *ko, *_NONE, hq, hkv, tokens, *self._dims, code, inverse, self.turns.data_ptr(), self.config.scale,
                          positions.dtype is torch.int64, positions.data_ptr()) + _NO_CACHE
        self._launch(_lib.lib().aspire_rotary, args, what)
        return q_out, k_out

    # -------------------------------------------------------------- operators
    def apply(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor):
        """``(q, k)`` turned at ``positions`` ``[T]``, as new tensors (``k`` may be None); differentiable, in reverse and in
        forward mode. Tokens at negative positions are copied."""
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) \
                or forward_ad._current_level >= 0 and _lib.has_tangent(q, k):
            return _Turn.apply(q, k, positions, self, False)
        return self._turn(q, k, positions, False, False, "RotaryEmbedding.apply")

    def apply_inplace(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor) -> None:
        """``apply`` on q and k themselves (not differentiable; no two of their rows may share memory)."""
        what = "RotaryEmbedding.apply_inplace"
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) \
                or forward_ad._current_level >= 0 and _lib.has_tangent(q, k):
            raise ValueError(f"{what}: not differentiable; use apply")
        self._turn(q, k, positions, False, True, what)

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_append_indptr: torch.Tensor,
               kv_cache: torch.Tensor, kv_page_indices: torch.Tensor, kv_page_indptr: torch.Tensor,
               kv_last_page_len: torch.Tensor, page_size: int, *, positions: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor:
        """Turn q (in place, or into ``q_out``, which it returns) and append the turned k and v to ``kv_cache``
        ``[P, 2, page, H_kv, D]`` where ``mylib::update_kv_padded`` would put them, in one launch. A token's position is
        its place in its row's sequence unless ``positions`` ``[T]`` gives another (negative: not turned). Tokens of no
        row are padding: their q passes unchanged, and nothing is written to the cache; nor is it for a token whose
        page id or list entry lies outside the pool or the list. No two tokens may share a slot."""
        what = "RotaryEmbedding.append"
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad) \
                or forward_ad._current_level >= 0 and _lib.has_tangent(q, k, v, q_out, kv_cache):
            raise ValueError(f"{what}: not differentiable")
        code, dtype = self._dtype(q, what), q.dtype
        if code == 2:
            raise ValueError(f"{what}: the cache holds bf16 or fp16")
        shape, qa = self._heads(q, dtype, what, "q")
        kv_shape, ka = self._heads(k, dtype, what, "k")
        v_shape, va = self._heads(v, dtype, what, "v")
        tokens, hkv = shape[0], kv_shape[1]
        qo = qa
        if q_out is None:
            q_out = q
        elif q_out is not q:
            out_shape, qo = self._heads(q_out, dtype, what, "q_out")
            if out_shape != shape:
                raise ValueError(f"{what}: q_out must have q's shape")
            if not _same_place(q, q_out):
                raise ValueError(f"{what}: q_out must be q itself or apart from it")
        if kv_shape[0] != tokens or v_shape != kv_shape:
            raise ValueError(f"{what}: q, k and v must have the same tokens, k and v the same heads")
        cache_shape, cs = kv_cache.shape, kv_cache.stride()
        if kv_cache.get_device() != self._index or kv_cache.dtype is not dtype \
                or cache_shape[1:] != (2, page_size, hkv, self._dims[0]) or cs[4] != 1:
            raise ValueError(f"{what}: kv_cache must be {dtype} [P, 2, {page_size}, {hkv}, {self._dims[0]}] on "
                             f"{self.device} with contiguous head dims")
        (ind, ind_len), (pages, num_pages) = self._list(kv_append_indptr, what), self._list(kv_page_indices, what)
        (ptr, ptr_len), (last, num_seq) = self._list(kv_page_indptr, what), self._list(kv_last_page_len, what)
        if ind_len <= num_seq or ptr_len <= num_seq:
            raise ValueError(f"{what}: kv_page_indptr and kv_append_indptr need len(kv_last_page_len) + 1 entries")
        at, wide = 0, False
        if positions is not None:
            positions = self._positions(positions, tokens, what)
            at, wide = positions.data_ptr(), positions.dtype is torch.int64
        args = _ARGS.pack(*qa, *qo, *ka, *_NONE, *va, shape[1], hkv, tokens, *self._dims, code, 0, self.turns.data_ptr(),
                          self.config.scale, wide, at, kv_cache.data_ptr(), cs[0], cs[1], cs[2], cs[3], cache_shape[0], num_pages, page_size,
                          num_seq, ind.data_ptr(), pages.data_ptr(), ptr.data_ptr(), last.data_ptr())
        self._launch(_lib.lib().aspire_rotary_append, args, what)
        return q_out


class _Turn(torch.autograd.Function):
    """The turn by the positions' angles, or back; each is the other's gradient. It is linear: tangents turn as values do."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        if forward_ad._current_level >= 0:  # for jvp, which runs at once
            ctx.save_for_forward(positions)
            ctx.shapes = None if q is None else q.shape, None if k is None else k.shape
        return rotary._turn(q, k, positions, inverse, False, "RotaryEmbedding.apply")

    @staticmethod
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        if dq is None and dk is None:
            return None, None, None, None, None
        if dq is not None and dq.stride(2) != 1:
            dq = dq.contiguous()
        if dk is not None and dk.stride(2) != 1:
            dk = dk.contiguous()
        if torch.is_grad_enabled() or forward_ad._current_level >= 0:  # a second derivative is wanted
            gq, gk = _Turn.apply(dq, dk, positions, ctx.rotary, not ctx.inverse)
        else:
            gq, gk = ctx.rotary._turn(dq, dk, positions, not ctx.inverse, False, "RotaryEmbedding.apply")
        return gq, gk, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        (positions,) = ctx.saved_tensors
        # an output that is not None needs a tangent; one of the two is there
        if tq is None and ctx.shapes[0] is not None:
            tq = tk.new_zeros(ctx.shapes[0])
        if tk is None and ctx.shapes[1] is not None:
            tk = tq.new_zeros(ctx.shapes[1])
        tq, tk = (t if t is None or t.stride(2) == 1 else t.contiguous() for t in (tq, tk))
        return _Turn.apply(tq, tk, positions, ctx.rotary, ctx.inverse)


__all__ = ["RotaryConfig", "RotaryEmbedding"]
