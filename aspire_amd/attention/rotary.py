"""Rotary positions in the forms that checkpoints have, alone and with the paged append (HIP).

``rope`` serves one form (interleaved pairs of whole 128-wide bf16 heads, in place, behind the q/k norm). Here a
``RotaryConfig`` says how a model turns its heads, and a ``RotaryEmbedding`` holds its frequencies on a device:

* pairs ``(i, i + R/2)`` (``layout="half"``) or ``(2i, 2i + 1)`` (``"interleaved"``) of the first ``R = rotary_dim``
  values of a head of up to 256; the others pass unchanged;
* frequencies ``f_i = theta^(-2i/R)``, or scaled for long contexts: ``"linear"`` (``f / factor``), ``"llama3"``
  (the smoothing of ``RopeConfig``), ``"yarn"`` (between the pairs that turn ``beta_fast`` and ``beta_slow`` times
  over the trained context ``f`` becomes ``f / factor`` linearly; cos and sin times ``0.1 ln(factor) + 1``), or
  divided by given ``pair_factors``;
* angles ``position * f_i`` are exact at any position (64-bit fixed point), cos and sin and the products fp32, one
  rounding to the output's type.

``apply`` is differentiable (the gradient turns back by the same angles); ``append`` is
``mylib::update_kv_padded`` (aspire/attention/kv_ops.py:63-187) with the turn on the way, one launch.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from dataclasses import dataclass

import torch

from aspire_amd import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
SCALINGS = ("none", "linear", "llama3", "yarn")
MAX_HEAD_DIM = 256


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

    def frequencies(self) -> list[float]:
        """Radians a position of each pair (64-bit)."""
        r = self.rotated
        base = [self.theta ** (-2.0 * i / r) for i in range(r // 2)]
        if self.pair_factors is not None:
            return [f / s for f, s in zip(base, self.pair_factors)]
        if self.scaling == "linear":
            return [f / self.factor for f in base]
        if self.scaling == "llama3":
            lo, hi, old = self.low_freq_factor, self.high_freq_factor, self.original_max_position
            keep = [min(max((old * f / (2 * math.pi) - lo) / (hi - lo), 0.0), 1.0) for f in base]
        elif self.scaling == "yarn":
            def at(turns):  # the pair that turns so often over the trained context
                return r * math.log(self.original_max_position / (2 * math.pi * turns)) / (2 * math.log(self.theta))
            first, last = max(math.floor(at(self.beta_fast)), 0), min(math.ceil(at(self.beta_slow)), r - 1)
            width = max(last - first, 0.001)
            keep = [1.0 - min(max((i - first) / width, 0.0), 1.0) for i in range(r // 2)]
        else:
            return base
        return [t * f + (1.0 - t) * f / self.factor for t, f in zip(keep, base)]


def _turns(frequencies) -> torch.Tensor:
    """Frequencies as 64-bit fixed-point fractions of a turn a position (int64 holding the bits)."""
    out = []
    for f in frequencies:
        t = int(math.fmod(f / (2 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64)
        out.append(t - (1 << 64) if t >> 63 else t)
    return torch.tensor(out, dtype=torch.int64)


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether ``b`` of ``a``'s shape can stand for it: no shared start, or the same layout."""
    return a.data_ptr() != b.data_ptr() or all(n == 1 or x == y for n, x, y in zip(a.shape, a.stride(), b.stride()))


def _on(device: torch.device):
    """The tensors' device as the current one for a launch."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


class RotaryEmbedding:
    """A model's rotary positions on one device."""

    def __init__(self, config: RotaryConfig, device="cuda"):
        self.config = config
        self.turns = _turns(config.frequencies()).to(device)
        self.device = self.turns.device
        self._args = dict(head_dim=config.head_dim, rotary_dim=config.rotated,
                          interleaved=int(config.layout == "interleaved"), amplitude=config.scale,
                          turns=self.turns.data_ptr())

    # ------------------------------------------------------------------ checks
    def _check(self, what: str, **tensors) -> torch.dtype:
        _lib.require_cuda(*tensors.values(), what=what)
        dtype = next(t.dtype for t in tensors.values() if t is not None)
        if dtype not in _DTYPES:
            raise ValueError(f"{what}: bf16, fp16 or fp32 tensors")
        for name, t in tensors.items():
            if t is None:
                continue
            if t.device != self.device:
                raise ValueError(f"{what}: {name} is on {t.device}, the frequencies on {self.device}")
            if t.dtype != dtype or t.dim() != 3 or t.shape[2] != self.config.head_dim:
                raise ValueError(f"{what}: {name} must be {dtype} [T, H, {self.config.head_dim}]")
            if t.stride(2) != 1 and t.numel():
                raise ValueError(f"{what}: {name} must have contiguous head dims")
        return dtype

    def _positions(self, positions: torch.Tensor, tokens: int, what: str) -> torch.Tensor:
        if positions.dim() != 1 or positions.shape[0] != tokens or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{what}: positions must be int32 or int64 [T]")
        if positions.device != self.device:
            raise ValueError(f"{what}: positions are on {positions.device}, the frequencies on {self.device}")
        return positions if positions.stride(0) == 1 else positions.contiguous()

    def _fill(self, dtype, tokens, inverse=False, positions=None) -> _lib.RotaryArgs:
        a = _lib.RotaryArgs(total_tokens=tokens, dtype=_DTYPES[dtype], inverse=int(inverse), **self._args)
        if positions is not None:
            a.positions, a.positions_64 = positions.data_ptr(), int(positions.dtype == torch.int64)
        return a

    def _turn(self, q, k, q_out, k_out, positions, inverse, what) -> None:
        first = q if q is not None else k
        tokens = first.shape[0]
        if k is not None and k.shape[0] != tokens:
            raise ValueError(f"{what}: q and k must have the same number of tokens")
        positions = self._positions(positions, tokens, what)
        a = self._fill(first.dtype, tokens, inverse, positions)
        if q is not None:
            a.q, a.q_stride_t, a.q_stride_h, a.num_qo_heads = q.data_ptr(), q.stride(0), q.stride(1), q.shape[1]
            a.q_out, a.q_out_stride_t, a.q_out_stride_h = q_out.data_ptr(), q_out.stride(0), q_out.stride(1)
        if k is not None:
            a.k, a.k_stride_t, a.k_stride_h, a.num_kv_heads = k.data_ptr(), k.stride(0), k.stride(1), k.shape[1]
            a.k_out, a.k_out_stride_t, a.k_out_stride_h = k_out.data_ptr(), k_out.stride(0), k_out.stride(1)
        with _on(self.device):
            _lib.check(_lib.lib().aspire_rotary(ctypes.byref(a), _lib.stream_of(first)), what)

    # -------------------------------------------------------------- operators
    def apply(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor):
        """``(q, k)`` turned at ``positions`` ``[T]``, as new tensors (``k`` may be None); differentiable. Tokens at
        negative positions are copied."""
        what = "RotaryEmbedding.apply"
        self._check(what, q=q, k=k)
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            out = _Turn.apply(q, k, positions, self, False)
            return out if k is not None else (out[0], None)
        return self._new(q, k, positions, False, what)

    def _new(self, q, k, positions, inverse, what):
        q_out, k_out = (None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
        self._turn(q, k, q_out, k_out, positions, inverse, what)
        return q_out, k_out

    def apply_inplace(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor) -> None:
        """``apply`` on q and k themselves (not differentiable; no two of their rows may share memory)."""
        what = "RotaryEmbedding.apply_inplace"
        self._check(what, q=q, k=k)
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            raise ValueError(f"{what}: not differentiable; use apply")
        self._turn(q, k, q, k, positions, False, what)

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_append_indptr: torch.Tensor,
               kv_cache: torch.Tensor, kv_page_indices: torch.Tensor, kv_page_indptr: torch.Tensor,
               kv_last_page_len: torch.Tensor, page_size: int, *, positions: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor:
        """Turn q (in place, or into ``q_out``, which it returns) and append the turned k and v to ``kv_cache``
        ``[P, 2, page, H_kv, D]`` where ``mylib::update_kv_padded`` would put them, in one launch. A token's position is
        its place in its row's sequence unless ``positions`` ``[T]`` gives another. Tokens of no row are
        padding: their q passes unchanged, and nothing is written to the cache; nor is it for a token whose
        page id or list entry lies outside the pool or the list."""
        what = "RotaryEmbedding.append"
        dtype = self._check(what, q=q, k=k, v=v, q_out=q_out)
        q_out = q if q_out is None else q_out
        tokens = q.shape[0]
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            raise ValueError(f"{what}: not differentiable")
        if dtype == torch.float32:
            raise ValueError(f"{what}: the cache holds bf16 or fp16")
        if k.shape[0] != tokens or v.shape != k.shape or q_out.shape != q.shape:
            raise ValueError(f"{what}: q, k and v must have the same tokens, k and v the same heads, q_out q's shape")
        if not _same_place(q, q_out):
            raise ValueError(f"{what}: q_out must be q itself or apart from it")
        if kv_cache.device != self.device or kv_cache.dtype != dtype or kv_cache.dim() != 5 \
                or tuple(kv_cache.shape[1:]) != (2, page_size, k.shape[1], self.config.head_dim) or kv_cache.stride(4) != 1:
            raise ValueError(f"{what}: kv_cache must be {dtype} [P, 2, {page_size}, {k.shape[1]}, "
                             f"{self.config.head_dim}] with contiguous head dims")
        lists = (kv_append_indptr, kv_page_indices, kv_page_indptr, kv_last_page_len)
        if any(t.device != self.device or t.dim() != 1 or t.dtype not in (torch.int32, torch.int64) for t in lists):
            raise ValueError(f"{what}: the index arrays must be 1-D int32 on {self.device}")
        num_seq = kv_last_page_len.shape[0]
        if kv_append_indptr.shape[0] < num_seq + 1 or kv_page_indptr.shape[0] < num_seq + 1:
            raise ValueError(f"{what}: kv_page_indptr and kv_append_indptr need len(kv_last_page_len) + 1 entries")
        if positions is not None:
            positions = self._positions(positions, tokens, what)
        ind, pages, ptr, last = (_lib.dense(t, torch.int32) for t in lists)
        a = self._fill(dtype, tokens, False, positions)
        a.q, a.q_stride_t, a.q_stride_h, a.num_qo_heads = q.data_ptr(), q.stride(0), q.stride(1), q.shape[1]
        a.q_out, a.q_out_stride_t, a.q_out_stride_h = q_out.data_ptr(), q_out.stride(0), q_out.stride(1)
        a.k, a.k_stride_t, a.k_stride_h, a.num_kv_heads = k.data_ptr(), k.stride(0), k.stride(1), k.shape[1]
        a.v, a.v_stride_t, a.v_stride_h = v.data_ptr(), v.stride(0), v.stride(1)
        a.kv_cache, a.num_pages, a.page_size, a.num_seq = kv_cache.data_ptr(), kv_cache.shape[0], page_size, num_seq
        a.cache_stride_p, a.cache_stride_kv, a.cache_stride_t, a.cache_stride_h = kv_cache.stride()[:4]
        a.append_indptr, a.kv_page_indices, a.num_page_indices = ind.data_ptr(), pages.data_ptr(), pages.shape[0]
        a.kv_page_indptr, a.kv_last_page_len = ptr.data_ptr(), last.data_ptr()
        with _on(self.device):
            _lib.check(_lib.lib().aspire_rotary_append(ctypes.byref(a), _lib.stream_of(q)), what)
        return q_out


class _Turn(torch.autograd.Function):
    """The turn by the positions' angles, or back; each is the other's gradient."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        return rotary._new(q, k, positions, inverse, "RotaryEmbedding.apply")

    @staticmethod
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        if dq is None and dk is None:
            return None, None, None, None, None
        dq, dk = (t if t is None or t.stride(2) == 1 else t.contiguous() for t in (dq, dk))
        gq, gk = _Turn.apply(dq, dk, positions, ctx.rotary, not ctx.inverse)
        return gq, gk, None, None, None


__all__ = ["RotaryConfig", "RotaryEmbedding"]
