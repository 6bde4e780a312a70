"""Linear layers with 4-bit weights on the HIP path (``aspire_linear_int4``).

The projections of ``aspire_amd.linear`` for checkpoints whose weights are 4-bit codes in groups along K, each with a
scale and, where the checkpoint has them, a zero point: ``w[n, k] = scales[n, k // group] * (codes[n, k] - zeros[n,
k // group])``. The weights are read as they are (an eighth of fp32's bytes) and never rounded to 16 bits: codes are
multiplied exactly, sums are fp32, and the output is rounded once. Up to 4,194,240 token rows, bf16 or fp16.

``Int4Weight`` holds a matrix in the kernels' layout, made once from a checkpoint's packed codes
(``from_packed``) or from a bf16 matrix (``quantize``). A few rows take 0.3 to 0.85 of the time of torch's product with bf16 weights, a prompt's
2,048 rows 1.05 to 1.4 of it.
"""

from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

from aspire_amd import _lib

GROUPS = (32, 64, 128)
_TYPES = (torch.bfloat16, torch.float16)


class Int4Weight:
    """``[N, K]`` 4-bit weights on a GPU, laid out in blocks of 16 rows x 128 columns."""

    def __init__(self, shape, group, codes, scales, zeros):
        self.shape, self.group = tuple(shape), group
        self.codes, self.scales, self.zeros = codes, scales, zeros  # see aspire_hip.h for the layouts

    @classmethod
    def from_packed(cls, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
                    group: int) -> "Int4Weight":
        """``packed`` uint8 ``[N, K / 2]`` (column 2j in the low half of byte j), ``scales`` bf16 or fp16
        ``[N, K / group]``, ``zeros`` uint8 ``[N, K / group]`` of 0 to 15 (None: 8 everywhere)."""
        n, k = packed.shape[0], packed.shape[1] * 2 if packed.dim() == 2 else 0
        if packed.dim() != 2 or packed.dtype != torch.uint8 or n == 0 or group not in GROUPS or k == 0 or k % group:
            raise ValueError(f"Int4Weight: packed must be uint8 [N, K / 2], group one of {GROUPS} and K a multiple of it")
        if scales.shape != (n, k // group) or scales.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("Int4Weight: scales must be bf16 or fp16 [N, K / group]")
        if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != torch.uint8):
            raise ValueError("Int4Weight: zeros must be uint8 [N, K / group]")
        if any(t is not None and t.device != packed.device for t in (scales, zeros)):
            raise ValueError("Int4Weight: packed, scales and zeros must be on one device")
        if zeros is not None and int(zeros.max()) > 15:
            raise ValueError("Int4Weight: zeros must be 0 to 15")
        tiles, blocks = (n + 15) // 16, (k + 127) // 128

        def fill(t, rows, cols):  # zeros behind the matrix' end
            if t.shape == (rows, cols):
                return t
            out = torch.zeros(rows, cols, dtype=t.dtype, device=t.device)
            out[: t.shape[0], : t.shape[1]] = t
            return out

        # bytes of a lane's word: [tile, row, block, word, lane / 16, byte] -> [tile, block, lane / 16, row, word, byte]
        b = fill(packed, tiles * 16, blocks * 64).reshape(tiles, 16, blocks, 4, 4, 4).permute(0, 2, 4, 1, 3, 5)
        b = b.contiguous()
        # nibble e of 8 goes to place e / 2 + 4 (e % 2): bytes (e1 e0)(e3 e2)(e5 e4)(e7 e6) -> (e2 e0)(e6 e4)(e3 e1)(e7 e5)
        lo, hi = b & 15, b >> 4
        codes = torch.empty_like(b)
        codes[..., 0] = lo[..., 0] | (lo[..., 1] << 4)
        codes[..., 1] = lo[..., 2] | (lo[..., 3] << 4)
        codes[..., 2] = hi[..., 0] | (hi[..., 1] << 4)
        codes[..., 3] = hi[..., 2] | (hi[..., 3] << 4)
        parts = 128 // group
        # [tile, row, block, group of it] -> [tile, block, row / 4, group, row % 4] and [tile, block, row, group]; clones, as one
        # block of 128 k has that order already, and contiguous() would hand the caller's own memory on
        scales = fill(scales, tiles * 16, blocks * parts).reshape(tiles, 4, 4, blocks, parts).permute(0, 3, 1, 4, 2)
        scales = scales.clone(memory_format=torch.contiguous_format)
        if zeros is not None:
            zeros = fill(zeros, tiles * 16, blocks * parts).reshape(tiles, 16, blocks, parts).transpose(1, 2)
            zeros = zeros.clone(memory_format=torch.contiguous_format)
        return cls((n, k), group, codes.view(tiles, blocks, 64, 16), scales, zeros)

    @classmethod
    def quantize(cls, w: torch.Tensor, *, group: int = 128, symmetric: bool = False) -> "Int4Weight":
        """The nearest 4-bit form of a matrix ``[N, K]``: each group's range (with 0 in it) in 15 steps, or with ``symmetric``
        its largest magnitude in 7."""
        if w.dim() != 2 or group not in GROUPS or w.shape[1] % group:
            raise ValueError(f"Int4Weight: w must be [N, K], group one of {GROUPS} and K a multiple of it")
        if not bool(torch.isfinite(w).all()):
            raise ValueError("Int4Weight: w must be finite")
        dtype = w.dtype if w.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
        v = w.float().reshape(w.shape[0], -1, group)
        if symmetric:
            scale, zero = v.abs().amax(-1) / 7, None
        else:
            lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
            scale = (hi - lo) / 15
        scale = scale.to(dtype)
        step = scale.float().clamp(min=torch.finfo(torch.float32).tiny)[..., None]
        if not symmetric:
            zero = (-lo[..., None] / step).round_().clamp_(0, 15)
        codes = ((v / step).round_() + (8 if zero is None else zero)).clamp_(0, 15).to(torch.uint8).view(w.shape)
        packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
        return cls.from_packed(packed, scale, None if zero is None else zero[..., 0].to(torch.uint8), group=group)

    @property
    def device(self):
        return self.codes.device

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.zeros) if t is not None)

    def to(self, device) -> "Int4Weight":
        move = lambda t: None if t is None else t.to(device)
        return Int4Weight(self.shape, self.group, move(self.codes), move(self.scales), move(self.zeros))

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The matrix ``[N, K]`` that the codes stand for."""
        (n, k), (tiles, blocks) = self.shape, self.codes.shape[:2]
        c = self.codes.view(tiles, blocks, 4, 16, 4, 4)
        nib = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2)              # places 0 .. 7 of a word
        nib = nib[..., [0, 4, 1, 5, 2, 6, 3, 7]]                              # in k's order
        codes = nib.permute(0, 3, 1, 4, 2, 5).reshape(tiles * 16, blocks * 128)
        spread = lambda t: t.reshape(tiles * 16, -1).float().repeat_interleave(self.group, dim=1)
        zeros = 8.0 if self.zeros is None else spread(self.zeros.transpose(1, 2))
        w = (codes.float() - zeros) * spread(self.scales.permute(0, 2, 4, 1, 3))
        return w[:n, :k].to(dtype)


# aspire_int4_args as one packed string (filling a ctypes structure takes longer than the launch)
_ARGS = struct.Struct("PqPPPPq7iPq")


def linear_int4(x: torch.Tensor, w: Int4Weight, out: torch.Tensor, *, swiglu: bool = False) -> torch.Tensor:
    """``out = x @ w.T`` (``[rows, N]``), or with ``swiglu`` ``silu(x @ w[:N/2].T) * (x @ w[N/2:].T)`` (``[rows, N/2]``, N a
    multiple of 32), for bf16 or fp16 ``x`` with 16-byte aligned rows; ``out`` of ``x``'s type with contiguous rows, apart
    from x. Past 16 rows, rows of x that lie 2^22 elements or more apart may be refused (ValueError; ``x.contiguous()`` is taken), as
    the last tokens of long sequences in one tensor do. Not differentiable. A row of x with an infinity or NaN (or bf16 values
    of 2^112 and more, whose sums may overflow on the way) gives no finite outputs; the other rows are not touched by it."""
    what = "linear_int4"
    if torch.is_grad_enabled() and x.requires_grad or forward_ad._current_level >= 0 and _lib.has_tangent(x, out, w.scales):
        raise ValueError(f"{what}: not differentiable")
    if not (x.is_cuda and out.is_cuda and w.codes.is_cuda):
        _lib.require_cuda(x, out, w.codes, what=what)
    n, k = w.shape
    shape, st, dtype, at = x.shape, x.stride(), x.dtype, x.data_ptr()
    if len(shape) != 2 or dtype not in _TYPES or shape[1] != k or st[1] != 1 or (st[0] % 8 and shape[0] > 1) or at % 16:
        raise ValueError(f"{what}: x must be bf16 or fp16 [rows, {k}] with 16-byte aligned rows")
    if swiglu and n % 32:
        raise ValueError(f"{what}: swiglu needs N a multiple of 32")
    rows, cols, to = shape[0], n // 2 if swiglu else n, out.stride()
    if out.dtype is not dtype or out.shape != (rows, cols) or to[1] != 1:
        raise ValueError(f"{what}: out must be {dtype} [{rows}, {cols}] with contiguous rows")
    index = w.codes.get_device()
    if x.get_device() != index or out.get_device() != index:
        raise ValueError(f"{what}: x, out and the weights must be on one device")
    L = _lib.lib()
    floats, ws = L.aspire_linear_int4_workspace(rows, n, k, w.group, swiglu), 0
    if floats:
        workspace = torch.empty(floats, dtype=torch.float32, device=x.device)
        ws = workspace.data_ptr()
    zeros = w.zeros
    args = _ARGS.pack(at, st[0] if rows > 1 else k, w.codes.data_ptr(), w.scales.data_ptr(),
                      0 if zeros is None else zeros.data_ptr(), out.data_ptr(), to[0] if rows > 1 else cols, rows, n, k, w.group,
                      swiglu, dtype is torch.float16, w.scales.dtype is torch.float16, ws, floats)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = L.aspire_linear_int4(args, stream)
    else:
        with torch.cuda.device(index):
            rc = L.aspire_linear_int4(args, stream)
    if rc:
        _lib.check(rc, what)
    return out


__all__ = ["GROUPS", "Int4Weight", "linear_int4"]
