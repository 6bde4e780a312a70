"""The 4-bit weights' layout, and the host-side checks of the products (no GPU)."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwad

from aspire_amd import _lib, linear_int4
from aspire_amd.linear_int4 import Int4Weight
from int4_cases import TILES, choice, representatives


@pytest.mark.parametrize("n,k,group,zeros", [(16, 128, 128, False), (40, 96, 32, True), (1, 320, 64, True)])
def test_layout_is_the_documented_one(n, k, group, zeros):
    g = torch.Generator().manual_seed(n + k)
    packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g)
    scales = torch.rand(n, k // group, generator=g).to(torch.float16)
    z = torch.randint(0, 16, (n, k // group), dtype=torch.uint8, generator=g) if zeros else None
    w = Int4Weight.from_packed(packed, scales, z, group=group)
    tiles, blocks = (n + 15) // 16, (k + 127) // 128
    words = w.codes.contiguous().view(torch.int32).view(tiles, blocks, 64, 4).tolist()
    code = lambda r, c: int(packed[r, c // 2]) >> (4 * (c % 2)) & 15 if r < n and c < k else 0
    for t in range(tiles):
        for b in range(blocks):
            for l in range(64):
                for c in range(4):
                    for e in range(8):
                        got = words[t][b][l][c] >> (4 * (e // 2) + 16 * (e % 2)) & 15
                        assert got == code(16 * t + l % 16, 128 * b + 32 * c + 8 * (l // 16) + e)
    parts = 128 // group
    assert w.scales.shape == (tiles, blocks, 4, parts, 4) and w.scales.is_contiguous()
    for t in range(tiles):
        for b in range(blocks):
            for row in range(16):
                for g in range(parts):
                    inside = 16 * t + row < n and b * parts + g < k // group
                    want = scales[16 * t + row, b * parts + g] if inside else 0
                    assert w.scales[t, b, row // 4, g, row % 4] == want
                    if zeros and inside:
                        assert w.zeros[t, b, row, g] == z[16 * t + row, b * parts + g]
    c = torch.stack([packed & 15, packed >> 4], dim=-1).view(n, k).float()
    spread = lambda t: t.float().repeat_interleave(group, dim=1)
    assert torch.equal(w.dequantize(), (c - (spread(z) if zeros else 8)) * spread(scales))


@pytest.mark.parametrize("change", [
    dict(packed=torch.zeros(4, 64)), dict(packed=torch.zeros(64, dtype=torch.uint8)), dict(group=48), dict(group=256),
    dict(scales=torch.zeros(4, 1, dtype=torch.bfloat16)), dict(scales=torch.zeros(4, 2)),
    dict(zeros=torch.zeros(4, 1, dtype=torch.uint8)), dict(zeros=torch.zeros(4, 2, dtype=torch.int32)),
    dict(zeros=torch.full((4, 2), 16, dtype=torch.uint8)), dict(packed=torch.zeros(4, 40, dtype=torch.uint8)),
])
def test_refused_weights(change):
    kw = dict(packed=torch.zeros(4, 64, dtype=torch.uint8), scales=torch.zeros(4, 2, dtype=torch.bfloat16), zeros=None, group=64)
    Int4Weight.from_packed(**kw)
    with pytest.raises(ValueError):
        Int4Weight.from_packed(**{**kw, **change})


def test_views_give_the_same_weights():
    """Packed codes, scales and zeros that are slices of larger or transposed tensors."""
    g = torch.Generator().manual_seed(5)
    packed = torch.randint(0, 256, (40, 2 * 96), dtype=torch.uint8, generator=g)[:, ::2][:, :64]
    scales = torch.rand(2, 40, generator=g).to(torch.bfloat16).t()
    z = torch.randint(0, 16, (2, 40), dtype=torch.uint8, generator=g).t()
    a = Int4Weight.from_packed(packed, scales, z, group=64)
    b = Int4Weight.from_packed(packed.contiguous(), scales.contiguous(), z.contiguous(), group=64)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.zeros, b.zeros)
    w = torch.randn(128, 32, generator=g).t()
    assert torch.equal(Int4Weight.quantize(w, group=64).codes, Int4Weight.quantize(w.contiguous(), group=64).codes)


def test_packed_arguments_match_the_structure():
    """The string that the entry point gets in place of the structure: every field at its place."""
    values = list(range(1, 17))
    a = _lib.Int4Args.from_buffer_copy(linear_int4._ARGS.pack(*values))
    assert ctypes.sizeof(_lib.Int4Args) == linear_int4._ARGS.size
    assert [getattr(a, f[0]) for f in a._fields_] == values


def test_refused_matrices():
    for w, group in ((torch.zeros(4, 100), 64), (torch.zeros(64), 64), (torch.zeros(4, 128), 16),
                     (torch.full((4, 64), float("nan")), 64)):
        with pytest.raises(ValueError):
            Int4Weight.quantize(w, group=group)


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libaspire_hip.so not built")
def test_entry_point_refuses_on_the_host():
    L = _lib.lib()

    def call(**kw):
        a = _lib.Int4Args(x=4096, x_stride=256, weights=4096, scales=4096, zeros=4096, out=4096, out_stride=64, rows=4, n=64,
                          k=256, group=64)
        for name, value in kw.items():
            setattr(a, name, value)
        return L.aspire_linear_int4(ctypes.byref(a), None)

    for kw in (dict(rows=-1), dict(rows=1 << 22), dict(n=-1), dict(k=0), dict(k=250), dict(k=1 << 22, x_stride=1 << 22), dict(rows=400, n=1 << 14, out_stride=1 << 14, x_stride=1 << 22), dict(group=16), dict(group=0), dict(x=None),
               dict(weights=None), dict(scales=None), dict(out=None), dict(x=4104), dict(x_stride=260), dict(x_stride=248),
               dict(out_stride=63), dict(n=48, swiglu=1), dict(scales=4100), dict(zeros=4097)):
        assert call(**kw) == _lib.ASPIRE_ERR_INVALID, kw
    assert call(rows=0) == _lib.ASPIRE_OK and call(n=0) == _lib.ASPIRE_OK
    assert L.aspire_linear_int4(None, None) == _lib.ASPIRE_ERR_INVALID


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k", [128, 256])
def test_weights_keep_their_own_copy(k, group):
    """A loader's buffers, whatever their offset, are free when the weights are made: with one block of k the layout
    has the order of the checkpoint's own scales and zero points."""
    n, parts = 32, k // group
    g = torch.Generator().manual_seed(k + group)
    packed = torch.randint(0, 256, (n * k // 2 + 1,), dtype=torch.uint8, generator=g)[1:].view(n, k // 2)
    scales = torch.rand(n * parts + 1, generator=g).to(torch.bfloat16)[1:].view(n, parts)
    zeros = torch.randint(0, 16, (n * parts + 1,), dtype=torch.uint8, generator=g)[1:].view(n, parts)
    w = Int4Weight.from_packed(packed, scales, zeros, group=group)
    before = w.dequantize().clone()
    for mine, given in ((w.codes, packed), (w.scales, scales), (w.zeros, zeros)):
        assert mine.untyped_storage().data_ptr() != given.untyped_storage().data_ptr() and mine.data_ptr() % 16 == 0
        given.zero_()
    assert torch.equal(w.dequantize(), before)


def test_dual_tensors_are_refused():
    """There is no derivative in forward mode either."""
    w = Int4Weight.quantize(torch.ones(16, 64), group=64)
    x, out = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 16, dtype=torch.bfloat16)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))
        scaled = Int4Weight(w.shape, w.group, w.codes, dual(w.scales), w.zeros)
        for args in ((dual(x), w, out), (x, w, dual(out)), (x, scaled, out)):
            with pytest.raises(ValueError, match="not differentiable"):
                linear_int4.linear_int4(*args)


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libaspire_hip.so not built")
@pytest.mark.parametrize("n,ks", [(16, (32, 1024, 2048, 4096)), (32, (64, 1024, 8192)), (96, (4096,)), (4096, (4096, 1 << 21)),
                                  (151936, (4096,)), ((1 << 23) * 16 - 16, (128,))])
def test_launches_stay_within_their_limits(n, ks):
    """65,535 workgroups in y and z, fewer than 2^32 threads in x: the stream kernel has 16 rows in z, the tiles theirs in y."""
    for rows in (1, 16, 17, 65535 * 16, 65535 * 16 + 1, (1 << 22) - 64):
        for k in ks:
            for group in (32, 64, 128):
                for swiglu in (0, 1):
                    if k % group or (swiglu and n % 32):
                        continue
                    tile, cols, splits = choice(rows, n, k, group, swiglu)
                    assert splits >= 1
                    if tile == 0:
                        assert (rows + 15) // 16 <= 65535 and splits <= 65535
                    else:
                        assert (rows + tile - 1) // tile <= 65535
                        assert 2 * ((n + cols - 1) // cols) * splits * 512 < 1 << 32


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libaspire_hip.so not built")
def test_choice_of_refused_sizes():
    for args in ((0, 16, 128, 32, 0), (-1, 16, 128, 32, 0), (1, 0, 128, 32, 0), (1, 16, 0, 32, 0), (1, (1 << 30) + 1, 128, 32, 0),
                 (1 << 22, 16, 128, 32, 0), (1, 16, 1 << 22, 32, 0), (1, 16, 128, 48, 0), (1, 16, 96, 64, 0), (1, 48, 128, 32, 1),
                 (1, 1 << 27, 128, 32, 0)):
        assert choice(*args) == (0, 0, 0)
    _lib.lib().aspire_linear_int4_choice(1, 16, 128, 32, 0, None)


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libaspire_hip.so not built")
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("swiglu", [0, 1])
def test_every_kernel_has_a_product_that_runs_it(group, swiglu):
    """The rule picks every tile, with and without splits, and every number of a stream wave's blocks, and no other kernel: what
    the GPU test of these products runs is all there is. Gate and up tiles of 128 columns and up to 64 rows pair in
    the join alone; a stream wave has 4 blocks or more where k is split (7 and 8 avoid the split)."""
    stream = {(0, held, False) for held in range(1, 7 if group == 32 else 9)}
    stream |= {(0, held, True) for held in range(4 if group == 32 else 5, 7)}
    tiles = {tile + (split,) for tile in TILES for split in (False, True)
             if split or not (swiglu and tile[1] == 128 and tile[0] <= 64)}
    assert set(representatives(group, swiglu)) == stream | tiles
