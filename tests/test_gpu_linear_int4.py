"""Products with 4-bit weights against the weights that the codes stand for, in 64 bits."""

import pytest
import torch

from aspire_amd.linear_int4 import Int4Weight, linear_int4
from helpers import say
from int4_cases import representatives

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
# both sides of every row class, rows that end inside a 16-row tile
ROWS = [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 257]


def weights(n, k, group, zeros, dtype, gpu, exact=False):
    """Packed codes, scales, zeros, and the matrix they stand for in 64 bits."""
    g = torch.Generator(device=gpu).manual_seed(n * 7 + k + group)
    packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=gpu, generator=g)
    if exact:  # powers of two
        scales = torch.pow(2.0, torch.randint(-3, 1, (n, k // group), device=gpu, generator=g).float()).to(dtype)
    else:
        scales = ((torch.rand(n, k // group, device=gpu, generator=g) + 0.5) * k ** -0.5 / 4).to(dtype)
    z = torch.randint(0, 16, (n, k // group), dtype=torch.uint8, device=gpu, generator=g) if zeros else None
    c = torch.stack([packed & 15, packed >> 4], dim=-1).view(n, k).double()
    spread = lambda t: t.double().repeat_interleave(group, dim=1)
    return packed, scales, z, (c - (spread(z) if zeros else 8.0)) * spread(scales)


def product_bound(x, scales, group, k):
    """What fp32 sums may be off by. In a group the sum of (offset + c) x and, for bf16, that of x times the offset are taken
    off each other; the offset with its code is at most 143 (fp16: the weights are exact, at most 15). Each of a
    group's additions rounds by 2^-24 of a partial sum of at most 143 sum |x|, twice, and two more for zero point and
    scale; adding up the groups rounds k / group + 8 times (waves, tail) by 2^-24 of at most 15 sum s |x|."""
    a = x.double().abs().view(x.shape[0], -1, group).sum(-1) @ scales.double().t()
    top = 143 if x.dtype == BF else 15
    return a * 2.0 ** -24 * (top * 2 * (group + 2) + 15 * (k // group + 8))


def close(got, ref, bound):
    """Within ``bound`` and half a step of the output's type (fp16: 2^-25 below its normal range)."""
    off = (got.double() - ref).abs()
    limit = bound + torch.finfo(got.dtype).eps / 2 * (ref.abs() + bound) + (2.0 ** -25 if got.dtype == HF else 0)
    assert not (off > limit).any(), f"worst {float((off - limit).max())}"


SHAPES = [
    # n, k, group, zeros, padding of x's rows and of out's
    (16, 32, 32, False, 0, 0),       # one group
    (1, 128, 128, True, 0, 0),       # one column
    (40, 96, 32, True, 8, 8),        # a block that ends early, a tile that ends early
    (35, 320, 64, True, 0, 1),       # odd columns: single stores
    (256, 1152, 128, False, 16, 4),
    (4001, 1024, 32, True, 0, 3),
    (6144, 2176, 64, False, 0, 0),
    (1056, 12288, 128, True, 0, 0),  # a long walk over k
    (4112, 5120, 128, False, 0, 0),  # 5 to 8 blocks a wave, walked over more tiles than workgroups
    (4112, 6080, 64, True, 0, 0),
    (4112, 6144, 32, True, 0, 0),
    (4112, 7168, 128, True, 0, 0),
    (4112, 8000, 64, False, 0, 0),
    (8224, 2944, 128, True, 0, 0),   # 2, 3 and 4
    (8224, 1920, 32, True, 0, 0),
    (8224, 4000, 32, False, 0, 0),
    (8224, 4096, 64, True, 0, 0),
    (24608, 640, 128, True, 0, 0),   # many columns
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k,group,zeros,xpad,opad", SHAPES)
def test_products(gpu, n, k, group, zeros, xpad, opad, dtype):
    """Sums of whole numbers, which fp32 holds exactly, are right to the last bit; real ones within their rounding.
    Nothing is written beside the output."""
    whole, real = (weights(n, k, group, zeros, dtype, gpu, exact=e) for e in (True, False))
    packs = [Int4Weight.from_packed(*w[:3], group=group) for w in (whole, real)]
    for rows in ROWS:
        say("int4", rows, n, k, group, zeros, dtype)
        g = torch.Generator(device=gpu).manual_seed(rows)
        buf = torch.full((rows, k + xpad), float("nan"), device=gpu).to(dtype)
        out = torch.full((rows + 1, n + opad), 7.0, dtype=dtype, device=gpu)
        x = buf[:, :k]
        # (offset + c) x, at most 143 * 2 a term, stays below 2^24 in a group; the sum of all in units of 1/8 too
        x.copy_(torch.randint(-2, 3, (rows, k), device=gpu, generator=g))
        linear_int4(x, packs[0], out[:rows, :n])
        assert torch.equal(out[:rows, :n], (x.double() @ whole[3].t()).to(dtype))
        x.copy_(torch.randn(rows, k, device=gpu, generator=g))
        linear_int4(x, packs[1], out[:rows, :n])
        close(out[:rows, :n], x.double() @ real[3].t(), product_bound(x, real[1], group, k))
        assert (out[rows:] == 7).all() and (out[:, n:] == 7).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k,group,zeros", [(32, 128, 128, True), (1056, 2208, 32, True), (2080, 640, 64, False), (8256, 8192, 64, True),
                                             (24576, 512, 128, True)])
def test_swiglu(gpu, n, k, group, zeros, dtype):
    packed, scales, z, w = weights(n, k, group, zeros, dtype, gpu)
    scales = (scales.float() * 2).to(dtype)  # gates on both sides of silu's bend
    w = w * 2
    pack = Int4Weight.from_packed(packed, scales, z, group=group)
    for rows in ROWS:
        say("int4 swiglu", rows, n, k, group, zeros, dtype)
        x = torch.randn(rows, k, device=gpu, generator=torch.Generator(device=gpu).manual_seed(rows)).to(dtype)
        out = torch.full((rows, n // 2 + 4), 7.0, dtype=dtype, device=gpu)
        linear_int4(x, pack, out[:, : n // 2], swiglu=True)
        y, b = x.double() @ w.t(), product_bound(x, scales, group, k)
        (gate, up), (bg, bu) = y.chunk(2, dim=1), b.chunk(2, dim=1)
        silu = gate * torch.sigmoid(gate)
        # |silu'| <= 1.1; expf, the sum, the quotient and the product round by at most 8 * 2^-24 of silu * up
        ds = 1.1 * bg
        close(out[:, : n // 2], silu * up, ds * up.abs() + silu.abs() * bu + ds * bu + 8 * 2.0 ** -24 * (silu * up).abs())
        assert (out[:, n // 2 :] == 7).all()


def test_scales_of_the_other_type(gpu):
    """fp16 scales with bf16 tokens and the other way round, as checkpoints come."""
    say("int4 scale types")
    for xt, st in ((BF, HF), (HF, BF)):
        packed, scales, z, w = weights(96, 512, 64, True, st, gpu)
        x = torch.randn(20, 512, device=gpu).to(xt)
        out = torch.empty(20, 96, dtype=xt, device=gpu)
        linear_int4(x, Int4Weight.from_packed(packed, scales, z, group=64), out)
        close(out, x.double() @ w.t(), product_bound(x, scales, 64, 512))


def test_rows_far_apart(gpu):
    """A last token of each of a few long sequences: row strides past 2^22 values, which tiles past 16 rows refuse."""
    say("int4 far rows")
    packed, scales, z, w = weights(8208, 256, 64, True, BF, gpu)
    pack = Int4Weight.from_packed(packed, scales, z, group=64)
    hidden = torch.zeros(17, 20000, 256, dtype=BF, device=gpu)   # 5,120,000 values a row
    x = hidden[:, -1]
    x.copy_(torch.randn(17, 256, device=gpu))
    for rows in (1, 5, 16):
        out = linear_int4(x[:rows], pack, torch.empty(rows, 8208, dtype=BF, device=gpu))
        assert torch.equal(out, linear_int4(x[:rows].contiguous(), pack, torch.empty_like(out)))
    with pytest.raises(ValueError):
        linear_int4(x, pack, torch.empty(17, 8208, dtype=BF, device=gpu))


def test_fewer_blocks_than_splits(gpu):
    """One block of k where the gate and up tiles pair in the join of two splits: an empty split."""
    say("int4 empty split")
    for dtype in (BF, HF):
        packed, scales, z, w = weights(8224, 64, 32, True, dtype, gpu)
        pack = Int4Weight.from_packed(packed, scales, z, group=32)
        x = torch.randn(33, 64, device=gpu).to(dtype)
        out = linear_int4(x, pack, torch.empty(33, 4112, dtype=dtype, device=gpu), swiglu=True)
        gate, up = (x.double() @ w.t()).chunk(2, dim=1)
        bg, bu = product_bound(x, scales, 32, 64).chunk(2, dim=1)
        silu = gate * torch.sigmoid(gate)
        close(out, silu * up, 1.1 * bg * (up.abs() + bu) + silu.abs() * bu + 8 * 2.0 ** -24 * (silu * up).abs())


def test_rows_do_not_mix(gpu):
    """A row with an infinity or NaN is not finite; the other rows are what they were."""
    say("int4 special values")
    for dtype in (BF, HF):
        packed, scales, z, w = weights(80, 256, 64, True, dtype, gpu)
        pack = Int4Weight.from_packed(packed, scales, z, group=64)
        for rows in (3, 40, 200):
            x = torch.randn(rows, 256, device=gpu).to(dtype)
            clean = linear_int4(x, pack, torch.empty(rows, 80, dtype=dtype, device=gpu))
            x[1, 7], x[rows - 1, 200] = float("inf"), float("nan")
            out = linear_int4(x, pack, torch.empty(rows, 80, dtype=dtype, device=gpu))
            keep = torch.ones(rows, dtype=torch.bool, device=gpu)
            keep[1] = keep[rows - 1] = False
            assert torch.equal(out[keep], clean[keep]) and not torch.isfinite(out[~keep]).any()


def test_results_do_not_depend_on_the_batch_within_a_class(gpu):
    """The same row gives the same bits alone and among others of its row class, and on every call."""
    say("int4 repeatable")
    packed, scales, z, w = weights(512, 1024, 128, True, BF, gpu)
    pack = Int4Weight.from_packed(packed, scales, z, group=128)
    x = torch.randn(200, 1024, device=gpu).to(BF)
    for rows in (16, 200):
        first = linear_int4(x[:rows], pack, torch.empty(rows, 512, dtype=BF, device=gpu))
        for _ in range(3):
            assert torch.equal(first, linear_int4(x[:rows], pack, torch.empty_like(first)))
    alone = linear_int4(x[3:4], pack, torch.empty(1, 512, dtype=BF, device=gpu))
    assert torch.equal(alone[0], linear_int4(x[:16], pack, torch.empty(16, 512, dtype=BF, device=gpu))[3])


def test_quantize_and_dequantize(gpu):
    """A quantized matrix is within half a step of the matrix, whole numbers of steps come back exactly."""
    say("int4 quantize")
    w = torch.randn(48, 256, device=gpu).to(BF)
    for symmetric in (False, True):
        q = Int4Weight.quantize(w, group=32, symmetric=symmetric)
        v = w.float().view(48, 8, 32)
        step = v.abs().amax(-1) / 7 if symmetric else (v.amax(-1).clamp(min=0) - v.amin(-1).clamp(max=0)) / 15
        # half a step of the weight, half a step of the zero point, and the step's own rounding (2^-8) over 15 steps
        limit = (step * (0.5 + 0.5 + 15 * 2.0 ** -8) * 1.001)[..., None].expand(-1, -1, 32).reshape(48, 256)
        assert ((q.dequantize() - w.float()).abs() <= limit).all()
        assert q.nbytes() == 48 * 128 + 48 * 8 * (2 if symmetric else 3)
    steps = torch.randint(-7, 8, (32, 128), device=gpu)
    steps[:, 0] = 7
    q = Int4Weight.quantize((steps * 0.25).to(BF), group=128, symmetric=True)
    assert torch.equal(q.dequantize(), steps * 0.25)
    zero = Int4Weight.quantize(torch.zeros(16, 64, device=gpu), group=64)
    assert not zero.dequantize().any()


def test_graph_and_streams(gpu):
    say("int4 graph")
    packed, scales, z, w = weights(512, 512, 128, True, BF, gpu)
    pack = Int4Weight.from_packed(packed, scales, z, group=128)
    for rows in (4, 150):
        x = torch.randn(rows, 512, device=gpu).to(BF)
        outs = [torch.empty(rows, n, dtype=BF, device=gpu) for n in (512, 256)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            linear_int4(x, pack, outs[0])
            linear_int4(x, pack, outs[1], swiglu=True)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            linear_int4(x, pack, outs[0])
            linear_int4(x, pack, outs[1], swiglu=True)
        for _ in range(4):
            x.copy_(torch.randn_like(x))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], linear_int4(x, pack, torch.empty_like(outs[0])))
            assert torch.equal(outs[1], linear_int4(x, pack, torch.empty_like(outs[1]), swiglu=True))


def test_refusals(gpu):
    say("int4 refusals")
    packed, scales, z, w = weights(48, 256, 64, True, BF, gpu)
    pack = Int4Weight.from_packed(packed, scales, z, group=64)
    x, out = torch.randn(4, 256, device=gpu).to(BF), torch.empty(4, 48, dtype=BF, device=gpu)
    bad = pytest.raises(ValueError)
    for args in ((x[:, :128], pack, out), (x.float(), pack, out), (x, pack, out.half()), (x, pack, out[:3]), (x[0], pack, out),
                 (x, pack, out[:, :40]), (x.t().contiguous().t(), pack, out), (x, pack, out.t().contiguous().t()),
                 (torch.empty(4, 257, dtype=BF, device=gpu)[:, :256], pack, out),
                 (torch.empty(4 * 256 + 1, dtype=BF, device=gpu)[1:].view(4, 256), pack, out),
                 (x.clone().requires_grad_(), pack, out)):
        with bad:
            linear_int4(*args)
    with bad:
        linear_int4(x, pack, out[:, :24], swiglu=True)  # 48 rows: tiles of gate and up rows mix
    with pytest.raises(RuntimeError):
        linear_int4(x.cpu(), pack, out)
    with pytest.raises(RuntimeError):
        linear_int4(x, pack.to("cpu"), out)
    assert linear_int4(x[:0], pack, out[:0]).shape == (0, 48)


def test_more_rows_than_the_stream_kernel_takes(gpu):
    """16 x 65,535 rows and more against a single tile of columns: every copy of the same rows gives the same bits."""
    rows = 4096 * 257
    say("int4 rows", rows)
    packed, scales, z, w = weights(16, 1024, 64, True, BF, gpu)
    pack = Int4Weight.from_packed(packed, scales, z, group=64)
    base = torch.randn(4096, 1024, device=gpu).to(BF)
    out = linear_int4(base.repeat(257, 1), pack, torch.full((rows, 16), float("nan"), dtype=BF, device=gpu)).view(257, 4096, 16)
    assert (out == out[0]).all()
    close(out[0], base.double() @ w.t(), product_bound(base, scales, 64, 1024))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_kernel_that_the_rule_picks(gpu, group, swiglu, dtype):
    """The least product for each tile, split and number of a stream wave's blocks, and the least that goes round a tile's
    ring; scales of both types. Sums of whole numbers: (192 + c - z) x and 192 x of a group stay below 399 * 2 * 128 <
    2^24, and all groups below 15 * 2 * 18,432 * 8 < 2^24 in units of the smallest scale, an eighth of the largest, so fp32 holds every one
    exactly. With swiglu expf, the sum, the quotient and the product round by at most 8 * 2^-24 of the result; for gates below
    -88.7 expf(-gate) is infinite, and silu 0 in place of less than 88.8 exp(-88.7) < 2^-121."""
    for i, (kernel, shapes) in enumerate(representatives(group, int(swiglu)).items()):
        for rows, n, k in shapes:
            say("int4 kernel", kernel, rows, n, k, group, swiglu, dtype)
            for st in (BF, HF):
                packed, _, z, _ = weights(n, k, group, i % 2 == 0, st, gpu, exact=True)
                g = torch.Generator(device=gpu).manual_seed(rows + n + k)
                top = -4 if swiglu else 0  # gates on both sides of silu's bend
                scales = torch.pow(2.0, torch.randint(top - 3, top + 1, (n, k // group), device=gpu, generator=g).float()).to(st)
                pack = Int4Weight.from_packed(packed, scales, z, group=group)
                w = pack.dequantize(torch.float64)
                x = torch.full((rows, k + 8), float("nan"), dtype=dtype, device=gpu)[:, :k]
                x.copy_(torch.randint(-2, 3, (rows, k), device=gpu, generator=g))
                cols = n // 2 if swiglu else n
                out = torch.full((rows + 1, cols + 3), 7.0, dtype=dtype, device=gpu)
                linear_int4(x, pack, out[:rows, :cols], swiglu=swiglu)
                ref = x.double() @ w.t()
                if swiglu:
                    gate, up = ref.chunk(2, dim=1)
                    ref = gate * torch.sigmoid(gate) * up
                    close(out[:rows, :cols], ref, 8 * 2.0 ** -24 * ref.abs() + 2.0 ** -121 * up.abs())
                else:
                    assert torch.equal(out[:rows, :cols], ref.to(dtype))
                assert (out[rows:] == 7).all() and (out[:, cols:] == 7).all()
                again = torch.empty(rows, cols, dtype=dtype, device=gpu)
                assert torch.equal(linear_int4(x, pack, again, swiglu=swiglu), out[:rows, :cols])
