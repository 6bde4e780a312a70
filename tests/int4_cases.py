"""Which kernel a 4-bit product runs on, and products that reach every one that the rule can pick."""

from __future__ import annotations

import ctypes
from functools import lru_cache

from aspire_amd import _lib

ROWS = (1, 2, 11, 16, 17, 31, 33, 40, 48, 49, 64, 65, 100, 129, 208, 225, 257, 300, 512, 700, 1025)
COLUMNS = (16, 32, 96, 512, 1056, 2080, 4128, 6144, 8224, 12320, 16384, 24608, 32800, 57376)
DEPTHS = (32, 64, 128, 192, 384, 640, 1152, 1984, 2176, 2944, 3584, 4096, 5120, 6144, 7168, 8192, 9216, 12288, 14336, 18432)
TILES = ((32, 128), (32, 256), (48, 128), (48, 256), (64, 128), (64, 256), (112, 256), (128, 128), (128, 256))
MOST_STEPS = 5  # stages of a ring


def choice(rows, n, k, group, swiglu):
    """Rows and columns of a tile (0, 0: the stream kernel), and the splits of k."""
    out = (ctypes.c_int32 * 3)()
    _lib.lib().aspire_linear_int4_choice(rows, n, k, group, swiglu, out)
    return tuple(out)


def kernel_of(rows, n, k, group, swiglu):
    """The tile, or the blocks that a wave of the stream kernel holds, and whether k is split; and a workgroup's blocks."""
    tile, cols, splits = choice(rows, n, k, group, swiglu)
    steps = -(-((k + 127) // 128) // splits)
    return ((tile, cols) if tile else (0, -(-steps // 8))) + (splits > 1,), steps


@lru_cache(None)
def representatives(group, swiglu):
    """``{kernel: [(rows, n, k), ...]}``: the least product for each kernel, and for a tile the least that goes round its ring."""
    least = {}
    for n in COLUMNS:
        for k in DEPTHS:
            if k % group or (swiglu and n % 32):
                continue
            for rows in ROWS:
                kernel, steps = kernel_of(rows, n, k, group, swiglu)
                for long in (False, True):
                    if kernel[0] == 0 and long or long and steps <= MOST_STEPS + 1:
                        continue
                    cost = (rows + 300) * n * k
                    if cost < least.get((kernel, long), (float("inf"),))[0]:
                        least[kernel, long] = cost, (rows, n, k)
    found = {}
    for (kernel, _), (_, shape) in sorted(least.items()):
        if shape not in found.setdefault(kernel, []):
            found[kernel].append(shape)
    return found
