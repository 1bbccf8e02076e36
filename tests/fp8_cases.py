"""Sizes that reach each kernel of uqm_fp8_linear."""

from __future__ import annotations

import ctypes

from uma_qmoe_amd import _native


def plan(rows, out_features, in_features):
    """(weight rows, tokens, waves) of a workgroup that the call takes."""
    got = [ctypes.c_int32() for _ in range(3)]
    rc = _native.library().uqm_fp8_linear_plan(rows, out_features, in_features, *map(ctypes.byref, got))
    _native.check(rc, "uqm_fp8_linear_plan")
    return tuple(v.value for v in got)


# (weight rows, tokens, waves), then tokens x out_features x in_features: a ragged
# size in each direction with a short last block, and whole blocks with 16-byte outputs
PLANNED = [
    ((16, 16, 4), 17, 70, 272), ((16, 16, 4), 32, 64, 256),
    ((16, 16, 8), 31, 70, 1040), ((16, 16, 8), 16, 128, 1024),
    ((32, 32, 4), 53, 8275, 144), ((32, 32, 4), 72, 7024, 128),
    ((32, 32, 8), 18, 9755, 800), ((32, 32, 8), 32, 4800, 2048),
    ((64, 32, 8), 8108, 35, 928), ((64, 32, 8), 841, 576, 896),
    ((64, 64, 4), 84, 11126, 272), ((64, 64, 4), 154, 6744, 128),
    ((64, 64, 8), 33, 11331, 1952), ((64, 64, 8), 133, 4928, 2048),
    ((128, 128, 8), 1100, 4501, 400), ((128, 128, 8), 286, 6552, 128),
    ((128, 256, 8), 665, 10446, 1344), ((128, 256, 8), 1024, 7680, 1536),
    ((256, 256, 8), 6172, 2433, 272), ((256, 256, 8), 4096, 2304, 256),
]

# the last tile has one row and one token, so that its buffers are shorter than the
# blocks that are loaded ahead, and their scales than a panel of 8
ONE_ROW = [
    ((128, 128, 8), 6529, 257, 16), ((128, 128, 8), 6529, 257, 128), ((128, 128, 8), 6529, 257, 144),
    ((128, 256, 8), 13569, 1025, 1040), ((256, 256, 8), 15105, 1537, 128), ((256, 256, 8), 14081, 513, 144),
    ((256, 256, 8), 13057, 513, 1040),
]
