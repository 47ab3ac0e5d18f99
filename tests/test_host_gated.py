"""Gated projections without a device: what their module refuses, and that the exact tests' shapes reach every kernel and tile that calls go to."""

import ctypes as C
import random

import pytest

import lucid_amd as L
import lucid_amd.nn as nn
import lucid_amd.nn.quantized as nnq
from lucid_amd import _C


@pytest.mark.parametrize("group_size", [0, 1, 16, 48, 256, -32])
def test_the_module_refuses_groups_that_its_forward_does_not_take(group_size):
    with pytest.raises(ValueError, match="group_size must be 32, 64 or 128"):
        nnq.QuantizedGatedLinearMLX(768, 8, group_size=group_size)
    with pytest.raises(ValueError, match="group_size must be 32, 64 or 128"):
        nnq.QuantizedGatedLinearMLX.from_float(nn.Linear(768, 8), nn.Linear(768, 8), group_size=group_size)


def tile(M, N, K, bits, dtype):
    """(kernel of many rows or not, rows and columns of a block) of a call."""
    out = [C.c_int() for _ in range(3)]
    _C.call("lq_wq_gated_tile", M, N, K, bits, dtype, *map(C.byref, out))
    return tuple(v.value for v in out)


# Shapes of the tiles that the lists of test_hip_wq_gated.py do not reach: blocks of 32 rows x 128 columns of float32
MORE = [(1229, 1651, 1120, 32), (552, 1945, 2752, 64), (399, 4892, 1088, 64), (1243, 1640, 1280, 128), (710, 2764, 352, 32), (645, 3052, 384, 64), (273, 6900, 512, 64)]


def test_the_exact_tests_reach_every_tile():
    from test_hip_wq_gated import SHAPES, WIDE

    shapes = SHAPES + [(M, N, K, gs) for M, N in WIDE for K, gs in ((160, 32), (320, 64), (640, 128))] + MORE
    types = [(dtype, bits) for dtype in (_C.F32, _C.F16) for bits in (4, 8)]
    reached = {(dtype, bits, gs) + tile(M, N, K, bits, dtype) for M, N, K, gs in shapes for dtype, bits in types}
    rng, missing = random.Random(0), {}
    for _ in range(20000):
        M, N, K = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 14)), 32 * int(2 ** rng.uniform(0, 9))
        for dtype, bits in types:
            t = tile(M, N, K, bits, dtype)
            for gs in (32, 64, 128):
                if K % gs == 0 and (dtype, bits, gs) + t not in reached:
                    missing[(dtype, bits, gs) + t] = (M, N, K)
    assert not missing


def test_tiles_of_what_is_no_call_are_refused():
    i = C.c_int()
    for args, error in (((0, 8, 64, 4, _C.F32), L.ShapeMismatch), ((1, -1, 64, 4, _C.F32), L.ShapeMismatch), ((1, 8, 0, 4, _C.F32), L.ShapeMismatch),
                        ((1, 8, 64, 2, _C.F32), ValueError), ((1, 8, 64, 4, _C.BF16), L.DtypeMismatch)):
        with pytest.raises(error, match="wq_gated_tile"):
            _C.call("lq_wq_gated_tile", *args, C.byref(i), C.byref(i), C.byref(i))
    with pytest.raises(ValueError, match="wq_gated_tile"):
        _C.call("lq_wq_gated_tile", 1, 8, 64, 4, _C.F32, C.byref(i), None, C.byref(i))
