"""The group terms (b + 2^(bits-1) s) (sum of x) of the gated projections where they cancel: they are float32 terms whatever x's type and
however many rows a call has."""

import numpy as np
import pytest

import oracle.wq_group as W
from lucid_amd.quantization import _qgemm
from test_hip_wq_gated import bound, hip, some_columns

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N", [(1, 40), (16, 300), (685, 8410)])
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_group_terms_keep_float32(M, N, gs, bits, dtype):
    """Four groups, the second and the fourth the first and the third with the other sign but for a few units of 2^-20 in b, under the same x: what is left of
    the gate is those units times the groups' sums of x.  b + 2^(bits-1) s is a multiple of 2^-20 below 1/2 and a sum of x at most 8, so that no sum passes
    2^24 units and float32 is exact; the way up is its bias of one.  So the result is the exact number, rounded to its type once."""
    rng = np.random.default_rng(M + gs + bits)
    half, K = 1 << (bits - 1), 4 * gs
    x = np.zeros((M, 4, gs))
    for g in (0, 2):
        for _ in range(8):
            x[np.arange(M), g, rng.integers(0, gs, M)] = 1
        x[:, g + 1] = x[:, g]
    assert x.sum(-1).max() <= 8
    codes = rng.integers(half - 3, half + 4, (N, 4, gs))
    codes[:, 1::2] = codes[:, ::2]
    s = np.where(np.arange(4) % 2, -1.0, 1.0) * 2.0 ** -9 * rng.integers(1, 3, (N, 2)).repeat(2, 1)
    units = rng.integers(-(1 << 19) + 1, 1 << 19, (N, 2)).repeat(2, 1)
    units[:, 1::2] = rng.integers(0, 40, (N, 2)) - units[:, ::2]
    b = units * 2.0 ** -20 - half * s
    per = 32 // bits
    packed = (codes.astype(np.uint32).reshape(N, K // per, per) << (np.arange(per, dtype=np.uint32) * np.uint32(bits))).sum(-1, dtype=np.uint64).astype(np.uint32).view(np.int32)
    assert np.array_equal(b, b.astype(np.float32)) and np.array_equal(W.unpack(packed, bits), codes.reshape(N, K))
    none = np.zeros((N, 4), np.float32)
    y = _qgemm.quantized_gated_matmul(hip(x.reshape(M, K).astype(dtype)), tuple(map(hip, (packed, s.astype(np.float32), b.astype(np.float32)))),
                                      (hip(np.zeros_like(packed)), hip(none), hip(none)), "relu", gs, bits, up_bias=hip(np.ones(N, np.float32))).numpy()
    w = W.unpack(packed, bits).astype(np.float64) * s.repeat(gs, 1) + b.repeat(gs, 1)
    want = np.maximum(x.reshape(M, K) @ w.T, 0)
    assert np.array_equal(want * 2 ** 20, np.rint(want * 2 ** 20)) and want.max() > 2.0 ** -15
    assert np.array_equal(y, want.astype(dtype))


@pytest.mark.parametrize("M,N,K,gs", [(16, 512, 1024, 128), (333, 8200, 1152, 128), (685, 8410, 512, 64), (412, 4875, 1056, 32)])
@pytest.mark.parametrize("bits,dtype", [(4, np.float16), (8, np.float16), (4, np.float32)])
@pytest.mark.parametrize("outliers", [True, False])
def test_weights_off_centre(M, N, K, gs, bits, dtype, outliers):
    """A weight of one among small ones in most groups, or all weights about one, under x of a mean: the groups' middles are far from zero and their terms
    cancel against the codes'.  Within the bound of float32 sums alone."""
    rng = np.random.default_rng(M + bits)
    x = (rng.standard_normal((M, K)) + 0.7).astype(dtype)
    w = [(0.02 * rng.standard_normal((N, K))).astype(np.float32) for _ in range(2)]
    for v in w:
        if outliers:
            at = rng.random((N, K)) < 1 / gs
            v[at] = rng.choice([-1.0, 1.0], (N, K))[at]
        else:
            v += rng.choice([-1.0, 1.0], (N, K // gs)).repeat(gs, 1)
    parts = [W.quantize(v, gs, bits) for v in w]
    y = _qgemm.quantized_gated_matmul(hip(x), *(tuple(map(hip, p)) for p in parts), "silu", gs, bits).numpy()
    cols = some_columns(N)
    want, e = bound(x.astype(np.float64), [tuple(a[cols] for a in p) for p in parts], gs, bits, "silu", [np.zeros(len(cols))] * 2)
    info = np.finfo(dtype)
    y = y[:, cols].astype(np.float64)
    near = abs(y - want) <= e + (abs(want) + e) * info.eps / 2 + info.tiny * info.eps
    # what rounds to infinity lies half a step above the largest number or beyond
    beyond = np.isinf(y) & (np.sign(y) == np.sign(want)) & (abs(want) + e >= float(info.max) * (1 + info.eps / 4))
    assert (near | beyond).all()
