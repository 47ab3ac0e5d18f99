"""The restatement of the key / value cache against the oracle's quantizer (which the reference's known answers pin) and
against a softmax written out."""

import numpy as np
import pytest

import oracle as O
import oracle.kv_cache as K


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("symmetric", [True, False])
def test_rows_are_quantized_as_the_row_quantizer_does(bits, symmetric):
    rng = np.random.default_rng(bits + symmetric)
    x = (rng.standard_normal((40, 96)) * rng.lognormal(0, 3, (40, 1))).astype(np.float32)
    x[0], x[1], x[2, :5] = 0, 3, 1e-30
    x[3] = np.abs(x[3])
    qmin, qmax = K.grid(bits)
    u, scale, zero = K.quantize(x, bits, symmetric)
    mn, mx = O.minmax(x, ch_axis=0)
    s, z = O.calc_qparams(mn, mx, symmetric, qmin, qmax, True)
    assert np.array_equal(scale, s) and np.array_equal(zero, z)
    assert np.array_equal(u.astype(int) + qmin, O.quantize(x, s, z, qmin, qmax, ch_axis=0))
    back = K.values(K.pack(u, bits), scale, zero, bits)
    # half a step; an affine zero point is rounded too and a value at an end of the range is clipped by what that moved: one step
    assert np.all(np.abs(back - x) <= scale[:, None] * (0.5 if symmetric else 1.0) * (1 + 1e-5) + (0.5 * scale[:, None] if symmetric else 0))


def test_attention_is_a_softmax_over_the_seen_keys():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((3, 2, 16)), rng.standard_normal((4, 1, 16, 16)), rng.standard_normal((4, 1, 16, 16))
    table = np.array([[2, 0, -1], [3, 3, 3]])
    got = K.attention(q, k, v, table, [0, 2, 2], [20, 0], 0.25)
    keys, vals = (np.concatenate([a[2, 0], a[0, 0, :4]]) for a in (k, v))
    for i in range(2):
        n = 19 + i
        e = np.exp(0.25 * q[i] @ keys[:n].T)
        assert np.allclose(got[i], e / e.sum(-1, keepdims=True) @ vals[:n])
    assert not got[2].any()  # a row of no sequence
    got = K.attention(q, k, v, table, [0, 1, 3], [0, 33], 0.25, window=1)
    assert not got[0].any() and np.allclose(got[1], v[3, 0, 15]) and np.allclose(got[2], v[3, 0, 0])
