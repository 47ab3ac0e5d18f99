"""The residual connection with its norms against float64, within a bound of float32 arithmetic that is derived from the formulas."""

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn as nn
import lucid_amd.nn.functional as F
from lucid_amd import _C

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of float32, relative


def hip(a):
    return L.tensor(np.ascontiguousarray(a), device="hip")


def norm(v, e, weight, bias, layer, eps):
    """A norm of rows v known to within e -> the result, and how far float32 arithmetic may be from it.  Sums: a lane adds 32 values at most, lanes and
    wavefronts ten times more: 48 roundings of a sum of the magnitudes bound them, and the products in front."""
    mean = v.mean(-1, keepdims=True) if layer else np.zeros_like(v[..., :1])
    e_mean = e.mean(-1, keepdims=True) + 48 * U * abs(v).mean(-1, keepdims=True) if layer else 0.0
    c = v - mean
    e = e + e_mean + U * abs(c)
    power = (c * c).mean(-1, keepdims=True) + eps
    # the root's relative error is half of the sum's; the root, the inverse, the mean's factor round too
    e_power = (2 * abs(c) * e + e * e).mean(-1, keepdims=True) + 52 * U * power
    f = 1 / np.sqrt(power)
    e_f = f * (e_power / power + 4 * U)
    y = c * f * weight + bias
    return y, abs(weight) * (e * (f + e_f) + abs(c) * e_f) + 3 * U * (abs(c * f * weight) + abs(bias)) + U * abs(y)


def check(rows, cols, layer=False, post=False, gate_rows=0, scale=False, x_type=np.float32, r_type=np.float32, eps=1e-6, affine=True, bias=None, seed=0,
          x=None, r=None, in_place=False):
    rng = np.random.default_rng(seed + rows * 31 + cols)
    some = lambda *s: rng.standard_normal(s).astype(np.float32)
    x = (some(rows, cols) * (1 + 20 * (rng.random(cols) < 0.02))).astype(x_type) if x is None else x
    r = (3 * some(rows, cols) + 1).astype(r_type) if r is None else r
    bias = layer if bias is None else bias
    vec = {"weight": 1 + 0.3 * some(cols) if affine else None, "bias": some(cols) if bias else None, "scale": some(cols) if scale else None,
           "post_weight": 1 + 0.3 * some(cols) if post and affine else None, "post_bias": some(cols) if post and bias else None}
    gate = some(gate_rows, cols).astype(x_type) if gate_rows else None
    xd, rd = hip(x), hip(r)
    out = dict(out=xd, residual_out=rd) if in_place else {}
    y, r2 = F.residual_norm(xd, rd, norm="layer" if layer else "rms", eps=eps, post=post, gate=hip(gate) if gate_rows else None,
                            **{n: hip(v) if v is not None else None for n, v in vec.items()}, **out)
    assert y.shape == x.shape and y.dtype.np == x_type and r2.dtype.np == r_type
    d = {n: v.astype(np.float64) if v is not None else (0.0 if "bias" in n else 1.0) for n, v in vec.items()}
    t, e = x.astype(np.float64), np.zeros((rows, cols))
    if post:
        t, e = norm(t, e, d["post_weight"], d["post_bias"], layer, eps)
    g = d["scale"] * (np.repeat(gate.astype(np.float64), rows // gate_rows, 0) if gate_rows else 1.0)
    e, t = abs(g) * e + 2 * U * abs(t * g), t * g
    want_r = r.astype(np.float64) + t
    e = e + U * abs(want_r)
    want_y, e_y = norm(want_r, e, d["weight"], d["bias"], layer, eps)
    half = lambda v, dt: abs(v) * np.finfo(dt).eps / 2 + np.finfo(dt).tiny * np.finfo(dt).eps  # (a rounding, and of the smallest numbers a step)
    assert (abs(r2.numpy() - want_r) <= e + half(abs(want_r) + e, r_type)).all()
    assert (abs(y.numpy() - want_y) <= e_y + half(abs(want_y) + e_y, x_type)).all()
    return y.numpy(), r2.numpy()


# rows of every number of threads and of values a thread, whole and not
WIDTHS = [1, 2, 3, 5, 16, 255, 256, 257, 512, 513, 768, 1000, 1024, 1025, 2047, 2048, 2501, 2910, 3000, 4095, 4096, 4097, 5999, 6140, 6146, 8191, 8192, 8195, 16384, 16385, 32767, 32768]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("layer,post", [(False, False), (True, True)])
def test_every_width(cols, layer, post):
    check(5, cols, layer, post, gate_rows=5, scale=True)


@pytest.mark.parametrize("types", [(np.float32, np.float32), (np.float16, np.float16), (np.float16, np.float32)])
@pytest.mark.parametrize("rows,cols", [(1, 4096), (3, 768), (197, 771), (6, 5001), (1025, 128)])
@pytest.mark.parametrize("layer,post,gate,scale", [(False, True, 0, False), (True, False, 1, False), (False, False, 1, True), (True, True, 0, True)])
def test_types_and_forms(types, rows, cols, layer, post, gate, scale):
    check(rows, cols, layer, post, gate, scale, *types)


@pytest.mark.parametrize("gate_rows", [1, 2, 3, 4, 6, 12])
def test_a_gate_of_fewer_rows(gate_rows):
    check(12, 130, gate_rows=gate_rows, x_type=np.float16)


@pytest.mark.parametrize("layer", [False, True])
def test_without_weights_and_with_a_bias_of_rms(layer):
    check(4, 300, layer, True, affine=False, bias=False)
    check(4, 300, layer, True, affine=False, bias=True)


@pytest.mark.parametrize("types", [(np.float32, np.float32), (np.float16, np.float16), (np.float16, np.float32)])
def test_in_the_places_of_x_and_residual(types):
    y, r = check(37, 1030, True, True, 37, True, *types)
    y2, r2 = check(37, 1030, True, True, 37, True, *types, in_place=True)
    assert np.array_equal(y, y2) and np.array_equal(r, r2)


@pytest.mark.parametrize("cols", [5, 258, 1233, 4555, 9002, 20003])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("types", [(np.float32, np.float32), (np.float16, np.float16), (np.float16, np.float32)])
def test_ragged_rows_in_their_own_places(cols, post, types):
    check(70, cols, layer=True, post=post, x_type=types[0], r_type=types[1], in_place=True)


def test_rows_of_zeros_and_of_one_value():
    x, r = np.zeros((3, 700), np.float32), np.zeros((3, 700), np.float32)
    r[1], r[2] = 1e4, -3e-3
    for layer in (False, True):
        check(3, 700, layer, True, x=x, r=r, eps=1e-5)


def test_a_mean_far_from_zero():
    """A variance about the mean, not the difference of two large numbers."""
    rng = np.random.default_rng(0)
    r = (1000 + rng.standard_normal((9, 2048))).astype(np.float32)
    check(9, 2048, True, x=np.zeros((9, 2048), np.float32), r=r)


def test_what_is_not_finite_stays_in_its_row():
    rng = np.random.default_rng(1)
    x, r = (rng.standard_normal((6, 900)).astype(np.float32) for _ in range(2))
    clean_y, clean_r = (t.numpy() for t in F.residual_norm(hip(x), hip(r)))
    x[1, 5], r[3, 899], x[4, 0] = np.nan, np.inf, -np.inf
    y, r2 = (t.numpy() for t in F.residual_norm(hip(x), hip(r)))
    for i in (0, 2, 5):
        assert np.array_equal(y[i], clean_y[i]) and np.array_equal(r2[i], clean_r[i])
    assert np.isnan(y[1]).all() and np.isnan(y[3, 899]) and np.isnan(y[4, 0])
    assert np.isnan(r2[1, 5]) and r2[3, 899] == np.inf and r2[4, 0] == -np.inf


def test_rms_norm_and_its_module():
    rng = np.random.default_rng(2)
    for dt, shape in ((np.float32, (3, 5, 77)), (np.float16, (2, 4096)), (np.float32, (0, 8))):
        x = rng.standard_normal(shape).astype(dt)
        m = nn.RMSNorm(shape[-1])
        w = (1 + 0.2 * rng.standard_normal(shape[-1])).astype(np.float32)
        m.register_buffer("weight", L.tensor(w))
        want, e = norm(x.astype(np.float64), np.zeros(shape), w.astype(np.float64), 0.0, False, 1e-6)
        for y in (m(hip(x)), F.rms_norm(hip(x), shape[-1], hip(w))):
            assert y.shape == shape and y.dtype.np == dt
            assert (abs(y.numpy() - want) <= e + (abs(want) + e) * np.finfo(dt).eps / 2 + np.finfo(dt).tiny * np.finfo(dt).eps).all()


def test_no_rows_and_no_columns():
    for shape in ((0, 5), (3, 0), (0, 0)):
        y, r = F.residual_norm(hip(np.zeros(shape, np.float32)), hip(np.zeros(shape, np.float32)), gate=hip(np.zeros(shape, np.float32)))
        assert y.shape == shape and r.shape == shape


def test_replayed_from_a_graph():
    rng = np.random.default_rng(3)
    new = lambda: rng.standard_normal((50, 640)).astype(np.float16)
    x, r = hip(new()), hip(new())
    F.residual_norm(x, r, post=True)
    with L.graph.capture() as g:
        y, r2 = F.residual_norm(x, r, post=True)
    for _ in range(3):
        x.copy_from(new()), r.copy_from(new())
        g.replay()
        L.synchronize()
        want = [t.numpy() for t in F.residual_norm(x, r, post=True)]
        assert np.array_equal(y.numpy(), want[0]) and np.array_equal(r2.numpy(), want[1])


@pytest.mark.parametrize("rows,cols", [((1 << 22) + 3, 4100), ((1 << 24) + 5, 1028)])
def test_rows_of_more_threads_than_a_launch_has_along_an_axis(rows, cols):
    """34 GB of one number, in place; each value's norm is 1 within half a step of float16."""
    x = L.Tensor.empty((rows, cols), L.float16, "hip")
    _C.call("lq_fill_bytes", x.data_ptr, 0x3c, x.nbytes, None)
    F.rms_norm(x, cols, eps=0.0, out=x)
    for at in (0, 1 << 20, 1 << 21, (1 << 21) + 1, rows // 2, (rows - 3) // 2, rows - 3):
        assert (x.row_range(at, at + 3).numpy() == 1.0).all()
