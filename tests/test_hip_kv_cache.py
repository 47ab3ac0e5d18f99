"""Quantized key / value cache on the device: rows written and read back, to the bit."""

import ctypes as C

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.quantization as Q
import oracle.kv_cache as K
from lucid_amd import _C

pytestmark = pytest.mark.gpu

SCHEMES = {True: Q.per_channel_symmetric, False: Q.per_channel_affine}
DTYPES = {8: Q.qint8, 4: Q.qint4}


def hip(a):
    return L.tensor(np.ascontiguousarray(a), device="hip")


def ids(a):
    return hip(np.asarray(a, np.int32))


def make(pages, page, heads, dim, symmetric, bits):
    return Q.PagedKVCache(pages, page, heads, dim, SCHEMES[symmetric], DTYPES[bits])


def buffers(c):
    return {n: getattr(c, n).numpy() for n in ("k_codes", "v_codes", "k_scale", "v_scale", "k_zero", "v_zero") if getattr(c, n) is not None}


def expected(c, before, k, v, slots):
    """The buffers after a write, from the oracle."""
    want = {n: b.copy() for n, b in before.items()}
    for t, s in enumerate(slots):
        if not 0 <= s < c.num_slots:
            continue
        for name, x in (("k", k), ("v", v)):
            u, scale, zero = K.quantize(x[t].astype(np.float32), c.qdtype.bits, c.qscheme.is_symmetric)
            at = (s // c.page_size, slice(None), s % c.page_size)
            want[name + "_codes"][at] = K.pack(u, c.qdtype.bits).view(np.int8)
            want[name + "_scale"][at] = scale
            if name + "_zero" in want:
                want[name + "_zero"][at] = zero
    return want


def same(got, want):
    for n in want:
        g, w = got[n], want[n]
        assert np.array_equal(g, w, equal_nan=g.dtype.kind == "f"), n


CASES = [(8, True, 128, 8, 16, np.float16, 37), (8, False, 64, 12, 32, np.float32, 100), (4, True, 128, 2, 16, np.float32, 1),
         (4, False, 32, 1, 48, np.float16, 65), (8, True, 16, 3, 16, np.float32, 33), (8, False, 80, 5, 64, np.float16, 7),
         (8, True, 256, 1, 16, np.float16, 9), (4, False, 224, 4, 16, np.float32, 20), (8, False, 112, 7, 16, np.float32, 300),
         (4, True, 96, 2, 128, np.float16, 130), (8, True, 48, 2, 16, np.float16, 17), (4, False, 160, 1, 16, np.float16, 5)]


@pytest.mark.parametrize("bits,symmetric,dim,heads,page,dtype,tokens", CASES)
def test_write_and_read_are_exact(bits, symmetric, dim, heads, page, dtype, tokens):
    rng = np.random.default_rng(dim + tokens)
    pages = tokens // page + 3
    c = make(pages, page, heads, dim, symmetric, bits)
    # what no token is written to stays as it was
    junk = {n: rng.integers(-128, 128, b.shape).astype(b.dtype) for n, b in buffers(c).items()}
    for n, b in junk.items():
        getattr(c, n).copy_from(b)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    if tokens > 3:
        slots[rng.permutation(tokens)[:3]] = [-1, pages * page, -(1 << 31)]
    k, v = ((rng.standard_normal((tokens, heads, dim)) * rng.lognormal(0, 2, (tokens, heads, 1))).astype(dtype) for _ in range(2))
    if tokens > 8:
        k[4], v[5], k[6] = 0, 2.5, np.abs(k[6])
    Q.kv_cache_write(c, hip(k), hip(v), ids(slots))
    got, want = buffers(c), expected(c, junk, k, v, slots)
    same(got, want)
    there = (slots >= 0) & (slots < pages * page)
    at = np.where(there, slots, 0)
    for dt in (L.float32, L.float16):
        for y, name in zip(Q.kv_cache_read(c, ids(slots), dt), "kv"):
            rows = [want[name + p][at // page, :, at % page] for p in ("_codes", "_scale")]
            zero = None if symmetric else want[name + "_zero"][at // page, :, at % page]
            x = K.values(rows[0], rows[1], zero, bits) * there[:, None, None]
            with np.errstate(over="ignore"):
                assert np.array_equal(y.numpy(), x.astype(dt.np)), (name, dt)


def test_rows_are_those_of_the_row_quantizer():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((64, 2, 128)).astype(np.float32)
    for bits in (8, 4):
        for symmetric in (True, False):
            c = make(4, 16, 2, 128, symmetric, bits)
            Q.kv_cache_write(c, hip(x), hip(-x), ids(np.arange(64)))
            for name, y in (("k", x), ("v", -x)):
                codes, scale, zero = Q.quantize_rows_dynamic(hip(y.reshape(128, 128)), SCHEMES[symmetric], DTYPES[bits])
                at = lambda t: t.reshape(4, 16, 2, -1).transpose(0, 2, 1, 3)
                u = K.unpack(getattr(c, name + "_codes").numpy(), bits).astype(int) + K.grid(bits)[0]
                assert np.array_equal(u, at(codes.numpy()))
                assert np.array_equal(getattr(c, name + "_scale").numpy(), at(scale.numpy())[..., 0])
                if not symmetric:
                    assert np.array_equal(getattr(c, name + "_zero").numpy(), at(zero.numpy())[..., 0])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("symmetric", [True, False])
def test_rows_of_special_values(bits, symmetric):
    """Infinities, NaN, subnormals, the largest floats, scales at the floor, and values on the border of two codes."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((48, 1, 64)).astype(np.float32)
    x[0, 0, 5], x[1, 0, 63], x[2, 0, 0], x[3, 0, 8] = np.inf, -np.inf, np.nan, np.inf
    x[3, 0, 9], x[3, 0, 10] = -np.inf, np.nan
    x[4], x[5], x[6], x[7] = x[4] * 1e-42, x[5] * 1e-9, x[6] * 1e37, np.clip(x[7] * 1e38, -3.4e38, 3.4e38)
    x[8, 0, :], x[9, 0, :], x[10, 0, :], x[11, 0, :] = 3.4028235e38, -3.4028235e38, -0.0, 1e-45
    x[12, 0, 1:], x[13, 0, 0], x[14, 0, 0] = 0, 1e30, -1e30
    x[15] *= np.float32(2.0 ** 119)
    for r in range(16, 48):  # quotients n + 1/2 and their neighbours: of a scale that is a power of two, and of any
        top = np.float32(127.5 if bits == 8 else 7.5) * np.float32(2.0 ** (r - 30) if r < 32 else rng.lognormal(0, 2))
        step = top / np.float32(127.5 if bits == 8 else 7.5)
        n = rng.integers(-K.grid(bits)[1] - 1, K.grid(bits)[1] + 1, 64)
        x[r, 0] = np.nextafter(((n + np.float32(0.5)) * step).astype(np.float32), rng.choice([-np.inf, 0, np.inf], 64).astype(np.float32))
        x[r, 0, 0] = top if r % 2 else -top
    c = make(3, 16, 1, 64, symmetric, bits)
    before = buffers(c)
    Q.kv_cache_write(c, hip(x), hip(x[::-1]), ids(np.arange(48)))
    same(buffers(c), expected(c, before, x, x[::-1], np.arange(48)))
    h = np.where(np.abs(x) < 6e4, x, 60000 * np.sign(x)).astype(np.float16)
    h[20, 0, 3], h[21, 0, 4] = np.inf, np.nan
    Q.kv_cache_write(c, hip(h), hip(h[::-1]), ids(np.arange(48)))
    same(buffers(c), expected(c, before, h, h[::-1], np.arange(48)))


def test_all_quotients_of_a_row_are_rounded_as_the_division():
    """Many values against many scales: the steps that stand in for the division give its result."""
    rng = np.random.default_rng(8)
    x = rng.uniform(-1, 1, (20000, 1, 128)).astype(np.float32) * rng.lognormal(0, 6, (20000, 1, 1)).astype(np.float32)
    c = make(1250, 16, 1, 128, False, 8)
    Q.kv_cache_write(c, hip(x), hip(x[::-1]), ids(np.arange(20000)))
    u, scale, zero = K.quantize(x, 8, False)
    assert np.array_equal(c.k_codes.numpy().view(np.uint8).reshape(u.shape), u)
    assert np.array_equal(c.k_scale.numpy().ravel(), scale.ravel()) and np.array_equal(c.k_zero.numpy().ravel(), zero.ravel())


@pytest.mark.parametrize("bits", [8, 4])
def test_float16_rows_of_every_maximum(bits):
    """Symmetric rows, one for each positive finite float16 as the largest value: the shorter way to the quotient gives the division's result."""
    rng = np.random.default_rng(bits)
    top = np.arange(1, 0x7c00, dtype=np.uint16)
    x = (rng.integers(0, 1 << 16, (len(top), 1, 128)) % (top[:, None, None].astype(np.int64) + 1)).astype(np.uint16)  # (by their bits: all sizes alike)
    near = rng.random(x.shape) < 0.5
    x = np.where(near, top[:, None, None] - np.minimum(top[:, None, None], rng.integers(0, 4096, x.shape)), x).astype(np.uint16)
    x[:, 0, 0] = top
    x = (x | (rng.integers(0, 2, x.shape) << 15).astype(np.uint16)).view(np.float16)
    c = make(1984, 16, 1, 128, True, bits)
    Q.kv_cache_write(c, hip(x), hip(x[::-1]), ids(np.arange(len(top))))
    for name, y in (("k", x), ("v", x[::-1])):
        u, scale, _ = K.quantize(y.astype(np.float32), bits, True)
        got = getattr(c, name + "_codes").numpy().view(np.uint8).reshape(-1, 128 * bits // 8)[:len(top)]
        assert np.array_equal(got, K.pack(u, bits).reshape(got.shape))
        assert np.array_equal(getattr(c, name + "_scale").numpy().ravel()[:len(top)], scale.ravel())


def test_packed_rows_and_an_empty_call():
    rng = np.random.default_rng(5)
    for dtype in (np.float32, np.float16):
        x = rng.standard_normal((3, 7, (6 + 2 * 2) * 64)).astype(dtype)
        slots = rng.permutation(32)[:21].astype(np.int32)
        a, b = make(2, 16, 2, 64, False, 4), make(2, 16, 2, 64, False, 4)
        Q.kv_cache_write_qkv(a, hip(x), 6, ids(slots))
        y = x.reshape(21, 10, 64)
        Q.kv_cache_write(b, hip(y[:, 6:8]), hip(y[:, 8:]), ids(slots))
        same(buffers(a), buffers(b))
        before = buffers(a)
        Q.kv_cache_write(a, L.Tensor.empty((0, 2, 64), L.float32), L.Tensor.empty((0, 2, 64), L.float32), L.Tensor.empty((0,), L.int32))
        k, v = Q.kv_cache_read(a, L.Tensor.empty((0,), L.int32))
        assert k.shape == v.shape == (0, 2, 64)
        same(buffers(a), before)


def test_a_cache_of_more_than_2_to_the_32_bytes():
    heads, dim, page = 8, 128, 64
    pages = (5 << 30) // (heads * dim * page)
    c = make(pages, page, heads, dim, True, 8)
    rng = np.random.default_rng(2)
    x = rng.standard_normal((40, heads, dim)).astype(np.float16)
    slots = np.concatenate([pages * page - 1 - np.arange(20), np.arange(20) * (c.num_slots // 20)]).astype(np.int32)
    Q.kv_cache_write(c, hip(x), hip(-x), ids(slots))
    u, scale, zero = K.quantize(x.astype(np.float32), 8, True)
    k, v = Q.kv_cache_read(c, ids(slots))
    assert np.array_equal(k.numpy(), K.values(u, scale, zero, 8))
    u, scale, zero = K.quantize(-x.astype(np.float32), 8, True)
    assert np.array_equal(v.numpy(), K.values(u, scale, zero, 8))


def test_a_captured_write_and_read_replays_on_another_stream():
    rng = np.random.default_rng(6)
    c = make(4, 16, 2, 64, True, 8)
    k, v, slots = hip(np.zeros((8, 2, 64), np.float32)), hip(np.zeros((8, 2, 64), np.float32)), ids(np.zeros(8))
    Q.kv_cache_write(c, k, v, slots)
    with L.graph.capture() as g:
        Q.kv_cache_write(c, k, v, slots)
        yk, yv = Q.kv_cache_read(c, slots)
    stream = C.c_void_p()
    _C.call("lq_stream_create", C.byref(stream))
    try:
        for rep in range(4):
            x, at = rng.standard_normal((2, 8, 2, 64)).astype(np.float32), rng.permutation(64)[:8].astype(np.int32)
            k.copy_from(x[0]), v.copy_from(x[1]), slots.copy_from(at)
            if rep % 2:
                _C.call("lq_graph_launch", g.id, stream)
                _C.call("lq_sync", stream)
            else:
                g.replay()
            for y, z in ((yk, x[0]), (yv, x[1])):
                u, scale, zero = K.quantize(z, 8, True)
                assert np.array_equal(y.numpy(), K.values(u, scale, zero, 8)), rep
    finally:
        L.synchronize()
        _C.call("lq_stream_destroy", stream)


def test_refusals():
    c = make(2, 16, 2, 64, True, 8)
    x, s = hip(np.zeros((3, 2, 64), np.float32)), ids([0, 1, 2])
    for bad, error in (((x, x, ids([0, 1])), L.ShapeMismatch), ((x, hip(np.zeros((3, 2, 64), np.float16)), s), L.DtypeMismatch),
                       ((hip(np.zeros((3, 2, 64), np.int32)),) * 2 + (s,), L.DtypeMismatch), ((x, hip(np.zeros((3, 2, 32), np.float32)), s), L.ShapeMismatch),
                       ((x, x, hip(np.zeros(3, np.int64))), L.DtypeMismatch), ((x.cpu(), x, s), L.DeviceMismatch), ((x, x, s.cpu()), L.DeviceMismatch),
                       ((x.reshape(3, 128), x, s), L.ShapeMismatch)):
        with pytest.raises(error):
            Q.kv_cache_write(c, *bad)
    with pytest.raises(L.ShapeMismatch):
        Q.kv_cache_write_qkv(c, hip(np.zeros((3, 5 * 64), np.float32)), 2, s)
    with pytest.raises(L.DtypeMismatch):
        Q.kv_cache_read(c, s, L.int8)
    with pytest.raises(L.ShapeMismatch):
        Q.kv_cache_read(c, s, out=(x, hip(np.zeros((2, 2, 64), np.float32))))
    with pytest.raises(L.ShapeMismatch):
        Q.kv_cache_read(c, ids([[0, 1]]))
    import copy
    with pytest.raises(TypeError):
        copy.deepcopy(c)
