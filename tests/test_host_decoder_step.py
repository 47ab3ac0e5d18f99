"""What the operators around a decoder's attention refuse, without a device: Python's checks, and those of the C entry points (the pointers
given are never followed)."""

import ctypes as C

import pytest

import lucid_amd as L
import lucid_amd.nn.functional as F
import lucid_amd.nn.quantized as nnq
import lucid_amd.quantization as Q
from lucid_amd import _C
from lucid_amd.quantization import _qgemm
from test_host_kv_cache import struct

P = 4096  # an aligned address that nothing reads


class Claimed(L.Tensor):
    """A device tensor of a shape and a type with no memory behind it."""

    def __init__(self, shape, dt=L.float32, ptr=P):
        super().__init__(shape, dt, "hip")
        object.__setattr__(self, "_claimed", ptr)

    data_ptr = property(lambda self: self._claimed)


class BareCache(Q.PagedKVCache):
    """Its sizes and addresses alone."""

    __slots__ = ()

    def __init__(self, **kw):
        s = struct(**kw)
        for n in ("num_pages", "page_size", "kv_heads", "head_dim"):
            object.__setattr__(self, n, getattr(s, n))
        object.__setattr__(self, "_struct", s)
        object.__setattr__(self, "_ref", C.byref(s))


i32, f32, f16, i8 = L.int32, L.float32, L.float16, L.int8
HOST = L.tensor([1.0, 2.0])


# ---------------------------------------------------------------- pages
@pytest.mark.parametrize("kw,error", [
    (dict(num_pages=0), L.ShapeMismatch), (dict(page_size=24), L.ShapeMismatch), (dict(num_pages=1 << 27), L.ShapeMismatch),
    (dict(head_dim=72), NotImplementedError), (dict(bits=2), NotImplementedError), (dict(k_scale=None), ValueError), (dict(v_codes=P + 8), ValueError),
    (dict(k_zero=P), ValueError)])
def test_c_entries_refuse_a_bad_cache(kw, error):
    c = C.byref(struct(**kw))
    with pytest.raises(error, match="kv_cache_copy"):
        _C.call("lq_kv_cache_copy", c, P, P, 1, None)
    with pytest.raises(error, match="kv_cache_compact"):
        _C.call("lq_kv_cache_compact", c, P, 1, 1, P, 1, P, None)


@pytest.mark.parametrize("args,error", [
    ((None, P, 1), ValueError), ((P, None, 1), ValueError), ((P, P, 1 << 31), L.ShapeMismatch), ((P, P, 1 << 60), L.ShapeMismatch)])
def test_c_copy_refuses(args, error):
    with pytest.raises(error, match="kv_cache_copy"):
        _C.call("lq_kv_cache_copy", C.byref(struct()), *args, None)


@pytest.mark.parametrize("at,value,error", [
    (1, None, ValueError), (2, -1, L.ShapeMismatch), (3, -1, L.ShapeMismatch), (4, None, ValueError), (5, 1 << 31, L.ShapeMismatch), (5, 1 << 40, L.ShapeMismatch),
    (6, None, ValueError)])
def test_c_compact_refuses(at, value, error):
    args = [C.byref(struct()), P, 4, 1, P, 64, P, None]
    args[at] = value
    with pytest.raises(error, match="kv_cache_compact"):
        _C.call("lq_kv_cache_compact", *args)


def test_nothing_to_move_is_no_call():
    c = C.byref(struct())
    _C.call("lq_kv_cache_copy", c, None, None, 0, None)
    for width, batch, kept in ((4, 1, 0), (4, 0, 5), (0, 1, 5)):
        _C.call("lq_kv_cache_compact", c, None, width, batch, None, kept, None, None)


@pytest.mark.parametrize("src,dst,error", [
    (HOST, Claimed((2,), i32), L.DeviceMismatch), (Claimed((2,), f32), Claimed((2,), i32), L.DtypeMismatch), (Claimed((2, 1), i32), Claimed((2,), i32), L.ShapeMismatch),
    (Claimed((2,), i32), Claimed((3,), i32), L.ShapeMismatch), (Claimed((2,), i32), Claimed((2,), L.int64), L.DtypeMismatch), ([1], [2], L.ShapeMismatch)])
def test_copy_refuses(src, dst, error):
    with pytest.raises(error, match="kv_cache_copy"):
        Q.kv_cache_copy(BareCache(), src, dst)


@pytest.mark.parametrize("table,keep,starts,error", [
    (Claimed((2,), i32), Claimed((5,), i32), Claimed((3,), i32), L.ShapeMismatch), (Claimed((2, 4), f32), Claimed((5,), i32), Claimed((3,), i32), L.DtypeMismatch),
    (Claimed((2, 4), i32), Claimed((5, 1), i32), Claimed((3,), i32), L.ShapeMismatch), (Claimed((2, 4), i32), Claimed((5,), L.int64), Claimed((3,), i32), L.DtypeMismatch),
    (Claimed((2, 4), i32), Claimed((5,), i32), Claimed((2,), i32), L.ShapeMismatch), (Claimed((2, 4), i32), Claimed((5,), i32), HOST, L.DeviceMismatch)])
def test_compact_refuses(table, keep, starts, error):
    with pytest.raises(error, match="kv_cache_compact"):
        Q.kv_cache_compact(BareCache(), table, keep, starts)


def test_what_is_no_cache():
    for call in (lambda: Q.kv_cache_copy(None, None, None), lambda: Q.kv_cache_compact("cache", None, None, None)):
        with pytest.raises(TypeError, match="PagedKVCache"):
            call()


# ---------------------------------------------------------------- residual norm
def norm_args(**kw):
    d = dict(x=P, r=P, gate=None, scale=None, weight=None, bias=None, post_weight=None, post_bias=None, y=P, r_out=P, rows=2, gate_rows=0, cols=8,
             x_dtype=_C.F32, r_dtype=_C.F32, layer=0, post=0, eps=1e-6)
    assert set(kw) <= set(d)
    return C.byref(_C.ResidualNormArgs(*{**d, **kw}.values()))


@pytest.mark.parametrize("kw,error", [
    (dict(x=None), ValueError), (dict(y=None), ValueError), (dict(rows=-1), L.ShapeMismatch), (dict(cols=-1), L.ShapeMismatch), (dict(cols=32769), NotImplementedError),
    (dict(rows=1 << 31), L.ShapeMismatch), (dict(layer=2), ValueError), (dict(x_dtype=_C.BF16), L.DtypeMismatch), (dict(r_dtype=_C.F16), L.DtypeMismatch),
    (dict(gate=P), ValueError), (dict(gate_rows=1), ValueError), (dict(gate=P, gate_rows=-1), ValueError), (dict(gate=P, gate_rows=3), L.ShapeMismatch)])
def test_c_residual_norm_refuses(kw, error):
    with pytest.raises(error, match="residual_norm"):
        _C.call("lq_residual_norm", norm_args(**kw), None)


@pytest.mark.parametrize("kw", [
    dict(y=0x1004), dict(y=0x1000, r_out=0x1000), dict(y=0x101c, r_out=0x3000), dict(y=0x4000, r_out=0x2020), dict(y=0x4000, r_out=0x403f), dict(y=0x3000, r_out=0x3000),
    dict(y=0x1000, r_out=0x2000, x_dtype=_C.F16, r=0x1000), dict(y=0x4000, r_out=0x1000, x_dtype=_C.F16), dict(y=0x5010, r_out=0x2000, gate=0x5000, gate_rows=2),
    dict(y=0x5000, r_out=0x2000, gate=0x5000, gate_rows=1)])
def test_c_residual_norm_refuses_results_on_what_is_read(kw):
    with pytest.raises(ValueError, match="residual_norm: a result lies"):
        _C.call("lq_residual_norm", norm_args(**{"x": 0x1000, "r": 0x2000, "r_out": 0x2000, **kw}), None)


def test_c_entries_refuse_no_arguments():
    with pytest.raises(ValueError, match="residual_norm"):
        _C.call("lq_residual_norm", None, None)
    with pytest.raises(ValueError, match="quantized_gated_matmul"):
        _C.call("lq_wq_gated_matmul", None, None)


def test_no_rows_are_no_call():
    _C.call("lq_residual_norm", norm_args(rows=0, x=None, y=None), None)
    _C.call("lq_residual_norm", norm_args(cols=0, x=None, y=None), None)


X = Claimed((3, 8))


@pytest.mark.parametrize("args,kw,error", [
    ((HOST, HOST), {}, L.DeviceMismatch), ((X, HOST), {}, L.DeviceMismatch), ((X, None), {}, L.ShapeMismatch), ((Claimed((3, 8), i8), X), {}, L.DtypeMismatch),
    ((X, Claimed((3, 9))), {}, L.ShapeMismatch), ((X, Claimed((3, 8), f16)), {}, L.DtypeMismatch), ((X, X), dict(norm="batch"), ValueError),
    ((X, X), dict(weight=Claimed((9,))), L.ShapeMismatch), ((X, X), dict(weight=Claimed((8,), f16)), L.DtypeMismatch), ((X, X), dict(weight=HOST), L.DeviceMismatch),
    ((X, X), dict(bias=Claimed((8, 1))), L.ShapeMismatch), ((X, X), dict(scale=Claimed((1,))), L.ShapeMismatch), ((X, X), dict(post_weight=Claimed((8,))), ValueError),
    ((X, X), dict(post=True, post_bias=Claimed((7,))), L.ShapeMismatch), ((X, X), dict(gate=Claimed((2, 8))), L.ShapeMismatch),
    ((X, X), dict(gate=Claimed((0, 8))), L.ShapeMismatch), ((X, X), dict(gate=Claimed((3, 4))), L.ShapeMismatch), ((X, X), dict(gate=Claimed((3, 8), f16)), L.DtypeMismatch),
    ((X, X), dict(out=Claimed((8, 3))), L.ShapeMismatch), ((X, X), dict(out=Claimed((3, 8), f16)), L.DtypeMismatch),
    ((X, X), dict(out=Claimed((3, 8), ptr=64), residual_out=Claimed((3, 8), f16)), L.DtypeMismatch),
    ((X, X), dict(out=Claimed((3, 8), ptr=64), residual_out=Claimed((3, 8), ptr=64)), ValueError)])
def test_residual_norm_refuses(args, kw, error):
    with pytest.raises(error, match="residual_norm"):
        F.residual_norm(*args, **kw)


def test_rms_norm_refuses():
    for args, error in (((HOST, 2), L.DeviceMismatch), ((X, 9), L.ShapeMismatch), ((X, 8, Claimed((9,))), L.ShapeMismatch), ((Claimed((2, 8), i32), 8), L.DtypeMismatch)):
        with pytest.raises(error, match="rms_norm"):
            F.rms_norm(*args)


# ---------------------------------------------------------------- drafts
@pytest.mark.parametrize("at,value,error", [
    (0, None, ValueError), (2, _C.BF16, L.DtypeMismatch), (3, -1, L.ShapeMismatch), (4, 0, L.ShapeMismatch), (4, (1 << 24) + 1, L.ShapeMismatch), (5, None, ValueError),
    (6, None, ValueError), (7, -1, L.ShapeMismatch), (7, 65536, L.ShapeMismatch), (8, None, ValueError), (9, None, ValueError), (10, None, ValueError),
    (11, None, ValueError), (10, 3 * P, ValueError)])
def test_c_verify_refuses(at, value, error):
    args = [P, P, _C.F32, 4, 100, 3 * P, P, 2, P, P, 5 * P, P, None]
    args[at] = value
    with pytest.raises(error, match="verify_drafts"):
        _C.call("lq_verify_drafts", *args)


def drafts(**kw):
    d = dict(target=Claimed((4, 100)), tokens=Claimed((4,), i32), starts=Claimed((3,), i32), uniforms=Claimed((4,)), last_uniforms=Claimed((2,)), draft=None, out=None)
    return {**d, **kw}


@pytest.mark.parametrize("kw,error", [
    (dict(target=HOST), L.ShapeMismatch), (dict(target=Claimed((4, 100), i8)), L.DtypeMismatch), (dict(tokens=Claimed((5,), i32)), L.ShapeMismatch),
    (dict(tokens=Claimed((4,), L.int64)), L.DtypeMismatch), (dict(starts=Claimed((0,), i32)), L.ShapeMismatch), (dict(starts=Claimed((3,))), L.DtypeMismatch),
    (dict(uniforms=Claimed((3,))), L.ShapeMismatch), (dict(uniforms=Claimed((4,), f16)), L.DtypeMismatch), (dict(last_uniforms=Claimed((3,))), L.ShapeMismatch),
    (dict(draft=Claimed((4, 99))), L.ShapeMismatch), (dict(draft=Claimed((4, 100), f16)), L.DtypeMismatch), (dict(draft=HOST), L.DeviceMismatch),
    (dict(out=(Claimed((3,), i32), Claimed((2,), i32))), L.ShapeMismatch), (dict(out=(Claimed((4,), i32), Claimed((2,)))), L.DtypeMismatch)])
def test_verify_refuses(kw, error):
    with pytest.raises(error, match="verify_drafts"):
        F.verify_drafts(**drafts(**kw))


# ---------------------------------------------------------------- gated projections
def gated_args(**kw):
    two = lambda v: (C.c_void_p * 2)(*v)
    d = dict(x=P, out=2 * P, packed=(P, P), scales=(P, P), biases=(P, P), bias=(None, None), M=2, N=8, K=64, group_size=32, bits=4, act=0, dtype=_C.F32)
    assert set(kw) <= set(d)
    return C.byref(_C.WqGatedArgs(*(two(v) if isinstance(v, tuple) else v for v in {**d, **kw}.values())))


@pytest.mark.parametrize("kw,error", [
    (dict(x=None), ValueError), (dict(out=None), ValueError), (dict(out=P), ValueError), (dict(out=P + 2 * 64 * 4 - 16), ValueError), (dict(out=P - 2 * 8 * 4 + 16), ValueError), (dict(x=P + 4), ValueError), (dict(packed=(P, None)), ValueError), (dict(packed=(P + 8, P)), ValueError),
    (dict(scales=(None, P)), ValueError), (dict(scales=(P, P + 2)), ValueError), (dict(biases=(P, None)), ValueError), (dict(M=-1), L.ShapeMismatch), (dict(N=-1), L.ShapeMismatch), (dict(K=0), L.ShapeMismatch),
    (dict(K=96, group_size=64), L.ShapeMismatch), (dict(K=1 << 30), L.ShapeMismatch), (dict(group_size=16), ValueError), (dict(bits=2), ValueError), (dict(act=4), ValueError),
    (dict(act=-1), ValueError), (dict(dtype=_C.BF16), L.DtypeMismatch)])
def test_c_gated_refuses(kw, error):
    with pytest.raises(error, match="quantized_gated_matmul"):
        _C.call("lq_wq_gated_matmul", gated_args(**kw), None)


def weight(n=8, k=64, gs=32, bits=4):
    return Claimed((n, k * bits // 32), i32), Claimed((n, k // gs)), Claimed((n, k // gs))


def gated(**kw):
    d = dict(x=Claimed((2, 64)), gate=weight(), up=weight(), activation="silu", group_size=32, bits=4)
    return {**d, **kw}


@pytest.mark.parametrize("kw,error", [
    (dict(x=HOST), L.DeviceMismatch), (dict(x=Claimed((2, 64), i8)), L.DtypeMismatch), (dict(x=Claimed((2, 96))), L.ShapeMismatch), (dict(x=Claimed((), f32)), L.ShapeMismatch),
    (dict(activation="swish"), ValueError), (dict(bits=3), ValueError), (dict(group_size=48), ValueError), (dict(up=weight(9)), L.ShapeMismatch),
    (dict(up=weight(8, 96)), L.ShapeMismatch), (dict(gate=weight(8, 64, 64)), L.ShapeMismatch), (dict(gate=(weight()[0], HOST, HOST)), L.DeviceMismatch),
    (dict(gate=(Claimed((8, 8), f32), *weight()[1:])), L.DtypeMismatch), (dict(up=(weight()[0], Claimed((8, 2), f16), weight()[2])), L.DtypeMismatch),
    (dict(gate=(Claimed((64,), i32), *weight()[1:])), L.ShapeMismatch), (dict(gate_bias=Claimed((9,))), L.ShapeMismatch), (dict(up_bias=Claimed((8,), f16)), L.DtypeMismatch),
    (dict(up_bias=HOST), L.DeviceMismatch), (dict(out=Claimed((2, 9))), L.ShapeMismatch), (dict(out=Claimed((2, 8), f16)), L.DtypeMismatch)])
def test_gated_refuses(kw, error):
    with pytest.raises(error):
        _qgemm.quantized_gated_matmul(**gated(**kw))


def test_gated_module_refuses():
    import lucid_amd.nn as nn
    for args, kw in (((64, 8), dict(bits=3)), ((65, 8), {}), ((64, 8), dict(activation="tanh"))):
        with pytest.raises(ValueError):
            nnq.QuantizedGatedLinearMLX(*args, **kw)
    with pytest.raises(L.ShapeMismatch):
        nnq.QuantizedGatedLinearMLX.from_float(nn.Linear(64, 8), nn.Linear(64, 9))


def test_arguments_as_bytes_are_the_structs():
    """What the wrappers pack lies where the header's structs have it."""
    for cls, packer in ((_C.ResidualNormArgs, _C.RESIDUAL_NORM_ARGS), (_C.WqGatedArgs, _C.WQ_GATED_ARGS)):
        n = len(packer.unpack(bytes(packer.size)))
        values = [i + 1 for i in range(n)]
        got, flat = cls.from_buffer_copy(packer.pack(*values)), []
        for field, _ in cls._fields_:
            v = getattr(got, field)
            flat += list(v) if isinstance(v, C.Array) else [v]
        assert C.sizeof(cls) == packer.size and flat == values
