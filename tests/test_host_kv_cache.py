"""What the key / value cache and its attention refuse, without a device: Python's checks, and those of the C entry points (the
pointers given are never followed)."""

import ctypes as C

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn.functional as F
import lucid_amd.quantization as Q
from lucid_amd import _C

P = 4096  # an aligned address that nothing reads


def struct(**kw):
    d = dict(k_codes=P, v_codes=P, k_scale=P, v_scale=P, k_zero=None, v_zero=None, num_pages=4, page_size=16, kv_heads=2, head_dim=64, bits=8)
    d.update(kw)
    return _C.KvCache(*d.values())


@pytest.mark.parametrize("kw,error", [
    (dict(num_pages=0), L.ShapeMismatch), (dict(kv_heads=0), L.ShapeMismatch), (dict(page_size=0), L.ShapeMismatch),
    (dict(page_size=24), L.ShapeMismatch), (dict(num_pages=1 << 27, page_size=16), L.ShapeMismatch), (dict(head_dim=8), NotImplementedError),
    (dict(head_dim=272), NotImplementedError), (dict(head_dim=72), NotImplementedError), (dict(head_dim=48, bits=4), NotImplementedError),
    (dict(bits=2), NotImplementedError), (dict(k_codes=None), ValueError), (dict(v_scale=None), ValueError), (dict(k_zero=P), ValueError),
    (dict(v_codes=P + 8), ValueError), (dict(k_zero=P, v_zero=P + 4), ValueError)])
def test_c_entries_refuse_a_bad_cache(kw, error):
    c = C.byref(struct(**kw))
    with pytest.raises(error):
        _C.call("lq_kv_cache_write", c, P, P, _C.F32, 128, 128, P, 1, None)
    with pytest.raises(error):
        _C.call("lq_kv_cache_read", c, P, 1, P, P, _C.F32, None)
    with pytest.raises(error):
        _C.call("lq_paged_attention", c, P, 128, P, _C.F32, 1, 2, 1, P, 1, P, P, 1.0, 1, 0, 0, None)


@pytest.mark.parametrize("at,value,error", [
    (1, None, ValueError), (1, P + 4, ValueError), (2, None, ValueError), (3, _C.I8, L.DtypeMismatch), (3, _C.BF16, L.DtypeMismatch),
    (4, 124, L.ShapeMismatch), (4, 130, ValueError), (5, 64, L.ShapeMismatch), (6, None, ValueError), (7, 1 << 40, L.ShapeMismatch),
    (7, 1 << 25, L.ShapeMismatch)])
def test_c_write_refuses(at, value, error):
    args = [C.byref(struct()), P, P, _C.F32, 128, 128, P, 1, None]
    args[at] = value
    with pytest.raises(error, match="kv_cache_write"):
        _C.call("lq_kv_cache_write", *args)


@pytest.mark.parametrize("at,value,error", [
    (1, None, ValueError), (2, 1 << 40, L.ShapeMismatch), (2, 1 << 25, L.ShapeMismatch), (3, None, ValueError), (4, P + 8, ValueError), (5, _C.F64, L.DtypeMismatch)])
def test_c_read_refuses(at, value, error):
    args = [C.byref(struct()), P, 1, P, P, _C.F16, None]
    args[at] = value
    with pytest.raises(error, match="kv_cache_read"):
        _C.call("lq_kv_cache_read", *args)


@pytest.mark.parametrize("at,value,error", [
    (1, None, ValueError), (1, P + 8, ValueError), (2, 192, L.ShapeMismatch), (2, 258, ValueError), (3, None, ValueError),
    (4, _C.I32, L.DtypeMismatch), (5, -1, ValueError), (5, 1 << 24, L.ShapeMismatch), (6, 3, L.ShapeMismatch), (6, 0, L.ShapeMismatch),
    (7, -1, ValueError), (8, None, ValueError), (9, -1, ValueError), (9, 1 << 27, L.ShapeMismatch), (10, None, ValueError),
    (11, None, ValueError), (14, -1, ValueError), (15, -2, ValueError)])
def test_c_attention_refuses(at, value, error):
    args = [C.byref(struct()), P, 256, P, _C.F32, 1, 4, 1, P, 1, P, P, 1.0, 1, 0, 0, None]
    args[at] = value
    with pytest.raises(error, match="paged_attention"):
        _C.call("lq_paged_attention", *args)


def test_c_entries_without_tokens_do_nothing():
    c = C.byref(struct())
    _C.call("lq_kv_cache_write", c, None, None, _C.F32, 0, 0, None, 0, None)
    _C.call("lq_kv_cache_read", c, None, 0, None, None, _C.F32, None)
    _C.call("lq_paged_attention", c, None, 0, None, _C.F32, 0, 4, 1, P, 1, P, P, 1.0, 1, 0, 0, None)


@pytest.mark.parametrize("args,error", [
    ((0, 16, 2, 64), L.ShapeMismatch), ((4, 8, 2, 64), L.ShapeMismatch), ((4, 40, 2, 64), L.ShapeMismatch), ((4, 16, 0, 64), L.ShapeMismatch),
    ((1 << 27, 16, 1, 16), L.ShapeMismatch), ((4, 16, 2, 20), NotImplementedError), ((4, 16, 2, 512), NotImplementedError),
    ((4, 16, 2, 48, Q.per_channel_affine, Q.qint4), NotImplementedError), ((4, 16, 2, 64, Q.per_tensor_affine), ValueError),
    ((4, 16, 2, 64, Q.per_channel_affine, Q.quint8), NotImplementedError), ((4, 16, 2, 64, "per_channel_affine"), ValueError)])
def test_a_cache_refuses_what_no_kernel_takes(args, error):
    with pytest.raises(error, match="PagedKVCache"):
        Q.PagedKVCache(*args)


def test_operators_want_a_cache():
    x = L.tensor(np.zeros((1, 2, 64), np.float32))
    for f in (lambda: Q.kv_cache_write(None, x, x, x), lambda: Q.kv_cache_write_qkv(x, x, 2, x), lambda: Q.kv_cache_read({}, x),
              lambda: F.paged_attention(x, None, x, x, x), lambda: F.paged_attention_qkv(x, 2, "cache", x, x, x)):
        with pytest.raises(TypeError, match="PagedKVCache"):
            f()


def bare_cache(kv_heads=2, head_dim=64):
    """A cache whose buffers do not exist: for checks that come before anything is read."""
    c = object.__new__(Q.PagedKVCache)
    s = struct(kv_heads=kv_heads, head_dim=head_dim)
    values = dict(num_pages=4, page_size=16, kv_heads=kv_heads, head_dim=head_dim, qscheme=Q.per_channel_symmetric, qdtype=Q.qint8, _struct=s, _ref=C.byref(s))
    for n, v in values.items():
        object.__setattr__(c, n, v)
    return c


@pytest.mark.parametrize("num_heads,width", [(-1, 3 * 64), (-3, 64), (-4, 0), (-(1 << 40), 64)])
def test_packed_rows_of_fewer_than_no_queries_are_refused(num_heads, width):
    """Keys of (num_heads + 2 kv_heads) heads a row lie num_heads heads from its start: with num_heads = -1, before the buffer."""
    x, s = L.tensor(np.zeros((2, width), np.float32)), L.tensor(np.zeros(2, np.int32))
    with pytest.raises(L.ShapeMismatch, match="kv_cache_write_qkv.*query heads"):
        Q.kv_cache_write_qkv(bare_cache(), x, num_heads, s)
    with pytest.raises(L.ShapeMismatch, match="paged_attention_qkv.*query heads"):
        F.paged_attention_qkv(x, num_heads, bare_cache(), s, s, s)


def test_packed_attention_without_queries_is_refused_before_it_asks_for_memory():
    x, s = L.tensor(np.zeros((2, 256), np.float32)), L.tensor(np.zeros(2, np.int32))
    with pytest.raises(L.ShapeMismatch, match="paged_attention_qkv.*query heads"):
        F.paged_attention_qkv(x, 0, bare_cache(), s, s, s)


@pytest.mark.parametrize("name", ["num_pages", "page_size", "kv_heads", "head_dim", "qscheme", "qdtype", "k_codes", "v_scale", "k_zero", "_struct"])
def test_a_cache_keeps_the_buffers_that_its_calls_write_to(name):
    """The calls go by the addresses and sizes of the construction: another buffer in a buffer's place would free memory that they still write to."""
    c = bare_cache()
    with pytest.raises(AttributeError, match=name):
        setattr(c, name, None)
    with pytest.raises(AttributeError, match=name):
        delattr(c, name)
    assert c.num_slots == 64 and c.kv_heads == 2
