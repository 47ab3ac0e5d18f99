"""The quantized key / value cache of a decoder: pages of codes that new tokens are quantized into and that
``nn.functional.paged_attention`` reads.  No counterpart in Lucid; a row (a token's key or value of one head) is
quantized as ``quantize_rows_dynamic`` quantizes it.
"""

from __future__ import annotations

import ctypes as C

from .. import _C
from .. import _tensor as T
from .._tensor import Tensor
from ._qscheme import QDtype, QScheme, per_channel_symmetric, qint4, qint8

_FLOATS = (T.float32, T.float16)


class PagedKVCache:
    """Device buffers of ``num_pages`` pages of ``page_size`` tokens with ``kv_heads`` heads of ``head_dim``.

    Slot ``s`` is place ``s % page_size`` of page ``s // page_size``; which pages a sequence has is the program's to say
    (``page_table`` of ``paged_attention``).  Every row has a scale of its own, and a zero point where ``qscheme`` is
    ``per_channel_affine``; ``qdtype`` is ``qint8`` or ``qint4``.  ``page_size`` is a multiple of 16, ``head_dim`` one of 16
    (``qint4``: 32), at most 256.

    ``k_codes`` / ``v_codes`` are bytes (int8-tagged) ``(num_pages, kv_heads, page_size, head_dim * bits // 8)`` that hold
    code - quant_min, two 4-bit codes in a byte, the first in the low half; ``k_scale``, ``v_scale``, ``k_zero``, ``v_zero`` are
    float32 ``(num_pages, kv_heads, page_size)``, the last two ``None`` for a symmetric cache.  A row stands for
    ``(code - zero) * scale``.  All buffers begin as zeros: a slot that was never written stands for zeros.  They belong to
    the cache: their contents may be written, the attributes are read-only."""

    __slots__ = ("num_pages", "page_size", "kv_heads", "head_dim", "qscheme", "qdtype", "k_codes", "v_codes", "k_scale", "v_scale",
                 "k_zero", "v_zero", "_struct", "_ref")

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, qscheme: QScheme = per_channel_symmetric,
                 qdtype: QDtype = qint8) -> None:
        if qdtype is not qint8 and qdtype is not qint4:
            raise NotImplementedError(f"PagedKVCache: qint8 and qint4 are built, got {qdtype!r}")
        if not isinstance(qscheme, QScheme) or not qscheme.is_per_channel:
            raise ValueError(f"PagedKVCache: every row has its own scale; qscheme is per_channel_symmetric or per_channel_affine, got {qscheme}")
        keep = lambda **kw: [object.__setattr__(self, n, v) for n, v in kw.items()]
        keep(num_pages=int(num_pages), page_size=int(page_size), kv_heads=int(kv_heads), head_dim=int(head_dim), qscheme=qscheme, qdtype=qdtype)
        step = 128 // qdtype.bits
        if self.num_pages < 1 or not 1 <= self.kv_heads <= 65535 or self.page_size < 16 or self.page_size % 16:
            raise _C.ShapeMismatch(f"PagedKVCache: {num_pages} pages of {page_size} tokens with {kv_heads} heads (pages are multiples of 16)")
        if self.num_pages * self.page_size > 0x7fffffff:
            raise _C.ShapeMismatch(f"PagedKVCache: {num_pages} pages of {page_size} tokens are more than 2^31 - 1 slots")
        if self.head_dim < step or self.head_dim > 256 or self.head_dim % step:
            raise NotImplementedError(f"PagedKVCache: head_dim {head_dim}; {qdtype.name} takes multiples of {step} up to 256")
        rows = (self.num_pages, self.kv_heads, self.page_size)

        def zeros(shape, dt):
            t = Tensor.empty(shape, dt, "hip")
            _C.call("lq_fill_bytes", t.data_ptr, 0, t.nbytes, None)
            return t

        codes = [zeros((*rows, self.head_dim * qdtype.bits // 8), T.int8) for _ in range(2)]
        scales = [zeros(rows, T.float32) for _ in range(2)]
        zero_points = [None, None] if qscheme.is_symmetric else [zeros(rows, T.float32) for _ in range(2)]
        pointers = [t.data_ptr if t is not None else None for t in codes + scales + zero_points]
        struct = _C.KvCache(*pointers, self.num_pages, self.page_size, self.kv_heads, self.head_dim, qdtype.bits)
        keep(k_codes=codes[0], v_codes=codes[1], k_scale=scales[0], v_scale=scales[1], k_zero=zero_points[0], v_zero=zero_points[1], _struct=struct,
             _ref=C.byref(struct))

    # The calls go by the addresses and sizes in _struct, for as long as the cache lives.
    def __setattr__(self, name, value):
        raise AttributeError(f"PagedKVCache: {name} is read-only (write into the buffers, or make another cache)")

    def __delattr__(self, name):
        raise AttributeError(f"PagedKVCache: {name} is read-only")

    @property
    def num_slots(self) -> int:
        return self.num_pages * self.page_size

    @property
    def nbytes(self) -> int:
        buffers = (self.k_codes, self.v_codes, self.k_scale, self.v_scale, self.k_zero, self.v_zero)
        return sum(t.nbytes for t in buffers if t is not None)

    def __repr__(self) -> str:
        return (f"PagedKVCache({self.num_pages}, {self.page_size}, kv_heads={self.kv_heads}, head_dim={self.head_dim}, "
                f"{self.qscheme.value}, {self.qdtype.name})")

    def _no_copy(self, *_):
        raise TypeError("PagedKVCache: the buffers belong to one cache (copy the tensors)")

    __copy__ = __deepcopy__ = __reduce__ = _no_copy


def _check_cache(name: str, cache) -> None:
    if not isinstance(cache, PagedKVCache):
        raise TypeError(f"{name} expects a PagedKVCache, got {type(cache).__name__}")


# (what a call checks of its tensors is a good part of what a small call takes: the usual case in one line)
def _check_ids(name: str, what: str, t, shape) -> None:
    if t.__class__ is Tensor and t.device == "hip" and t.dtype is T.int32 and t.shape == shape:
        return
    if not isinstance(t, Tensor) or t.device != "hip":
        raise _C.DeviceMismatch(f"{name}: {what} must be a tensor on the 'hip' device")
    if t.dtype != T.int32:
        raise _C.DtypeMismatch(f"{name}: {what} is int32, got {t.dtype}")
    if t.shape != shape:
        raise _C.ShapeMismatch(f"{name}: {what} has shape {t.shape}, expected {shape}")


def _check_rows(name: str, what: str, t, shape) -> None:
    if t.__class__ is Tensor and t.device == "hip" and (t.dtype is T.float16 or t.dtype is T.float32) and t.shape == shape:
        return
    if not isinstance(t, Tensor) or t.device != "hip":
        raise _C.DeviceMismatch(f"{name}: {what} must be a tensor on the 'hip' device")
    if t.dtype not in _FLOATS:
        raise _C.DtypeMismatch(f"{name}: {what} is float32 or float16, got {t.dtype}")
    if t.shape != shape:
        raise _C.ShapeMismatch(f"{name}: {what} has shape {t.shape}, expected {shape}")


def _written(t: Tensor) -> None:
    """A call has written `t`: what told of the values before (codes on a grid, a kept range) goes."""
    t._grid = t._range = None


def kv_cache_write(cache: PagedKVCache, k: Tensor, v: Tensor, slots: Tensor) -> None:
    """Quantizes keys and values ``(tokens, kv_heads, head_dim)`` (float32 or float16) into the slots ``slots`` (int32
    ``(tokens,)``).  A slot that is negative or beyond the cache is skipped: what pads a batch.  The others are distinct; of
    tokens that share a slot, codes and scale may come from different ones."""
    _check_cache("kv_cache_write", cache)
    if not isinstance(k, Tensor) or k.ndim != 3:
        raise _C.ShapeMismatch("kv_cache_write: k is a (tokens, kv_heads, head_dim) tensor")
    shape = (k.shape[0], cache.kv_heads, cache.head_dim)
    _check_rows("kv_cache_write", "k", k, shape)
    _check_rows("kv_cache_write", "v", v, shape)
    if v.dtype != k.dtype:
        raise _C.DtypeMismatch(f"kv_cache_write: k is {k.dtype}, v {v.dtype}")
    _check_ids("kv_cache_write", "slots", slots, shape[:1])
    width = cache.kv_heads * cache.head_dim
    _C.call("lq_kv_cache_write", cache._ref, k.data_ptr, v.data_ptr, k.dtype.code, width, width, slots.data_ptr, shape[0], None)


def kv_cache_write_qkv(cache: PagedKVCache, qkv: Tensor, num_heads: int, slots: Tensor) -> None:
    """``kv_cache_write`` of the keys and values in the packed output of a qkv Linear: ``qkv`` is
    ``(..., (num_heads + 2 * kv_heads) * head_dim)``, queries first, then keys, then values; ``slots`` has an entry per row."""
    _check_cache("kv_cache_write_qkv", cache)
    num_heads = int(num_heads)
    if num_heads < 0:  # (the keys would begin before the row)
        raise _C.ShapeMismatch(f"kv_cache_write_qkv: {num_heads} query heads")
    row = (num_heads + 2 * cache.kv_heads) * cache.head_dim
    if not isinstance(qkv, Tensor) or qkv.ndim < 2 or qkv.shape[-1] != row:
        raise _C.ShapeMismatch(f"kv_cache_write_qkv: qkv has rows of {num_heads} + 2 * {cache.kv_heads} heads of {cache.head_dim}, {row} values")
    _check_rows("kv_cache_write_qkv", "qkv", qkv, qkv.shape)
    tokens = qkv.numel // row
    _check_ids("kv_cache_write_qkv", "slots", slots, (tokens,))
    k = qkv.data_ptr + num_heads * cache.head_dim * qkv.dtype.itemsize
    v = k + cache.kv_heads * cache.head_dim * qkv.dtype.itemsize
    _C.call("lq_kv_cache_write", cache._ref, k, v, qkv.dtype.code, row, row, slots.data_ptr, tokens, None)


def kv_cache_read(cache: PagedKVCache, slots: Tensor, dtype=T.float32, out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
    """``(k, v)``, each ``(tokens, kv_heads, head_dim)``: the values that the rows at ``slots`` (int32 ``(tokens,)``) stand for, zeros
    where a slot is negative or beyond the cache.  ``dtype`` is float32 or float16; ``out`` takes the results (and says the type)."""
    _check_cache("kv_cache_read", cache)
    if not isinstance(slots, Tensor) or slots.ndim != 1:
        raise _C.ShapeMismatch("kv_cache_read: slots is a (tokens,) tensor")
    _check_ids("kv_cache_read", "slots", slots, slots.shape)
    shape = (slots.shape[0], cache.kv_heads, cache.head_dim)
    if out is None:
        dt = T.as_dtype(dtype)
        if dt not in _FLOATS:
            raise _C.DtypeMismatch(f"kv_cache_read: float32 or float16, got {dt}")
        k, v = Tensor.empty(shape, dt, "hip"), Tensor.empty(shape, dt, "hip")
    else:
        k, v = out
        _check_rows("kv_cache_read", "out[0]", k, shape)
        _check_rows("kv_cache_read", "out[1]", v, shape)
        if v.dtype != k.dtype:
            raise _C.DtypeMismatch(f"kv_cache_read: out is {k.dtype} and {v.dtype}")
    _C.call("lq_kv_cache_read", cache._ref, slots.data_ptr, shape[0], k.data_ptr, v.data_ptr, k.dtype.code, None)
    _written(k), _written(v)
    return k, v


def kv_cache_copy(cache: PagedKVCache, src: Tensor, dst: Tensor) -> None:
    """Copies page ``src[i]`` into page ``dst[i]`` (int32 ``(pages,)``), keys, values and their scales and zero points: what forks a
    sequence, whose whole pages both then share and whose last one each has for itself.  A pair with a page that is negative or
    beyond the cache is skipped: what pads a list.  A page may be copied several times; the destinations are distinct, and none is
    another pair's source."""
    _check_cache("kv_cache_copy", cache)
    if not isinstance(src, Tensor) or src.ndim != 1:
        raise _C.ShapeMismatch("kv_cache_copy: src is a (pages,) tensor")
    _check_ids("kv_cache_copy", "src", src, src.shape)
    _check_ids("kv_cache_copy", "dst", dst, src.shape)
    _C.call("lq_kv_cache_copy", cache._ref, src.data_ptr, dst.data_ptr, src.shape[0], None)


def kv_cache_compact(cache: PagedKVCache, page_table: Tensor, keep: Tensor, starts: Tensor) -> None:
    """Moves the tokens that sequences keep to their beginnings, so that the pages behind them are free.

    Sequence ``b`` keeps the places ``keep[starts[b]:starts[b + 1]]`` (int32 ``(kept,)``, from 0 and rising within a sequence; ``starts`` int32
    ``(batch + 1,)``, rising from 0 to ``kept``) of its pages ``page_table[b]`` (int32 ``(batch, pages)``); the ``i``-th of them becomes
    its token ``i``, and its length the number of them (``kv_lens`` of ``paged_attention``).  What lies behind stays as it was.  A token
    whose old or new place is beyond ``page_table``, or on a page that is negative or beyond the cache, is not moved; one that stays
    in its place is neither read nor written, so sequences may share pages of such tokens.  Other pages belong to one sequence."""
    _check_cache("kv_cache_compact", cache)
    if not isinstance(page_table, Tensor) or page_table.ndim != 2:
        raise _C.ShapeMismatch("kv_cache_compact: page_table is a (batch, pages) tensor")
    _check_ids("kv_cache_compact", "page_table", page_table, page_table.shape)
    if not isinstance(keep, Tensor) or keep.ndim != 1:
        raise _C.ShapeMismatch("kv_cache_compact: keep is a (kept,) tensor")
    _check_ids("kv_cache_compact", "keep", keep, keep.shape)
    batch, width = page_table.shape
    _check_ids("kv_cache_compact", "starts", starts, (batch + 1,))
    if max(batch, width) > 0x7fffffff:  # (ctypes takes the low 32 bits of a longer int)
        raise _C.ShapeMismatch(f"kv_cache_compact: {batch} sequences of {width} pages")
    _C.call("lq_kv_cache_compact", cache._ref, page_table.data_ptr, width, batch, keep.data_ptr, keep.shape[0], starts.data_ptr, None)
