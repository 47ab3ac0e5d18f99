"""Attention over the pages of a quantized key / value cache against float64."""

import ctypes as C

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn.functional as F
import lucid_amd.quantization as Q
import oracle.kv_cache as K
from lucid_amd import _C
from test_hip_kv_cache import DTYPES, SCHEMES, hip, ids

pytestmark = pytest.mark.gpu


class Batch:
    """Sequences of `chunks` new tokens and `lengths` tokens in all, in pages that lie anywhere, a few of them nobody's."""

    def __init__(self, chunks, lengths, heads, kv_heads, dim, page=16, bits=8, symmetric=True, dtype=np.float16, seed=0, tail=0, wide=0,
                 gain=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.dim, self.bits, self.symmetric, self.dtype = heads, kv_heads, dim, bits, symmetric, dtype
        used = [-(-n // page) for n in lengths]
        pages = sum(used) + 3
        self.table = np.full((len(chunks), max(used + [0]) + wide), -1, np.int32)
        order = iter(rng.permutation(pages))
        for b, n in enumerate(used):
            self.table[b, :n] = [next(order) for _ in range(n)]
        self.q_starts, self.kv_lens = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32), np.asarray(lengths, np.int32)
        self.cache = Q.PagedKVCache(pages, page, kv_heads, dim, SCHEMES[symmetric], DTYPES[bits])
        self.pages = {}
        for name in "kv":
            x = (rng.standard_normal((pages, kv_heads, page, dim)) * gain).astype(np.float32) * (1 + 3 * (rng.random((kv_heads, 1, dim)) < 0.06))
            self.put(name, *K.quantize(x.astype(np.float32), bits, symmetric))
        self.q = (1.5 * rng.standard_normal((sum(chunks) + tail, heads, dim))).astype(dtype)

    def put(self, name, u, scale, zero):
        getattr(self.cache, name + "_codes").copy_from(K.pack(u, self.bits).view(np.int8))
        getattr(self.cache, name + "_scale").copy_from(scale)
        if not self.symmetric:
            getattr(self.cache, name + "_zero").copy_from(zero)
        self.pages[name] = K.values(K.pack(u, self.bits), scale, zero, self.bits)

    def run(self, **kw):
        return F.paged_attention(hip(self.q), self.cache, ids(self.table), ids(self.q_starts), ids(self.kv_lens), **kw).numpy()

    def want(self, scale=None, causal=True, window=None):
        scale = 1 / np.sqrt(self.dim) if scale is None else scale
        return K.attention(self.q, self.pages["k"], self.pages["v"], self.table, self.q_starts, self.kv_lens, scale, causal, window)

    def check(self, got, scale=None, causal=True, window=None):
        want = self.want(scale, causal, window)
        scale = 1 / np.sqrt(self.dim) if scale is None else scale
        assert got.dtype == self.dtype and got.shape == want.shape and np.isfinite(got).all()
        # Rounding, in float32 unless said.  A score is a sum of dim products whose partial sums stay below a = scale sum |q k|: each
        # addition adds 2^-24 of it, which as independent errors makes sqrt(dim) 2^-24 a (4 deviations below); float32 queries are two
        # float16 of 22 bits, 2^-23 a more.  Scale and maximum round three times, the exponential twice: 8 units of 1 + |score|.  A
        # probability that is off by e moves the result by 2 e max|v| at most; sums of n terms add sqrt(n) 2^-24 max|v| (4 deviations).
        n, vmax, u = int(self.kv_lens.max(initial=0)), np.abs(self.pages["v"]).max(), 2.0 ** -24
        k = np.abs(self.pages["k"]).max((0, 2))
        group = self.heads // self.kv_heads
        a = max((np.abs(self.q[:, h].astype(np.float64)) * k[h // group]).sum(-1).max(initial=0) for h in range(self.heads)) * abs(scale)
        tol = u * vmax * (2 * (4 * np.sqrt(self.dim) * a + 2 * a + 8 * (1 + a)) + 4 * np.sqrt(n) + 8)
        if self.dtype == np.float16:  # the result, and each probability against the sum of them: half a step, 2^-11
            tol = tol + 2.0 ** -11 * (np.abs(want) + vmax) + 2.0 ** -25
        assert np.all(np.abs(got - want) <= tol), (np.abs(got - want).max(), np.max(tol))
        # and on the whole: the same errors as root mean squares.  A score's partial sums are about sqrt(scores' square mean) large
        ref = np.sqrt(np.mean(want ** 2))
        if ref:
            spread = abs(scale) * np.sqrt(np.mean(self.q.astype(np.float64) ** 2) * np.mean(self.pages["k"] ** 2) * self.dim)
            vrms = np.sqrt(np.mean(self.pages["v"] ** 2))
            rel = u * 2 * ((4 * np.sqrt(self.dim) + 10) * (1 + spread) + np.sqrt(n) + 8) * vrms / ref
            if self.dtype == np.float16:  # rounded values are off by 2^-11 / sqrt(3) of themselves at most in the mean
                rel += 2.0 ** -11 / np.sqrt(3) * (1 + vrms / ref)
            off = np.sqrt(np.mean((got - want) ** 2)) / ref
            assert off <= rel, (off, rel)
        return want


GRID = [  # chunks, lengths, heads, kv_heads, dim, page, bits, symmetric, dtype
    ([1], [1], 1, 1, 64, 16, 8, True, np.float32), ([1], [197], 12, 12, 64, 16, 8, True, np.float32),
    ([1, 1, 1], [5, 700, 33], 8, 2, 128, 16, 8, True, np.float16), ([1] * 9, [31, 32, 33, 63, 64, 65, 127, 128, 129], 4, 1, 128, 32, 4, False, np.float16),
    ([1, 1], [3000, 1111], 16, 1, 64, 48, 4, True, np.float32), ([1], [4097], 7, 1, 128, 64, 8, False, np.float16),
    ([5, 3, 8], [600, 3, 1200], 8, 2, 128, 16, 8, True, np.float32), ([2, 1, 7], [100, 1, 50], 6, 3, 80, 16, 8, False, np.float16),
    ([17, 40], [40, 300], 4, 4, 96, 16, 4, False, np.float32), ([33], [777], 5, 1, 112, 16, 8, True, np.float16),
    ([100, 1, 300], [100, 400, 500], 4, 2, 128, 16, 8, True, np.float16), ([130, 65], [1000, 65], 2, 1, 128, 64, 4, False, np.float16),
    ([200], [333], 3, 3, 64, 16, 8, False, np.float32), ([129, 2], [640, 640], 8, 1, 256, 32, 8, True, np.float16),
    ([150], [150], 2, 2, 256, 16, 4, False, np.float32), ([70, 20], [90, 2000], 2, 1, 16, 16, 8, True, np.float32),
    ([257], [600], 2, 1, 32, 128, 4, True, np.float16), ([64, 64], [300, 64], 4, 1, 160, 16, 8, False, np.float16),
    ([90], [91], 20, 1, 48, 16, 8, False, np.float32), ([1], [600], 48, 1, 64, 16, 8, True, np.float16), ([3], [513], 40, 2, 224, 16, 4, True, np.float32)]


@pytest.mark.parametrize("case", range(len(GRID)))
def test_against_float64(case):
    b = Batch(*GRID[case], seed=case)
    b.check(b.run())
    b.check(b.run(max_chunk=int(np.diff(b.q_starts).max())))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 100, 5000])
@pytest.mark.parametrize("chunks,lengths", [([1, 1], [300, 20]), ([9, 4], [500, 4]), ([150, 3], [700, 900])])
def test_windows(window, chunks, lengths, dtype):
    b = Batch(chunks, lengths, 4, 2, 64, dtype=dtype, seed=window)
    b.check(b.run(window=window), window=window)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("chunks,lengths", [([1, 1], [300, 20]), ([9, 4], [500, 2]), ([150, 3, 20], [700, 900, 6])])
def test_all_keys(chunks, lengths, dtype):
    b = Batch(chunks, lengths, 4, 2, 64, dtype=dtype, seed=4)
    b.check(b.run(causal=False), causal=False)
    b.check(b.run(causal=False, window=40, scale=-0.3), causal=False, window=40, scale=-0.3)


@pytest.mark.parametrize("chunks,lengths", [([0, 1, 0, 2], [10, 0, 0, 40]), ([3, 5], [0, 2]), ([0], [0]), ([200, 0, 90], [100, 7, 0])])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_empty_sequences_and_rows_that_see_nothing(chunks, lengths, dtype):
    b = Batch(chunks, lengths, 2, 1, 64, dtype=dtype, seed=2, tail=5, wide=2)
    want = b.check(b.run())
    assert not want[sum(chunks):].any()
    b.check(b.run(window=3), window=3)


@pytest.mark.parametrize("chunks,lengths", [([1, 1, 1], [300, 40, 20]), ([5, 100], [50, 333])])
def test_rows_of_no_sequence_are_zeros_whatever_the_memory_held(chunks, lengths):
    b = Batch(chunks, lengths, 4, 2, 128, seed=3, tail=67)
    out = hip(np.full(b.q.shape, np.nan, np.float16))
    y = F.paged_attention(hip(b.q), b.cache, ids(b.table), ids(b.q_starts), ids(b.kv_lens), out=out)
    assert y is out
    b.check(out.numpy())
    starts = b.q_starts + 3  # rows before the first sequence as well
    out.copy_from(np.full(b.q.shape, np.nan, np.float16))
    F.paged_attention(hip(b.q), b.cache, ids(b.table), ids(starts), ids(b.kv_lens), out=out)
    b.q_starts = starts
    b.check(out.numpy())
    none = F.paged_attention(hip(b.q), b.cache, L.Tensor.empty((0, 4), L.int32), ids([0]), L.Tensor.empty((0,), L.int32), out=out)
    assert not none.numpy().any()
    none = F.paged_attention(hip(b.q), b.cache, L.Tensor.empty((len(chunks), 0), L.int32), ids(b.q_starts), ids(b.kv_lens), out=out)
    assert not none.numpy().any()


@pytest.mark.parametrize("tokens,width,max_chunk", [(1, 4, None), (3, 4, 1), (3, 100, None), (60, 4, 60), (200, 100, 200), (700, 0, None)])
def test_a_batch_of_no_sequences_gives_zeros(tokens, width, max_chunk):
    b = Batch([1], [20], 4, 2, 64, seed=4)
    out = hip(np.full((tokens, 4, 64), np.nan, np.float16))
    F.paged_attention(hip(np.ones((tokens, 4, 64), np.float16)), b.cache, L.Tensor.empty((0, width), L.int32), ids([0]),
                      L.Tensor.empty((0,), L.int32), max_chunk=max_chunk, out=out)
    assert not out.numpy().any()


@pytest.mark.parametrize("chunks,lengths", [([1, 1], [500, 100]), ([6, 3], [400, 90]), ([130, 70], [600, 200])])
def test_what_nobody_sees_may_be_anything(chunks, lengths):
    """NaN scales behind the lengths, before the window and in pages of others; pages that are not there."""
    for window in (None, 64):
        b = Batch(chunks, lengths, 4, 2, 64, dtype=np.float32, symmetric=False, seed=9)
        b.table[0, 2], b.table[0, 5], b.table[1, 0] = -1, 1 << 20, -(1 << 31)
        seen = np.zeros((b.cache.num_pages, 16), bool)
        for s, (n, length) in enumerate(zip(chunks, lengths)):
            for j in range(length):
                p = b.table[s, j // 16]
                if 0 <= p < b.cache.num_pages and (window is None or j > length - n - window):
                    seen[p, j % 16] = True
        want = b.want(window=window)
        for name in ("k_scale", "v_scale", "k_zero", "v_zero"):
            t = getattr(b.cache, name)
            t.copy_from(np.where(seen[:, None], t.numpy(), np.nan))
        got = b.run(window=window)
        assert np.isfinite(got).all()
        b.pages = {n: np.where(seen[:, None, :, None], p, 0) for n, p in b.pages.items()}
        assert np.array_equal(b.want(window=window), want)
        b.check(got, window=window)


def test_nan_and_infinite_keys_and_values_show():
    b = Batch([1, 2, 100], [40, 60, 300], 2, 1, 64, dtype=np.float32, seed=5)
    k, v = b.cache.k_scale.numpy().copy(), b.cache.v_scale.numpy().copy()
    k[b.table[0, 1]], v[b.table[1, 0]] = np.nan, np.inf
    b.cache.k_scale.copy_from(k), b.cache.v_scale.copy_from(v)
    got = b.run()
    assert np.isnan(got[0]).all()
    assert not np.isfinite(got[1:3]).any()
    assert np.isfinite(got[3:]).all()
    b.q[3:] = np.nan
    assert np.isnan(b.run()[3:]).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("chunk", [1, 90])
def test_values_of_very_different_sizes(dtype, chunk):
    """Rows of the cache whose scales are 2^-40 to 2^20 of each other, and scores up to some hundreds."""
    b = Batch([chunk, chunk], [700, 350], 4, 2, 64, dtype=dtype, seed=6)
    u, scale, zero = (K.unpack(b.cache.v_codes.numpy(), 8), b.cache.v_scale.numpy(), None)
    b.put("v", u, (scale * 2.0 ** b.rng.integers(-40, 1, scale.shape)).astype(np.float32), zero)
    b.check(b.run())
    b.put("v", u, (scale * 2.0 ** np.sort(b.rng.integers(-60, -10, scale.shape), 2)).astype(np.float32), zero)
    if dtype == np.float32:
        b.check(b.run())
    b.put("v", u, scale, zero)
    b.check(b.run(scale=4.0), scale=4.0)
    b.check(b.run(scale=0.0), scale=0.0)


def test_float32_queries_of_very_different_sizes():
    b = Batch([3, 100], [400, 350], 4, 2, 64, dtype=np.float32, seed=7)
    q = b.q.copy()
    for gain in (1e-30, 1e-6, 1e4, 1e30):
        b.q = (q * np.float32(gain)).astype(np.float32)
        b.check(b.run(scale=0.125 / gain), scale=0.125 / gain)
    b.q = q * np.where(np.arange(64) % 2, np.float32(1e-5), np.float32(1))
    b.check(b.run())
    b.q = q * 0
    b.check(b.run())


def test_a_length_beyond_the_table_is_cut():
    for chunks in ([1, 2], [100, 3]):
        b = Batch(chunks, [160, 64], 2, 2, 64, seed=8)
        b.kv_lens = np.array([100_000, 2**31 - 1], np.int32)
        b.check(b.run())
        b.kv_lens = np.array([-5, 64], np.int32)
        b.check(b.run())


LONG = [  # one long sequence before many keys, as blocks of twice as many rows; equal lengths; more sequences than lanes
    ([300], [1300], 4, 1, 128, 64, 8, True, np.float16), ([260], [1100], 8, 2, 96, 16, 4, False, np.float32),
    ([512], [2100], 2, 1, 128, 32, 4, True, np.float16), ([300], [2000], 4, 1, 80, 48, 8, False, np.float32),
    ([130] * 5, [900] * 5, 2, 1, 64, 16, 8, True, np.float16), ([120, 130, 110], [1500, 1499, 1450], 1, 1, 128, 16, 4, False, np.float16),
    ([100] * 70, [100 + 13 * i for i in range(70)], 1, 1, 32, 16, 8, True, np.float32)]


@pytest.mark.parametrize("case", range(len(LONG)))
def test_long_chunks(case):
    b = Batch(*LONG[case], seed=case, tail=3)
    b.check(b.run())
    b.check(b.run(window=333), window=333)
    b.check(b.run(causal=False, scale=-0.05), causal=False, scale=-0.05)


@pytest.mark.parametrize("batch,longest,kv_heads,dtype", [(65, 40, 1, np.float32), (200, 900, 2, np.float16), (1100, 60, 4, np.float16),
                                                          (1500, 700, 1, np.float32), (4300, 30, 1, np.float16)])
def test_many_sequences_a_few_without_new_tokens(batch, longest, kv_heads, dtype):
    rng = np.random.default_rng(batch)
    chunks = rng.choice([0, 1, 1, 1, 3], batch)
    b = Batch(list(chunks), list(rng.integers(1, longest + 1, batch)), kv_heads, kv_heads, 32, dtype=dtype, seed=1, tail=2)
    b.check(b.run())
    b.check(b.run(max_chunk=3, window=25), window=25)
    # most of them idle
    keep = (rng.random(batch) < 0.03).astype(int)
    keep[batch // 2] = 2
    b.q_starts = np.concatenate([[0], np.cumsum(keep)]).astype(np.int32)
    b.check(b.run())


def test_a_prompt_whose_tiles_fill_the_device_is_its_halves():
    b = Batch([4096], [4096], 64, 16, 16, seed=7)
    whole = b.run().astype(np.float64)
    q, n = b.q, 2048
    for at in (0, n):
        b.q, b.q_starts, b.kv_lens = q[at:at + n], np.array([0, n], np.int32), np.array([at + n], np.int32)
        half = b.run().astype(np.float64)
        # both are off by half a step of the result and half a step of each probability at most, and by a float32 score's few units
        tol = 2 * 2.0 ** -11 * (np.abs(half) + np.abs(b.pages["v"]).max()) + 1e-5
        assert np.all(np.abs(whole[at:at + n] - half) <= tol)


@pytest.mark.parametrize("chunks,lengths", [([1, 1, 1], [300, 900, 20]), ([5, 30], [50, 1400]), ([150, 1], [700, 900]), ([300], [1300])])
def test_the_result_may_take_the_queries_place(chunks, lengths):
    b = Batch(chunks, lengths, 4, 1, 128, seed=9, tail=2)
    q = hip(b.q)
    F.paged_attention(q, b.cache, ids(b.table), ids(b.q_starts), ids(b.kv_lens), out=q)
    assert np.array_equal(q.numpy(), b.run())


def test_packed_queries():
    b = Batch([5, 60], [80, 90], 6, 2, 64, seed=1)
    packed = np.concatenate([b.q, b.rng.standard_normal((65, 4, 64)).astype(np.float16)], 1).reshape(5, 13, 640)
    y = F.paged_attention_qkv(hip(packed), 6, b.cache, ids(b.table), ids(b.q_starts), ids(b.kv_lens)).numpy()
    assert y.shape == (5, 13, 384)
    assert np.array_equal(y.reshape(b.q.shape), b.run())


def test_a_call_gives_the_same_bits_each_time():
    for chunks, lengths in (([1] * 8, [900, 2000, 30, 4000, 5, 77, 1000, 1]), ([200, 3], [1500, 4000])):
        b = Batch(chunks, lengths, 8, 2, 128, seed=2)
        first = b.run()
        for _ in range(3):
            assert np.array_equal(b.run(), first)
        b.check(first)


def test_a_cache_of_more_than_2_to_the_32_bytes():
    heads, dim, page = 8, 128, 64
    pages = (5 << 30) // (heads * dim * page)
    c = Q.PagedKVCache(pages, page, heads, dim)
    rng = np.random.default_rng(2)
    n = 640
    where = np.array([pages - 1, 0, pages // 2, pages - 2, 17, pages - 9, pages // 3, 5, pages - 50, 1], np.int32)
    x = rng.standard_normal((2, n, heads, dim)).astype(np.float16)
    slots = where[np.arange(n) // page] * page + np.arange(n) % page
    Q.kv_cache_write(c, hip(x[0]), hip(x[1]), ids(slots))
    k, v = (K.values(*K.quantize(y.astype(np.float32), 8, True)[:2], None, 8).reshape(10, page, heads, dim).transpose(0, 2, 1, 3) for y in x)
    for chunk in (1, 150):
        q = rng.standard_normal((chunk, heads, dim)).astype(np.float16)
        got = F.paged_attention(hip(q), c, ids(where[None]), ids([0, chunk]), ids([n])).numpy()
        want = K.attention(q, k, v, np.arange(10)[None], [0, chunk], [n], dim ** -0.5)
        assert np.abs(got - want).max() <= 2.0 ** -11 * (np.abs(want).max() + np.abs(v).max()) + 1e-5


@pytest.mark.parametrize("chunks,lengths", [([1] * 4, [3000, 100, 1500, 9]), ([180, 6], [900, 2500])])
def test_captured_calls_replay_beside_eager_ones(chunks, lengths):
    """Two graphs captured on streams of their own, replayed at once, with eager calls of other sizes between."""
    b, other = Batch(chunks, lengths, 8, 2, 128, seed=3), Batch([1, 4], [5000, 300], 8, 2, 128, seed=4)
    want, eager = b.run(), other.run()
    t = [hip(b.q), ids(b.table), ids(b.q_starts), ids(b.kv_lens)]
    outs, graphs, streams = [], [], []
    for _ in range(2):
        with L.graph.capture() as g:
            outs.append(F.paged_attention(t[0], b.cache, *t[1:]))
        graphs.append(g)
        s = C.c_void_p()
        _C.call("lq_stream_create_nonblocking", C.byref(s))
        streams.append(s)
    try:
        for rep in range(4):
            b.q = np.ascontiguousarray(b.q[::-1])
            t[0].copy_from(b.q)
            L.synchronize()
            for g, s in zip(graphs, streams):
                _C.call("lq_graph_launch", g.id, s)
            assert np.array_equal(other.run(), eager)
            for s in streams:
                _C.call("lq_sync", s)
            want = b.run()
            for y in outs:
                assert np.array_equal(y.numpy(), want), rep
            # lengths are read when the graph runs: another step of the same sequences
            t[3].copy_from(np.maximum(b.kv_lens - rep, np.diff(b.q_starts)).astype(np.int32))
            graphs[0].replay()
            b.kv_lens = t[3].numpy()
            assert np.array_equal(outs[0].numpy(), b.run()), rep
            b.check(outs[0].numpy())
    finally:
        L.synchronize()
        for s in streams:
            _C.call("lq_stream_destroy", s)


def test_calls_on_two_streams_share_nothing():
    batches = [Batch([1] * 3, [6000, 100, 2000], 8, 2, 64, seed=1), Batch([1, 2], [300, 7000], 8, 2, 64, seed=2)]
    want = [b.run() for b in batches]
    args = [(hip(b.q), b.cache, ids(b.table), ids(b.q_starts), ids(b.kv_lens)) for b in batches]
    streams = []
    for _ in batches:
        s = C.c_void_p()
        _C.call("lq_stream_create", C.byref(s))
        streams.append(s)
    L.synchronize()
    prev, outs = _C.current_stream(), [[], []]
    try:
        for _ in range(8):
            for i, s in enumerate(streams):
                _C.set_current_stream(s)
                outs[i].append(F.paged_attention(*args[i]))
        for s in streams:
            _C.call("lq_sync", s)
    finally:
        _C.set_current_stream(prev)
    for i, ys in enumerate(outs):
        for y in ys:
            assert np.array_equal(y.numpy(), want[i])
    for s in streams:
        _C.call("lq_stream_destroy", s)


def test_refusals():
    b = Batch([2, 3], [20, 30], 4, 2, 64, seed=1)
    q, table, starts, lens = hip(b.q), ids(b.table), ids(b.q_starts), ids(b.kv_lens)
    for args, kw, error in [
            ((q.reshape(5, 256), b.cache, table, starts, lens), {}, L.ShapeMismatch), ((hip(b.q[:, :3]), b.cache, table, starts, lens), {}, L.ShapeMismatch),
            ((hip(b.q[:, :, :32]), b.cache, table, starts, lens), {}, L.ShapeMismatch), ((q.cpu(), b.cache, table, starts, lens), {}, L.DeviceMismatch),
            ((hip(b.q.astype(np.int32)), b.cache, table, starts, lens), {}, L.DtypeMismatch), ((q, b.cache, ids([1, 2]), starts, lens), {}, L.ShapeMismatch),
            ((q, b.cache, hip(b.table.astype(np.int64)), starts, lens), {}, L.DtypeMismatch), ((q, b.cache, table, ids([0, 5]), lens), {}, L.ShapeMismatch),
            ((q, b.cache, table, starts, ids([1, 2, 3])), {}, L.ShapeMismatch), ((q, b.cache, table, starts, lens), dict(window=0), ValueError),
            ((q, b.cache, table, starts, lens), dict(max_chunk=0), ValueError), ((q, b.cache, table, starts.cpu(), lens), {}, L.DeviceMismatch),
            ((q, b.cache, table, starts, lens), dict(out=hip(b.q[:4])), L.ShapeMismatch),
            ((q, b.cache, table, starts, lens), dict(out=hip(b.q.astype(np.float32))), L.DtypeMismatch)]:
        with pytest.raises(error):
            F.paged_attention(*args, **kw)
    with pytest.raises(L.ShapeMismatch):
        F.paged_attention_qkv(hip(np.zeros((5, 7 * 64), np.float16)), 4, b.cache, table, starts, lens)
    empty = F.paged_attention(L.Tensor.empty((0, 4, 64), L.float16), b.cache, table, starts, lens)
    assert empty.shape == (0, 4, 64)


def held_by_a_graph(calls):
    """Bytes of the pool that a graph of these calls holds."""
    used = C.c_size_t()
    L.synchronize()
    _C.call("lq_empty_cache")  # (a kept block of up to twice the size would be taken for one that is asked for)
    _C.call("lq_memory_stats", C.byref(used), None)
    before = used.value
    with L.graph.capture() as g:
        for call in calls:
            call()
    _C.call("lq_memory_stats", C.byref(used), None)
    return g, used.value - before


@pytest.mark.parametrize("chunks,lengths", [([1] * 4, [3000, 100, 1500, 9]), ([180, 6], [900, 2500])])
def test_a_captured_step_of_many_layers_holds_one_set_of_pieces(chunks, lengths):
    b = Batch(chunks, lengths, 8, 2, 128, seed=3)
    t = [hip(b.q), ids(b.table), ids(b.q_starts), ids(b.kv_lens)]
    outs = [hip(np.zeros_like(b.q)) for _ in range(12)]
    call = lambda y: lambda: F.paged_attention(t[0], b.cache, *t[1:], out=y)
    want = b.run()
    one, alone = held_by_a_graph([call(outs[0])])
    all_, together = held_by_a_graph([call(y) for y in outs])
    assert alone and together == alone
    for g in (one, all_, all_):
        for y in outs:
            y.copy_from(np.zeros_like(b.q))
        g.replay()
        L.synchronize()
        for y in outs[:1 if g is one else 12]:
            assert np.array_equal(y.numpy(), want)


def test_room_for_pieces_does_not_grow_with_the_heads():
    """Tiles of several parts have at most 4 parts for each of the 512 places of blocks, over all heads; a part is 128 rows of 64 columns, a maximum and a
    sum each, in float32.  Beside them some rounding."""
    b = Batch([70] * 100, [420] * 100, 64, 64, 16, dtype=np.float16, seed=3)
    t = [hip(b.q), ids(b.table), ids(b.q_starts), ids(b.kv_lens)]
    out = hip(np.zeros_like(b.q))
    g, nbytes = held_by_a_graph([lambda: F.paged_attention(t[0], b.cache, *t[1:], out=out)])
    assert nbytes <= (4 * 512 + 256) * 128 * (64 + 2) * 4
    g.replay()
    L.synchronize()
    assert np.array_equal(out.numpy(), b.run())
