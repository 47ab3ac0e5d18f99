"""How far attention over the pages may be off, row by row: a row is held to what it sees itself."""

import numpy as np
import pytest

import oracle.kv_cache as K
from test_hip_paged_attention import GRID, LONG, Batch

pytestmark = pytest.mark.gpu


def rms(x):
    return np.sqrt(np.mean(np.square(x, dtype=np.float64)))


@pytest.mark.parametrize("bits,symmetric,dim,chunks,lengths,max_chunk", [
    (8, True, 128, [300], [2000], None), (8, False, 64, [200, 150], [900, 600], None), (4, False, 128, [512], [512], None), (4, True, 256, [130], [700], None),
    (8, True, 128, [40, 40], [900, 700], 1), (8, True, 128, [40, 40], [900, 700], 300)])  # the last two: one batch on both sides of the launch rule
def test_a_float16_result_is_off_by_its_own_rounding(bits, symmetric, dim, chunks, lengths, max_chunk):
    """Probabilities have 22 bits and all else float32, so that a float16 result is the float64 one rounded, but for values that lie within some
    2^-20 of a tie.  As root mean squares: what the rounding to float16 itself does to the float64 result, 5 % for those, and 2^-18 of the result for
    the scores' errors."""
    b = Batch(chunks, lengths, 8, 2, dim, 16, bits, symmetric, seed=dim + bits)
    want, got = b.want(), b.run(max_chunk=max_chunk)
    rounding = rms(want.astype(np.float16).astype(np.float64) - want)
    assert rms(got - want) <= 1.05 * rounding + 2.0 ** -18 * rms(want), (rms(got - want), rounding)


def bounds(b, scale=None, causal=True, window=None):
    """The float64 result and how far each element may be off, from what its own row sees.

    u = 2^-24.  A row's scores: sums of dim products whose partial sums stay below a = scale sum |q k| (the largest of the seen keys), as
    independent errors 4 sqrt(dim) u a at four deviations; float32 queries are two float16 of 22 bits, 2 u a; scale, maximum and exponential
    round 8 units of 1 + a.  With e for all of that, probabilities off by a factor 1 + e move column d by e (sum_j p_j |v_jd| + |o_d|).  A
    weight p_j v_scale_j is held to u of the row's largest one, its product with a code (of which a row has one of half the range at least)
    adds u times twice that to each of n terms, as does their sum: 4 sqrt(n) + 8 units of 2 max_j p_j max_d |v_jd|.  A float16 result is rounded
    by 2^-11 of itself, or 2^-25."""
    scale, u = 1 / np.sqrt(b.dim) if scale is None else scale, 2.0 ** -24
    q, group, page = b.q.astype(np.float64), b.heads // b.kv_heads, b.cache.page_size
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(len(b.kv_lens)):
        lo, hi, length = int(b.q_starts[s]), int(b.q_starts[s + 1]), int(b.kv_lens[s])
        j = np.arange(length)
        k, v = (b.pages[n][b.table[s][j // page], :, j % page].astype(np.float64) for n in "kv")
        place = length - (hi - lo) + np.arange(hi - lo)[:, None]
        seen = (j <= place) if causal else np.ones((hi - lo, length), bool)
        if window is not None:
            seen = seen & (j > place - window)
        some = seen.any(1)
        for h in range(b.heads if length and hi > lo else 0):
            kh, vh = k[:, h // group], v[:, h // group]
            with np.errstate(all="ignore"):
                sc = np.where(seen, q[lo:hi, h] @ kh.T * scale, -np.inf)
                a = np.where(seen, np.abs(q[lo:hi, h]) @ np.abs(kh).T * abs(scale), 0).max(1, keepdims=True)
                p = np.exp(sc - sc.max(1, keepdims=True))
                p = np.where(some[:, None], p / p.sum(1, keepdims=True), 0)
            held = seen.any(0)  # (what nobody sees may be anything)
            p, vh = p[:, held], vh[held]
            o = p @ vh
            e = u * (4 * np.sqrt(b.dim) * a + 2 * a + 8 * (1 + a))
            n = seen.sum(1, keepdims=True)
            t = e * (p @ np.abs(vh) + np.abs(o)) + u * (4 * np.sqrt(n) + 8) * 2 * (p * np.abs(vh).max(1)).max(1, keepdims=True, initial=0)
            if b.dtype == np.float16:
                t = t + 2.0 ** -11 * np.abs(o) + 2.0 ** -25
            want[lo:hi, h], tol[lo:hi, h] = o, t
    return want, tol


def held(b, got, **kw):
    want, tol = bounds(b, **kw)
    assert got.shape == want.shape and got.dtype == b.dtype and np.isfinite(got).all()
    off = np.abs(got - want)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert (off <= tol).all(), (worst, got[worst], want[worst], tol[worst])


def scaled(b, factor):
    """The batch's values, those of token j of sequence s times factor(s, j, head), a power of two."""
    u = K.unpack(b.cache.v_codes.numpy(), b.bits)
    scale = b.cache.v_scale.numpy().copy()
    zero = None if b.symmetric else b.cache.v_zero.numpy()
    for s, length in enumerate(b.kv_lens):
        for j in range(length):
            at = (b.table[s, j // b.cache.page_size], slice(None), j % b.cache.page_size)
            scale[at] *= factor(s, j)
    b.put("v", u, scale.astype(np.float32), zero)


SIZES = [([1, 3], [300, 700]), ([16, 5], [333, 40]), ([90], [700]), ([150, 100], [200, 900]), ([300], [1300])]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("chunks,lengths", SIZES)
def test_a_row_does_not_feel_values_that_it_does_not_see(chunks, lengths, dtype):
    """The last token of each chunk has values 2^12 to 2^30 times the others': causality keeps them from the rows before it.  A key that has
    left the window of all but the first row, likewise."""
    for r in (12, 16) if dtype == np.float16 else (12, 17, 22, 30):
        for bits, symmetric in ((8, True), (4, False)):
            b = Batch(chunks, lengths, 4, 2, 64, bits=bits, symmetric=symmetric, dtype=dtype, seed=r)
            scaled(b, lambda s, j: 2.0 ** (r * (j == lengths[s] - 1) - 4))
            held(b, b.run())
            b = Batch(chunks, lengths, 4, 2, 64, bits=bits, symmetric=symmetric, dtype=dtype, seed=r)
            scaled(b, lambda s, j: 2.0 ** (r * (j == lengths[s] - chunks[s] - 19) - 4))  # the first key of the first row's window of 20
            held(b, b.run(window=20), window=20)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("chunks,lengths", SIZES)
def test_an_infinite_scale_is_felt_by_those_that_see_it_alone(chunks, lengths, dtype):
    b = Batch(chunks, lengths, 4, 2, 64, dtype=dtype, seed=3)
    scale = b.cache.v_scale.numpy().copy()
    for s, n in enumerate(lengths):
        scale[b.table[s, (n - 1) // 16], :, (n - 1) % 16] = np.inf
    want, tol = bounds(b)
    b.cache.v_scale.copy_from(scale)
    got = b.run()
    last = b.q_starts[1:] - 1
    assert not np.isfinite(got[last]).all(-1).any()
    others = np.setdiff1d(np.arange(len(got)), last)
    assert (np.abs(got - want) <= tol)[others].all()


@pytest.mark.parametrize("chunks,lengths", SIZES)
def test_weights_of_all_sizes_keep_their_bits(chunks, lengths):
    """Scales that differ from key to key, from page to page, grow, fall, or are zero here and there; so far apart that their ratio is beyond
    a float32's exponents."""
    rng = np.random.default_rng(len(chunks) + chunks[0])
    jumble = rng.integers(-30, 31, (2, 2000))
    for factor in (lambda s, j: 2.0 ** jumble[s, j], lambda s, j: 2.0 ** jumble[s, j // 16], lambda s, j: 2.0 ** (j // 16 % 60 - 30), lambda s, j: 2.0 ** (30 - j // 16 % 60),
                   lambda s, j: 2.0 ** (j % 64 // 8), lambda s, j: float(jumble[s, j] % 3 > 0), lambda s, j: 2.0 ** (-40 if j % 300 else 85),
                   lambda s, j: 2.0 ** (85 if j < 40 else -40), lambda s, j: 2.0 ** (100 if j == 7 else -12)):
        b = Batch(chunks, lengths, 4, 2, 64, dtype=np.float32, seed=5)
        scaled(b, factor)
        held(b, b.run())
        held(b, b.run(scale=1.0, window=100), scale=1.0, window=100)


@pytest.mark.parametrize("case", range(len(GRID + LONG)))
def test_each_row_against_what_it_sees(case):
    b = Batch(*(GRID + LONG)[case], seed=case, tail=2)
    held(b, b.run())
    held(b, b.run(causal=False, window=70), causal=False, window=70)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("chunks,lengths", [([200], [100]), ([20, 3], [7, 40]), ([300, 150], [40, 600]), ([5], [0])])
def test_windows_beyond_all_keys(chunks, lengths, dtype):
    """As no window at all, also where a chunk is longer than its sequence."""
    b = Batch(chunks, lengths, 4, 2, 64, dtype=dtype, seed=1)
    for causal in (True, False):
        want = b.run(causal=causal)
        held(b, want, causal=causal)
        for window in (max(lengths) + max(chunks), (1 << 30) + 1, (1 << 31) - 1):
            assert np.array_equal(b.run(causal=causal, window=window), want), window


def test_a_longest_chunk_of_more_than_32_bits_is_one_beyond_all_tokens():
    b = Batch([40, 40], [700, 600], 8, 2, 128, seed=1)
    want = b.run(max_chunk=(1 << 31) - 1)
    assert not np.array_equal(want, b.run(max_chunk=1))  # (the other kernel: results differ by rounding)
    for n in (1 << 31, (1 << 32) + 1, 1 << 70):
        assert np.array_equal(b.run(max_chunk=n), want)


def test_a_window_of_more_than_32_bits_is_one_beyond_all_keys():
    b = Batch([40, 3], [100, 60], 4, 2, 64, seed=1)
    want = b.run()
    for n in (1 << 31, (1 << 32) - 1, (1 << 32) + 1, (1 << 32) + 5, 1 << 70):
        assert np.array_equal(b.run(window=n), want), n
    for bad in (-1, -(1 << 32) + 5):
        with pytest.raises(ValueError):
            b.run(window=bad)
        with pytest.raises(ValueError):
            b.run(max_chunk=bad)


@pytest.mark.parametrize("chunks,lengths", SIZES)
def test_queries_near_the_largest_float_of_keys_near_the_smallest(chunks, lengths):
    """Queries 2^118 times as large, the scale twice, keys 2^-119 times (their scales, 2^-7 and more here, stay normal numbers): every score is what it was,
    to the bit, though the scaled sum of a query's products with codes passes 2^128."""
    for bits, symmetric in ((8, True), (8, False), (4, False)):
        b = Batch(chunks, lengths, 4, 2, 64, bits=bits, symmetric=symmetric, dtype=np.float32, seed=2)
        want = b.run(scale=1.0)
        held(b, want, scale=1.0)
        b.q = b.q * np.float32(2.0 ** 118)
        assert b.cache.k_scale.numpy().min() >= 2.0 ** -7
        b.cache.k_scale.copy_from(b.cache.k_scale.numpy() * np.float32(2.0 ** -119))
        assert np.array_equal(b.run(scale=2.0), want)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("chunks,lengths,max_chunk", [
    ([300, 1, 300], [310, 400, 700], 300), ([300, 280, 299], [300, 280, 900], 300),  # alike: long chunks alone, one of them a token
    ([1200, 1, 0, 900], [1300, 700, 20, 900], 1200), ([1200, 1, 0, 900], [1300, 700, 20, 900], None), ([700] + [1] * 9, [900] + [300] * 9, 700),
    ([0, 0, 600, 3], [5, 0, 600, 64], 600), ([2100] + [1] * 4, [2100] + [90] * 4, None), ([2] * 70 + [260], [40] * 70 + [300], 260), ([60, 1] * 3, [99, 98] * 3, 7)])
def test_prompts_beside_single_tokens(chunks, lengths, max_chunk, dtype):
    """Batches whose sequences go to either kernel, or all to one, with rows of none behind them."""
    for kw in ({}, dict(window=130)):
        b = Batch(chunks, lengths, 4, 1, 64, bits=4 if len(kw) else 8, dtype=dtype, seed=len(chunks), tail=3)
        held(b, b.run(max_chunk=max_chunk, **kw), **kw)


KINDS = {"16 rows": ([1, 1], [300, 45]), "32 rows": ([5, 2], [200, 64]), "chunks": ([40, 70], [40, 300]), "one prompt": ([260], [1100])}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 224, 256])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("bits", [8, 4])
def test_every_kernel(bits, symmetric, dtype, dim, kind):
    """Each kernel for codes, scheme, type, head dims up to 64, 128 and 256 and rows of a sequence at a whole and a cut head dim: pages within a step and
    beyond it, a window, all keys."""
    chunks, lengths = KINDS[kind]
    b = Batch(chunks, lengths, 4, 1, dim, 16 if dim % 64 else 64, bits, symmetric, dtype, seed=dim + bits, tail=1)
    kw = (dict(), dict(window=21), dict(causal=False, scale=-0.4 / np.sqrt(dim)))[(dim // 32 + bits + symmetric) % 3]
    held(b, b.run(max_chunk=max(chunks), **kw), **kw)
