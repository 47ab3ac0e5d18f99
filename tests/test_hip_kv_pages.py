"""Pages of the key / value cache copied, and sequences moved together, to the byte."""

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn.functional as F
import lucid_amd.quantization as Q
from test_hip_kv_cache import buffers, hip, ids, make, same

pytestmark = pytest.mark.gpu


def filled(rng, *shape):
    c = make(*shape)
    for n, b in buffers(c).items():
        getattr(c, n).copy_from(rng.integers(-128, 128, b.shape).astype(b.dtype))
    return c


# pages of many blocks and of less than one, every kind of row
CACHES = [(8, True, 128, 8, 16), (8, False, 64, 12, 32), (4, True, 128, 2, 16), (4, False, 32, 1, 48), (8, True, 16, 1, 16), (8, False, 80, 5, 64),
          (8, True, 256, 3, 128), (4, False, 224, 4, 16), (4, True, 96, 2, 16), (8, False, 48, 7, 16)]


def copied(before, src, dst):
    want = {n: b.copy() for n, b in before.items()}
    pages = len(before["k_scale"])
    for s, d in zip(src, dst):
        if 0 <= s < pages and 0 <= d < pages:
            for n in want:
                want[n][d] = before[n][s]
    return want


@pytest.mark.parametrize("bits,symmetric,dim,heads,page", CACHES)
@pytest.mark.parametrize("pairs", [1, 7, 40])
def test_copied_pages(bits, symmetric, dim, heads, page, pairs):
    rng = np.random.default_rng(dim + pairs)
    c = filled(rng, 2 * pairs + 2, page, heads, dim, symmetric, bits)
    before = buffers(c)
    order = rng.permutation(2 * pairs + 2)
    src, dst = order[:pairs].copy(), order[pairs:2 * pairs].copy()
    src[pairs // 2] = src[0]  # one page twice
    if pairs > 4:
        src[1], dst[2], src[3], dst[4] = -1, -(1 << 31), 2 * pairs + 2, 0x7fffffff
    Q.kv_cache_copy(c, ids(src), ids(dst))
    same(buffers(c), copied(before, src, dst))


def compacted(before, page, table, keep, starts):
    want = {n: b.copy() for n, b in before.items()}
    pages = len(before["k_scale"])
    for b in range(len(starts) - 1):
        for i, p in enumerate(keep[starts[b]:starts[b + 1]]):
            if not (0 <= p < len(table[b]) * page and i < len(table[b]) * page):
                continue
            s, d = table[b][p // page], table[b][i // page]
            if 0 <= s < pages and 0 <= d < pages:
                for n in want:
                    want[n][d, :, i % page] = before[n][s, :, p % page]
    return want


def sequences(rng, lengths, page, extra=2):
    used = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(used) + extra)
    table, at = np.full((len(lengths), max(max(used), 1)), -1, np.int32), 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return sum(used) + extra, table


def check(c, table, keep, starts):
    before = buffers(c)
    Q.kv_cache_compact(c, ids(table), ids(keep), ids(starts))
    same(buffers(c), compacted(before, c.page_size, table, keep, starts))


@pytest.mark.parametrize("bits,symmetric,dim,heads,page", CACHES)
@pytest.mark.parametrize("lengths,part", [([1], 1.0), ([300], 0.5), ([17, 0, 1, 200, 64], 0.9), ([700, 31], 0.1), ([129] * 9, 0.99)])
def test_compacted_sequences(bits, symmetric, dim, heads, page, lengths, part):
    rng = np.random.default_rng(dim + sum(lengths))
    pages, table = sequences(rng, lengths, page)
    c = filled(rng, pages, page, heads, dim, symmetric, bits)
    keep = [np.sort(rng.permutation(n)[:max(min(n, 1), round(part * n))]) for n in lengths]
    check(c, table, np.concatenate(keep), np.cumsum([0] + [len(k) for k in keep]))


@pytest.mark.parametrize("n", [63, 64, 65, 255, 256, 257, 513, 1000, 5000])
@pytest.mark.parametrize("kind", ["first evicted", "a window", "sinks and a window", "every other", "all", "none of the second half", "one each"])
def test_what_sequences_keep(n, kind):
    """Rows that move by one, by the most, not at all; a tile's old places taken by tiles far behind it."""
    rng = np.random.default_rng(n)
    keep = {"first evicted": np.arange(1, n), "a window": np.arange(n - n // 3, n), "every other": np.arange(0, n, 2), "all": np.arange(n),
            "sinks and a window": np.concatenate([np.arange(4), np.arange(n // 2, n)]), "none of the second half": np.arange(n // 2),
            "one each": np.arange(n - 1, n)}[kind]
    pages, table = sequences(rng, [n, n], 16)
    c = filled(rng, pages, 16, 2, 64, True, 8)
    check(c, table, np.concatenate([keep, keep]), [0, len(keep), 2 * len(keep)])


@pytest.mark.parametrize("bits,symmetric,dim,heads", [(8, True, 16, 1), (8, False, 64, 3), (4, False, 32, 1), (4, True, 128, 2), (8, False, 80, 1)])
@pytest.mark.parametrize("part", [0.3, 0.98])
def test_many_sequences_and_long_ones(bits, symmetric, dim, heads, part):
    """Sequences that end on both sides of a tile, and many that have none to themselves."""
    rng = np.random.default_rng(dim + heads)
    lengths = list(rng.integers(0, 20, 560)) + [1023, 1024, 1025, 1400, 4000, 2049, 1]
    pages, table = sequences(rng, lengths, 16)
    c = filled(rng, pages, 16, heads, dim, symmetric, bits)
    keep = [np.sort(rng.permutation(n)[:round(part * n)]) for n in lengths]
    keep[-5], keep[-3] = np.arange(1, 1025), np.concatenate([np.arange(1024), np.arange(1030, 4000)])
    check(c, table, np.concatenate(keep), np.cumsum([0] + [len(k) for k in keep]))


def test_places_that_are_none():
    """Beyond the table, on a page that is negative or beyond the cache, old or new: not moved.  Entries of no sequence are not looked at."""
    rng = np.random.default_rng(2)
    c = filled(rng, 6, 16, 3, 32, False, 8)
    table = np.array([[0, 6, 1], [-1, 2, 3], [4, -(1 << 31), 5]], np.int32)
    keep = np.array([1, 15, 17, 33, 40, 48, 3, 20, 37, 47, 1 << 30, 0x7fffffff, -1, 1, 3, 33, 35, 99], np.int32)
    check(c, table, keep, [0, 6, 12, 17])


def test_shared_pages_whose_rows_stay():
    rng = np.random.default_rng(3)
    c = filled(rng, 5, 16, 2, 64, True, 4)
    table = np.array([[0, 1, 2], [0, 1, 3]], np.int32)
    keep = [np.concatenate([np.arange(32), [35, 40, 41]]), np.concatenate([np.arange(32), [33, 47]])]
    check(c, table, np.concatenate(keep), [0, 35, 69])


def test_more_rows_kept_than_the_cache_has():
    """Sequences that share most of their pages keep more between them than there are rows."""
    rng = np.random.default_rng(6)
    c = filled(rng, 8, 16, 2, 32, False, 8)
    table = np.array([[0, 1, 2 + b] for b in range(6)], np.int32)
    keep = [np.concatenate([np.arange(32), np.sort(32 + rng.permutation(16)[:5])]) for _ in range(6)]
    assert 6 * 37 > 8 * 16
    check(c, table, np.concatenate(keep), np.arange(7) * 37)


def test_nothing_to_move():
    rng = np.random.default_rng(4)
    c = filled(rng, 3, 16, 1, 16, True, 8)
    before = buffers(c)
    Q.kv_cache_copy(c, ids([]), ids([]))
    Q.kv_cache_compact(c, ids(np.zeros((0, 3))), ids([]), ids([0]))
    Q.kv_cache_compact(c, ids(np.zeros((2, 0))), ids([1, 2]), ids([0, 1, 2]))
    Q.kv_cache_compact(c, ids([[0, 1]]), ids([]), ids([0, 0]))
    same(buffers(c), before)


def test_calls_on_two_streams_and_in_graphs():
    """Two graphs captured on one stream, replayed in turn with eager calls between; their lists change between replays."""
    rng = np.random.default_rng(5)
    caches = [filled(rng, 80, 16, 4, 64, i == 0, 8) for i in range(2)]
    states = []
    for i, c in enumerate(caches):
        lengths = [500, 90] if i else [1200]
        _, table = sequences(rng, lengths, 16, 0)
        states.append([c, lengths, table, ids(table), None, None])
    def new_keep(lengths):
        keep = [np.sort(rng.permutation(n)[:n // 2]) for n in lengths]
        return np.concatenate(keep), np.cumsum([0] + [len(k) for k in keep])
    graphs = []
    for s in states:
        keep, starts = new_keep(s[1])
        s[4], s[5] = ids(keep), ids(starts)
        Q.kv_cache_compact(s[0], s[3], s[4], s[5])
        with L.graph.capture() as g:
            Q.kv_cache_compact(s[0], s[3], s[4], s[5])
        graphs.append(g)
    for rep in range(4):
        for s, g in zip(states, graphs):
            keep, starts = new_keep(s[1])
            s[4].copy_from(np.asarray(keep, np.int32)), s[5].copy_from(np.asarray(starts, np.int32))
            before = buffers(s[0])
            g.replay()
            L.synchronize()
            same(buffers(s[0]), compacted(before, 16, s[2], keep, starts))
            keep, starts = new_keep(s[1])
            check(s[0], s[2], keep, starts)


def test_a_forked_sequence_goes_its_own_way():
    """Two sequences share whole pages, each has its own copy of the last one; both attend to what they wrote since."""
    rng = np.random.default_rng(6)
    c = Q.PagedKVCache(6, 16, 2, 64)
    rows = lambda n, h: rng.standard_normal((n, h, 64)).astype(np.float32)
    k, v = rows(40, 2), rows(40, 2)
    Q.kv_cache_write(c, hip(k), hip(v), ids(np.arange(40)))
    Q.kv_cache_copy(c, ids([2]), ids([4]))
    k2, v2, q = rows(2, 2), rows(2, 2), rows(2, 4)
    Q.kv_cache_write(c, hip(k2), hip(v2), ids([40, 4 * 16 + 8]))
    both = F.paged_attention(hip(q), c, ids([[0, 1, 2], [0, 1, 4]]), ids([0, 1, 2]), ids([41, 41])).numpy()
    for b in range(2):
        alone = Q.PagedKVCache(3, 16, 2, 64)
        Q.kv_cache_write(alone, hip(np.concatenate([k, k2[b:b + 1]])), hip(np.concatenate([v, v2[b:b + 1]])), ids(np.arange(41)))
        want = F.paged_attention(hip(q[b:b + 1]), alone, ids([[0, 1, 2]]), ids([0, 1]), ids([41])).numpy()
        # (the same rows; sums may be divided otherwise: 41 terms of at most the largest value, twice)
        assert np.abs(both[b] - want[0]).max() <= 2 * 41 * 2.0 ** -24 * np.abs(v).max() + 2.0 ** -22 * np.abs(v).max() * 16


def test_attention_after_compaction_is_that_of_the_kept():
    rng = np.random.default_rng(7)
    c, alone = Q.PagedKVCache(12, 16, 2, 64), Q.PagedKVCache(12, 16, 2, 64)
    k, v = (rng.standard_normal((150, 2, 64)).astype(np.float32) for _ in range(2))
    q = hip(rng.standard_normal((3, 4, 64)).astype(np.float32))
    pages = rng.permutation(12)[:10]
    slots = pages[np.arange(150) // 16] * 16 + np.arange(150) % 16
    Q.kv_cache_write(c, hip(k), hip(v), ids(slots))
    keep = np.sort(rng.permutation(150)[:70])
    Q.kv_cache_compact(c, ids([pages]), ids(keep), ids([0, 70]))
    Q.kv_cache_write(alone, hip(k[keep]), hip(v[keep]), ids(slots[:70]))
    args = ids([pages]), ids([0, 3]), ids([70])
    assert np.array_equal(F.paged_attention(q, c, *args).numpy(), F.paged_attention(q, alone, *args).numpy())
