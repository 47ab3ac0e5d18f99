"""Drafted tokens verified on the device against the rule in float64, token by token."""

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn.functional as F

pytestmark = pytest.mark.gpu


def hip(a, dt=None):
    return L.tensor(np.ascontiguousarray(a, dt), device="hip")


def drawn(weights, w):
    """The lowest token of positive weight whose running sum passes w times the sum, else the last of positive weight, else -1."""
    with np.errstate(invalid="ignore"):
        weights = np.where((weights > 0) & (weights < np.inf), weights, 0.0)
    total = np.cumsum(weights)
    over = np.nonzero((weights > 0) & (total > float(w) * total[-1]))[0]
    some = np.nonzero(weights > 0)[0]
    return over[0] if len(over) else some[-1] if len(some) else -1


def verified(target, tokens, starts, uniforms, last, draft, new):
    target = target.astype(np.float64)
    vocab, counts = target.shape[1], []
    new = new.copy()
    for b in range(len(starts) - 1):
        rows = range(starts[b], starts[b + 1])
        got = []
        for i in rows:
            p = target[i]
            if i + 1 == starts[b + 1]:
                got.append(drawn(p, last[b]))
                break
            x = tokens[i + 1]
            q = draft[i].astype(np.float64) if draft is not None else (np.arange(vocab) == x).astype(np.float64)
            if 0 <= x < vocab and float(uniforms[i]) * (q[x] if draft is not None else 1.0) < p[x]:
                got.append(x)
                continue
            if draft is not None:
                with np.errstate(invalid="ignore"):
                    rest = np.where((p > 0) & (p < np.inf) | ~np.isfinite(p), p, 0.0) - np.where((q > 0) & (q < np.inf), q, 0.0)
            else:
                rest = np.where(q > 0, 0.0, p)
            with np.errstate(invalid="ignore"):
                some = ((rest > 0) & (rest < np.inf)).any()
            got.append(drawn(rest if some else p, last[b]))
            break
        new[rows.start:rows.stop] = -1
        new[rows.start:rows.start + len(got)] = got
        counts.append(len(got))
    return new, np.array(counts, np.int32)


def check(target, tokens, starts, uniforms, last, draft=None):
    rows = len(tokens)
    before = np.full(rows, 77, np.int32)
    out = hip(before), hip(np.full(len(starts) - 1, 99, np.int32))
    args = (hip(target), hip(tokens, np.int32), hip(starts, np.int32), hip(uniforms, np.float32), hip(last, np.float32))
    new, counts = F.verify_drafts(*args, draft=hip(draft) if draft is not None else None, out=out)
    assert new is out[0] and counts is out[1]
    want = verified(target, tokens, starts, np.float32(uniforms), np.float32(last), draft, before)
    assert np.array_equal(counts.numpy(), want[1])
    assert np.array_equal(new.numpy(), want[0])
    return want


def some(rng, counts, vocab, dtype, given, sharp=3.0, near=0.7):
    rows = sum(counts)
    logits = sharp * rng.standard_normal((rows, vocab))
    soft = lambda z: (np.exp(z - z.max(-1, keepdims=True)) / np.exp(z - z.max(-1, keepdims=True)).sum(-1, keepdims=True)).astype(dtype)
    target, draft = soft(logits), soft(logits + near * rng.standard_normal((rows, vocab)))
    tokens = np.zeros(rows, np.int32)
    for i in range(rows - 1):
        tokens[i + 1] = min(vocab - 1, np.searchsorted(np.cumsum(draft[i].astype(np.float64)), rng.random() * draft[i].astype(np.float64).sum())) if given else draft[i].argmax()
    return target, tokens, np.cumsum([0] + counts), rng.random(rows), rng.random(len(counts)), draft if given else None


COUNTS = [[1], [6], [2, 1, 0, 5, 3], [0, 0], [0, 4, 0], [5] * 16, [300, 2], [1] * 70, [257]]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("vocab", [1, 7, 8, 9, 15, 64, 1000])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("given", [True, False])
def test_sequences_of_all_kinds(counts, vocab, dtype, given):
    rng = np.random.default_rng(sum(counts) + vocab)
    check(*some(rng, counts, vocab, dtype, given))


@pytest.mark.parametrize("vocab", [2047, 2049, 8191, 8192, 8193, 32000, 50001, 131072, 262145])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_large_vocabularies(vocab, dtype):
    rng = np.random.default_rng(vocab)
    for given in (True, False):
        check(*some(rng, [3, 1, 4], vocab, dtype, given))


def test_long_drafts_that_are_accepted():
    """The same distribution on both sides: only rounding of u could refuse, and does not."""
    rng = np.random.default_rng(0)
    target, tokens, starts, u, last, _ = some(rng, [700, 256, 257], 50, np.float32, True, near=0.0)
    new, counts = check(target, tokens, starts, u, last, target)
    assert counts.tolist() == [700, 256, 257]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_on_the_borders(dtype):
    """Probabilities and numbers that are multiples of 1/16: u q = p is a refusal, a running sum that equals w times the sum is not past it."""
    rng = np.random.default_rng(1)
    for rep in range(20):
        rows = [3] * 40
        parts = lambda: np.stack([np.bincount(rng.integers(0, 6, 16), minlength=9)[:9] / 16 for _ in range(sum(rows))]).astype(dtype)
        target, draft = parts(), parts()
        u, last = rng.integers(0, 16, sum(rows)) / 16, rng.integers(0, 16, len(rows)) / 16
        check(target, rng.integers(0, 9, sum(rows)).astype(np.int32), np.cumsum([0] + rows), u, last, draft if rep % 2 else None)


def test_numbers_of_one_and_beyond():
    rng = np.random.default_rng(2)
    target, tokens, starts, u, last, draft = some(rng, [2] * 6, 5000, np.float32, True)
    u[:] = [0, 1, 2, -1, np.nan, 0, np.inf, 0, 1, 0, -0.0, 0]
    last[:] = [0, 1, 1.5, np.nan, -1, np.float32(1 - 2.0 ** -24)]
    check(target, tokens, starts, u, last, draft)


def test_probabilities_that_are_none():
    """Zeros, rows of nothing, negative numbers, infinities and NaN count as nothing."""
    rng = np.random.default_rng(3)
    target, tokens, starts, u, last, draft = some(rng, [2] * 12, 3000, np.float32, True)
    target[0] = 0
    target[2], target[4, ::3], target[6, 1000:] = -1, np.nan, np.inf
    target[8] = draft[8] / 2           # nothing of p - q is positive: from p
    draft[10], draft[12, 5:], draft[14] = np.nan, np.inf, -3
    target[16], target[17] = 0, 0      # no weight at all, wherever it ends
    target[18, :] = 0
    target[18, 2999] = 1e-30
    u[::2] = np.where(rng.random(12) < 0.5, 0.999, u[::2])
    check(target, tokens, starts, u, last, draft)
    check(target, tokens, starts, u, last)


def test_tokens_outside_the_vocabulary_are_refused():
    rng = np.random.default_rng(4)
    target, tokens, starts, u, last, draft = some(rng, [3] * 5, 100, np.float32, True)
    tokens[[1, 4, 7, 10, 13]] = [-1, 100, 0x7fffffff, -(1 << 31), 99]
    for d in (draft, None):
        check(target, tokens, starts, u, last, d)


def test_rows_of_no_sequence_stay():
    rng = np.random.default_rng(5)
    target, tokens, _, u, last, draft = some(rng, [4, 3, 9], 300, np.float32, True)
    check(target, tokens, np.array([2, 5, 5, 9]), u, last, draft)


def test_all_tokens_are_distributed_as_the_targets():
    """Over a grid of numbers, the first new token falls on each token as often as p says, whatever q is."""
    p, q = np.array([0.5, 0.25, 0.125, 0.125, 0.0]), np.array([0.125, 0.5, 0.25, 0.0, 0.125])
    n = 32
    drafted, u, w = (a.ravel() for a in np.meshgrid(np.repeat(np.arange(5), (q * 8).astype(int)), (np.arange(n) + 0.5) / n, (np.arange(n) + 0.5) / n, indexing="ij"))
    rows = 2 * len(u)
    tokens = np.zeros(rows, np.int32)
    tokens[1::2] = drafted
    uniforms = np.zeros(rows)
    uniforms[::2] = u
    new, _ = check(np.tile(p, (rows, 1)).astype(np.float32), tokens, np.arange(0, rows + 1, 2), uniforms, w, np.tile(q, (rows, 1)).astype(np.float32))
    share = np.bincount(new[::2], minlength=5) / len(u)
    assert np.abs(share - p).max() <= 1 / n  # (a border of u or w within a cell of the grid)


def test_replayed_from_graphs_and_on_its_own_memory():
    rng = np.random.default_rng(6)
    graphs = []
    for vocab in (40000, 900):
        case = some(rng, [4, 2, 7], vocab, np.float32, True)
        t = [hip(case[0]), hip(case[1], np.int32), hip(case[2], np.int32), hip(case[3], np.float32), hip(case[4], np.float32)]
        d = hip(case[5])
        F.verify_drafts(*t, draft=d)
        with L.graph.capture() as g:
            out = F.verify_drafts(*t, draft=d)
        graphs.append((g, t, d, out, vocab))
    for _ in range(3):
        for g, t, d, out, vocab in graphs:
            case = some(rng, [4, 2, 7], vocab, np.float32, True)
            for dst, src in zip(t, case):
                dst.copy_from(np.asarray(src, dst.dtype.np))
            d.copy_from(case[5])
            g.replay()
            L.synchronize()
            want = verified(case[0], case[1], case[2], np.float32(case[3]), np.float32(case[4]), case[5], np.full(13, -1, np.int32))
            assert np.array_equal(out[0].numpy(), want[0]) and np.array_equal(out[1].numpy(), want[1])
            check(*case)
