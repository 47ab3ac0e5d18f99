"""A decoder's steps with drafted tokens as a program runs them: a block of residual norms, attention over the quantized cache and a gated feed-forward on
packed weights, probabilities, verified drafts; sequences that are forked and that evict tokens between the steps.  Every stage is held to float64
(or to the byte) on what it was given, so that what one operator hands to the next is seen."""

import ctypes as C

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn as nn
import lucid_amd.nn.functional as F
import lucid_amd.nn.quantized as nnq
import lucid_amd.quantization as Q
from lucid_amd import _C
from lucid_amd.quantization import _qgemm
import oracle.kv_cache as K
import oracle.wq_group as W
from test_hip_kv_cache import buffers, same
from test_hip_kv_pages import compacted, copied, filled
from test_hip_residual_norm import norm
from test_hip_verify_drafts import verified
from test_hip_wq_gated import bound

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HEADS, KV_HEADS, DIM, PAGE, HIDDEN, VOCAB, GROUP = 4, 2, 64, 16, 320, 500, 64
WIDTH = HEADS * DIM


def hip(a):
    return L.tensor(np.ascontiguousarray(a), device="hip")


def ids(a):
    return hip(np.asarray(a, np.int32))


class Decoder:
    def __init__(self, bits):
        rng = self.rng = np.random.default_rng(bits)
        some = lambda *s: rng.standard_normal(s).astype(np.float32)
        self.bits, self.embedding = bits, 2 * some(VOCAB, WIDTH)
        self.qkv, self.proj, self.head = nn.Linear(WIDTH, (HEADS + 2 * KV_HEADS) * DIM), nn.Linear(WIDTH, WIDTH), nn.Linear(WIDTH, VOCAB)
        self.first = nn.RMSNorm(WIDTH)
        self.norms = [(1 + 0.2 * some(WIDTH)) for _ in range(4)]
        self.first.register_buffer("weight", hip(self.norms[0]))
        gate, up, down = nn.Linear(WIDTH, HIDDEN), nn.Linear(WIDTH, HIDDEN), nn.Linear(HIDDEN, WIDTH)
        self.float_mlp = gate, up, down
        self.mlp = nnq.QuantizedGatedLinearMLX.from_float(gate, up, bits=bits, group_size=GROUP)
        self.down = nnq.QuantizedLinearMLX.from_float(down, bits=bits, group_size=GROUP)
        self.cache = Q.PagedKVCache(24, PAGE, KV_HEADS, DIM, Q.per_channel_affine, Q.qint8)
        self.free, self.tables, self.lengths = list(rng.permutation(24)), [], []

    def new_sequence(self):
        self.tables.append([])
        self.lengths.append(0)

    def table(self):
        t = np.full((len(self.tables), max(map(len, self.tables))), -1, np.int32)
        for b, pages in enumerate(self.tables):
            t[b, :len(pages)] = pages
        return t

    def step(self, tokens):
        """A step of a list of tokens of each sequence, the probabilities behind each of them."""
        counts, slots = [len(t) for t in tokens], []
        for b, n in enumerate(counts):
            for place in range(self.lengths[b], self.lengths[b] + n):
                if place // PAGE == len(self.tables[b]):
                    self.tables[b].append(int(self.free.pop()))
                slots.append(self.tables[b][place // PAGE] * PAGE + place % PAGE)
        lens, starts = [n + c for n, c in zip(self.lengths, counts)], np.cumsum([0] + counts)
        x = hip(self.embedding[np.concatenate(tokens).astype(int)])
        y = self.first(x)
        self.near_norm(y.numpy(), x.numpy(), 0)
        packed = self.qkv(y)
        Q.kv_cache_write_qkv(self.cache, packed, HEADS, ids(slots))
        a = F.paged_attention_qkv(packed, HEADS, self.cache, ids(self.table()), ids(starts), ids(lens), max_chunk=max(counts))
        self.near_attention(a.numpy(), packed.numpy(), counts, lens)
        o = self.proj(a)
        y2, r = F.residual_norm(o, x, hip(self.norms[1]), post=True, post_weight=hip(self.norms[2]))
        t, e = norm(o.numpy().astype(np.float64), 0 * o.numpy(), self.norms[2], 0.0, False, 1e-6)
        want_r = x.numpy() + t
        assert (abs(r.numpy() - want_r) <= e + 2 * U * abs(want_r)).all()
        self.near_norm(y2.numpy(), r.numpy(), 1)
        h = self.mlp(y2)
        parts = [W.quantize(m.weight.numpy(), GROUP, self.bits) for m in self.float_mlp[:2]]
        want, e = bound(y2.numpy().astype(np.float64), parts, GROUP, self.bits, "silu", [m.bias.numpy() for m in self.float_mlp[:2]])
        assert (abs(h.numpy() - want) <= e + abs(want) * U).all()
        y3, _ = F.residual_norm(self.down(h), r, hip(self.norms[3]), residual_out=r)
        self.near_norm(y3.numpy(), r.numpy(), 3)
        logits = self.head(y3).numpy().astype(np.float64)
        p = np.exp(logits - logits.max(-1, keepdims=True))
        return starts, (p / p.sum(-1, keepdims=True)).astype(np.float32)

    def near_norm(self, y, v, which):
        # (v is the residual as it was rounded: the norm saw it within a rounding)
        want, e = norm(v.astype(np.float64), U * abs(v), self.norms[which], 0.0, False, 1e-6)
        assert (abs(y - want) <= e + U * abs(want)).all()

    def near_attention(self, got, packed, counts, lens):
        """Each token over its sequence's rows as the cache has them; the bound of an attention of float32 (a score's products and sums, the exponential's
        argument, the sum of the values), at sizes of at most 100 keys."""
        held = buffers(self.cache)
        at = 0
        for b, (n, length) in enumerate(zip(counts, lens)):
            place = np.arange(length)
            pages = np.array(self.tables[b])[place // PAGE]
            k, v = (K.values(held[w + "_codes"][pages, :, place % PAGE].view(np.uint8), held[w + "_scale"][pages, :, place % PAGE],
                             held[w + "_zero"][pages, :, place % PAGE], 8).astype(np.float64) for w in "kv")
            for i in range(n):
                q = packed[at + i, :WIDTH].astype(np.float64).reshape(KV_HEADS, -1, DIM)
                seen = length - n + i + 1
                s = q @ k[:seen].transpose(1, 2, 0) / np.sqrt(DIM)
                p = np.exp(s - s.max(-1, keepdims=True))
                want = (p / p.sum(-1, keepdims=True) @ v[:seen].transpose(1, 0, 2)).reshape(-1)
                size, top = (abs(q) @ abs(k[:seen]).transpose(1, 2, 0)).max() / np.sqrt(DIM), abs(v[:seen]).max()
                e = U * (4 * np.sqrt(DIM) * size + 2 * size + 8 * (1 + abs(s).max()))
                assert abs(got[at + i] - want).max() <= 2 * e * top + 4 * np.sqrt(seen + 1) * U * top
            at += n

    def fork(self, b):
        """A new sequence with b's whole pages and a copy of its last one."""
        self.new_sequence()
        whole, rest = divmod(self.lengths[b], PAGE)
        self.tables[-1], self.lengths[-1] = self.tables[b][:whole], self.lengths[b]
        if rest:
            page, before = int(self.free.pop()), buffers(self.cache)
            Q.kv_cache_copy(self.cache, ids([self.tables[b][whole], -1]), ids([page, -1]))
            same(buffers(self.cache), copied(before, [self.tables[b][whole]], [page]))
            self.tables[-1].append(page)

    def evict(self, shared):
        """Every sequence keeps the tokens of the shared beginning and some of the others."""
        keep = [np.concatenate([np.arange(min(shared, n)), np.sort(shared + self.rng.permutation(max(0, n - shared))[:max(0, n - shared) // 2])]).astype(int)
                for n in self.lengths]
        starts, before = np.cumsum([0] + [len(k) for k in keep]), buffers(self.cache)
        Q.kv_cache_compact(self.cache, ids(self.table()), ids(np.concatenate(keep)), ids(starts))
        same(buffers(self.cache), compacted(before, PAGE, self.table(), np.concatenate(keep), starts))
        for b, k in enumerate(keep):
            self.lengths[b] = len(k)
            used = -(-len(k) // PAGE)
            self.free += [p for p in self.tables[b][used:] if not any(p in t for i, t in enumerate(self.tables) if i != b)]
            self.tables[b] = self.tables[b][:used]


@pytest.mark.parametrize("bits,given", [(4, True), (8, False)])
def test_steps_with_drafts_forks_and_evictions(bits, given):
    d = Decoder(bits)
    rng = d.rng
    for n in (37, 5):
        d.new_sequence()
    prompts = [rng.integers(0, VOCAB, n) for n in (37, 5)]
    starts, p = d.step(prompts)
    d.lengths = [37, 5]
    last = [int(p[s - 1].argmax()) for s in starts[1:]]
    d.fork(0)
    last.append(int(rng.integers(0, VOCAB)))
    told = 0
    for turn in range(5):
        # drafts: as many as three a sequence, likely ones
        drafts = [list(rng.integers(0, VOCAB, n)) for n in rng.integers(0, 4, len(d.tables))]
        tokens = [[t] + more for t, more in zip(last, drafts)]
        starts, p = d.step(tokens)
        flat = np.concatenate(tokens).astype(np.int32)
        # the drafts' own distribution: some that the target would have, some that it would not
        q = None
        if given:
            q = np.full_like(p, 1 / VOCAB)
            for i in range(len(flat) - 1):
                q[i, flat[i + 1]] = p[i, flat[i + 1]] * rng.choice([0.5, 3.0])
        else:
            p[np.arange(len(flat) - 1), flat[1:]] += rng.choice([0.0, 0.7], len(flat) - 1).astype(np.float32)
        u, w = rng.random(len(flat)).astype(np.float32), rng.random(len(tokens)).astype(np.float32)
        new, counts = (t.numpy() for t in F.verify_drafts(hip(p), ids(flat), ids(starts), hip(u), hip(w), draft=hip(q) if given else None))
        want = verified(p, flat, starts, u, w, q, np.full(len(flat), -1, np.int32))
        assert np.array_equal(new, want[0]) and np.array_equal(counts, want[1])
        # what was accepted stays in the cache; the next step writes over the rest
        d.lengths = [n + int(c) for n, c in zip(d.lengths, counts)]
        last = [int(new[s + c - 1]) for s, c in zip(starts, counts)]
        told += int(counts.sum()) - len(tokens)
        if turn == 2:
            d.evict(32)
    assert told > 0  # (some drafts were accepted)


def test_each_call_on_two_streams_at_once():
    """Every call that takes scratch, on two streams of different inputs without a wait between: each has what it gives alone."""
    rng = np.random.default_rng(9)
    some = lambda *s: rng.standard_normal(s).astype(np.float32)
    parts = [[tuple(map(hip, W.quantize(some(n, 512), 64, 4))) for _ in range(2)] for n in (700, 90)]
    calls = [[], []]
    for i in (0, 1):
        for rows, dtype in ((3, np.float32), (20, np.float32), (300, np.float32), (300, np.float16)):
            x = hip(some(rows + i, 512).astype(dtype))
            calls[i].append(lambda x=x, w=parts[i]: _qgemm.quantized_gated_matmul(x, *w, group_size=64, bits=4))
        vocab, n = (60000, 700)[i], 12
        p, q = (hip(rng.random((n, vocab)).astype(np.float32)) for _ in range(2))
        t, starts, u, w = ids(rng.integers(0, vocab, n)), ids([0, 5, 6, n]), hip(rng.random(n).astype(np.float32)), hip(rng.random(3).astype(np.float32))
        calls[i].append(lambda p=p, q=q, t=t, s=starts, u=u, w=w: F.verify_drafts(p, t, s, u, w, draft=q)[0])
        calls[i].append(lambda p=p, t=t, s=starts, u=u, w=w: F.verify_drafts(p, t, s, u, w)[0])
        x, r = hip(some(50 + i, 1000)), hip(some(50 + i, 1000))
        calls[i].append(lambda x=x, r=r: F.residual_norm(x, r, norm="layer", post=True)[0])
    alone = [[f().numpy() for f in c] for c in calls]
    # a cache each, compacted again and again: a row is evicted at a time
    tokens, turns = (900, 3000), 4
    caches, befores = [], []
    for i in (0, 1):
        pages = tokens[i] // PAGE + 1
        c, table = filled(rng, pages, PAGE, KV_HEADS, DIM, False, 8), ids([rng.permutation(pages)])
        want = buffers(c)
        for turn in range(turns):
            keep = np.delete(np.arange(tokens[i] - turn), turn * 7)
            want = compacted(want, PAGE, table.numpy(), keep, [0, len(keep)])
            calls[i].append(lambda c=c, t=table, k=ids(keep), s=ids([0, len(keep)]): Q.kv_cache_compact(c, t, k, s))
        caches.append(c), befores.append(want)
    streams = []
    for _ in range(2):
        s = C.c_void_p()
        _C.call("lq_stream_create", C.byref(s))
        streams.append(s)
    L.synchronize()
    prev, got = _C.current_stream(), [[], []]
    try:
        for a, b in zip(*calls):
            for i, f in enumerate((a, b)):
                _C.set_current_stream(streams[i])
                got[i].append(f())
        for s in streams:
            _C.call("lq_sync", s)
    finally:
        _C.set_current_stream(prev)
    for i in (0, 1):
        for g, want in zip(got[i], alone[i]):
            assert np.array_equal(g.numpy(), want)
        same(buffers(caches[i]), befores[i])
