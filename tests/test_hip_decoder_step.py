"""A decoder's attention block as a program runs it, prompts in chunks and then token by token: a qkv Linear, quantization.kv_cache_write_qkv,
functional.paged_attention_qkv, an output Linear, against the block in float64."""

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn as nn
import lucid_amd.nn.functional as F
import lucid_amd.quantization as Q
import oracle.kv_cache as K
from test_hip_kv_cache import DTYPES, SCHEMES, hip, ids

pytestmark = pytest.mark.gpu


class Block:
    """The block, its pages and the tokens of two sequences so far."""

    def __init__(self, heads, kv_heads, dim, page, bits, symmetric, window):
        self.rng = np.random.default_rng(heads * dim + bits)
        self.heads, self.kv_heads, self.dim, self.page, self.bits, self.symmetric, self.window = heads, kv_heads, dim, page, bits, symmetric, window
        self.width, out = heads * dim, (heads + 2 * kv_heads) * dim
        self.qkv, self.proj = nn.Linear(self.width, out), nn.Linear(self.width, self.width)
        self.cache = Q.PagedKVCache(14, page, kv_heads, dim, SCHEMES[symmetric], DTYPES[bits])
        self.free, self.tables, self.rows = list(self.rng.permutation(14)), [[], []], [[], []]

    def step(self, counts, padding):
        """`counts` new tokens of the sequences and `padding` rows behind them -> what the block gives for all of them, and the packed rows."""
        x = (3 * self.rng.standard_normal((sum(counts) + padding, self.width))).astype(np.float32)
        slots = []
        for b, n in enumerate(counts):
            for place in range(len(self.rows[b]), len(self.rows[b]) + n):
                if place // self.page == len(self.tables[b]):
                    self.tables[b].append(int(self.free.pop()))
                slots.append(self.tables[b][place // self.page] * self.page + place % self.page)
        slots += [-1] * padding
        table = np.full((2, max(map(len, self.tables))), -1, np.int32)
        for b, t in enumerate(self.tables):
            table[b, :len(t)] = t
        packed = self.qkv(hip(x))
        host = packed.numpy()
        at = 0
        for b, n in enumerate(counts):
            self.rows[b] += list(host[at:at + n])
            at += n
        Q.kv_cache_write_qkv(self.cache, packed, self.heads, ids(slots))
        y = F.paged_attention_qkv(packed, self.heads, self.cache, ids(table), ids(np.cumsum([0] + counts)), ids([len(r) for r in self.rows]),
                                  window=self.window, max_chunk=max(counts))
        return host, y.numpy(), self.proj(y).numpy()

    def want(self, host, counts):
        """The block in float64, each token over its sequence's rows, quantized as the cache has them -> the result and a bound of its error."""
        y, bound = np.zeros((len(host), self.width)), 0.0
        group, at = self.heads // self.kv_heads, 0
        for b, n in enumerate(counts):
            rows = np.array(self.rows[b], np.float32).reshape(len(self.rows[b]), self.heads + 2 * self.kv_heads, self.dim)
            k, v = (K.values(K.pack(u, self.bits), s, z, self.bits).astype(np.float64)
                    for u, s, z in (K.quantize(np.ascontiguousarray(part), self.bits, self.symmetric)
                                    for part in (rows[:, self.heads:self.heads + self.kv_heads], rows[:, self.heads + self.kv_heads:])))
            for i in range(n):
                here = len(rows) - n + i
                lo = max(0, here - self.window + 1) if self.window else 0
                q = rows[here, :self.heads].astype(np.float64).reshape(self.kv_heads, group, self.dim)
                keys, values = k[lo:here + 1].transpose(1, 2, 0), v[lo:here + 1].transpose(1, 0, 2)
                s = q @ keys / np.sqrt(self.dim)
                p = np.exp(s - s.max(-1, keepdims=True))
                y[at + i] = (p / p.sum(-1, keepdims=True) @ values).reshape(-1)
                # a score is a sum of dim products in float32, of partial sums below `a` (4 deviations), of a query of 22 bits; scale, maximum and
                # exponential round 8 units of 1 + |score|; a probability off by e moves the result by 2 e max|v|; sums of n terms add sqrt(n)
                a, top = (abs(q) @ abs(keys)).max() / np.sqrt(self.dim), abs(values).max()
                e = 2.0 ** -24 * (4 * np.sqrt(self.dim) * a + 2 * a + 8 * (1 + abs(s).max()))
                bound = max(bound, 2 * e * top + 4 * np.sqrt(here + 1) * 2.0 ** -24 * top)
            at += n
        return y, bound


@pytest.mark.parametrize("heads,kv_heads,dim,page,bits,symmetric,window", [
    (4, 2, 64, 16, 8, True, None), (6, 1, 32, 48, 8, False, 50), (4, 4, 64, 32, 4, False, None), (8, 2, 128, 64, 4, True, 33)])
def test_prompts_in_chunks_then_token_by_token(heads, kv_heads, dim, page, bits, symmetric, window):
    block = Block(heads, kv_heads, dim, page, bits, symmetric, window)
    weight, bias = block.proj.weight.numpy().astype(np.float64), block.proj.bias.numpy().astype(np.float64)
    # a chunk each, one of a sequence beside a token of the other, neither, tokens with padding behind them, two at a time
    for counts, padding in (([60, 37], 0), ([1, 70], 3), ([0, 1], 0), ([1, 1], 0), ([1, 0], 5), ([2, 2], 1), ([1, 1], 0)):
        host, y, out = block.step(counts, padding)
        want, bound = block.want(host, counts)
        assert np.abs(y - want).max() <= bound
        assert not y[sum(counts):].any()
        # the Linear: a sum of `width` products in float32 of rows that are off by the bound
        lin = want @ weight.T + bias
        assert np.abs(out - lin).max() <= (bound + 2.0 ** -24 * (np.sqrt(block.width) + 2) * 4 * np.abs(want).max()) * np.abs(weight).sum(1).max() + 2.0 ** -23


def test_results_in_a_tensors_place_leave_nothing_of_what_it_was():
    """A tensor that kept the range of what it held, or its codes on a grid, is the new result alone afterwards: what quantizes it next goes by the new
    values."""
    from lucid_amd._tensor import Grid

    rng = np.random.default_rng(1)
    cache = Q.PagedKVCache(2, 16, 2, 64)
    k, v, q = (hip(rng.standard_normal((20, h, 64)).astype(np.float32)) for h in (2, 2, 4))
    slots, table, starts, lens = ids(np.arange(20)), ids([[0, 1]]), ids([0, 20]), ids([20])
    Q.kv_cache_write(cache, k, v, slots)
    lin = nn.quantized.dynamic.Linear.from_float(nn.Linear(64, 64))

    def small(*shape):  # values of 1e-3 with their range
        return F.gelu(hip(np.full(shape, 1e-3, np.float32)), track_range=True)

    def on_grid(*shape):
        one = lambda a: hip(np.asarray(a))
        return L.Tensor.on_grid(shape, Grid(one(np.ones(shape, np.int8)), one(np.float32(1e-3)), one(np.float32(0)), Q.qint8, 0))

    for make in (small, on_grid):
        out = make(20, 4, 64)
        F.paged_attention(q, cache, table, starts, lens, out=out)
        pair = make(20, 2, 64), make(20, 2, 64)
        Q.kv_cache_read(cache, slots, out=pair)
        for y in (out, *pair):
            assert y._range is None and y._grid is None
            assert np.array_equal(lin(y).numpy(), lin(hip(y.numpy())).numpy())
        assert np.array_equal(out.numpy(), F.paged_attention(q, cache, table, starts, lens).numpy())
        assert all(np.array_equal(a.numpy(), b.numpy()) for a, b in zip(pair, Q.kv_cache_read(cache, slots)))
