"""Gated projections at shapes of which it is asserted that they go to the kernel of many rows: every tile on exact numbers, all activations against float64, rows of
all sizes, views, two streams, calls of several chunks."""

import ctypes as C

import numpy as np
import pytest

import lucid_amd as L
import oracle.wq_group as W
from lucid_amd import _C
from lucid_amd.quantization import _qgemm
from test_hip_wq_gated import ACTS, bound, exact_numbers, hip, some_columns, weight64
from test_host_gated import MORE, tile

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of float32, relative


def many(M, N, K, bits, dtype):
    return tile(M, N, K, bits, _C.F16 if dtype is np.float16 else _C.F32)[0] == 1


@pytest.mark.parametrize("M,N,K,gs", MORE)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_tiles_that_few_shapes_have(M, N, K, gs, bits, dtype):
    exact_numbers(M, N, K, gs, bits, dtype, some_columns(N))


@pytest.mark.parametrize("dtype,M,N,K,gs", [(np.float32, 333, 8200, 1152, 128), (np.float32, 340, 9000, 160, 32), (np.float32, 399, 4892, 1088, 64),
                                            (np.float16, 333, 8200, 1152, 128), (np.float16, 325, 11009, 160, 32), (np.float16, 670, 4475, 640, 64)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("biases", [(True, True), (True, False), (False, True)])
def test_activations_and_biases(dtype, M, N, K, gs, bits, act, biases):
    assert many(M, N, K, bits, dtype)
    rng = np.random.default_rng(M + bits)
    x = (rng.standard_normal((M, K)) * (1 + 9 * (rng.random(K) < 0.02)) + 0.3).astype(dtype)
    parts = [W.quantize((0.03 * rng.standard_normal((N, K))).astype(np.float32), gs, bits) for _ in range(2)]
    bias = [(0.2 * rng.standard_normal(N)).astype(np.float32) if b else None for b in biases]
    y = _qgemm.quantized_gated_matmul(hip(x), *(tuple(map(hip, p)) for p in parts), act, gs, bits, *(None if b is None else hip(b) for b in bias)).numpy()
    cols = some_columns(N)
    want, e = bound(x.astype(np.float64), [tuple(a[cols] for a in p) for p in parts], gs, bits, act, [np.zeros(len(cols)) if b is None else b[cols] for b in bias])
    info = np.finfo(dtype)
    assert (abs(y[:, cols] - want) <= e + (abs(want) + e) * info.eps / 2 + info.tiny * info.eps).all()


@pytest.mark.parametrize("M,N,K,gs", [(340, 9000, 160, 32), (333, 8200, 1152, 128), (399, 4892, 1088, 64)])
@pytest.mark.parametrize("bits", [4, 8])
def test_rows_of_all_sizes_side_by_side(M, N, K, gs, bits):
    """Each float32 row keeps its own bits: rows of 1e-15 to 1e15, of zeros, of numbers next to nothing, with one value far above the others."""
    assert many(M, N, K, bits, np.float32)
    rng = np.random.default_rng(M)
    x = rng.standard_normal((M, K)) * 10.0 ** rng.integers(-15, 16, (M, 1))
    x[0], x[M - 1], x[1, 7], x[M // 2, K - 1], x[5] = 0, 0, 3e4 * abs(x[1]).max(), 3e4 * abs(x[M // 2]).max(), 2.0 ** -149
    x = x.astype(np.float32)
    parts = [W.quantize((0.03 * rng.standard_normal((N, K))).astype(np.float32), gs, bits) for _ in range(2)]
    y = _qgemm.quantized_gated_matmul(hip(x), *(tuple(map(hip, p)) for p in parts), "relu", gs, bits).numpy()
    cols = some_columns(N)
    want, e = bound(x.astype(np.float64), [tuple(a[cols] for a in p) for p in parts], gs, bits, "relu", [np.zeros(len(cols))] * 2)
    assert (abs(y[:, cols] - want) <= e + abs(want) * U + 2.0 ** -149).all()


@pytest.mark.parametrize("dtype,M,N,K,gs", [(np.float32, 340, 9000, 160, 32), (np.float32, 399, 4892, 1088, 64), (np.float16, 325, 11009, 160, 32), (np.float16, 670, 4475, 640, 128)])
@pytest.mark.parametrize("bits", [4, 8])
def test_rows_out_of_the_middle(dtype, M, N, K, gs, bits):
    """Weights that are some rows of larger ones, whose scales lie at any multiple of four bytes; x and the result likewise."""
    assert many(M, N, K, bits, dtype)
    rng = np.random.default_rng(M + K)
    parts = [W.quantize(rng.standard_normal((N + 9, K)).astype(np.float32), gs, bits) for _ in range(2)]
    x = rng.standard_normal((M + 3, K)).astype(dtype)
    want = _qgemm.quantized_gated_matmul(hip(x[1:M + 1]), *[tuple(hip(p[5:N + 5]) for p in w) for w in parts], "sigmoid", gs, bits).numpy()
    filled = np.full((M + 2, N), 7, dtype)
    out = hip(filled)
    _qgemm.quantized_gated_matmul(hip(x).row_range(1, M + 1), *[tuple(hip(p).row_range(5, N + 5) for p in w) for w in parts], "sigmoid", gs, bits,
                                  out=out.row_range(1, M + 1))
    filled[1:M + 1] = want
    assert np.array_equal(out.numpy(), filled)


def test_on_two_streams_at_once():
    """The operands that a call lays out are its stream's: calls of different sizes on two streams without a wait between, each with what it gives alone."""
    rng = np.random.default_rng(3)
    shapes = [(np.float32, 340, 9000, 160, 32), (np.float16, 333, 8200, 1152, 128), (np.float32, 333, 8200, 1152, 128), (np.float16, 325, 11009, 160, 32)]
    made = []
    for dtype, M, N, K, gs in shapes:
        assert many(M, N, K, 4, dtype)
        made.append((hip(rng.standard_normal((M, K)).astype(dtype)), [tuple(map(hip, W.quantize(rng.standard_normal((N, K)).astype(np.float32), gs, 4))) for _ in range(2)], gs))
    call = lambda i: _qgemm.quantized_gated_matmul(made[i][0], *made[i][1], "gelu", made[i][2], 4)
    alone = [call(i).numpy() for i in range(4)]
    orders, got = ([0, 1, 2, 3] * 3, [2, 3, 1, 0] * 3), [[], []]
    streams = []
    for _ in range(2):
        s = C.c_void_p()
        _C.call("lq_stream_create", C.byref(s))
        streams.append(s)
    L.synchronize()
    prev = _C.current_stream()
    try:
        for a, b in zip(*orders):
            for i, which in enumerate((a, b)):
                _C.set_current_stream(streams[i])
                got[i].append(call(which))
        for s in streams:
            _C.call("lq_sync", s)
    finally:
        _C.set_current_stream(prev)
    for i in (0, 1):
        for which, y in zip(orders[i], got[i]):
            assert np.array_equal(y.numpy(), alone[which])


def test_replayed_from_two_graphs_beside_eager_calls():
    rng = np.random.default_rng(4)
    graphs = []
    for dtype, M, N, K, gs in ((np.float32, 340, 9000, 160, 32), (np.float16, 670, 4475, 640, 64)):
        assert many(M, N, K, 4, dtype)
        parts = [tuple(map(hip, W.quantize(rng.standard_normal((N, K)).astype(np.float32), gs, 4))) for _ in range(2)]
        x = hip(rng.standard_normal((M, K)).astype(dtype))
        call = lambda x=x, parts=parts, gs=gs: _qgemm.quantized_gated_matmul(x, *parts, group_size=gs, bits=4)
        call()
        with L.graph.capture() as g:
            y = call()
        graphs.append((g, x, y, call))
    for _ in range(3):
        for g, x, y, call in graphs:
            x.copy_from(rng.standard_normal(x.shape).astype(x.dtype.np))
            g.replay()
            want = call().numpy()
            L.synchronize()
            assert np.array_equal(y.numpy(), want)


# more rows than a launch has of either kernel: 2^29 values of float16, 2^28 of float32 of the one, 2^28 values of the other's
@pytest.mark.parametrize("dtype,M,N,K,to_many", [(np.float32, 70000, 130, 4096, True), (np.float16, 140000, 70, 4096, True), (np.float32, 280000, 20, 1024, False),
                                                 (np.float16, 33000, 40, 8192, False)])
def test_rows_in_several_chunks(dtype, M, N, K, to_many):
    """Small whole numbers, as in exact_numbers, of a block of rows again and again: a row that a chunk leaves out or takes from elsewhere shows."""
    assert many(M, N, K, 4, dtype) == to_many and M * K > (1 << (29 if dtype is np.float16 and to_many else 28))
    rng = np.random.default_rng(5)
    block, parts, proj = rng.integers(-3, 4, (1009, K)).astype(dtype), [], []
    block[rng.random(block.shape) < 0.7] = 0
    for scale in (1.0, 2.0 ** -6):
        packed = rng.integers(0, 1 << 32, (N, K // 8), dtype=np.uint64).astype(np.uint32).view(np.int32)
        s = np.full((N, K // 128), scale, np.float32)
        b = (-8 * s + scale * rng.integers(-2, 3, s.shape)).astype(np.float32)
        parts.append(tuple(map(hip, (packed, s, b))))
        proj.append(block.astype(np.float64) @ weight64(packed, s, b, 128, 4).T)
        assert abs(proj[-1]).max() < 2 ** 18 * scale
    with np.errstate(over="ignore"):
        want = (np.maximum(proj[0], 0) * proj[1]).astype(np.float32).astype(dtype)
    rows = np.arange(M) % 1009
    y = _qgemm.quantized_gated_matmul(hip(np.tile(block, (-(-M // 1009), 1))[:M]), *parts, "relu", 128, 4)
    assert np.array_equal(y.numpy(), want[rows])
