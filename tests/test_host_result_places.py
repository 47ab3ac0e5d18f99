"""Results that lie on what a call reads are refused, without a device: by the C entry points, whose pointers are never followed, and through the
wrappers."""

import pytest

import lucid_amd as L
import lucid_amd.nn.functional as F
from lucid_amd import _C
from lucid_amd.quantization import _qgemm
from test_host_decoder_step import Claimed, gated_args, norm_args

VECTORS = ("scale", "weight", "bias", "post_weight", "post_bias")


# ---------------------------------------------------------------- residual norm: 2 rows of 8 float32 are 0x40 bytes, a vector 0x20
@pytest.mark.parametrize("vector", VECTORS)
@pytest.mark.parametrize("result", ["y", "r_out"])
@pytest.mark.parametrize("at", [0x7000, 0x7020, 0x703c, 0x6fe4])
def test_c_residual_norm_refuses_results_on_its_vectors(vector, result, at):
    places = {"x": 0x1000, "r": 0x2000, "y": 0x3000, "r_out": 0x4000, "post": 1, result: 0x7000, vector: at}
    with pytest.raises(ValueError, match="residual_norm: a result lies"):
        _C.call("lq_residual_norm", norm_args(**places), None)


@pytest.mark.parametrize("vector", VECTORS)
@pytest.mark.parametrize("result", ["out", "residual_out"])
def test_residual_norm_of_one_row_refuses_results_in_a_vectors_place(vector, result):
    x, r, v = Claimed((1, 8), ptr=0x1000), Claimed((1, 8), ptr=0x2000), Claimed((8,), ptr=0x7000)
    places = {"out": Claimed((1, 8), ptr=0x3000), "residual_out": Claimed((1, 8), ptr=0x4000), result: Claimed((1, 8), ptr=0x7000)}
    with pytest.raises(ValueError, match="residual_norm: a result lies"):
        F.residual_norm(x, r, post=True, **{vector: v}, **places)


def test_rms_norm_refuses_its_weights_place():
    with pytest.raises(ValueError, match="residual_norm: a result lies"):
        F.rms_norm(Claimed((1, 8), ptr=0x1000), 8, Claimed((8,), ptr=0x7000), out=Claimed((1, 8), ptr=0x7000))


# ---------------------------------------------------------------- drafts: 4 rows of 100 float32, 2 sequences
READ = {"target": (0, 0x10000, 4 * 100 * 4), "draft": (1, 0x20000, 4 * 100 * 4), "tokens": (5, 0x30000, 16), "starts": (6, 0x40000, 12), "uniforms": (8, 0x50000, 16),
        "last": (9, 0x60000, 8)}


def verify_call(**kw):
    args = [0x10000, 0x20000, _C.F32, 4, 100, 0x30000, 0x40000, 2, 0x50000, 0x60000, 0x70000, 0x80000, None]
    for at, value in kw.values():
        args[at] = value
    _C.call("lq_verify_drafts", *args)


@pytest.mark.parametrize("what", list(READ))
@pytest.mark.parametrize("result,size", [(10, 16), (11, 8)])
def test_c_verify_refuses_results_on_what_is_read(what, result, size):
    _, at, n = READ[what]
    for place in (at, at + n - 4, at - size + 4):
        with pytest.raises(ValueError, match="verify_drafts: a result lies"):
            verify_call(result=(result, place))


@pytest.mark.parametrize("at", [0x70000, 0x7000c, 0x6fffc])
def test_c_verify_refuses_one_result_on_the_other(at):
    with pytest.raises(ValueError, match="verify_drafts: a result lies"):
        verify_call(counts=(11, at))


def test_verify_refuses_rows_beside_those_that_are_read():
    """Rows of one tensor for the drafted and the new tokens, of another for starts and counts."""
    i32 = L.int32
    t = dict(target=Claimed((4, 100), ptr=0x10000), tokens=Claimed((4,), i32, 0x30000), starts=Claimed((3,), i32, 0x40000), uniforms=Claimed((4,), ptr=0x50000),
             last_uniforms=Claimed((2,), ptr=0x60000))
    new, counts = Claimed((4,), i32, 0x70000), Claimed((2,), i32, 0x80000)
    for out in ((Claimed((4,), i32, 0x30004), counts), (Claimed((4,), i32, 0x2fff8), counts), (new, Claimed((2,), i32, 0x40008)), (new, Claimed((2,), i32, 0x70008))):
        with pytest.raises(ValueError, match="verify_drafts: a result lies"):
            F.verify_drafts(**t, out=out)


# ---------------------------------------------------------------- gated projections: 2 x 8 float32 of K = 64 in 4 bits, groups of 32
OPERANDS = {"x": (0x10000, 2 * 64 * 4), "packed": (0x20000, 8 * 32), "scales": (0x30000, 8 * 2 * 4), "biases": (0x40000, 8 * 2 * 4), "bias": (0x50000, 8 * 4)}


def gated_places():
    """Where each operand lies: the gate's, and the way up's 0x8000 behind."""
    return {n: at if n == "x" else (at, at + 0x8000) for n, (at, _) in OPERANDS.items()}


@pytest.mark.parametrize("what,second", [("x", False)] + [(n, s) for n in list(OPERANDS)[1:] for s in (False, True)])
def test_c_gated_refuses_a_result_on_what_is_read(what, second):
    at, size = OPERANDS[what][0] + 0x8000 * second, OPERANDS[what][1]
    for place in (at, at + size - 4, at - 2 * 8 * 4 + 4):
        with pytest.raises(ValueError, match="quantized_gated_matmul: the result cannot"):
            _C.call("lq_wq_gated_matmul", gated_args(**gated_places(), out=place), None)


@pytest.mark.parametrize("bias", ["gate_bias", "up_bias"])
def test_gated_refuses_a_result_in_a_biass_place(bias):
    at = lambda base: (Claimed((8, 8), L.int32, base), Claimed((8, 2), ptr=base + 0x1000), Claimed((8, 2), ptr=base + 0x2000))
    with pytest.raises(ValueError, match="quantized_gated_matmul: the result cannot"):
        _qgemm.quantized_gated_matmul(Claimed((1, 64), ptr=0x10000), at(0x20000), at(0x30000), group_size=32, bits=4, out=Claimed((1, 8), ptr=0x40000),
                                      **{bias: Claimed((8,), ptr=0x40000)})
