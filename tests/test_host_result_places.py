"""Results that lie on what a call reads are refused, without a device: by the C entry points, whose pointers are never followed, and through the
wrappers."""

import ctypes as C

import pytest

import lucid_amd as L
import lucid_amd.nn.functional as F
from lucid_amd import _C
from test_host_decoder_step import Claimed, norm_args

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
