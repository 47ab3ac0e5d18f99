"""How far attention over the pages may be off, row by row: a row is held to what it sees itself."""

import numpy as np
import pytest

from test_hip_paged_attention import Batch

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
