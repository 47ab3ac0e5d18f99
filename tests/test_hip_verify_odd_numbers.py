"""Verified drafts at the numbers that are no probabilities, acceptance and drawing told apart, and of no rows."""

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn.functional as F
from test_hip_verify_drafts import hip

pytestmark = pytest.mark.gpu
INF, NAN = np.inf, np.nan


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [5, 40, 9000])
@pytest.mark.parametrize("u,p,q,accepted", [(0.5, INF, 0.25, True), (0.5, INF, INF, False), (0.0, INF, INF, False), (0.5, NAN, 0.25, False), (0.5, 0.25, NAN, False),
                                            (0.5, 0.25, INF, False), (0.5, 0.0, -1.0, True), (0.0, 0.0, -1.0, False), (0.5, -0.5, -2.0, True), (0.5, -INF, 0.25, False),
                                            (0.5, 0.25, -INF, True)])
def test_acceptance_compares_the_numbers_as_they_are_and_drawing_counts_them_as_nothing(dtype, vocab, u, p, q, accepted):
    """A sequence of one draft, token 3, and rows of 0 but at tokens 3 and 4: refused, or behind it, the token drawn is the only one of positive finite weight."""
    target, draft = np.zeros((2, vocab), dtype), np.zeros((2, vocab), dtype)
    target[0, 3], draft[0, 3], target[0, 4], target[1, 2], target[1, 1] = p, q, 0.125, 0.5, NAN
    args = [hip(target), hip([0, 3], np.int32), hip([0, 2], np.int32), hip([u, 0], np.float32), hip([0.75], np.float32)]
    new, counts = F.verify_drafts(*args, draft=hip(draft))
    if accepted:
        assert new.numpy().tolist() == [3, 2] and counts.numpy().tolist() == [2]
        return
    # what is left of p - q: token 4, and where q counts as nothing a p of 0.25 at token 3, which 0.75 of the sum 0.375 passes
    assert new.numpy().tolist() == [4, -1] and counts.numpy().tolist() == [1]


def test_drafts_of_no_rows():
    """A step in which no sequence has a token, results given or not."""
    ids, f32 = lambda n: L.tensor(np.zeros(n, np.int32), device="hip"), lambda *s: L.tensor(np.zeros(s, np.float32), device="hip")
    for batch in (0, 3):
        for out in (None, (ids(0), L.tensor(np.full(batch, 9, np.int32), device="hip"))):
            new, counts = F.verify_drafts(f32(0, 50), ids(0), ids(batch + 1), f32(0), f32(batch), out=out)
            assert new.shape == (0,) and counts.numpy().tolist() == [0] * batch
