"""nn.RMSNorm as a program has it: made on the host, called again and again, captured."""

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn as nn
import lucid_amd.nn.functional as F

pytestmark = pytest.mark.gpu


def test_its_weight_goes_to_the_device_once():
    rng = np.random.default_rng(0)
    m, w = nn.RMSNorm(96), (1 + 0.2 * rng.standard_normal(96)).astype(np.float32)
    m.load_state_dict({"weight": L.tensor(w)})
    x = L.tensor(rng.standard_normal((7, 96)).astype(np.float32), device="hip")
    want = F.rms_norm(x, 96, L.tensor(w, device="hip")).numpy()
    assert np.array_equal(m(x).numpy(), want)
    at = m.weight.data_ptr
    assert m.weight.device == "hip" and np.array_equal(m.state_dict()["weight"].numpy(), w)
    assert np.array_equal(m(x).numpy(), want) and m.weight.data_ptr == at
    F.residual_norm(x, x, m.weight, eps=m.eps)
    # other numbers, of the host, in its place
    m.load_state_dict({"weight": L.tensor(2 * w)})
    assert np.array_equal(m(x).numpy(), 2 * want)
    m.register_buffer("weight", L.tensor(w))
    assert np.array_equal(m(x).numpy(), want)


def test_captured_after_a_call():
    rng = np.random.default_rng(1)
    m = nn.RMSNorm(640)
    x = L.tensor(rng.standard_normal((5, 640)).astype(np.float16), device="hip")
    m(x)
    with L.graph.capture() as g:
        y = m(x)
    for _ in range(3):
        x.copy_from(rng.standard_normal((5, 640)).astype(np.float16))
        g.replay()
        L.synchronize()
        assert np.array_equal(y.numpy(), m(x).numpy())
