"""The way back of a gated block of float16: through float32, as the documents say."""

import numpy as np
import pytest

import lucid_amd as L
import lucid_amd.nn as nn
import lucid_amd.nn.functional as F
import lucid_amd.nn.quantized as nnq
import oracle.wq_group as W
from test_hip_wq_gated import bound, hip, weight64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 9, 70])
def test_a_float16_block_goes_back_through_float32(rows):
    gate, up, down = nn.Linear(256, 672), nn.Linear(256, 672, bias=False), nn.Linear(672, 256)
    m, back = nnq.QuantizedGatedLinearMLX.from_float(gate, up, bits=4, group_size=32), nnq.QuantizedLinearMLX.from_float(down, bits=8, group_size=32)
    rng = np.random.default_rng(rows)
    x, r = rng.standard_normal((rows, 256)).astype(np.float16), rng.standard_normal((rows, 256)).astype(np.float32)
    h = m(hip(x))
    assert h.dtype is L.float16
    want, e = bound(x.astype(np.float64), [W.quantize(lin.weight.numpy(), 32, 4) for lin in (gate, up)], 32, 4, "silu", [gate.bias.numpy(), np.zeros(672)])
    assert (abs(h.numpy() - want) <= e + (abs(want) + e) * 2.0 ** -11 + 2.0 ** -25).all()
    with pytest.raises(L.DtypeMismatch):
        back(h)
    o = back(h.to(L.float32))
    w = weight64(*W.quantize(down.weight.numpy(), 32, 8), 32, 8)
    assert (abs(o.numpy() - (h.numpy().astype(np.float64) @ w.T + down.bias.numpy())) <= 1e-4 * max(1.0, abs(o.numpy()).max())).all()
    y, s = F.residual_norm(o, hip(r))
    want = (o.numpy() + r).astype(np.float64)
    assert np.array_equal(s.numpy(), o.numpy() + r)
    assert (abs(y.numpy() * np.sqrt((want ** 2).mean(-1, keepdims=True) + 1e-6) - want) <= 2.0 ** -20 * abs(want) + 1e-30).all()
