"""Gated projections without a device: what their module refuses."""

import pytest

import lucid_amd.nn as nn
import lucid_amd.nn.quantized as nnq


@pytest.mark.parametrize("group_size", [0, 1, 16, 48, 256, -32])
def test_the_module_refuses_groups_that_its_forward_does_not_take(group_size):
    with pytest.raises(ValueError, match="group_size must be 32, 64 or 128"):
        nnq.QuantizedGatedLinearMLX(768, 8, group_size=group_size)
    with pytest.raises(ValueError, match="group_size must be 32, 64 or 128"):
        nnq.QuantizedGatedLinearMLX.from_float(nn.Linear(768, 8), nn.Linear(768, 8), group_size=group_size)
