"""``QuantizedLinearMLX`` (``lucid/nn/quantized/mlx_linear.py:21-200``): a Linear whose
weight is group-wise int4 / int8 packed and decoded inside the matmul.  The name is
Lucid's; on this backend the kernels are HIP.  Buffers as in Lucid:
``packed_weight`` int32 ``(out, in*bits/32)``, ``scales`` / ``biases`` float32
``(out, in/group_size)``, ``bias`` float32 ``(out,)`` or None; attributes ``bits``,
``group_size``, ``relu``.
"""

from __future__ import annotations

import numpy as np

from ... import _C
from ... import _tensor as T
from ..._tensor import Tensor
from ...quantization import _qgemm
from ..module import Module


class QuantizedLinearMLX(Module):
    def __init__(self, in_features: int, out_features: int, bias: bool = True, bits: int = 8,
                 group_size: int = 64, relu: bool = False) -> None:
        super().__init__()
        if bits not in (4, 8):
            raise ValueError(f"bits must be 4 or 8, got {bits}")
        if in_features % group_size:
            raise ValueError(f"group_size {group_size} must divide in_features {in_features}")
        self.in_features, self.out_features = in_features, out_features
        self.bits, self.group_size, self.relu = bits, group_size, relu
        self.register_buffer("packed_weight", T.tensor(
            np.zeros((out_features, in_features * bits // 32), np.int32), device="hip"))
        g = in_features // group_size
        self.register_buffer("scales", T.tensor(np.zeros((out_features, g), np.float32), device="hip"))
        self.register_buffer("biases", T.tensor(np.zeros((out_features, g), np.float32), device="hip"))
        self.register_buffer("bias", T.tensor(np.zeros(out_features, np.float32), device="hip") if bias else None)

    def forward(self, x: Tensor) -> Tensor:
        if not isinstance(x, Tensor) or x.device != "hip":
            raise _C.DeviceMismatch("QuantizedLinearMLX: input must be a tensor on the 'hip' device")
        y = _qgemm.quantized_matmul(x, self.packed_weight, self.scales, self.biases, transpose=True,
                                    group_size=self.group_size, bits=self.bits)
        if self.bias is not None or self.relu:
            M = y.numel // self.out_features
            _C.call("lq_bias_act_f32", y.data_ptr, self.bias.data_ptr if self.bias is not None else None,
                    M, self.out_features, int(self.relu), None)
        return y

    @classmethod
    def from_float(cls, mod, bits: int = 8, group_size: int = 64, relu: bool = False) -> "QuantizedLinearMLX":
        """Pack a float ``Linear``'s weight (``mlx_linear.py`` ``from_float``)."""
        q = cls(mod.in_features, mod.out_features, bias=mod.bias is not None, bits=bits,
                group_size=group_size, relu=relu)
        packed, scales, biases = _qgemm.quantize(mod.weight.to("hip"), group_size, bits)
        q.register_buffer("packed_weight", packed)
        q.register_buffer("scales", scales)
        q.register_buffer("biases", biases)
        if mod.bias is not None:
            q.register_buffer("bias", mod.bias.to("hip"))
        return q

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bits={self.bits}, "
                f"group_size={self.group_size}")


class QuantizedGatedLinearMLX(Module):
    """Both projections of a gated feed-forward block, ``act(gate(x)) * up(x)``, on group-wise int4 / int8 weights in one call
    (``_qgemm.quantized_gated_matmul``).  Buffers: ``gate_packed_weight``, ``gate_scales``, ``gate_biases``, ``gate_bias`` and the same of ``up``, each as
    ``QuantizedLinearMLX`` has it.  ``x`` is float32 or float16, and the result has its type.  A ``QuantizedLinearMLX`` takes a float32 result back, as the
    Linears of this package are float32; a float16 one goes through ``.to(float32)`` first."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, bits: int = 8, group_size: int = 64,
                 activation: str = "silu") -> None:
        super().__init__()
        if bits not in (4, 8):
            raise ValueError(f"bits must be 4 or 8, got {bits}")
        if group_size not in (32, 64, 128):
            raise ValueError(f"group_size must be 32, 64 or 128, got {group_size}")
        if in_features % group_size:
            raise ValueError(f"group_size {group_size} must divide in_features {in_features}")
        if activation not in _qgemm._GATES:
            raise ValueError(f"activation must be one of {', '.join(_qgemm._GATES)}, got {activation!r}")
        self.in_features, self.out_features = in_features, out_features
        self.bits, self.group_size, self.activation = bits, group_size, activation
        zeros = lambda shape, dt: T.tensor(np.zeros(shape, dt), device="hip")
        for name in ("gate", "up"):
            self.register_buffer(f"{name}_packed_weight", zeros((out_features, in_features * bits // 32), np.int32))
            self.register_buffer(f"{name}_scales", zeros((out_features, in_features // group_size), np.float32))
            self.register_buffer(f"{name}_biases", zeros((out_features, in_features // group_size), np.float32))
            self.register_buffer(f"{name}_bias", zeros(out_features, np.float32) if bias else None)

    def forward(self, x: Tensor) -> Tensor:
        return _qgemm.quantized_gated_matmul(x, (self.gate_packed_weight, self.gate_scales, self.gate_biases),
                                             (self.up_packed_weight, self.up_scales, self.up_biases), self.activation, self.group_size, self.bits,
                                             self.gate_bias, self.up_bias)

    @classmethod
    def from_float(cls, gate, up, bits: int = 8, group_size: int = 64, activation: str = "silu") -> "QuantizedGatedLinearMLX":
        """Pack the weights of two float ``Linear`` of one shape."""
        if (gate.in_features, gate.out_features) != (up.in_features, up.out_features):
            raise _C.ShapeMismatch(f"gate is {gate.in_features} -> {gate.out_features}, up {up.in_features} -> {up.out_features}")
        q = cls(gate.in_features, gate.out_features, bias=gate.bias is not None or up.bias is not None, bits=bits, group_size=group_size,
                activation=activation)
        for name, mod in (("gate", gate), ("up", up)):
            for part, t in zip(("packed_weight", "scales", "biases"), _qgemm.quantize(mod.weight.to("hip"), group_size, bits)):
                q.register_buffer(f"{name}_{part}", t)
            if mod.bias is not None:
                q.register_buffer(f"{name}_bias", mod.bias.to("hip"))
        return q

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bits={self.bits}, group_size={self.group_size}, "
                f"activation={self.activation}")
