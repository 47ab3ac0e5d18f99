"""Group-wise weight-only int4 / int8 (``lucid/quantization/_qgemm.py:24-320``):
``quantize`` packs a float weight, ``dequantize`` inverts it, ``quantized_matmul``
contracts a float activation against the packed weight.  Lucid runs these on MLX
(Metal); here they are HIP kernels with the same signatures, defaults and shapes.
The packed tensor is int32-tagged (Lucid has no uint32 dtype either,
``QuantizedMatmul.cpp:53-63``).
"""

from __future__ import annotations

from .. import _C
from .. import _tensor as T
from .._tensor import Tensor


def is_available() -> bool:
    """True when the HIP library and a device are present (``_qgemm.py:24-66``)."""
    return _C.is_available()


def _check(name: str, *ts: Tensor) -> None:
    for t in ts:
        if not isinstance(t, Tensor) or t.device != "hip":
            raise _C.DeviceMismatch(f"{name}: operands must be tensors on the 'hip' device")


def quantize(w: Tensor, group_size: int = 64, bits: int = 8) -> tuple[Tensor, Tensor, Tensor]:
    """``(packed_weight, scales, biases)`` of a float32 ``(out, in)`` weight."""
    _check("quantize", w)
    if w.dtype != T.float32 or w.ndim != 2:
        raise _C.DtypeMismatch(f"quantize expects a 2-d float32 weight, got {w.dtype} {w.shape}")
    N, K = w.shape
    packed = Tensor.empty((N, K * bits // 32), T.int32, "hip")
    scales = Tensor.empty((N, K // group_size), T.float32, "hip")
    biases = Tensor.empty((N, K // group_size), T.float32, "hip")
    _C.call("lq_wq_quantize", w.data_ptr, N, K, int(group_size), int(bits), packed.data_ptr,
            scales.data_ptr, biases.data_ptr, None)
    return packed, scales, biases


def dequantize(wq: Tensor, scales: Tensor, biases: Tensor, group_size: int = 64, bits: int = 8) -> Tensor:
    """Float32 ``(out, in)`` weight ``c * s + beta``."""
    _check("dequantize", wq, scales, biases)
    N = wq.shape[0]
    K = wq.shape[1] * 32 // bits
    out = Tensor.empty((N, K), T.float32, "hip")
    _C.call("lq_wq_dequantize", wq.data_ptr, scales.data_ptr, biases.data_ptr, N, K, int(group_size),
            int(bits), out.data_ptr, None)
    return out


def quantized_matmul(x: Tensor, wq: Tensor, scales: Tensor, biases: Tensor, transpose: bool = True,
                     group_size: int = 64, bits: int = 8) -> Tensor:
    """``x @ w_hat.T`` (``transpose=True``, the Linear layout); float32 in and out."""
    _check("quantized_matmul", x, wq, scales, biases)
    if not transpose:
        raise NotImplementedError("quantized_matmul on hip: only transpose=True (x @ w_hat.T) is built")
    if x.dtype != T.float32:
        raise _C.DtypeMismatch(f"quantized_matmul expects a float32 activation, got {x.dtype}")
    N = wq.shape[0]
    K = wq.shape[1] * 32 // bits
    if x.shape[-1] != K:
        raise _C.ShapeMismatch(f"quantized_matmul: activation {x.shape} against a packed ({N}, {K}) weight")
    M = x.numel // K
    out = Tensor.empty((*x.shape[:-1], N), T.float32, "hip")
    _C.call("lq_wq_matmul", x.data_ptr, wq.data_ptr, scales.data_ptr, biases.data_ptr, M, N, K,
            int(group_size), int(bits), out.data_ptr, None)
    return out


_GATES = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


def quantized_gated_matmul(x: Tensor, gate: tuple[Tensor, Tensor, Tensor], up: tuple[Tensor, Tensor, Tensor], activation: str = "silu",
                           group_size: int = 64, bits: int = 8, gate_bias: Tensor | None = None, up_bias: Tensor | None = None,
                           out: Tensor | None = None) -> Tensor:
    """``act(x @ w_gate.T + gate_bias) * (x @ w_up.T + up_bias)``: both projections of a gated feed-forward block, its activation and its
    product in one call.  ``gate`` and ``up`` are what ``quantize`` gives of ``(out, in)`` weights of one shape; ``x`` ``(..., in)`` is float32 or
    float16 and so is the result ``(..., out)``, the biases are float32 ``(out,)``.  ``activation``: ``"silu"``, ``"gelu"`` (erf form), ``"relu"`` or
    ``"sigmoid"``.  Beyond its codes nothing of a weight is rounded but ``b + 2^(bits - 1) s`` of a group, to float32.  A value of a float32 ``x`` is off by at most
    ``2^-22`` of itself or ``2^-39`` of its row's largest; float16 results are rounded once.  ``out`` takes the result, apart from all that is read.  No counterpart in
    Lucid."""
    name = "quantized_gated_matmul"
    if activation not in _GATES:
        raise ValueError(f"{name}: activation {activation!r}; one of {', '.join(_GATES)}")
    _check(name, x, *gate, *up)
    dtype = x.dtype
    if dtype is not T.float16 and dtype is not T.float32:
        raise _C.DtypeMismatch(f"{name} expects a float32 or float16 activation, got {dtype}")
    if bits not in (4, 8) or group_size not in (32, 64, 128):
        raise ValueError(f"{name}: bits {bits}, group_size {group_size}; 4 or 8, and 32, 64 or 128")
    shape = gate[0].shape
    if len(shape) != 2:
        raise _C.ShapeMismatch(f"{name}: a packed weight is 2-d, got {shape}")
    N, K = shape[0], shape[1] * 32 // bits
    groups = (N, K // group_size)
    for what, (packed, scales, biases), bias in (("gate", gate, gate_bias), ("up", up, up_bias)):
        if packed.shape != shape or K % group_size or scales.shape != groups or biases.shape != groups:
            raise _C.ShapeMismatch(f"{name}: {what} is packed {packed.shape}, scales {scales.shape}, biases {biases.shape} in groups of {group_size}; "
                                   f"gate is packed {shape}")
        if packed.dtype is not T.int32 or scales.dtype is not T.float32 or biases.dtype is not T.float32:
            raise _C.DtypeMismatch(f"{name}: {what} is int32, float32 and float32, got {packed.dtype}, {scales.dtype} and {biases.dtype}")
        if bias is not None:
            _check(name, bias)
            if bias.dtype is not T.float32:
                raise _C.DtypeMismatch(f"{name}: {what}_bias is float32, got {bias.dtype}")
            if bias.shape != (N,):
                raise _C.ShapeMismatch(f"{name}: {what}_bias has shape {bias.shape}, expected {(N,)}")
    if not x.shape or x.shape[-1] != K:
        raise _C.ShapeMismatch(f"{name}: activation {x.shape} against packed ({N}, {K}) weights")
    shape = (*x.shape[:-1], N)
    if out is None:
        out = Tensor.empty(shape, dtype, "hip")
    else:
        _check(name, out)
        if out.dtype is not dtype:
            raise _C.DtypeMismatch(f"{name}: x is {dtype}, out {out.dtype}")
        if out.shape != shape:
            raise _C.ShapeMismatch(f"{name}: out has shape {out.shape}, expected {shape}")
    M = x.numel // K if K else 0
    if max(M, N, K) > 0x7fffffff:  # (more than an int says)
        raise _C.ShapeMismatch(f"{name}: {M} x {N} x {K}")
    args = _C.WQ_GATED_ARGS.pack(x.data_ptr, out.data_ptr, gate[0].data_ptr, up[0].data_ptr, gate[1].data_ptr, up[1].data_ptr, gate[2].data_ptr,
                                 up[2].data_ptr, 0 if gate_bias is None else gate_bias.data_ptr, 0 if up_bias is None else up_bias.data_ptr, M, N, K,
                                 group_size, bits, _GATES[activation], dtype.code)
    _C.call("lq_wq_gated_matmul", args, None)
    out._grid = out._range = None
    return out
