"""Dense layers over any number of positions on torch device tensors.

A projection with bias, activation and residual (`linear`), and the gated feed-forward
block with its gradient (`gated_ffn`, `gated_ffn_backward`), over the resident matrices
of the spine (BF16 bits, or int8 with a scale per row) at the lengths of a prompt or a
training batch.  The reference runs these steps through ATen (row_int8_linear,
native/provider_gate/provider_moe.cpp:507-516; situ, :524-533).

Every call enqueues gfx950 work on the current torch stream of the current device through
include/k3_hip_dense_abi.h and raises K3SpineError with the library's reason on a
non-zero status; arguments that do not fit raise ValueError.  There is no CPU path.
Tensors are contiguous and live on the current device.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .moe import _dtype_code, stream_handle

_BF16_BITS = (torch.int16, torch.uint16, torch.bfloat16)
ACTIVATIONS = {None: _lib.K3_DENSE_ACT_NONE, "none": _lib.K3_DENSE_ACT_NONE,
               "silu": _lib.K3_DENSE_ACT_SILU, "gelu": _lib.K3_DENSE_ACT_GELU}
GATES = {"situ": _lib.K3_ACT_SITU, "silu": _lib.K3_ACT_SILU}


def _check(t: torch.Tensor, dtypes, shape, what: str) -> None:
    dtypes = dtypes if isinstance(dtypes, tuple) else (dtypes,)
    if (t.device.type != "cuda" or t.dtype not in dtypes or not t.is_contiguous()
            or tuple(t.shape) != tuple(shape)):
        raise ValueError(f"{what} must be a contiguous {' / '.join(map(str, dtypes))} device "
                         f"tensor of shape {list(shape)}, got {t.dtype} {list(t.shape)} on "
                         f"{t.device}")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{what} is on {t.device}, the current device is "
                         f"cuda:{torch.cuda.current_device()}")


def _rows(x: torch.Tensor, columns: int, what: str) -> torch.Tensor:
    """x as [positions, columns]; a single row may come without its first dimension."""
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{what} must be float32 or bfloat16, got {x.dtype}")
    if x.dim() not in (1, 2):
        raise ValueError(f"{what} must be [columns] or [positions, columns]")
    x2 = x if x.dim() == 2 else x.view(1, -1) if x.is_contiguous() else x.reshape(1, -1)
    _check(x2, x.dtype, (x2.shape[0], columns), what)
    return x2


def _matrix(w: torch.Tensor, scales: torch.Tensor | None, what: str) -> int:
    """The K3_SPINE_MATRIX_* kind of w, its shape and scales checked."""
    if w.dim() != 2:
        raise ValueError(f"{what} must be 2-D [rows, columns]")
    _check(w, (*_BF16_BITS, torch.int8), w.shape, what)
    if w.dtype == torch.int8:
        if scales is None:
            raise ValueError(f"int8 {what} needs a scale per row")
        _check(scales, torch.float32, (w.shape[0],), f"{what} scales")
        return _lib.K3_SPINE_MATRIX_INT8
    if scales is not None:
        raise ValueError(f"BF16 {what} takes no row scales")
    return _lib.K3_SPINE_MATRIX_BF16


def _out(out: torch.Tensor | None, shape, dtype: torch.dtype, what: str) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device="cuda")
    _check(out, dtype, shape, what)
    return out


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _run(name: str, d, workspace: torch.Tensor | None) -> None:
    lib = _lib.load()
    need = getattr(lib, name + "_workspace_bytes")(C.byref(d))
    if need == 0:
        raise _lib.K3SpineError(_lib.K3_SPINE_E_INVALID, name + "_workspace_bytes")
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
    else:
        _check(workspace, torch.uint8, workspace.shape, "workspace")
    _lib.check_spine(getattr(lib, name)(C.byref(d), workspace.data_ptr(), workspace.numel(),
                                        stream_handle()), name)


def linear(weights: torch.Tensor, x: torch.Tensor, bias: torch.Tensor | None = None,
           activation: str | None = None, residual: torch.Tensor | None = None,
           row_scales: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None
           ) -> torch.Tensor:
    """out[p, r] = activation(row_scales[r] * sum_c weights[r, c] x[p, c] + bias[r])
    + residual[p, r], for any number of positions.

    weights: BF16 bits (int16, uint16 or bfloat16) or int8 with fp32 row_scales,
    [rows, columns]; x: fp32 or bfloat16 [positions, columns]; bias: fp32 [rows];
    activation: None, "silu" or "gelu" (the erf form); residual: [positions, rows] in the
    output's dtype, and may be `out` itself.  out_dtype: x's unless given.  Sums are fp32
    and rounded once.  workspace: uint8, at least linear_workspace's bytes, for a caller
    that keeps one (one per call that may run at the same time)."""
    d, out = _linear_descriptor(weights, x, bias, activation, residual, row_scales, out_dtype, out)
    _run("k3_hip_linear", d, workspace)
    return out


def _linear_descriptor(weights, x, bias, activation, residual, row_scales, out_dtype, out):
    kind = _matrix(weights, row_scales, "weights")
    rows, cols = weights.shape
    x2 = _rows(x, cols, "x")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None, 'silu' or 'gelu', got {activation!r}")
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"outputs are float32 or bfloat16, not {dtype}")
    shape = (x2.shape[0], rows)
    if bias is not None:
        _check(bias, torch.float32, (rows,), "bias")
    if residual is not None:
        _check(residual, dtype, shape, "residual")
    out = _out(out, shape, dtype, "out")
    d = _lib.K3HipLinearV1()
    d.abi_version, d.struct_bytes = _lib.K3_DENSE_ABI_V1, C.sizeof(d)
    d.matrix_kind, d.activation = kind, ACTIVATIONS[activation]
    d.x_dtype, d.out_dtype = _dtype_code(x2), _dtype_code(out)
    d.rows, d.columns, d.positions = rows, cols, x2.shape[0]
    d.weights, d.row_scales, d.bias = _ptr(weights), _ptr(row_scales), _ptr(bias)
    d.x, d.residual, d.out = _ptr(x2), _ptr(residual), _ptr(out)
    return d, out


def _gate_code(activation) -> int:
    if activation in GATES:
        return GATES[activation]
    if activation in GATES.values() and not isinstance(activation, bool):
        return int(activation)
    raise ValueError(f"activation must be 'silu' or 'situ', got {activation!r}")


def _pair(w_gate, w_up, gate_scales, up_scales) -> int:
    kind = _matrix(w_gate, gate_scales, "w_gate")
    if _matrix(w_up, up_scales, "w_up") != kind or w_up.shape != w_gate.shape:
        raise ValueError("w_gate and w_up must be of one kind and shape")
    return kind


def gated_ffn(w_gate: torch.Tensor, w_up: torch.Tensor, x: torch.Tensor,
              activation: str | int = "silu", keep: bool = False,
              gate_scales: torch.Tensor | None = None, up_scales: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None):
    """f(W_gate x, W_up x) for any number of positions, both projections, the activation
    and the product in one kernel: f(g, u) = silu(g) u ("silu", K3_ACT_SILU) or the K3
    SiTU 4 tanh(g/4) sigmoid(g) 25 tanh(u/25) ("situ", K3_ACT_SITU).

    w_gate, w_up: as linear's weights, [rows, columns]; x: fp32 or bfloat16 [positions,
    columns].  Returns h [positions, rows], or (h, g, u) with keep, g and u being the two
    projections for gated_ffn_backward; all in out_dtype (x's unless given)."""
    kind = _pair(w_gate, w_up, gate_scales, up_scales)
    rows, cols = w_gate.shape
    x2 = _rows(x, cols, "x")
    code = _gate_code(activation)
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"outputs are float32 or bfloat16, not {dtype}")
    shape = (x2.shape[0], rows)
    out = _out(out, shape, dtype, "out")
    g = torch.empty_like(out) if keep else None
    u = torch.empty_like(out) if keep else None
    d = _lib.K3HipGatedV1()
    d.abi_version, d.struct_bytes = _lib.K3_DENSE_ABI_V1, C.sizeof(d)
    d.matrix_kind, d.activation = kind, code
    d.x_dtype, d.out_dtype = _dtype_code(x2), _dtype_code(out)
    d.rows, d.columns, d.positions = rows, cols, x2.shape[0]
    d.gate, d.up = _ptr(w_gate), _ptr(w_up)
    d.gate_scales, d.up_scales = _ptr(gate_scales), _ptr(up_scales)
    d.x, d.out, d.out_gate, d.out_up = _ptr(x2), _ptr(out), _ptr(g), _ptr(u)
    _run("k3_hip_gated_ffn", d, workspace)
    return (out, g, u) if keep else out


def gated_ffn_backward(w_gate: torch.Tensor, w_up: torch.Tensor, x: torch.Tensor,
                       g: torch.Tensor, u: torch.Tensor, grad: torch.Tensor,
                       activation: str | int = "silu", workspace: torch.Tensor | None = None
                       ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradient of gated_ffn: (d_x [positions, columns], d_gate, d_up [rows, columns])
    from grad = d(loss)/d(h) and the kept projections g and u [positions, rows].

    The matrices are BF16 (int8 ones have no gradient here); x, g, u and grad are all
    fp32 or all bfloat16 and the results have that dtype."""
    if _pair(w_gate, w_up, None, None) != _lib.K3_SPINE_MATRIX_BF16:
        raise ValueError("the gradient takes BF16 matrices")
    rows, cols = w_gate.shape
    x2 = _rows(x, cols, "x")
    code = _gate_code(activation)
    shape = (x2.shape[0], rows)
    two = [t if t.dim() == 2 else t.reshape(1, -1) for t in (g, u, grad)]
    for t, name in zip(two, ("g", "u", "grad")):
        _check(t, x2.dtype, shape, name)
    d_x = torch.empty_like(x2)
    d_gate = torch.empty(rows, cols, dtype=x2.dtype, device="cuda")
    d_up = torch.empty_like(d_gate)
    d = _lib.K3HipGatedGradV1()
    d.abi_version, d.struct_bytes = _lib.K3_DENSE_ABI_V1, C.sizeof(d)
    d.activation, d.dtype = code, _dtype_code(x2)
    d.rows, d.columns, d.positions = rows, cols, x2.shape[0]
    d.gate, d.up, d.x = _ptr(w_gate), _ptr(w_up), _ptr(x2)
    d.g, d.u, d.grad = (_ptr(t) for t in two)
    d.d_x, d.d_gate, d.d_up = _ptr(d_x), _ptr(d_gate), _ptr(d_up)
    _run("k3_hip_gated_ffn_grad", d, workspace)
    return d_x, d_gate, d_up
