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

_MATRICES = (torch.bfloat16, torch.int8, torch.int16, torch.uint16)
_ROWS = (torch.float32, torch.bfloat16)
ACTIVATIONS = {None: _lib.K3_DENSE_ACT_NONE, "none": _lib.K3_DENSE_ACT_NONE,
               "silu": _lib.K3_DENSE_ACT_SILU, "gelu": _lib.K3_DENSE_ACT_GELU}
GATES = {"situ": _lib.K3_ACT_SITU, "silu": _lib.K3_ACT_SILU}


def _check(t: torch.Tensor, dtypes, shape, what: str) -> None:
    """t is a contiguous tensor of one of the dtypes and the shape on the current device.
    (One comparison after the other on purpose: a decode step's call is host bound.)"""
    fits = t.dtype in dtypes if isinstance(dtypes, tuple) else t.dtype is dtypes
    if fits and t.shape == shape and t.is_contiguous():
        at = t.get_device()
        if at >= 0:
            if at == torch._C._cuda_getDevice():
                return
            raise ValueError(f"{what} is on {t.device}, the current device is "
                             f"cuda:{torch.cuda.current_device()}")
    names = " / ".join(map(str, dtypes if isinstance(dtypes, tuple) else (dtypes,)))
    raise ValueError(f"{what} must be a contiguous {names} device tensor of shape "
                     f"{list(shape)}, got {t.dtype} {list(t.shape)} on {t.device}")


def _rows(x: torch.Tensor, columns: int, what: str) -> torch.Tensor:
    """x as [positions, columns]; a single row may come without its first dimension."""
    if x.dtype not in _ROWS:
        raise ValueError(f"{what} must be float32 or bfloat16, got {x.dtype}")
    if x.dim() == 1:
        x = x.reshape(1, -1)
    elif x.dim() != 2:
        raise ValueError(f"{what} must be [columns] or [positions, columns]")
    _check(x, x.dtype, (x.shape[0], columns), what)
    return x


def _matrix(w: torch.Tensor, scales: torch.Tensor | None, what: str) -> int:
    """The K3_SPINE_MATRIX_* kind of w, its shape and scales checked."""
    if w.dim() != 2:
        raise ValueError(f"{what} must be 2-D [rows, columns]")
    _check(w, _MATRICES, w.shape, what)
    if w.dtype is torch.int8:
        if scales is None:
            raise ValueError(f"int8 {what} needs a scale per row")
        _check(scales, torch.float32, (w.shape[0],), f"{what} scales")
        return _lib.K3_SPINE_MATRIX_INT8
    if scales is not None:
        raise ValueError(f"BF16 {what} takes no row scales")
    return _lib.K3_SPINE_MATRIX_BF16


def _out(out: torch.Tensor | None, x: torch.Tensor, rows: int, dtype: torch.dtype | None
         ) -> torch.Tensor:
    """The output [positions, rows]: `out`, or a new tensor of the dtype (x's unless given)."""
    if dtype is None:
        dtype = x.dtype if out is None else out.dtype
    if dtype not in _ROWS:
        raise ValueError(f"outputs are float32 or bfloat16, not {dtype}")
    if out is None:
        return torch.empty((x.shape[0], rows), dtype=dtype, device=x.device)
    _check(out, dtype, (x.shape[0], rows), "out")
    return out


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _run(name: str, d, workspace: torch.Tensor | None) -> None:
    lib = _lib.load()
    ref = C.byref(d)
    if workspace is not None:
        _check(workspace, torch.uint8, workspace.shape, "workspace")
        at, have = workspace.data_ptr(), workspace.numel()
    else:
        at, have = None, getattr(lib, name + "_workspace_bytes")(ref)
        if have == 0:
            raise _lib.K3SpineError(_lib.K3_SPINE_E_INVALID, name + "_workspace_bytes")
        if have > _lib.K3_DENSE_NO_WORKSPACE:
            workspace = torch.empty(have, dtype=torch.uint8, device="cuda")
            at = workspace.data_ptr()
    _lib.check_spine(getattr(lib, name)(ref, at, have, stream_handle()), name)


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
    kind = _matrix(weights, row_scales, "weights")
    rows, cols = weights.shape
    x2 = _rows(x, cols, "x")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None, 'silu' or 'gelu', got {activation!r}")
    out = _out(out, x2, rows, out_dtype)
    if bias is not None:
        _check(bias, torch.float32, (rows,), "bias")
    if residual is not None:
        _check(residual, out.dtype, out.shape, "residual")
    d = _lib.K3HipLinearV1(
        _lib.K3_DENSE_ABI_V1, C.sizeof(_lib.K3HipLinearV1), kind, ACTIVATIONS[activation],
        _dtype_code(x2), _dtype_code(out), rows, cols, x2.shape[0], 0, weights.data_ptr(),
        _ptr(row_scales), _ptr(bias), x2.data_ptr(), _ptr(residual), out.data_ptr())
    _run("k3_hip_linear", d, workspace)
    return out


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
    out = _out(out, x2, rows, out_dtype)
    g = torch.empty_like(out) if keep else None
    u = torch.empty_like(out) if keep else None
    d = _lib.K3HipGatedV1(
        _lib.K3_DENSE_ABI_V1, C.sizeof(_lib.K3HipGatedV1), kind, code, _dtype_code(x2),
        _dtype_code(out), rows, cols, x2.shape[0], 0, w_gate.data_ptr(), w_up.data_ptr(),
        _ptr(gate_scales), _ptr(up_scales), x2.data_ptr(), out.data_ptr(), _ptr(g), _ptr(u))
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
    d_gate = torch.empty((rows, cols), dtype=x2.dtype, device=x2.device)
    d_up = torch.empty_like(d_gate)
    d = _lib.K3HipGatedGradV1(
        _lib.K3_DENSE_ABI_V1, C.sizeof(_lib.K3HipGatedGradV1), code, _dtype_code(x2), rows, cols,
        x2.shape[0], 0, w_gate.data_ptr(), w_up.data_ptr(), x2.data_ptr(),
        *(t.data_ptr() for t in two), d_x.data_ptr(), d_gate.data_ptr(), d_up.data_ptr())
    _run("k3_hip_gated_ffn_grad", d, workspace)
    return d_x, d_gate, d_up
