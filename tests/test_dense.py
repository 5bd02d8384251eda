"""Dense layers without a GPU: refusals of the C ABI (before any device work) and of the
torch interface, workspace sizes, and the oracle against plain differences."""
import ctypes as C

import numpy as np
import pytest

from oracle import dense as D

A = 1 << 20  # addresses that are only looked at


def _linear(**kw):
    from deltafin_amd import _lib
    d = _lib.K3HipLinearV1()
    d.abi_version, d.struct_bytes = 1, C.sizeof(d)
    d.x_dtype = d.out_dtype = _lib.K3_DTYPE_F32
    d.rows, d.columns, d.positions = 64, 128, 5
    d.weights, d.x, d.out = A, 2 * A, 3 * A
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _gated(**kw):
    from deltafin_amd import _lib
    d = _lib.K3HipGatedV1()
    d.abi_version, d.struct_bytes = 1, C.sizeof(d)
    d.rows, d.columns, d.positions = 64, 128, 5
    d.gate, d.up, d.x, d.out = A, 2 * A, 3 * A, 4 * A
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _grad(**kw):
    from deltafin_amd import _lib
    d = _lib.K3HipGatedGradV1()
    d.abi_version, d.struct_bytes = 1, C.sizeof(d)
    d.rows, d.columns, d.positions = 64, 128, 5
    for i, name in enumerate(("gate", "up", "x", "g", "u", "grad", "d_x", "d_gate", "d_up")):
        setattr(d, name, (i + 1) * A)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _refused(name, d, match, ws=256 * A, bytes_=1 << 40):
    from deltafin_amd import _lib
    lib = _lib.load()
    rc = getattr(lib, name)(C.byref(d) if d is not None else None, ws, bytes_, None)
    assert rc == _lib.K3_SPINE_E_INVALID
    assert match in lib.k3_hip_spine_last_error().decode()


@pytest.mark.parametrize("kw,match", [
    (dict(abi_version=2), "descriptor version"), (dict(struct_bytes=80), "descriptor version"),
    (dict(reserved=1), "reserved"), (dict(rows=0), "must be 1.."), (dict(columns=0), "must be 1.."),
    (dict(positions=0), "must be 1.."), (dict(positions=(1 << 20) + 1), "must be 1.."),
    (dict(x_dtype=2), "x_dtype"), (dict(out_dtype=7), "out_dtype"),
    (dict(matrix_kind=2), "matrix kind"), (dict(activation=3), "activation"),
    (dict(weights=None), "null"), (dict(x=None), "null"), (dict(out=None), "null"),
    (dict(matrix_kind=1), "null"), (dict(row_scales=5 * A), "no row scales"),
    (dict(weights=A + 1), "weights is not aligned"), (dict(x=2 * A + 2), "x is not aligned"),
    (dict(bias=5 * A + 2), "bias is not aligned"), (dict(out=3 * A + 1), "out is not aligned"),
    (dict(out=2 * A + 64), "out overlaps x"), (dict(out=A), "out overlaps weights"),
    (dict(residual=3 * A + 16), "out overlaps residual"), (dict(bias=3 * A + 4), "out overlaps bias"),
])
def test_linear_refusals(kw, match):
    _refused("k3_hip_linear", _linear(**kw), match)


@pytest.mark.parametrize("kw,match", [
    (dict(abi_version=0), "descriptor version"), (dict(rows=0), "must be 1.."),
    (dict(activation=2), "activation"), (dict(up=None), "null"), (dict(matrix_kind=1), "null"),
    (dict(out_gate=5 * A), "kept together"), (dict(gate_scales=5 * A), "no row scales"),
    (dict(out_gate=4 * A, out_up=6 * A), "out_gate overlaps out"),
    (dict(out_gate=6 * A, out_up=6 * A + 16), "out_up overlaps out_gate"),
    (dict(out=3 * A), "out overlaps x"), (dict(x_dtype=9), "x_dtype"),
])
def test_gated_refusals(kw, match):
    _refused("k3_hip_gated_ffn", _gated(**kw), match)


@pytest.mark.parametrize("kw,match", [
    (dict(struct_bytes=1), "descriptor version"), (dict(columns=0), "must be 1.."),
    (dict(dtype=2), "dtype"), (dict(activation=5), "activation"), (dict(grad=None), "null"),
    (dict(d_up=None), "null"), (dict(d_x=3 * A), "d_x overlaps x"),
    (dict(d_up=8 * A), "d_up overlaps d_gate"), (dict(g=4 * A + 2), "g is not aligned"),
])
def test_grad_refusals(kw, match):
    _refused("k3_hip_gated_ffn_grad", _grad(**kw), match)


@pytest.mark.parametrize("name,make", [("k3_hip_linear", _linear), ("k3_hip_gated_ffn", _gated),
                                       ("k3_hip_gated_ffn_grad", _grad)])
def test_workspace_refusals(name, make):
    from deltafin_amd import _lib
    lib = _lib.load()
    need = getattr(lib, name + "_workspace_bytes")(C.byref(make(positions=50, columns=100)))
    assert need > _lib.K3_DENSE_NO_WORKSPACE
    _refused(name, make(positions=50, columns=100), "workspace", ws=None)
    _refused(name, make(positions=50, columns=100), "workspace", ws=256 * A + 16)
    _refused(name, make(positions=50, columns=100), "workspace", bytes_=need - 1)
    _refused(name, None, "null descriptor")
    assert getattr(lib, name + "_workspace_bytes")(None) == 0
    assert getattr(lib, name + "_workspace_bytes")(C.byref(make(rows=0))) == 0


def test_a_small_workspace_is_not_none():
    """The smallest scratch memory there is (one row's dg and du) is told from none at all."""
    from deltafin_amd import _lib
    lib = _lib.load()
    d = _grad(rows=8, columns=16, positions=1, dtype=_lib.K3_DTYPE_BF16)
    assert lib.k3_hip_gated_ffn_grad_workspace_bytes(C.byref(d)) > _lib.K3_DENSE_NO_WORKSPACE
    _refused("k3_hip_gated_ffn_grad", d, "workspace", ws=None,
             bytes_=_lib.K3_DENSE_NO_WORKSPACE)
    none = _linear(x_dtype=_lib.K3_DTYPE_BF16, positions=1)
    assert (lib.k3_hip_linear_workspace_bytes(C.byref(none)) == _lib.K3_DENSE_NO_WORKSPACE)


def test_workspace_counts_what_is_laid_out_again():
    """fp32 rows need their terms, odd widths a copy; BF16 rows in place need neither."""
    from deltafin_amd import _lib
    lib = _lib.load()
    size = lambda **kw: lib.k3_hip_linear_workspace_bytes(C.byref(_linear(
        rows=65536, columns=64, positions=4096, **kw)))
    bf16 = _lib.K3_DTYPE_BF16
    assert size(x_dtype=bf16) == _lib.K3_DENSE_NO_WORKSPACE
    assert size(x_dtype=bf16, x=2 * A + 2) >= 4096 * 64 * 2
    assert size() >= 3 * 4096 * 64 * 2
    assert size(x_dtype=bf16, weights=A + 2) >= 65536 * 64 * 2


def test_torch_interface_refuses_host_tensors():
    import torch

    from deltafin_amd import dense
    w, x = torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(2, 16)
    with pytest.raises(ValueError, match="device tensor"):
        dense.linear(w, x)
    with pytest.raises(ValueError, match="device tensor"):
        dense.gated_ffn(w, w, x)
    with pytest.raises(ValueError, match="device tensor"):
        dense.gated_ffn_backward(w, w, x, x, x, x)


@pytest.mark.parametrize("act", ["silu", "situ"])
def test_oracle_gradient_is_the_difference(act):
    """Central differences of sum(grad h): truncation of order step^2."""
    rng = np.random.default_rng(3)
    wg, wu = rng.standard_normal((2, 5, 7))
    x, grad = rng.standard_normal((4, 7)), rng.standard_normal((4, 5))
    (_, g, u), _ = D.gated(wg, wu, x, act)
    found, _ = D.gated_grad(wg, wu, x, g, u, grad, act)
    loss = lambda a, b, c: float((D.gated(a, b, c, act)[0][0] * grad).sum())
    step = 1e-5
    for which, at in ((2, x), (0, wg), (1, wu)):
        diff = np.zeros_like(at)
        for i in np.ndindex(at.shape):
            lo, hi = at.copy(), at.copy()
            lo[i] -= step
            hi[i] += step
            args = [wg, wu, x]
            args[which] = hi
            up = loss(*args)
            args[which] = lo
            diff[i] = (up - loss(*args)) / (2 * step)
        want = found[{2: 0, 0: 1, 1: 2}[which]]
        assert np.allclose(diff, want, rtol=1e-7, atol=1e-7)


def test_c_caller_probe(tmp_path):
    """The headers as a C11 caller sees them."""
    import subprocess
    from pathlib import Path

    from deltafin_amd import _lib
    root = Path(__file__).resolve().parents[1]
    exe = tmp_path / "dense_probe"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", f"-I{root / 'include'}",
                    str(root / "tests" / "c" / "dense_probe.c"), "-o", str(exe),
                    f"-L{_lib.LIB_PATH.parent}", "-lk3hipmoe",
                    f"-Wl,-rpath,{_lib.LIB_PATH.parent}"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip() == "ok"
