"""Sampling without a GPU: refusals of the C ABI and the oracle's own answers."""
import ctypes as C

import numpy as np
import pytest

from oracle.sampling import sample_row

A = 1 << 24


def _desc(**kw):
    from deltafin_amd import _lib
    d = _lib.K3HipSampleV1()
    d.abi_version, d.struct_bytes = 1, C.sizeof(d)
    d.rows, d.vocabulary = 4, 1000
    for i, name in enumerate(("logits", "u", "temperature", "top_k", "top_p", "min_p", "tokens")):
        setattr(d, name, (i + 1) * A)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,match", [
    (dict(abi_version=2), "descriptor version"), (dict(struct_bytes=72), "descriptor version"),
    (dict(reserved=3), "reserved"), (dict(logits_dtype=2), "neither fp32 nor BF16"),
    (dict(rows=0), "rows (0)"), (dict(rows=32769), "rows (32769)"),
    (dict(vocabulary=0), "vocabulary (0)"), (dict(vocabulary=(1 << 24) + 1), "vocabulary"),
    (dict(logits=None), "null"), (dict(u=None), "null"), (dict(tokens=None), "null"),
    (dict(logits=A + 2), "not aligned"), (dict(top_k=4 * A + 1), "not aligned"),
    (dict(tokens=A + 160), "tokens overlap"), (dict(tokens=3 * A), "tokens overlap"),
])
def test_refusals(kw, match):
    from deltafin_amd import _lib
    lib = _lib.load()
    rc = lib.k3_hip_sample(C.byref(_desc(**kw)), 256 * A, 1 << 40, None)
    assert rc == _lib.K3_SPINE_E_INVALID
    assert match in lib.k3_hip_spine_last_error().decode()


def test_workspace_refusals():
    from deltafin_amd import _lib
    lib = _lib.load()
    need = lib.k3_hip_sample_workspace_bytes(C.byref(_desc()))
    assert need >= 4 * 2048 * 12
    for ws, n in ((None, need), (256 * A + 8, need), (256 * A, need - 1)):
        assert lib.k3_hip_sample(C.byref(_desc()), ws, n, None) == _lib.K3_SPINE_E_INVALID
        assert "workspace" in lib.k3_hip_spine_last_error().decode()
    assert lib.k3_hip_sample(None, 256 * A, need, None) == _lib.K3_SPINE_E_INVALID
    assert lib.k3_hip_sample_workspace_bytes(None) == 0


def test_torch_interface_refuses_host_tensors():
    import torch

    from deltafin_amd import sampling
    with pytest.raises(ValueError, match="device tensor"):
        sampling.sample(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(ValueError, match="logits must be"):
        sampling.sample(torch.zeros(8), torch.zeros(1))


def test_oracle_by_hand():
    l = np.log([1.0, 4.0, 2.0, 1.0])  # order 1, 2, 0, 3; weights 1, .5, .25, .25 of the largest
    draw = lambda u, **kw: sample_row(l, u, **kw)[0]
    assert [draw(u) for u in (0.0, 0.49, 0.51, 0.74, 0.76, 0.87, 0.88, 0.999)] == [
        1, 1, 2, 2, 0, 0, 3, 3]
    assert [draw(u, top_k=2) for u in (0.66, 0.67)] == [1, 2]
    assert [draw(u, top_p=0.7) for u in (0.66, 0.67)] == [1, 2]
    assert draw(0.9, top_p=0.4) == 1 and draw(0.9, top_p=0.0) == 1
    assert draw(0.999, min_p=0.3) == 2
    assert draw(0.9, temperature=0.0) == 1
    assert sample_row([-np.inf, np.nan], 0.5)[0] == -1
    assert sample_row([0.0, np.inf, 5.0, np.inf], 0.6)[0] == 3
