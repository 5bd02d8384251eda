"""Float64 oracle of the dense layers (include/k3_hip_dense_abi.h) in numpy: a projection
with bias, activation and residual, the gated feed-forward block and its gradient, with
the bounds that fp32 sums and a final rounding allow.

SiTU is the reference's (situ, native/provider_gate/provider_moe.cpp:524-533).
"""
from __future__ import annotations

import math

import numpy as np

F32_HALF_STEP = 2.0 ** -24   # half an fp32 step, relative to the value
BF16_HALF_STEP = 2.0 ** -8   # half a BF16 step


def bf16_round(v: np.ndarray) -> np.ndarray:
    """Nearest BF16 values (ties to even) of fp32 ones, as fp32."""
    u = np.ascontiguousarray(v, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def sigmoid(z: np.ndarray) -> np.ndarray:
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1.0, e) / (1.0 + e)


_erf = np.vectorize(math.erf, otypes=[np.float64])


def activation(name, z: np.ndarray) -> np.ndarray:
    if name == "silu":
        return z * sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1.0 + _erf(z / math.sqrt(2.0)))
    return z


def linear(w, x, bias=None, act=None, residual=None, scales=None):
    """(out, bound): every argument holds the exact values that the call reads.  The bound
    is that of the fp32 arithmetic ahead of the output's own rounding: a sum of C products
    in any order is off by at most C half steps of the sum of magnitudes; scale, bias,
    activation (derivatives under 1.2, library functions to 8 half steps) and residual
    add a few half steps of what they produce."""
    w, x = np.asarray(w, np.float64), np.asarray(x, np.float64)
    z, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    if scales is not None:
        z, mag = z * scales, mag * np.abs(scales)
    bound = (x.shape[1] + 4) * mag
    if bias is not None:
        z = z + bias
        bound = bound + np.abs(bias) + np.abs(z)
    out = activation(act, z)
    if act not in (None, "none"):
        bound = 1.2 * bound + 16.0 * np.abs(z)
    if residual is not None:
        out = out + residual
        bound = bound + np.abs(out)
    return out, F32_HALF_STEP * bound


def gate(name, g, u):
    """(f, f_g, f_u) of the gated block's f."""
    s = sigmoid(g)
    if name == "silu":
        return g * s * u, u * (s + g * s * (1 - s)), g * s
    t, v = np.tanh(g / 4), np.tanh(u / 25)
    a, b = 4 * t * s, 25 * v
    return a * b, ((1 - t * t) * s + 4 * t * s * (1 - s)) * b, a * (1 - v * v)


def gated(wg, wu, x, act, gs=None, us=None):
    """((h, g, u), bounds of each) as linear's."""
    g, eg = linear(wg, x, scales=gs)
    u, eu = linear(wu, x, scales=us)
    h, fg, fu = gate(act, g, u)
    # first order in the errors of g and u, doubled for what the derivatives change
    # within them, and the functions' own roundings
    eh = 2 * (np.abs(fg) * eg + np.abs(fu) * eu) + eg * eu + 32 * F32_HALF_STEP * np.abs(h)
    return (h, g, u), (eh, eg, eu)


def gated_grad(wg, wu, x, g, u, grad, act, dtype="f32"):
    """((d_x, d_gate, d_up), bounds).  dg and du carry a few fp32 roundings (of the terms
    of f_g and f_u, at most 32 half steps of their magnitudes) and with BF16 one rounding
    to it; with fp32 the term split drops products under 2^-24 of a term's."""
    wg, wu, x = (np.asarray(a, np.float64) for a in (wg, wu, x))
    g, u, grad = (np.asarray(a, np.float64) for a in (g, u, grad))
    _, fg, fu = gate(act, g, u)
    s = sigmoid(g)
    # magnitudes of the summed parts of f_g (they can cancel) and of f_u
    if act == "silu":
        mg, mu = np.abs(u) * s * (1 + np.abs(g)), np.abs(g) * s
    else:
        t, v = np.tanh(g / 4), np.tanh(u / 25)
        mg = np.abs(25 * v) * s * (2 + 4 * np.abs(t))
        mu = 8 * np.abs(t) * s
    dg, du = grad * fg, grad * fu
    eg, eu = (32 * F32_HALF_STEP * np.abs(grad) * m for m in (mg, mu))
    if dtype == "bf16":
        eg, eu = eg + BF16_HALF_STEP * np.abs(dg), eu + BF16_HALF_STEP * np.abs(du)
    n_x, n_w = 2 * wg.shape[0] + 8, x.shape[0] + 8
    d_x = dg @ wg + du @ wu
    e_x = (eg @ np.abs(wg) + eu @ np.abs(wu)
           + n_x * F32_HALF_STEP * (np.abs(dg) @ np.abs(wg) + np.abs(du) @ np.abs(wu)))
    outs, errs = [d_x], [e_x]
    for d, e in ((dg, eg), (du, eu)):
        outs.append(d.T @ x)
        errs.append(e.T @ np.abs(x) + n_w * F32_HALF_STEP * (np.abs(d).T @ np.abs(x)))
    return outs, errs
