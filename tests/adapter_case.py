"""64-bit references and derived tolerances of the adapter and conditioning operators.

A BF16 rounding is off by at most 2^-8 of the value. An F32 sum of n products on the tensor cores is
taken to be off by at most n * 2^-23 of the sum of the products' magnitudes (one truncation per
addition). Tolerances add up the roundings of the operator, element by element; nothing is fitted.
"""
import numpy as np

import h3_oracle as o

HALF_BF16 = 2.0 ** -8
F32_STEP = 2.0 ** -23
NONE = 0xFFFFFFFF


def wide(bits):
    return o.from_bf16(bits).astype(np.float64)


def lora_reference(x, w, bias, down, up, scale, row_adapter):
    """(result, tolerance) of x.W^T + bias + scale[a] (x.down[a]^T).up[a]^T, all float64 arrays of the
    inputs' exact values; row_adapter: U32 per row."""
    rows, k = x.shape
    adapters, rank = down.shape[:2]
    y, mass = x @ w.T, np.abs(x) @ np.abs(w.T)
    if bias is not None:
        y, mass = y + bias, mass + np.abs(bias)
    rounded = np.zeros_like(y)
    for a in range(adapters):
        at = np.nonzero(row_adapter == a)[0]
        if not at.size:
            continue
        t = x[at] @ down[a].T * scale[a]
        t_mass = np.abs(x[at]) @ np.abs(down[a].T) * abs(scale[a])
        y[at] += t @ up[a].T
        mass[at] += t_mass @ np.abs(up[a].T)
        rounded[at] += np.abs(t) @ np.abs(up[a].T)
    # the low-rank row is rounded to BF16, every sum is F32, the result is rounded once to BF16
    before = HALF_BF16 * rounded + 2 * (k + rank + 8) * F32_STEP * mass
    return y, before + HALF_BF16 * (np.abs(y) + before)


def cross_reference(q, k, v, segments, scale, untouched):
    """(result, tolerance) with q [rows][heads][dim], k / v [key rows][kv heads][dim] in float64;
    `untouched` is what rows of no segment hold (tolerance 0 there)."""
    heads, dim = q.shape[1:]
    group = heads // k.shape[1]
    out, tol = untouched.astype(np.float64).copy(), np.zeros(q.shape)
    for q0, qn, k0, kn in segments:
        q0 = min(q0, q.shape[0]); qn = min(qn, q.shape[0] - q0)
        k0 = min(k0, k.shape[0]); kn = min(kn, k.shape[0] - k0)
        if not qn:
            continue
        if not kn:
            out[q0:q0 + qn] = 0.0
            continue
        for h in range(heads):
            qq, kk, vv = q[q0:q0 + qn, h], k[k0:k0 + kn, h // group], v[k0:k0 + kn, h // group]
            s = qq @ kk.T * scale
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            y, mass = p @ vv, p @ np.abs(vv)
            # scores: F32 sums of dim products, then one fused multiply-add in log2 units whose result
            # is at most a few hundred (2^-24 of it), then an exponential good to 2^-21
            score_off = (dim + 4) * F32_STEP * abs(scale) * (np.abs(qq) @ np.abs(kk.T)).max(1, keepdims=True)
            score_off = score_off + 2.0 ** -24 * np.abs(s).max(1, keepdims=True) * 2 + 2.0 ** -21
            before = (HALF_BF16 + 2 * score_off + 2 * (kn + 8) * F32_STEP) * mass
            out[q0:q0 + qn, h] = y
            tol[q0:q0 + qn, h] = before + HALF_BF16 * (np.abs(y) + before)
    return out, tol


def assert_within(got_bits, want, tol, name=""):
    got = wide(got_bits).reshape(want.shape)
    assert np.isfinite(got).all(), f"{name}: {int((~np.isfinite(got)).sum())} values are not finite"
    off = np.abs(got - want)
    bad = off > tol
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.size} outside, worst {float((off - tol).max()):.3g} "
                           f"over a tolerance of {float(tol.flat[(off - tol).argmax()]):.3g}")
