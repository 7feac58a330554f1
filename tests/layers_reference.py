"""Plain f64 forms of the operators of include/homura_cuda_layers.h, with the bounds the tests hold the kernels to.

The bounds are worst-case first-order error propagation. U is the unit roundoff of the computation type (2^-24 for f32,
2^-53 for f64); a result is finally rounded to its dtype, half a step: eps / 2 relative, and for F16 half of 2^-24
absolute among the subnormals."""
from __future__ import annotations

import math

import numpy as np

from homura_b200.host import BF16, F16, F32, F64, f32_to_half_bits, half_bits_to_f32

EPS = {F16: 2.0**-10, BF16: 2.0**-7, F32: 2.0**-23, F64: 2.0**-52}
TINY = {F16: 2.0**-25, BF16: 2.0**-134, F32: 2.0**-150, F64: 0.0}


def unit(dtype):
    return 2.0**-53 if dtype == F64 else 2.0**-24


def raw(values: np.ndarray, dtype: int) -> np.ndarray:
    """`values` rounded to the dtype, as stored."""
    if dtype == F64:
        return np.asarray(values, np.float64)
    f = np.asarray(values, np.float32)
    return f if dtype == F32 else f32_to_half_bits(f, dtype)


def value(stored: np.ndarray, dtype: int) -> np.ndarray:
    """The stored elements in f64."""
    if dtype in (F16, BF16):
        return half_bits_to_f32(stored, dtype).astype(np.float64)
    return stored.astype(np.float64)


def rounded(bound, want, dtype):
    """An error bound before the final rounding -> after it."""
    return bound + (EPS[dtype] / 2) * (np.abs(want) + bound) + TINY[dtype]


def within(got, want, bound, what):
    got, want, bound = (np.asarray(v, np.float64) for v in (got, want, bound))
    assert got.shape == want.shape, f"{what}: shape {got.shape}, expected {want.shape}"
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), f"{what}: NaN in other places ({np.isnan(got).sum()} against {nan.sum()})"
    inf = np.isinf(want)
    assert (got[inf] == want[inf]).all(), f"{what}: infinities differ"
    ok = ~nan & ~inf
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
    bad = ok & ~(off <= bound)
    if bad.any():
        i = tuple(int(v[0]) for v in np.nonzero(bad))
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} beyond the bound; first at {i}: got {got[i]!r}, want {want[i]!r}, "
                             f"off {off[i]:.3g}, bound {np.broadcast_to(bound, off.shape)[i]:.3g}")


# ---- gated linear recurrence ----

def gates(gate, sigmoid):
    """(a, 1 - a)"""
    if not sigmoid:
        return gate, 1.0 - gate
    with np.errstate(over="ignore"):
        e = np.exp(-np.abs(gate))
    small, large = e / (1 + e), 1 / (1 + e)
    return np.where(gate > 0, large, small), np.where(gate > 0, small, large)


def gate_error(gate, sigmoid, dtype):
    """Relative error of the kernel's a and 1 - a: the exponential and the quotient of f32 or f64 are good to a few units;
    for half types the argument's rounding (|g| units), ex2.approx (2^-22), the sum and rcp.approx (2^-23) add up."""
    u = unit(dtype)
    if not sigmoid:
        return np.full(gate.shape, u)
    if dtype in (F16, BF16):
        return (12 + 2 * np.abs(gate)) * u
    return np.full(gate.shape, 8 * u)


def recurrence(gate, x, initial, dtype, sigmoid=False, complement=False, reverse=False):
    """(h, its bound before rounding, last, its bound) of [batch, time, channels] f64 arrays."""
    if reverse:
        h, e, last, el = recurrence(gate[:, ::-1], x[:, ::-1], initial, dtype, sigmoid, complement)
        return h[:, ::-1], e[:, ::-1], last, el
    u = unit(dtype)
    a, left = gates(gate, sigmoid)
    da = gate_error(gate, sigmoid, dtype)
    add = left * x if complement else x
    h, e = np.zeros_like(x), np.zeros_like(x)
    state = np.zeros((x.shape[0], x.shape[2])) if initial is None else initial.copy()
    err = np.zeros_like(state)
    for t in range(x.shape[1]):
        # a step rounds the gate, u, a product of gates and the fused sum; folding a run of steps first rounds each of
        # them at most twice more
        with np.errstate(over="ignore", invalid="ignore"):
            err = np.abs(a[:, t]) * err + (da[:, t] + 4 * u) * np.abs(a[:, t] * state) + (da[:, t] + 6 * u) * np.abs(add[:, t])
            state = a[:, t] * state + add[:, t]
            err = err + 2 * u * np.abs(state)
        h[:, t], e[:, t] = state, err
    return h, e, state, err


def recurrence_backward(gate, x, out, initial, dout, dlast, dtype, sigmoid=False, complement=False, reverse=False):
    """(dgate, bound, dx, bound, dinitial, bound)"""
    if reverse:
        flip = lambda v: None if v is None else v[:, ::-1]
        dg, eg, dx, ex, di, ei = recurrence_backward(flip(gate), flip(x), flip(out), initial, flip(dout), dlast, dtype, sigmoid, complement)
        return dg[:, ::-1], eg[:, ::-1], dx[:, ::-1], ex[:, ::-1], di, ei
    u = unit(dtype)
    a, left = gates(gate, sigmoid)
    da = gate_error(gate, sigmoid, dtype)
    b, time, c = dout.shape
    g, e = np.zeros_like(dout), np.zeros_like(dout)
    state = np.zeros((b, c)) if dlast is None else dlast.copy()
    err = np.zeros_like(state)
    coefficient, ce = np.ones((b, c)), np.zeros((b, c))
    for t in range(time - 1, -1, -1):
        err = np.abs(coefficient) * err + (ce + 4 * u) * np.abs(coefficient * state) + 4 * u * np.abs(dout[:, t])
        state = coefficient * state + dout[:, t]
        err = err + 2 * u * np.abs(state)
        g[:, t], e[:, t] = state, err
        coefficient, ce = a[:, t], da[:, t]
    start = np.zeros((b, 1, c)) if initial is None else initial[:, None]
    before = np.concatenate([start, out[:, :-1]], 1) if time else out
    h = before - x if complement else before
    size = np.abs(before) + (np.abs(x) if complement else 0.0)
    dgate = g * h
    eg = e * np.abs(h) + 4 * u * np.abs(g) * size
    if sigmoid:
        eg = eg * np.abs(a * left) + np.abs(dgate * a * left) * (2 * da + 4 * u)
        dgate = dgate * a * left
    dx, ex = (g * left, e * np.abs(left) + np.abs(g * left) * (da + 2 * u)) if complement else (g, e)
    if time:
        dinitial = a[:, 0] * g[:, 0]
        ei = np.abs(a[:, 0]) * e[:, 0] + np.abs(dinitial) * (da[:, 0] + 2 * u)
    else:
        dinitial, ei = state, err
    return dgate, eg, dx, ex, dinitial, ei


# ---- group norm ----

_erf = np.vectorize(math.erf, otypes=[np.float64])


def activation(kind, z):
    """(act(z), act'(z))"""
    with np.errstate(over="ignore", invalid="ignore"):
        if kind == "relu":
            return np.where(np.isnan(z), z, np.maximum(z, 0.0)), (z > 0).astype(np.float64)
        if kind == "silu":
            s = gates(z, True)[0]
            return z * s, s * (1 + z * (1 - s))
        if kind == "gelu":
            cdf = 0.5 * (1 + (_erf(z / math.sqrt(2)) if z.size else z))
            return z * cdf, cdf + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        if kind == "gelu_tanh":
            k = math.sqrt(2 / math.pi)
            t = np.tanh(k * (z + 0.044715 * z**3))
            return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    return z, np.ones_like(z)


def activation_error(kind, z, dtype):
    """Absolute error of the kernel's act(z) and act'(z) at an exact z: a few units of 1 + |z| (the exponential's argument
    carries its own rounding: |z| units, |z|^2 for gelu's density, whose factor e^(-z^2/2) keeps the product below one unit
    each; gelu_tanh's inner polynomial carries 4 units of up to |z| (1 + z^2), beyond |z| = 5 times a vanishing slope); f32 goes through ex2.approx
    (2 units), rcp.approx (1) and, for gelu, a fit of erfc good to 1.2e-7 (2 units), which 16 hold; half types four times
    that, for none of it is seen after their rounding."""
    if kind in (None, "none", "relu"):
        return np.zeros_like(z), np.zeros_like(z)
    u = unit(dtype) * (4 if dtype in (F16, BF16) else 1)
    size = 1 + np.minimum(np.abs(z), 1e3)
    return 16 * u * size, 32 * u * size


STEEP, BENT = 1.13, 1.0  # the largest |act'| and (times 1.3 below) |act''| of silu, gelu and gelu_tanh
DEPTH = 100              # roundings on the way of a value through a sum of f32: 8 rows, 64 + 5 of a warp, its merges


def group_norm(x, weight, bias, groups, eps, kind, dtype):
    """(y, bound before rounding, mean, bound, rstd, bound) of [samples, positions, channels]."""
    n, s, c = x.shape
    u = unit(dtype)
    g = x.reshape(n, s, groups, -1)
    count = g.shape[1] * g.shape[3]
    with np.errstate(invalid="ignore", over="ignore"):
        mean = g.sum((1, 3)) / count
        dev = g - mean[:, None, :, None]
        var = (dev * dev).sum((1, 3)) / count
        rstd = 1 / np.sqrt(var + eps)
        emean = DEPTH * u * np.abs(g).sum((1, 3)) / count
        # the deviations are taken from a rounded mean (its square error adds) and summed to DEPTH roundings
        evar = (DEPTH + 4) * u * var + 4 * emean * np.sqrt(var) * DEPTH * u + emean**2
        erstd = rstd * (0.5 * evar / (var + eps) + 4 * u)
        xhat = dev * rstd[:, None, :, None]
        exhat = (emean * rstd)[:, None, :, None] + np.abs(xhat) * (erstd / rstd + 3 * u)[:, None, :, None]
        xhat, exhat = xhat.reshape(x.shape), exhat.reshape(x.shape)
        w = np.ones(c) if weight is None else weight
        b = np.zeros(c) if bias is None else bias
        z = xhat * w + b
        ez = exhat * np.abs(w) + 3 * u * (np.abs(xhat * w) + np.abs(b))
        y = activation(kind, z)[0]
        ey = STEEP * ez + activation_error(kind, z, dtype)[0]
    return y, ey, mean, emean + u * np.abs(mean), rstd, erstd


def group_norm_backward(x, dout, mean, rstd, weight, bias, groups, kind, dtype):
    """(dsrc, bound, dweight, bound, dbias, bound) with the moments taken as given."""
    n, s, c = x.shape
    u = unit(dtype)
    cg = c // groups
    wide = lambda v: np.repeat(v, cg, 1)[:, None, :]
    xhat = (x - wide(mean)) * wide(rstd)
    exhat = 3 * u * np.abs(xhat)
    w = np.ones(c) if weight is None else weight
    b = np.zeros(c) if bias is None else bias
    z = xhat * w + b
    ez = exhat * np.abs(w) + 3 * u * (np.abs(xhat * w) + np.abs(b))
    slope = activation(kind, z)[1]
    dz = dout * slope
    edz = np.abs(dout) * (1.3 * BENT * ez * (kind not in (None, "none", "relu")) + activation_error(kind, z, dtype)[1]) + 3 * u * np.abs(dz)
    if kind == "relu":
        edz = edz + np.abs(dout) * (np.abs(z) <= ez)  # the sign of z is not decided there
    p, ep = dz * w, edz * np.abs(w) + u * np.abs(dz * w)
    q, eq = p * xhat, ep * np.abs(xhat) + np.abs(p) * exhat
    depth = DEPTH + min(s, 300)
    mean_of = lambda v: v.reshape(n, s, groups, cg).mean((1, 3))
    m1, m2 = mean_of(p), mean_of(q)
    em1 = mean_of(ep) + depth * u * mean_of(np.abs(p))
    em2 = mean_of(eq) + depth * u * mean_of(np.abs(q))
    m1, m2, em1, em2 = (wide(v) for v in (m1, m2, em1, em2))
    dsrc = wide(rstd) * (p - m1 - xhat * m2)
    e = np.abs(wide(rstd)) * (ep + em1 + np.abs(xhat) * em2 + exhat * np.abs(m2) + 5 * u * (np.abs(p) + np.abs(m1) + np.abs(xhat * m2)))
    dweight, dbias = (dz * xhat).sum((0, 1)), dz.sum((0, 1))
    edw = (edz * np.abs(xhat) + np.abs(dz) * exhat).sum((0, 1)) + depth * u * np.abs(dz * xhat).sum((0, 1))
    edb = edz.sum((0, 1)) + depth * u * np.abs(dz).sum((0, 1))
    return dsrc, e, dweight, edw, dbias, edb


# ---- dropout ----

def philox_words(n, seed, offset):
    """The first n 32-bit words of the Philox4x32-10 blocks from `offset` on (Salmon et al., Random123)."""
    m = np.uint64(0xFFFFFFFF)
    with np.errstate(over="ignore"):
        block = np.arange(-(-n // 4), dtype=np.uint64) + np.uint64(offset % 2**64)
        c = [block & m, block >> np.uint64(32), np.zeros_like(block), np.zeros_like(block)]
        k0, k1 = seed & 0xFFFFFFFF, seed >> 32
        for _ in range(10):
            p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & m]
            k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)[:n]


def dropout(x, residual, p, seed, offset, dtype):
    """(y, bound before rounding, kept) in row-major order of x's logical positions."""
    kept = (philox_words(x.size, seed, offset) >= np.uint64(int(np.rint(p * 2.0**32)))).reshape(x.shape)
    u = unit(dtype)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        y = np.where(kept, x / (1 - p) if p < 1 else 0.0, 0.0)
        bound = np.where(kept, 3 * u * np.abs(y), 0.0)
        if residual is not None:
            y = y + residual
            bound = bound + 2 * u * np.abs(y)
    return y, np.where(np.isfinite(bound), bound, 0.0), kept
