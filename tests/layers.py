"""Plain 64-bit forms of the layers' products and what their kernels may be off by, shared by the tests of 8-bit matrices and gated units."""
import math

import numpy as np

TYPE_IDS = {"f64": 0, "f32": 1, "bf16": 2, "f16": 3}
UNIT = {"f64": 2.0 ** -53, "f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # half a step, relative
TINY = {"f64": 0.0, "f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}       # the smallest step
CALC = {"f64": 2.0 ** -53, "f32": 2.0 ** -24, "bf16": 2.0 ** -24, "f16": 2.0 ** -24}  # half a step of what values are computed in
BYTES = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}


def encode(a, t):
    """fp64 values as the type's bytes (bf16 as uint16, rounded to nearest even)."""
    a = np.asarray(a, np.float64)
    if t == "f64":
        return a.copy()
    if t == "f32":
        return a.astype(np.float32)
    if t == "f16":
        return a.astype(np.float16)
    u = a.astype(np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r).astype(np.uint16)


def decode(b, t):
    if t == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


def quantise(Y):
    """(whole numbers, scales) of the rows of Y: max * (1 / 127) in fp32, exact quotients to the nearest, ties to even. fp64 quotients of fp32 operands and
    of the fp64 values are what the definition says."""
    with np.errstate(all="ignore"):
        big = np.max(np.abs(Y), axis=1) if Y.shape[1] else np.zeros(Y.shape[0])
        s = big.astype(np.float32) * (np.float32(1) / np.float32(127))
        s[~np.isfinite(big.astype(np.float32))] = np.nan
        q = np.where(s[:, None] > 0, np.clip(np.rint(Y / s.astype(np.float64)[:, None]), -127, 127), 0.0)
    return np.nan_to_num(q).astype(np.int8), s


def act(x, kind):
    """(value, derivative) of an activation in 64 bits."""
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-x))
    erf = np.vectorize(math.erf, otypes=[float])
    if kind == "sigmoid":
        return s, s * (1 - s)
    if kind == "silu":
        return x * s, s + x * s * (1 - s)
    if kind == "gelu":
        p = 0.5 * (1 + erf(x / math.sqrt(2)))
        return x * p, p + x * np.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = np.tanh(c * (x + 0.044715 * x ** 3))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)
    if kind == "relu":
        return np.maximum(x, 0), (x > 0).astype(float)
    return x, np.ones_like(x)


def gated_bound(g, u, dg, du, kind, t):
    """How far act(g) * u may be off where g and u are off by dg and du. Slopes are at most 1.13 in magnitude (1.0998 silu, 1.1290 gelu), second derivatives at
    most 1.1 (so a slope at a point dg away adds 1.1 dg * dg). The value itself: exp, erf and tanh within 4 units of the computing type, their argument's rounding
    times the slope, at most 6 further operations: 16 half steps of (1 + |g|), which is above the value and above any intermediate."""
    c = CALC[t]
    v, s = act(g, kind)
    dv = np.abs(s) * dg + 1.1 * dg * dg + 16 * c * (1 + np.abs(g))
    return np.abs(u) * dv + np.abs(v) * du + dv * du + 2 * c * np.abs(v * u) + UNIT[t] * (np.abs(v * u) + np.abs(u) * dv + np.abs(v) * du) + TINY[t]
