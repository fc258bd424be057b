"""numpy restatement (float64, unsigned integers) of the group norm with activation and dropout, of the dropout by units, and of
the random words they go by."""
import math

import numpy as np

EPS_OF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # half a step of a rounding


def philox4x32_10(counter, key):
    """counter (..., 4), key (2,): 32-bit words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011)."""
    a, b, c, d = (np.asarray(counter, np.uint64)[..., q] for q in range(4))
    k0, k1 = int(key[0]), int(key[1])
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p, q = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (q >> np.uint64(32)) ^ b ^ np.uint64(k0), q & low, (p >> np.uint64(32)) ^ d ^ np.uint64(k1), p & low
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack([a, b, c, d], -1).astype(np.uint32)


def keep_factor(units, p, rng):
    """What dropout multiplies the given units (an array of their numbers) by."""
    units = np.asarray(units, np.uint64)
    seed, offset = (int(v) % 2 ** 64 for v in rng)
    block = units >> np.uint64(3)
    counter = np.stack([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF),
                        np.full_like(block, offset >> 32)], -1)
    words = philox4x32_10(counter, (seed & 0xFFFFFFFF, seed >> 32))
    at = (units & np.uint64(7)).astype(np.int64)
    word = np.take_along_axis(words, (at >> 1)[..., None], -1)[..., 0] >> (16 * (at & 1)).astype(np.uint32) & np.uint32(0xFFFF)
    t = math.floor(65536 * p + 0.5)
    return np.where(word >= t, 65536 / (65536 - t) if t < 65536 else 0.0, 0.0)


def _phi(z):
    return 0.5 * np.vectorize(math.erfc, otypes=[float])(-z * math.sqrt(0.5))


def activation(z, kind):
    """(act(z), act'(z))"""
    if kind == "relu":
        return np.maximum(z, 0), (z > 0).astype(float)
    if kind == "silu":
        s = 1 / (1 + np.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if kind == "gelu":
        return z * _phi(z), _phi(z) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, np.ones_like(z)


def group_norm_act(x, lengths, groups, weight, bias, eps, residual, act, p, rng, grad):
    """Everything in float64: a dict of y, dx, dw, db, dresidual, and of the parts that error bounds are made of."""
    n, c = x.shape
    w = np.ones(c) if weight is None else weight
    b = np.zeros(c) if bias is None else bias
    keep = keep_factor(np.arange(n * c), p, rng).reshape(n, c) if p else np.ones((n, c))
    out = {k: np.zeros((n, c)) for k in ("y", "dx", "dresidual", "z", "xh", "rstd", "m1", "m2", "gh")}
    at = 0
    for length in list(lengths) + [0]:
        rows = slice(at, at + length)
        at += length
        if length == 0:
            continue
        v = x[rows].reshape(length, groups, -1)
        mean = v.mean((0, 2), keepdims=True)
        rstd = 1 / np.sqrt(((v - mean) ** 2).mean((0, 2), keepdims=True) + eps)
        xh = ((v - mean) * rstd).reshape(length, c)
        z = xh * w + b + (0 if residual is None else residual[rows])
        y, slope = activation(z, act)
        gz = grad[rows] * slope * keep[rows]
        gh = gz * w
        by_group = lambda t: np.broadcast_to(t.reshape(length, groups, -1).mean((0, 2), keepdims=True), v.shape).reshape(length, c)
        out["m1"][rows], out["m2"][rows] = by_group(gh), by_group(gh * xh)
        out["y"][rows], out["dresidual"][rows], out["z"][rows], out["xh"][rows], out["gh"][rows] = y * keep[rows], gz, z, xh, gh
        out["rstd"][rows] = np.broadcast_to(rstd, v.shape).reshape(length, c)
        out["dx"][rows] = out["rstd"][rows] * (gh - out["m1"][rows] - xh * out["m2"][rows])
    out["dw"], out["db"] = (out["dresidual"] * out["xh"]).sum(0), out["dresidual"].sum(0)
    return out


def dropout(x, p, rng, unit, lengths, residual, relu, grad):
    """(y, dx, dresidual) in float64."""
    n, c = x.shape
    if unit == "element":
        keep = keep_factor(np.arange(n * c), p, rng).reshape(n, c)
    else:
        sample = np.repeat(np.arange(len(lengths)), lengths)
        keep = keep_factor(sample[:, None] * c + np.arange(c) if unit == "channel" else sample[:, None], p, rng) * np.ones((n, c))
    y = np.where(keep > 0, x, 0) * keep + (0 if residual is None else residual)
    g = np.where(y > 0, grad, 0) if relu else grad
    return np.maximum(y, 0) if relu else y, g * keep, g
