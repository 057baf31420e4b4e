"""Plain numpy forms in 64 bits of the operators of transformer layers (jittor_amd/layers.py), and bounds of their errors in 32 bits.
Shared by test_layers.py and test_gpu_layers.py."""
import math

import numpy as np

from jittor_amd.dtypes import bf16_bits_to_f32

ULP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}      # relative error of rounding to nearest
TINY = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25, "float32": 2.0 ** -150}  # and below the normal range
E = 2.0 ** -24


def to_type(a, dtype):
    """(storage, exact values of it in 64 bits)"""
    a = np.asarray(a, np.float32)
    if dtype == "bfloat16":
        bits = a.view(np.uint32)
        odd = bits >> 16 & 1
        raw = np.where(np.isnan(a), np.uint32(0x7FC00000), bits + 0x7FFF + odd) >> 16
        raw = raw.astype(np.uint16).reshape(a.shape)
        return raw, bf16_bits_to_f32(raw).astype(np.float64)
    a = a.astype(np.float16) if dtype == "float16" else a
    return a, a.astype(np.float64)


# ---- dropout ------------------------------------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 of one counter of four words and a key of two, in Python integers."""
    c, k, low = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def numbers(n, seed, offset):
    """The 32 bits of elements 0 .. n - 1."""
    seed, offset, low = seed & (1 << 64) - 1, offset & (1 << 64) - 1, 0xFFFFFFFF
    u = []
    for g in range((n + 7) // 8):
        blocks = [philox([g & low, (g >> 32) | block << 31, offset & low, offset >> 32], [seed & low, seed >> 32]) for block in (0, 1)]
        for j in range(8):
            hi, lo = ((b[j // 2] >> 16 * (j % 2)) & 0xFFFF for b in blocks)
            u.append(hi << 16 | lo)
    return np.array(u[:n], np.uint64)


def kept(n, p, seed, offset):
    return numbers(n, seed, offset) >= round(p * 2.0 ** 32)


# ---- norms of heads and rotation ------------------------------------------------------------------------------------
def angles_of(table, positions, sections, lead):
    """(cos, sin) [tokens, pairs] from the table and positions [axes, tokens]; NaN for rows that are not there."""
    axis = np.repeat(np.arange(len(sections)), sections)
    at = positions[axis].T                                                   # [tokens, pairs]
    there = (at >= 0) & (at < len(table))
    t = np.where(there[..., None], table[np.where(there, at, 0), np.arange(table.shape[1])], np.nan)
    return t[..., 0], t[..., 1]


def turn(z, cos, sin, paired):
    """z [tokens, heads, dim]"""
    y = z.copy()
    if cos is None:
        return y
    n = cos.shape[1]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if paired else (slice(0, n), slice(n, 2 * n))
    c, s = cos[:, None], sin[:, None]
    y[..., a], y[..., b] = z[..., a] * c - z[..., b] * s, z[..., a] * s + z[..., b] * c
    return y


def pair_size(z, cos, paired):
    """For each element |a| + |b| of its pair: what an error of the turned values is relative to."""
    m = np.abs(z)
    if cos is None:
        return m
    n = cos.shape[1]
    out = m.copy()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if paired else (slice(0, n), slice(n, 2 * n))
    out[..., a] = out[..., b] = m[..., a] + m[..., b]
    return out


def head_norm(x, scale, cos, sin, eps, paired):
    """Forward of heads of one kind: x [tokens, heads, dim]."""
    if scale is None:
        return turn(x, cos, sin, paired)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return turn(x * r * scale, cos, sin, paired)


def head_norm_grad(x, scale, cos, sin, eps, paired, dy):
    """(dx, dscale) and the sizes their errors are relative to."""
    dz = turn(dy, cos, None if sin is None else -sin, paired)
    size = pair_size(dy, cos, paired)
    if scale is None:
        return dz, None, size, None
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = x * r
    dn = dz * scale
    dx = r * (dn - n * (dn * n).mean(-1, keepdims=True))
    sdn = size * np.abs(scale)
    return dx, (dz * n).sum((0, 1)), r * (sdn + np.abs(n) * (sdn * np.abs(n)).mean(-1, keepdims=True)), (size * np.abs(n)).sum((0, 1))


# ---- gated projections ------------------------------------------------------------------------------------------------
def activation(name, g):
    """The activation and its derivative."""
    with np.errstate(over="ignore"):
        s = 1.0 / (1.0 + np.exp(-g))
    if name == "relu":
        return np.maximum(g, 0.0), (g > 0).astype(np.float64)
    if name == "sigmoid":
        return s, s * (1.0 - s)
    if name == "silu":
        return g * s, s * (1.0 + g * (1.0 - s))
    below = 0.5 * np.vectorize(math.erfc)(-g / math.sqrt(2.0))
    return g * below, below + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)


def gated(x, w, name):
    """y and the bound of its error in 32 bits, before it is rounded.  The products' errors: K additions of at most E relative to the sum of
    magnitudes.  |act'| is below 1.2; an activation in 32 bits is good to 16 E of its argument's size."""
    f = len(w) // 2
    both = x @ w.T
    off = (x.shape[1] + 2) * E * (np.abs(x) @ np.abs(w).T)
    (g, u), (eg, eu) = (both[:, :f], both[:, f:]), (off[:, :f], off[:, f:])
    a, _ = activation(name, g)
    ea = 1.2 * eg + 16 * E * np.maximum(np.abs(a), np.abs(g) * E + 2.0 ** -126)
    return a * u, ea * np.abs(u) + np.abs(a) * eu + ea * eu + 2 * E * np.abs(a * u)


def gated_grad(x, w, name, dy, dtype):
    """(dx, dw) and bounds of their errors.  d is rounded to the operands' type before the products; |act''| is below 1.2 too, except that
    relu's derivative jumps: gates nearer to zero than their error may fall on either side."""
    f = len(w) // 2
    both = x @ w.T
    off = (x.shape[1] + 2) * E * (np.abs(x) @ np.abs(w).T)
    (g, u), (eg, eu) = (both[:, :f], both[:, f:]), (off[:, :f], off[:, f:])
    a, da = activation(name, g)
    d = np.concatenate([dy * u * da, dy * a], 1)
    slope = np.where(np.abs(g) <= eg, 1.0, 0.0) if name == "relu" else 1.2 * eg
    ea, eda = 1.2 * eg + 16 * E * (np.abs(a) + np.abs(g) * E), slope + 16 * E * (np.abs(da) + 1.0)
    ed = np.concatenate([np.abs(dy) * (eu * (np.abs(da) + eda) + np.abs(u) * eda), np.abs(dy) * ea], 1) + (ULP[dtype] + 4 * E) * np.abs(d) + TINY[dtype]
    dx, dw = d @ w, d.T @ x
    return (dx, (ed + 2 * f * 2 * E * np.abs(d)) @ np.abs(w) + E * np.abs(dx)), (dw, (ed + 2 * len(x) * E * np.abs(d)).T @ np.abs(x) + E * np.abs(dw))
