"""Attention over behaviour lists in 64 bits: the rotation with norms, linear attention and attention on shared prefixes, each with a bound on
what a kernel may be off.

u = 2^-24 is half a step of fp32. Exponentials, roots and quotients of the kernels are taken to be right to 2^-21 relative; a result is
rounded once to its own type (half a step). Where a kernel rounds an operand to fewer bits on the way, its share stands beside the bound."""
import numpy as np

from ssm_oracle import HALF, TINY, U, close  # noqa: F401


def rope(x, positions, freqs, weight, eps, norm, adjacent, dtype):
    """x [rows, heads, d]. The mean is a sum of d squares (off by (d + 2) u relative), its root and quotient by 2^-21 and half of that; cosines and
    sines are off by 2^-21 (2 units in the last place and the angle's rounding to fp32, at most pi u)."""
    rows, heads, d = x.shape
    t, e = x.copy(), np.zeros_like(x)
    if norm:
        t = t / np.sqrt((t * t).mean(-1, keepdims=True) + eps) * (weight if weight is not None else 1.0)
        e = np.abs(t) * ((d / 2 + 4) * U + 2.0 ** -20)
    half = 0 if freqs is None else len(freqs)
    y, ey = t.copy(), e.copy()
    if half:
        w = positions.astype(np.float64)[:, None, None] * freqs
        i, j = (2 * np.arange(half), 2 * np.arange(half) + 1) if adjacent else (np.arange(half), half + np.arange(half))
        a, b = t[..., i], t[..., j]
        y[..., i], y[..., j] = a * np.cos(w) - b * np.sin(w), b * np.cos(w) + a * np.sin(w)
        size = np.abs(a) + np.abs(b)
        off = e[..., i] + e[..., j] + size * (2.0 ** -21 + 3 * U + np.abs(w) * 2.0 ** -51)
        ey[..., i] = ey[..., j] = off
    return y, ey + HALF[dtype] * (np.abs(y) + ey) + TINY[dtype]


def linear(q, k, v, log_decay, scale, lists, h0, dtype):
    """q [rows, H, dk], k [rows, Hkv, dk], v [rows, Hkv, dv], h0: [H, dk, dv] a list. Returns y, its bound, the last states and theirs.

    `A` is the state with |k| |v| for k v. fp32 goes row by row: a row's three roundings are of the state's own size, (the decay less 1) is known to
    2^-21 of itself, and y is a sum of dk products. 16-bit types go by rows or by chunks of 64: there the state's operands are known to 2^-22 of
    themselves, what a matrix instruction adds is cut off (2^-23 of the running sum, 12 of them a chunk), and of what y is made of scores and states are
    rounded to TF32 (half a step, 2^-12). A decay over n rows is exp(n log_decay), off by (n |log_decay| + 2) u and 2^-21."""
    rows, H, dk = q.shape
    share, dv = H // k.shape[1], v.shape[2]
    y, ey = np.full((rows, H, dv), np.nan), np.full((rows, H, dv), np.nan)
    last, elast = [], []
    ld = np.minimum(log_decay, 0.0)
    g = np.exp(ld)[:, None, None]
    with np.errstate(invalid="ignore"):
        lost = np.where(np.isinf(ld), 0.0, (-np.expm1(ld) * 2.0 ** -21 + 2.0 ** -21 * np.minimum(1.0, -ld)))[:, None, None]
    half_type = dtype != "f32"
    for (r0, r1), h in zip(lists, h0):
        S, A, E = h.copy(), np.abs(h), np.zeros_like(h)
        for t in range(r0, r1):
            kk, vv = np.repeat(k[t], share, 0), np.repeat(v[t], share, 0)
            kv = kk[:, :, None] * vv[:, None, :]
            E = g * E + lost * A + 3 * U * (g * A + np.abs(kv)) + (2.0 ** -19 * np.abs(kv) if half_type else 0)
            S, A = g * S + kv, g * A + np.abs(kv)
            out = scale * np.einsum("hk,hkv->hv", q[t], S)
            sized = abs(scale) * np.einsum("hk,hkv->hv", np.abs(q[t]), A)
            off = abs(scale) * np.einsum("hk,hkv->hv", np.abs(q[t]), E) + sized * ((dk + 4) * U + (2.0 ** -12 + 2.0 ** -17 if half_type else 0))
            y[t], ey[t] = out, off + HALF[dtype] * (np.abs(out) + off) + TINY[dtype]
        last.append(S)
        elast.append(E + 2.0 ** -126)
    return y, ey, last, elast
