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
    rounded once, of fp16 to fp16 (half a step: it keeps 10 bits behind the leading one, so neighbours are 2^-10 of a value just above a power of two
    apart and a rounding is off by 2^-11 of it; every term of y has one such rounding, of its score or of the state), of bf16 to two bf16 terms (2^-17). A decay over n rows is exp(n log_decay), off by (n |log_decay| + 2) u and 2^-21."""
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
            off = abs(scale) * np.einsum("hk,hkv->hv", np.abs(q[t]), E) + sized * ((dk + 4) * U + ({'f16': 2.0 ** -11, 'bf16': 2.0 ** -16}.get(dtype, 0) + (2.0 ** -17 if half_type else 0)))
            y[t], ey[t] = out, off + HALF[dtype] * (np.abs(out) + off) + TINY[dtype]
        last.append(S)
        elast.append(E + 2.0 ** -126)
    return y, ey, last, elast


def prefix(q, k, v, lists, own, prefixes, pk, pv, scale, dtype):
    """q [rows, H, d]; lists, own: (first, last) of every list's queries and own rows; prefixes: (first, last) of its prefix, None: none.
    Returns y and its bound.

    A score is a sum of d products in fp32, which a matrix instruction cuts off (2^-23 of the running sum a step of 16, at most d / 16 + 1 of them); its
    exponential turns what it is off by into as much of the weight; ex2 is right to 2^-21 and fp32 holds the exponent, as large as `e`, to 2^-23 of it.
    Weights are rounded to the inputs' type beside values (half a step, of fp16 at least 2^-25 of the largest, since a maximum in use is not above the largest), and sums of n
    weights or products are off by 2^-23 a step of 16, joined in order."""
    rows, H, d = q.shape
    share = H // (k if k is not None else pk).shape[1]
    y, e = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    for (r0, r1), (o0, o1), pre in zip(lists, own, prefixes):
        n = r1 - r0
        for r in range(r0, r1):
            seen = max((o1 - o0) - (n - 1 - (r - r0)), 0)
            parts = ([(pk[pre[0]:pre[1]], pv[pre[0]:pre[1]])] if pre else []) + ([(k[o0:o0 + seen], v[o0:o0 + seen])] if k is not None else [])
            kk = np.repeat(np.concatenate([a for a, _ in parts]), share, 1) if parts else np.zeros((0, H, d))
            vv = np.repeat(np.concatenate([b for _, b in parts]), share, 1) if parts else np.zeros((0, H, d))
            if len(kk) == 0:
                y[r], e[r] = 0, 0
                continue
            s = scale * np.einsum("hd,khd->hk", q[r], kk)
            off = scale * np.einsum("hd,khd->hk", np.abs(q[r]), np.abs(kk)) * ((d / 16 + 4) * 2.0 ** -23) + np.abs(s) * 2.0 ** -22
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            off_w = off + 2.0 ** -20
            out = np.einsum("hk,khd->hd", w, vv)
            size = np.abs(vv)
            lost = np.einsum("hk,khd->hd", w * (off_w + HALF[dtype] * (1 + off_w)), size) + (len(kk) / 16 + 8) * 2.0 ** -23 * np.einsum("hk,khd->hd", w, size)
            if dtype == "f16":
                lost = lost + 2.0 ** -25 * w.max(1, keepdims=True) * size.sum(0)
            lost = lost + np.abs(out) * (np.einsum("hk,hk->h", w, off_w)[:, None] + (len(kk) / 16 + 8) * 2.0 ** -23)
            y[r], e[r] = out, lost + HALF[dtype] * (np.abs(out) + lost) + TINY[dtype]
    return y, e
