"""The state-space layer's convolution and scan, and the projection with adapters, in 64 bits, each with a bound on what a kernel
that works in 32 bits may be off.

The bounds follow the formulas step by step with u = 2^-24 (half a step of fp32). Exponentials, quotients and logarithms of the
kernels are taken to be right to 2^-21 relative and softplus to 2^-20; a result is rounded once to its own type (half a step)."""
import numpy as np

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}        # below the normal numbers a step is this large


def _sigmoid(v):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-v))


def conv(x, w, bias, lists, states, silu, dtype):
    """lists: [(first, last)], states: [K - 1, D] a list. Returns y, its bound, the states after."""
    D, K = w.shape
    y, e, after = np.full(x.shape, np.nan), np.full(x.shape, np.nan), []
    for (r0, r1), st in zip(lists, states):
        ahead = np.concatenate([st, x[r0:r1]])
        after.append(ahead[len(ahead) - (K - 1):])
        n = r1 - r0
        terms = np.stack([ahead[j:j + n] * w[:, j] for j in range(K)])
        v = terms.sum(0) + bias
        ev = (K + 1) * U * (np.abs(terms).sum(0) + np.abs(bias))
        if silu:
            out = v * _sigmoid(v)
            ev = 1.1 * ev + 2.0 ** -20 * np.abs(out)
        else:
            out = v
        y[r0:r1], e[r0:r1] = out, ev + HALF[dtype] * (np.abs(out) + ev) + TINY[dtype]
    return y, e, after


def scan(x, delta, A, B, C, skip, z, bias, groups, softplus, lists, h0, dtype):
    """B, C [rows, groups, N]; h0: [D, N] a list. Returns y, its bound, the last states and theirs."""
    D, N = A.shape
    g = np.arange(D) // (D // groups)
    y, e, last, elast = np.full(x.shape, np.nan), np.full(x.shape, np.nan), [], []
    v = delta + bias
    with np.errstate(over="ignore"):
        d = np.where(v > 30, v + np.exp(-np.abs(v)), np.log1p(np.exp(np.minimum(v, 30)))) if softplus else v
    ed = (d * 2.0 ** -20 + _sigmoid(v) * U * np.abs(v)) if softplus else U * np.abs(v)
    for (r0, r1), h in zip(lists, h0):
        h = h.copy()
        eh = np.zeros_like(h)
        for t in range(r0, r1):
            dt, edt = d[t][:, None], ed[t][:, None]
            q = dt * A
            with np.errstate(over="ignore", invalid="ignore"):
                a = np.exp(q)
                ea = a * (np.abs(A) * edt + 3 * U * np.abs(q) + 2.0 ** -21)
                b = dt * x[t][:, None] * B[t][g]
                eb = np.abs(x[t][:, None] * B[t][g]) * edt + 4 * U * np.abs(b)
                eh = a * eh + ea * np.abs(h) + eb
                h = a * h + b
                eh = eh + U * np.abs(h)
                out = (C[t][g] * h).sum(1)
                eo = (np.abs(C[t][g]) * eh).sum(1) + (N + 2) * U * np.abs(C[t][g] * h).sum(1)
                s = skip * x[t]
                out, eo = out + s, eo + 2 * U * np.abs(s) + U * np.abs(out + s)
                if z is not None:
                    gate = z[t] * _sigmoid(z[t])
                    out, eo = out * gate, eo * np.abs(gate) + np.abs(out * gate) * 2.0 ** -20
            y[t], e[t] = out, eo + HALF[dtype] * (np.abs(out) + eo) + TINY[dtype]
        last.append(h)
        elast.append(eh + 2.0 ** -126)
    return y, e, last, elast


def lora(X, W, A, B, adapter, scale, bias, dtype):
    """W [K, N]. Sums of K products: a kernel adds at most K times (matrix instructions: K / 16 times, cut off to a step)."""
    K, r = X.shape[1], A.shape[1]
    y = X @ W + bias
    e = (K + 2) * U * (np.abs(X) @ np.abs(W) + np.abs(bias))
    for a in range(len(A)):
        m = adapter == a
        if not m.any():
            continue
        u = scale[a] * (X[m] @ A[a].T)
        eu = (K + 2) * U * np.abs(scale[a]) * (np.abs(X[m]) @ np.abs(A[a]).T) + 2.0 ** -21 * np.abs(u)
        y[m] += u @ B[a].T
        e[m] += eu @ np.abs(B[a]).T + (r + 2) * U * (np.abs(u) @ np.abs(B[a]).T)
    e = e + 2 * U * np.abs(y)
    return y, e + HALF[dtype] * (np.abs(y) + e) + TINY[dtype]


def close(got, want, bound, what=""):
    """Element by element; where the bound is not finite the sign of an overflow has no say, so those must not occur."""
    got, want, bound = (np.asarray(t, np.float64) for t in (got, want, bound))
    assert np.isfinite(want).all() and np.isfinite(bound).all(), what
    off = np.abs(got - want)
    bad = ~(off <= bound)
    if bad.any():
        i = tuple(int(k) for k in np.argwhere(bad)[0])
        raise AssertionError("%s: %d of %d off; first at %s: %r, %r wanted, bound %g (largest off / bound %.3g)" % (
            what, bad.sum(), bad.size, i, float(got[i]), float(want[i]), float(bound[i]), float(np.nanmax(off / bound))))
