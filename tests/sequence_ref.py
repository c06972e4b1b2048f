"""The linear recurrence, the products grouped by expert and their gradients
in 64 bits on the host, with bounds of what the kernels' roundings may add.

u = 2^-53.  An f32 result is rounded once (2^-24 of its value), a packed pair
to 2^-48 of its value: hi is off by at most 2^-24 of the value, and lo holds
the rest to 2^-24 of it.  The smallest subnormal's half, 2^-150, is what
either may lose below the normal range.
"""
import numpy as np

U = 2.0 ** -53
LONG = np.longdouble


def pair_of(x):
    """emitFromFloat: the packed pair [..., 2] of f64 values."""
    hi = x.astype(np.float32)
    with np.errstate(invalid="ignore"):
        lo = (x - hi.astype(np.float64)).astype(np.float32)
    return np.stack([hi, lo], axis=-1)


def value_of(p):
    return p[..., 0].astype(np.float64) + p[..., 1].astype(np.float64)


def as_type(x, kind):
    """(array handed to the kernel, its exact f64 values)."""
    if kind == "f64":
        return x, x
    if kind == "f32":
        y = x.astype(np.float32)
        return y, y.astype(np.float64)
    y = pair_of(x)
    return y, value_of(y)


def result_rounding(value, kind):
    """How far the one rounding to the result's type moves `value`."""
    v = np.abs(value)
    if kind == "f64":
        return 0.0 * v
    return v * (2.0 ** -24 if kind == "f32" else 2.0 ** -48) + 2.0 ** -150


def recurrence(a, b, h0=None):
    """h and the recurrence of the magnitudes, [B, T, D]."""
    B, T, D = a.shape
    h = np.zeros((B, D), LONG) if h0 is None else h0.astype(LONG)
    m = np.abs(h)
    out, mag = np.empty((B, T, D), LONG), np.empty((B, T, D), LONG)
    with np.errstate(invalid="ignore", over="ignore"):
        for t in range(T):
            h = a[:, t].astype(LONG) * h + b[:, t].astype(LONG)
            m = np.abs(a[:, t]).astype(LONG) * m + np.abs(b[:, t]).astype(LONG)
            out[:, t], mag[:, t] = h, m
    return out, mag


def recurrence_bound(mag, kind, value):
    """A term b_s a_{s+1} ... a_t passes at most t - s products of
    coefficients, as many FMAs and one more per joined chunk: 3 T + 4
    roundings bound them all, each u of the term's magnitude (the doubling
    covers the higher orders); then the result's rounding."""
    T = mag.shape[1]
    return ((3 * T + 4) * 2 * U * mag + result_rounding(value, kind)).astype(np.float64)


def recurrence_vjp(a, h, gh, h0=None):
    """(grad_a, grad_b, grad_h0) and their magnitudes."""
    B, T, D = a.shape
    a, h, gh = a.astype(LONG), h.astype(LONG), gh.astype(LONG)
    s = np.zeros((B, D), LONG) if h0 is None else h0.astype(LONG)
    ga, gb, ma, mb = (np.empty((B, T, D), LONG) for _ in range(4))
    c, m = np.zeros((B, D), LONG), np.zeros((B, D), LONG)
    with np.errstate(invalid="ignore", over="ignore"):
        for t in reversed(range(T)):
            g = gh[:, t] + c
            mg = np.abs(gh[:, t]) + m
            before = h[:, t - 1] if t else s
            ga[:, t], gb[:, t] = g * before, g
            ma[:, t], mb[:, t] = mg * np.abs(before), mg
            c, m = a[:, t] * g, np.abs(a[:, t]) * mg
    return (ga, gb, c), (ma, mb, m)


def vjp_bounds(values, mags, kind, T):
    """As recurrence_bound; grad_a and grad_h0 are one product more."""
    return [((3 * T + 6) * 2 * U * m + result_rounding(v, kind)).astype(np.float64)
            for v, m in zip(values, mags)]


def spans(sizes, M):
    """[(group, first row, end)] with negative sizes as 0 and groups ending at M."""
    at, out = 0, []
    for g, n in enumerate(sizes):
        end = min(M, at + max(int(n), 0))
        out.append((g, at, end))
        at = end
    return out


def _product_bound(a, b, c, kind):
    """Error of a[m, K] b[K, n] = c.  f64 sums: K + 2 roundings of the terms'
    magnitudes.  The tensor-core product keeps a row of a and a column of b to
    P bits below their largest value's next power of two (at most twice it),
    half a unit each, so an output is off by at most K of the units
    2^-P (2 max|a_i|) (2 max|b_j|) (and 2^35 / 2^P more from the rebuilt low
    limb), with P as planned for K: min(50, floor((110.2 - 2 - log2 K) / 2));
    then two roundings."""
    K = a.shape[1]
    terms = np.abs(a) @ np.abs(b)
    f64 = (K + 2) * 2 * U * terms
    P = min(50, int((110.2 - 2 - np.log2(max(K, 1))) // 2))
    chunks = -(-max(K, 1) // 32768)
    if chunks > 1:
        P = int((110.2 - 2 - 15) // 2)
    rowmax = np.abs(a).max(axis=1, initial=0.0)[:, None]
    colmax = np.abs(b).max(axis=0, initial=0.0)[None, :]
    unit = 4.0 * rowmax * colmax * 2.0 ** -P
    tensor = (K + 2.0 ** (35 - P) * chunks) * unit + (2 + chunks) * U * np.abs(c)
    rounding = result_rounding(c, "f64" if kind == "f64" else "packed")
    return np.maximum(f64, tensor) + rounding * 2 ** (chunks - 1)


def matmul_long(a, b):
    """a @ b to about twice f64: a's leading bits apart, so that each partial
    product's terms are exact in long double sums on the host for small
    sizes, f64 for large ones."""
    if a.shape[0] * a.shape[1] * b.shape[1] <= 1 << 24:
        return (a.astype(LONG) @ b.astype(LONG)).astype(np.float64)
    return a @ b


def ragged_dot(lhs, rhs, sizes, kind="f64"):
    """rhs [G, K, N] -> (out [M, N], bound)."""
    M, N = lhs.shape[0], rhs.shape[2]
    out, bound = np.zeros((M, N)), np.zeros((M, N))
    for g, s, e in spans(sizes, M):
        if e > s:
            out[s:e] = matmul_long(lhs[s:e], rhs[g])
            bound[s:e] = _product_bound(lhs[s:e], rhs[g], out[s:e], kind)
    return out, bound


def ragged_contract(lhs, rhs, sizes, kind="f64"):
    """-> (out [G, K, N], bound)."""
    M = lhs.shape[0]
    out = np.zeros((len(sizes), lhs.shape[1], rhs.shape[1]))
    bound = np.zeros_like(out)
    for g, s, e in spans(sizes, M):
        if e > s:
            out[g] = matmul_long(lhs[s:e].T, rhs[s:e])
            bound[g] = _product_bound(lhs[s:e].T, rhs[s:e], out[g], kind)
    return out, bound
