"""Plain implementations, in at least 64 bits, of layer norm, dropout and the gated block, with bounds on what a correct evaluation in a smaller
type may differ from them: every bound is a first-order count of roundings, u = half a unit in the last place of 1."""
import numpy as np

WIDE = np.longdouble


def unit(dtype):
    return np.finfo(dtype).eps / 2


# ---- dropout ---------------------------------------------------------------------------------------------------------------------
def philox4x32(counter, key, rounds=10):
    """counter: four arrays of 32-bit values (as uint64), key: two values; Salmon et al. 2011, with their constants."""
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ np.uint64(k0), b & low, (a >> shift) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def keeps(shape, p, seed, stream):
    n = int(np.prod(shape))
    i = np.arange((n + 3) // 4, dtype=np.uint64)
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    s = np.uint64(stream & 0xFFFFFFFFFFFFFFFF)
    words = philox4x32([i & low, i >> shift, np.full_like(i, s & low), np.full_like(i, s >> shift)], (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    return (np.stack(words, 1).reshape(-1)[:n] >= np.uint64(int(p * 2.0 ** 32))).reshape(shape)


def dropout(x, p, seed, stream, residual=None):
    """in x's own type: one rounding for the product, one for the sum, so a correct evaluation gives these very values"""
    t = x.dtype.type
    v = np.where(keeps(x.shape, p, seed, stream), x * t(1.0 / (1.0 - p)), t(0))
    return v if residual is None else residual + v


# ---- layer norm ------------------------------------------------------------------------------------------------------------------
def norm(x, gain, shift, eps):
    x = x.astype(WIDE)
    mu = x.mean(-1, keepdims=True)
    r = 1 / np.sqrt(((x - mu) ** 2).mean(-1, keepdims=True) + WIDE(eps))
    xh = (x - mu) * r
    y = xh * (1 if gain is None else gain.astype(WIDE)) + (0 if shift is None else shift.astype(WIDE))
    return y, xh, r


SUM = 96   # additions that a sum over a row passes through: at most 32 in a thread, the lanes, the warps and the chunks


def norm_errors(x, xh, r, u):
    """What xh may be off by: the mean by SUM u mean|x|, the differences by a rounding each, r by half of what the variance is."""
    return u * (SUM * np.abs(x.astype(WIDE)).mean(-1, keepdims=True) * r + (SUM / 2 + 6) * np.abs(xh))


def norm_bound(x, gain, y, xh, r, u):
    g = 1 if gain is None else np.abs(gain.astype(WIDE))
    return (norm_errors(x, xh, r, u) + u * np.abs(xh)) * g + 3 * u * (np.abs(y) + np.abs(xh) * g)


def norm_gradients(x, gain, e, eps, u):
    """(dx, bound), (dgain, bound), (dshift, bound)"""
    y, xh, r = norm(x, None, None, eps)
    off = norm_errors(x, xh, r, u)
    e = e.astype(WIDE)
    g = e if gain is None else e * gain.astype(WIDE)
    m1, m2 = g.mean(-1, keepdims=True), (g * xh).mean(-1, keepdims=True)
    dx = r * (g - m1 - xh * m2)
    a1, a2 = np.abs(g).mean(-1, keepdims=True), np.abs(g * xh).mean(-1, keepdims=True)
    m2_off = (SUM + 4) * u * a2 + (np.abs(g) * off).mean(-1, keepdims=True)
    dx_off = r * (4 * u * np.abs(g) + (SUM + 2) * u * a1 + off * np.abs(m2) + np.abs(xh) * m2_off + 4 * u * np.abs(xh * m2) + 2 * u * np.abs(m1)) + (SUM / 2 + 6) * u * np.abs(dx)
    axes = tuple(range(x.ndim - 1))
    rows = int(np.prod(x.shape[:-1])) + 4
    dgain_off = (np.abs(e) * off).sum(axes) + rows * u * np.abs(e * xh).sum(axes)
    return (dx, dx_off), ((e * xh).sum(axes), dgain_off), (e.sum(axes), rows * u * np.abs(e).sum(axes))


# ---- the gated block -------------------------------------------------------------------------------------------------------------
def gate(fun, g):
    """value and derivative, as the framework defines the functions"""
    g = g.astype(WIDE)
    if fun == "idy":
        return g, np.ones_like(g)
    if fun == "relu":
        s = np.where(g >= 0, WIDE(1), WIDE(0.01))
        return g * s, s
    if fun == "tanh":
        t = np.tanh(g)
        return t, 1 - t * t
    k = WIDE(1.702) if fun == "gelu" else WIDE(1)
    s = 1 / (1 + np.exp(-k * g))
    if fun == "sig":
        return s, s * (1 - s)
    return g * s, s + k * g * s * (1 - s)


SLOPE, CURVE = 1.2, 0.9   # no gate is steeper than 1.1, no derivative (but relu's step) than 1.702 / 2
PRODUCT = {np.dtype(np.float32): 1e-5, np.dtype(np.float64): 1e-12}   # a product's bound relative to sum |a||b|, as for every product of the framework


def gated(x, wg, wu, fun):
    """(y, bound) and what the gradients need"""
    tol, u_ = PRODUCT[x.dtype], unit(x.dtype)
    X, G, U = x.astype(WIDE), wg.astype(WIDE), wu.astype(WIDE)
    g, u = X @ G, X @ U
    g_off, u_off = tol * (np.abs(X) @ np.abs(G)), tol * (np.abs(X) @ np.abs(U))
    f, df = gate(fun, g)
    f_off = SLOPE * g_off + 4 * u_ * np.abs(f)
    y = f * u
    return (y, f_off * (np.abs(u) + u_off) + np.abs(f) * u_off + 2 * u_ * np.abs(y)), (g, u, g_off, u_off, f, df, f_off)


def gated_gradients(x, wg, wu, e, fun):
    """(dx, bound), (dwg, bound), (dwu, bound)"""
    tol, u_ = PRODUCT[x.dtype], unit(x.dtype)
    _, (g, u, g_off, u_off, f, df, f_off) = gated(x, wg, wu, fun)
    X, G, U, E = (a.astype(WIDE) for a in (x, wg, wu, e))
    df_off = CURVE * g_off + 8 * u_ * (1 + np.abs(df))
    if fun == "relu":
        df_off = df_off + np.where(np.abs(g) <= g_off, WIDE(0.99), WIDE(0))   # either side of the step
    dg, du = E * u * df, E * f
    dg_off = np.abs(E) * (u_off * (np.abs(df) + df_off) + np.abs(u) * df_off) + 4 * u_ * np.abs(dg)
    du_off = np.abs(E) * f_off + 2 * u_ * np.abs(du)
    dx = dg @ G.T + du @ U.T
    dx_off = (dg_off + tol * np.abs(dg)) @ np.abs(G.T) + (du_off + tol * np.abs(du)) @ np.abs(U.T) + 2 * u_ * np.abs(dx)
    A = np.abs(X.T)
    return (dx, dx_off), (X.T @ dg, A @ (dg_off + tol * np.abs(dg))), (X.T @ du, A @ (du_off + tol * np.abs(du)))


def assert_within(got, want_and_bound, what):
    want, bound = want_and_bound
    got = np.asarray(got).astype(WIDE).reshape(np.shape(want))
    off = np.abs(got - want)
    bad = ~(off <= bound + np.finfo(np.float64).tiny)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} values outside their bounds, worst {float((off / (bound + 1e-300)).max()):.3g} of the bound"
