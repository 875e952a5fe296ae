"""64-bit forms of the gated recurrent block's operators, each with a bound on the rounding of a
float32 computation of it (numpy, element by element, no code of the package).

Units: U = 2^-24 is half a step of float32.  A product, sum or fused product is off by at most 1 U, a
quotient by 2 steps (4 U), the fast exp(z) by 2 steps and, since it rounds its argument, 2 |z| U.  So
q = sigmoid(-f) = 1 / (1 + exp(f)) is off by at most (12 + 2 |f|) U of itself, and a = 1 - q by that and
half a unit of its own range, U."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # eps / 2
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -25}


def rounding(value, kind):
    """How far rounding `value` to a type may move it: eps / 2 relative, or half the smallest number
    (fp16's 2^-25; the float32 range of the others leaves nothing to speak of)."""
    return HALF_STEP[kind] * np.abs(value) + TINY[kind]


def sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def gated_scan(f, x, h0, gate, borders, dy=None, dh=None):
    """borders: (first, past) rows of each sequence; rows [L, C], h0 and dh [S, C].  Returns
    {name: (value, error bound before the rounding to the output's type)}."""
    L, C = f.shape
    a, q = sigmoid(f), sigmoid(-f)
    z = gate if gate is not None else None
    w = sigmoid(z) if z is not None else None
    silu = z * w if z is not None else np.ones_like(f)
    # q itself is off by q_err, and as exp(f) is what carries the error, min(a, q) by that share of it; a = 1 - q
    # by the same and its rounding.  Composing steps rounds the products of a and the partial states once more
    small, q_err = np.minimum(a, q), (12 + 2 * np.abs(f)) * U
    q_off = np.minimum(q, q_err * small + 8 * U * q)
    a_off = q_off + U
    fast = (14 + 2 * np.abs(z)) * U if z is not None else np.zeros_like(f)
    silu_err = fast * np.abs(silu)
    h, he = np.zeros((L, C)), np.zeros((L, C))
    before, be = np.zeros((L, C)), np.zeros((L, C))
    last, laste = np.zeros_like(h0), np.zeros_like(h0)
    inside = np.zeros((L, 1))
    for s, (b, e) in enumerate(borders):
        inside[b:e] = 1.0
        v, err = h0[s].copy(), np.zeros(C)
        for t in range(b, e):
            before[t], be[t] = v, err
            err = a[t] * err + a_off[t] * np.abs(v) + q_off[t] * np.abs(x[t]) + 4 * U * (a[t] * np.abs(v) + np.abs(x[t]))
            v = a[t] * v + q[t] * x[t]
            h[t], he[t] = v, err
        last[s], laste[s] = v, err
    out = {"y": (inside * h * silu, inside * (he * np.abs(silu) + np.abs(h) * silu_err + U * np.abs(h * silu))),
           "h": (last, laste)}
    if dy is None and dh is None:
        return out
    dy = np.zeros_like(f) if dy is None else dy
    dh = np.zeros_like(h0) if dh is None else dh
    e_t = dy * silu
    e_err = np.abs(dy) * silu_err + U * np.abs(e_t)
    lam, le = np.zeros((L, C)), np.zeros((L, C))
    dh0, dh0e = np.zeros_like(h0), np.zeros_like(h0)
    for s, (b, e) in enumerate(borders):
        m, me = dh[s].copy(), np.zeros(C)
        for t in range(e - 1, b - 1, -1):
            lam[t] = e_t[t] + m
            le[t] = e_err[t] + me + 2 * U * (np.abs(e_t[t]) + np.abs(m))
            m, me = a[t] * lam[t], a[t] * le[t] + (a_off[t] + 4 * U * a[t]) * np.abs(lam[t])
        dh0[s], dh0e[s] = m, me
    D = before - x
    De = be + U * (np.abs(before) + np.abs(x))
    df, dx = lam * D * a * q, lam * q
    out["dx"] = (dx, q * le + (q_off + 2 * U * q) * np.abs(lam))
    out["df"] = (df, np.abs(lam * a * q) * De + np.abs(D * a * q) * le + (a_off * q + a * q_off) * np.abs(lam * D)
                 + 6 * U * np.abs(df))
    out["dh0"] = (dh0, dh0e)
    if z is not None:
        slope = w * (1 + z * (1 - w))
        # 1 - w is off by `fast` at most, and 1 + z (1 - w) by that times |z| and its own rounding
        slope_err = w * (fast * np.abs(z) + 2 * fast * (1 + np.abs(z) * (1 - w)))
        out["dgate"] = (inside * dy * h * slope, inside * np.abs(dy) * (he * np.abs(slope) + np.abs(h) * slope_err
                                                                        + 2 * U * np.abs(h * slope)))
    return out


def silu_gated_linear(x, wg, wu, kind, dy=None):
    """Sums over K products in float32, in any order: off by at most (K + 16) 2 U of the sum of their
    sizes (2 U an addition: an accumulator may cut instead of rounding).  The fast exp rounds its
    argument too: off by (4 + 2 |g|) U.  float16 gradients dg, du are rounded after scaling by a power
    of two that brings the largest |dy| into [1, 2): numbers below 2^-14 of that keep 2^-25 of it."""
    C, F, R = x.shape[1], wg.shape[0], x.shape[0]
    g, u = x @ wg.T, x @ wu.T
    sum_err = lambda k: (k + 16) * 2 * U  # noqa: E731
    ge, ue = sum_err(C) * (np.abs(x) @ np.abs(wg).T), sum_err(C) * (np.abs(x) @ np.abs(wu).T)
    w = sigmoid(g)
    silu, slope = g * w, w * (1 + g * (1 - w))
    fast = (14 + 2 * np.abs(g)) * U
    se = 1.1 * ge + fast * np.abs(silu)  # |silu'| <= 1.1
    out = {"y": (silu * u, se * np.abs(u) + np.abs(silu) * ue + U * np.abs(silu * u))}
    if dy is None:
        return out
    dg, du = dy * u * slope, dy * silu
    # |silu''| <= 0.5; 1 - w is off by `fast` at most, and 1 + g (1 - w) by that times |g|
    slope_err = 0.5 * ge + w * (fast * np.abs(g) + 2 * fast * (1 + np.abs(g) * (1 - w)))
    dge = np.abs(dy) * (ue * np.abs(slope) + np.abs(u) * slope_err) + 4 * U * np.abs(dg)
    due = np.abs(dy) * se + 2 * U * np.abs(du)
    # the operands of the products that follow are rounded to the type once
    floor = TINY[kind] * (2.0 * np.abs(dy).max() if kind == "float16" and dy.size else 1.0)
    dge, due = dge + HALF_STEP[kind] * np.abs(dg) + floor, due + HALF_STEP[kind] * np.abs(du) + floor
    aw, au, ax = np.abs(wg), np.abs(wu), np.abs(x)
    out["dx"] = (dg @ wg + du @ wu, dge @ aw + due @ au + sum_err(2 * F) * (np.abs(dg) @ aw + np.abs(du) @ au))
    out["dwg"] = (dg.T @ x, dge.T @ ax + sum_err(R) * (np.abs(dg).T @ ax))
    out["dwu"] = (du.T @ x, due.T @ ax + sum_err(R) * (np.abs(du).T @ ax))
    return out


def philox_halves(n, seed, offset, block=0):
    """The 16-bit numbers of n places from place 8 `block` on: Philox4x32-10 in Python's own whole numbers."""
    low, out = 0xFFFFFFFF, []
    for j in range(block, block + (n + 7) // 8):
        c = [j & low, j >> 32, offset & low, (offset >> 32) & low]
        k = [seed & low, (seed >> 32) & low]
        for _ in range(10):
            p, r = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(r >> 32) ^ c[1] ^ k[0], r & low, (p >> 32) ^ c[3] ^ k[1], p & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        for word in c:
            out += [word & 0xFFFF, word >> 16]
    return np.array(out[:n], dtype=np.int64)


def within(got, value, bound, kind):
    """The largest share of its allowed error that any element of `got` uses (to be <= 1)."""
    allowed = bound + rounding(np.abs(value) + bound, kind)
    d = np.abs(np.asarray(got, dtype=np.float64) - value)
    return float((d / allowed).max()) if d.size else 0.0
