"""Plain float64 forms of the language-model operators, from their formulas,
with the error bounds that the tests hold the kernels to.

A bound is what the arithmetic allows in the type that the kernel sums in
(u = 2^-24 for float32, 2^-53 for float64): each operation is off by u of its
result, a sum of n terms by at most the longest chain of additions times u of
the sum of magnitudes, exp and log by a few u.
"""
import numpy as np

U = {"float": 2.0 ** -24, "float16": 2.0 ** -24, "double": 2.0 ** -53}
# rounding to the storage type: relative part, and the absolute part of subnormals
STORE = {"float": (2.0 ** -24, 0.0), "float16": (2.0 ** -11, 2.0 ** -25), "double": (2.0 ** -53, 0.0)}


def moved(x, axis):
    """Rows (column-major over the other axes) x elements along the 1-based axis."""
    return np.moveaxis(np.asarray(x), axis - 1, 0).reshape(x.shape[axis - 1], -1, order="F").T


def logprob(x, tokens, scale, top):
    """x: rows x V.  tokens count from 1.  (logprob, entropy, lse, index, top_logprob)."""
    x = np.asarray(x).astype(np.float64)
    rows, V = x.shape
    lp, H, lse = np.zeros(rows), np.zeros(rows), np.zeros(rows)
    index, tlp = np.zeros((rows, top), np.int64), np.zeros((rows, top))
    with np.errstate(all="ignore"):
        for r in range(rows):
            m = x[r].max()  # NaN when there is one
            if m == -np.inf:
                lse[r], H[r], log_s = -np.inf, 0.0, 0.0
            else:
                z = scale * (x[r] - m)
                e = np.exp(z)
                S = e.sum()
                log_s = np.log(S)
                lse[r] = scale * m + log_s
                H[r] = log_s - np.where(e == 0, 0.0, e * z).sum() / S
            t = int(tokens[r]) - 1
            if t == -1:
                lp[r] = 0.0
            elif not 0 <= t < V:
                lp[r] = np.nan
            else:
                lp[r] = -np.inf if m == -np.inf else scale * (x[r, t] - m) - log_s
            fine = np.flatnonzero(~np.isnan(x[r]))
            order = fine[np.argsort(-x[r, fine], kind="stable")][:top]
            index[r] = np.iinfo(np.int64).min
            tlp[r] = np.nan
            index[r, :len(order)] = order + 1
            tlp[r, :len(order)] = -np.inf if m == -np.inf else scale * (x[r, order] - m) - log_s
    return lp, H, lse, index, tlp


def logprob_bounds(ref, V, dtype):
    """Absolute bounds of (logprob, entropy, lse, top_logprob).  Terms below
    e^-17 of the maximum do not count, so z is off by at most 17 * 3 u; exp by
    4 u; the sum's longest chain is V / 32 additions and some merges."""
    u = U[dtype]
    lp, H, lse, _, tlp = ref
    S = (60 + V / 32 + 40) * u
    fin = lambda a: np.where(np.isfinite(a), np.abs(a), 0.0)  # noqa: E731
    # T / S: each z e is off like e, weighted by |z| <= 17 or so
    return (S + 4 * u * (fin(lp) + 1), 2 * S * (2 + np.log(V + 1.0) + fin(H)), S + 4 * u * fin(lse) + 4 * u,
            S + 4 * u * (fin(tlp) + 1))


def logprob_grad(x, tokens, lse, H, g, gH, gl, scale, lowest):
    """rows x V gradient from the stored lse and entropy."""
    x = np.asarray(x).astype(np.float64)
    rows, V = x.shape
    out = np.zeros((rows, V))
    with np.errstate(all="ignore"):
        for r in range(rows):
            if lse[r] <= lowest / 4:
                continue
            lp = scale * x[r] - lse[r]
            p = np.exp(lp)
            gt = 0.0
            t = int(tokens[r]) - 1 if tokens is not None else -1
            if g is not None and 0 <= t < V:
                gt = g[r]
            v = np.where(p == 0, 0.0, p * ((0 if gl is None else gl[r]) - gt
                                           - (0 if gH is None else gH[r] * (lp + H[r]))))
            if gt != 0.0:
                v[t] += gt
            out[r] = scale * v
    return out


def logprob_grad_bound(ref, x, lse, H, g, gH, gl, scale, dtype):
    u = U[dtype]
    x = np.asarray(x).astype(np.float64)
    a = lambda v: 0.0 if v is None else np.abs(np.asarray(v))[:, None]  # noqa: E731
    with np.errstate(all="ignore"):
        lp = scale * x - lse[:, None]
        p = np.exp(lp)
        rel = (np.abs(scale * x) + np.abs(lse[:, None]) + np.abs(lp)) * 2 * u + 16 * u
        mag = p * (a(g) + a(gl) + a(gH) * (np.abs(lp) + a(H)))
    mag = np.where(p == 0, 0.0, mag)
    rel = np.where(p == 0, 0.0, rel)
    r, s = STORE[dtype]
    # a p below the smallest normal float32 may be flushed
    return scale * (mag * (rel + 8 * u) + 8 * u * a(g) + 2e-38) + r * np.abs(ref) + s


def norm(r, b, w_pre, w_post, gate, alpha, eps, per):
    """rows x D each; gate groups x D or None.  (h, y, rstd_h, rstd_block)."""
    r, b = np.asarray(r, np.float64), np.asarray(b, np.float64)
    rb = None
    c = b
    if w_post is not None:
        rb = 1 / np.sqrt((b * b).mean(1) + eps)
        c = b * rb[:, None] * np.asarray(w_post, np.float64)
    if gate is not None:
        c = c * np.repeat(np.asarray(gate, np.float64), per, 0)
    h = alpha * r + c
    rh = 1 / np.sqrt((h * h).mean(1) + eps)
    return h, h * rh[:, None] * np.asarray(w_pre, np.float64), rh, rb, np.abs(alpha * r) + np.abs(c)


def norm_bounds(ref, w_pre, D, dtype):
    """(h, y, rstd_h, rstd_block).  mag bounds |alpha r| + |gate b'|."""
    u = U[dtype]
    h, y, rh, rb, mag = ref
    e = (D / 8 + 64) * u  # the mean of squares: chain of at most D/8 additions
    r, s = STORE[dtype]
    w = np.abs(np.asarray(w_pre, np.float64))
    herr = mag * (e + 8 * u)
    # rstd_h: half the relative error of mean(h^2), to which the errors of h add
    hrel = e + 2 * np.sqrt((herr ** 2).mean(1) / np.maximum((h * h).mean(1), 1e-300)) + 8 * u
    yerr = (herr + np.abs(h) * hrel[:, None]) * rh[:, None] * w
    return (herr + r * np.abs(h) + s, yerr + r * np.abs(y) + s, rh * hrel,
            None if rb is None else rb * (e + 8 * u))


def norm_grad(dh, dy, h, b, rh, rb, w_pre, w_post, gate, alpha, per):
    f = lambda a: np.asarray(a, np.float64)  # noqa: E731
    dy, h, b, wp = f(dy), f(h), f(b), f(w_pre)
    rh = f(rh)[:, None]
    hn = h * rh
    t = (0 if dh is None else f(dh)) + rh * (dy * wp - hn * (dy * wp * hn).mean(1, keepdims=True))
    g = np.repeat(f(gate), per, 0) if gate is not None else 1.0
    u = t * g
    bn, wo = b, 1.0
    if w_post is not None:
        rb, wo = f(rb)[:, None], f(w_post)
        bn = b * rb
        db = rb * (u * wo - bn * (u * wo * bn).mean(1, keepdims=True))
    else:
        db = u
    gates = 0 if gate is None else len(gate)
    dgate = (t * bn * wo).reshape(gates, per, -1).sum(1) if gates else None
    return (alpha * t, db, (dy * hn).sum(0), (u * bn).sum(0) if w_post is not None else None, dgate)


def norm_grad_bounds(args, dtype):
    """The same expressions over magnitudes, times the error of their chains."""
    dh, dy, h, b, rh, rb, w_pre, w_post, gate, alpha, per = args
    a = lambda v: None if v is None else np.abs(np.asarray(v, np.float64))  # noqa: E731
    D, rows = np.asarray(h).shape[1], np.asarray(h).shape[0]
    u = U[dtype]
    dh, dy, h, b, rh, rb, wp, wo, gate = (a(v) for v in (dh, dy, h, b, rh, rb, w_pre, w_post, gate))
    hn = h * rh[:, None]
    t = (0 if dh is None else dh) + rh[:, None] * (dy * wp + hn * (dy * wp * hn).mean(1, keepdims=True))
    g = np.repeat(gate, per, 0) if gate is not None else 1.0
    uu = t * g
    bn, w = b, 1.0
    if wo is not None:
        bn, w = b * rb[:, None], wo
        db = rb[:, None] * (uu * w + bn * (uu * w * bn).mean(1, keepdims=True))
    else:
        db = uu
    e = (D / 8 + 64) * u
    c = (rows + 64) * u + e  # column sums: at most one chain over all rows
    r, s = STORE[dtype]
    out = [abs(alpha) * t * (e + r) + s, db * (2 * e + r) + s, (dy * hn).sum(0) * c,
           (uu * bn).sum(0) * c if wo is not None else None,
           (t * bn * w).reshape(len(gate), per, -1).sum(1) * c if gate is not None else None]
    return out


def quant4_unpack(weights, K):
    """[16 ceil(K/32), M] int8 -> M x K values 0..15."""
    w = np.asarray(weights).view(np.uint8).T
    q = np.empty((w.shape[0], 2 * w.shape[1]), np.int64)
    q[:, 0::2] = w & 15
    q[:, 1::2] = w >> 4
    return q[:, :K]


def quant4_matvec(weights, scales, zeros, x, group, dtype_out):
    """(y, bound): M x n."""
    x = np.asarray(x, np.float64)
    x = x.reshape(x.shape[0], -1)
    K = x.shape[0]
    g = np.arange(K) // group
    q = quant4_unpack(weights, K)
    s = np.asarray(scales, np.float64).T[:, g]
    z = np.asarray(zeros, np.float64).T[:, g] if zeros is not None else 8.0
    y = ((q - z) * s) @ x
    r, sub = STORE[dtype_out]
    # the kernel may sum q x and the zero points apart; chains of at most K/8 additions
    mag = (np.abs(s) * (16 + np.abs(z))) @ np.abs(x)
    return y, mag * (K / 8 + 64) * U["float"] + r * np.abs(y) + sub


def assert_within(actual, expected, bound, what=""):
    """Equal where not finite, within `bound` elsewhere."""
    actual, expected = np.asarray(actual, np.float64), np.asarray(expected, np.float64)
    assert actual.shape == expected.shape, "%s: shape %s vs %s" % (what, actual.shape, expected.shape)
    fine = np.isfinite(expected)
    assert np.array_equal(np.isnan(actual), np.isnan(expected)), "%s: NaN in other places" % what
    inf = ~fine & ~np.isnan(expected)
    assert np.array_equal(actual[inf], expected[inf]), "%s: infinities differ" % what
    err = np.where(fine, np.abs(np.where(fine, actual, 0) - np.where(fine, expected, 0)), 0)
    bad = ~(err <= np.broadcast_to(bound, err.shape)) & fine
    if bad.any():
        k = np.unravel_index(int(np.argmax(np.where(bad, err, -1))), err.shape)
        raise AssertionError("%s: %d of %d outside the bound, at %s: %r, expected %r, bound %g" % (
            what, int(bad.sum()), err.size, k, actual[k], expected[k], np.broadcast_to(bound, err.shape)[k]))
