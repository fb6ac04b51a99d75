"""Rows of logits of which only some count, for tests that a kernel leaves none
of a long row out and takes none twice.

Row r has its peaks at every position of one residue class modulo `period`, so
that a period of rows has a peak at every position once.  All peaks lie within
half a nat of each other; the other logits are 120 below, which is exactly 0 in
the sums (e^-120 is below the smallest normal float32, and below half a unit in
the last place of a float64 sum).  One peak more or less then moves the sum by
a fraction 0.6 / n of it (n peaks a row), which the bounds below are far under:

  a sum of n terms in any order and grouping is off by (n + merges) u of it
  (adding exact zeros rounds nothing); each term by 2 u for the logit's
  difference, 2 u for its product with the scale (both times |z| <= 7: a
  kernel's reference may lie 8 bits below the maximum), 4 u for the exponential;
  at most 40 merges of partial sums, which scale a sum by an exponential each.
"""
import numpy as np

LOW = -120.0


def peaks(V, period, rows, rng, dtype, scale=1.0):
    """(first, values): row r's peaks stand at first[r], first[r] + period, ..., values[r]
    long (a row of fewer holds NaN at the end); exact in `dtype`."""
    first = np.arange(rows) % period
    n = -(-V // period)
    # within half a nat, on a grid that float16 has exactly
    values = rng.integers(0, 64, (rows, n)) / 128.0 / scale
    values = values.astype(dtype).astype(np.float64)
    values[first + (n - 1) * period >= V, n - 1] = np.nan
    return first, values


def dense(V, period, first, values, dtype):
    """rows x V logits."""
    x = np.full((len(first), V), LOW, dtype)
    for r, f in enumerate(first):
        v = values[r][~np.isnan(values[r])]
        x[r, f::period] = v
    return x


def statistics(values, scale, drop=None):
    """(lse, entropy) of rows with these peaks; drop: leaves out that many last ones."""
    lse, H = [], []
    for v in values:
        v = v[~np.isnan(v)]
        v = v[:len(v) - drop] if drop else v
        z = scale * (v - v.max())
        e = np.exp(z)
        S = e.sum()
        lse.append(scale * v.max() + np.log(S))
        H.append(np.log(S) - (e * z).sum() / S)
    return np.array(lse), np.array(H)


def bounds(values, lse, H, u):
    """(lse, entropy, logprob)."""
    n = values.shape[1]
    rel = (n + 40 * 8 + 7 * 4 + 4) * u
    # T / S: off by twice the relative error times |z| <= 7
    return rel + 4 * u * np.abs(lse) + 4 * u, rel + 14 * rel + 4 * u * (np.abs(H) + 8), rel + 4 * u * (np.abs(lse) + 1)
