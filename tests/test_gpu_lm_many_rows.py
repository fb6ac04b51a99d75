"""Alternatives of many short rows across the lanes, on both sides of the number of
rows from which a thread takes a row of its own."""
import numpy as np
import pytest
import torch

import lm_oracle as O

pytestmark = pytest.mark.gpu

NP = {"float": np.float32, "float16": np.float16}


@pytest.mark.parametrize("dtype", ["float", "float16"])
@pytest.mark.parametrize("rows", [9000, 9604, 18948, 28416, 42624, 47364])
@pytest.mark.parametrize("top", [1, 2, 3, 5, 7, 8])
def test_alternatives(acd, dtype, rows, top):
    """Smooth and coarse logits, ties at the last alternative, masked rows, NaN inside;
    indices exactly, log probabilities against the formula from those."""
    V = 140
    rng = np.random.default_rng(rows + top)
    x = (rng.standard_normal((rows, V)) * 3).astype(NP[dtype])
    x[: rows // 3] = np.rint(x[: rows // 3])
    x[10:40] = -np.inf
    x[20:40, 17] = 1
    x[30:40, 3] = 1
    x[50:60, ::5] = np.nan
    x[60:70] = 2
    x[rows - 5:] = np.arange(V)
    got = acd.token_logprob(acd.as_tensor(x, dtype=dtype), None, axis=2, top=top)
    wide = x.astype(np.float64)
    key = np.where(np.isnan(wide), -np.inf, wide)
    order = np.argsort(-key, axis=1, kind="stable")
    # NaN never: among -Inf logits they would come in the order of their index
    order[50:60] = [np.concatenate([r[~np.isnan(w[r])], r[np.isnan(w[r])]]) for r, w in zip(order[50:60], wide[50:60])]
    want = order[:, :top]
    assert np.array_equal(got.top_index.as_array(), want + 1)
    m = key.max(1, keepdims=True)
    nan = np.isnan(wide).any(1)
    with np.errstate(invalid="ignore", divide="ignore"):
        S = np.where(np.isneginf(key), 0, np.exp(key - m)).sum(1, keepdims=True)
        lp = np.take_along_axis(wide, want, 1) - m - np.log(S)
    lp[np.isneginf(m[:, 0])] = -np.inf
    lp[nan] = np.nan
    # a chain of at most V / 8 additions and 8 merges in S, then a subtraction
    u = 2.0 ** -24
    O.assert_within(got.top_logprob.as_array(), lp, (V / 8 + 100) * u + 8 * u * (np.where(np.isfinite(lp), np.abs(lp), 0) + 1))
