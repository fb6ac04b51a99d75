"""token_logprob on wide rows, every position of which counts in some row: see
lm_peaks.py.  Pieces, batches, tiles, segments and the shares of blocks and
clusters all end somewhere in a row; none may be left out or taken twice."""
import numpy as np
import pytest
import torch

import lm_peaks as P

pytestmark = pytest.mark.gpu

NP = {"float": np.float32, "float16": np.float16, "double": np.float64}
U = {"float": 2.0 ** -24, "float16": 2.0 ** -24, "double": 2.0 ** -53}

# dtype, layout, V, period, rows a call, alternatives.  Rows a call decide between a
# warp, a block and a cluster a row, and how a row is divided across the lanes.
CASES = [("float", "rows", 50001, 200, 3, 0), ("float", "rows", 50001, 200, 200, 5),
         ("float16", "rows", 131072, 1024, 1, 20), ("float16", "rows", 131071, 512, 16, 0),
         ("float16", "rows", 32767, 128, 128, 3), ("double", "rows", 40003, 160, 5, 2),
         ("float", "rows", 4099, 64, 2500, 0), ("float16", "rows", 8191, 64, 2500, 5),
         ("float", "strided", 4099, 64, 7, 3), ("float16", "strided", 9001, 64, 40, 0),
         ("float", "lanes", 50001, 200, 200, 0), ("float", "lanes", 50001, 200, 40, 5),
         ("float16", "lanes", 131071, 512, 64, 20), ("float16", "lanes", 32768, 128, 128, 0),
         ("float", "lanes", 4099, 64, 20000, 5), ("double", "lanes", 30011, 120, 121, 3),
         ("float", "lanes", 20011, 100, 5, 2)]


@pytest.mark.parametrize("dtype,layout,V,period,per,top", CASES)
def test_every_logit_counts_once(acd, dtype, layout, V, period, per, top):
    rng = np.random.default_rng(V)
    rows = max(period, per)
    first, values = P.peaks(V, period, rows, rng, NP[dtype])
    lse, H = P.statistics(values, 1.0)
    bl, bh, bp = (np.broadcast_to(b, rows) for b in P.bounds(values, lse, H, U[dtype]))
    # the peaks in place; tokens are peaks, the last one and the first one of a row among them
    T = {"float": torch.float32, "float16": torch.float16, "double": torch.float64}[dtype]
    which = rng.integers(0, (~np.isnan(values)).sum(1))
    which[::3] = (~np.isnan(values)).sum(1)[::3] - 1
    which[1::3] = 0
    tokens = first + which * period + 1
    token_value = values[np.arange(rows), which]
    x = torch.full((rows, V), P.LOW, dtype=T, device="cuda")
    n = values.shape[1]
    at = torch.from_numpy(first[:, None] + np.arange(n)[None, :] * period).cuda()
    ok = at < V
    r = torch.arange(rows, device="cuda")[:, None].expand(-1, n)
    x[r[ok], at[ok]] = torch.from_numpy(values).cuda().to(T)[ok]
    step = 2 if layout == "strided" else 1
    for r0 in range(0, rows, per):
        r1 = min(rows, r0 + per)
        part = x[r0:r1]
        m = r1 - r0
        if layout == "lanes":
            st = part.t().contiguous().reshape(-1)
            t, axis = acd.from_torch(st, (m, V), dtype), 2
        else:  # rows of odd width start at all offsets of a piece
            st = torch.full((m * V * step + 1,), float("nan"), dtype=T, device="cuda")
            st[: m * V * step: step] = part.reshape(-1)
            t, axis = acd.gpuTensor(st, (V, m), dtype, (step, step * V), 0), 1
        tok = acd.as_tensor(tokens[r0:r1], dtype="int64")
        got = acd.token_logprob(t, tok, axis=axis, top=top)
        f = lambda v: v.as_array().reshape(-1, order="F").astype(np.float64)  # noqa: E731
        e = lse[r0:r1]
        assert (np.abs(f(got.logsumexp) - e) <= bl[r0:r1]).all(), "lse of rows from %d" % r0
        assert (np.abs(f(got.entropy) - H[r0:r1]) <= bh[r0:r1]).all(), "entropy of rows from %d" % r0
        assert (np.abs(f(got.logprob) - (token_value[r0:r1] - e)) <= bp[r0:r1]).all(), "logprob of rows from %d" % r0
        if top:
            ix = got.top_index.as_array()
            ix = ix.T if axis == 1 else ix
            order = np.argsort(-np.where(np.isnan(values[r0:r1]), -np.inf, values[r0:r1]), axis=1, kind="stable")[:, :top]
            assert np.array_equal(ix, first[r0:r1, None] + order * period + 1), "alternatives of rows from %d" % r0
