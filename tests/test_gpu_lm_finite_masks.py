"""token_logprob_grad on rows far from 0: masked throughout by a large finite
value, shifted far up, and on the way there."""
import numpy as np
import pytest

import lm_oracle as O

pytestmark = pytest.mark.gpu

NP = {"float": np.float32, "float16": np.float16, "double": np.float64}
FILLS = {"float": [-1e9, -1e10, -1e30, -3.4028234663852886e38], "float16": [-65504.0],
         "double": [-1e17, -1e30, -1.7976931348623157e308]}
# at this lse (times a scale above 1) and below no digits are left for what log
# probabilities are made of
FAR = {"float": -2.0 ** 20, "float16": -2.0 ** 20, "double": -2.0 ** 49}


def gradient(acd, x, dtype, axis, tokens, lse, H, g, gH, gl, scale, stride=1, inplace=False):
    """x: rows x V in any layout that the kernels tell apart.  Returns rows x V."""
    sd = "double" if dtype == "double" else "float"
    a = np.asfortranarray(x.T) if axis == 1 else x
    t = acd.as_tensor(a, dtype=dtype)
    if stride != 1:  # every stride-th element of a larger tensor
        import torch
        st = torch.zeros(t.size * stride, dtype=t.storage.dtype, device="cuda")
        st[::stride] = t.storage[:t.size]
        t = acd.gpuTensor(st, a.shape, dtype, (stride, stride * a.shape[0]), 0)
    w = lambda v: None if v is None else acd.as_tensor(v, dtype=sd)  # noqa: E731
    got = acd.token_logprob_grad(t, acd.as_tensor(tokens, dtype="int64"), w(lse), w(H), w(g), w(gH), w(gl), axis=axis,
                                 scale=scale, inplace=inplace).as_array()
    return got.T if axis == 1 else got


@pytest.mark.parametrize("dtype", ["float", "float16", "double"])
@pytest.mark.parametrize("axis,rows,V,stride", [(1, 11, 600, 1), (1, 11, 601, 2), (2, 12, 600, 1), (2, 11, 33, 1),
                                                (2, 40, 3, 1), (1, 11, 32000, 1)])
@pytest.mark.parametrize("scale", [0.1, 0.7, 1.0, 1.3, 1.5, 50.0])
def test_rows_masked_throughout(acd, dtype, axis, rows, V, stride, scale):
    """Such a row's gradient is 0 where its lse has no digits left, and its
    formula's (lse as the forward call has rounded it) otherwise; its neighbours
    keep theirs."""
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((rows, V)) * 3).astype(NP[dtype])
    for k, fill in enumerate(FILLS[dtype]):
        x[2 * k + 1] = fill
    tokens = rng.integers(1, V + 1, rows)
    st = np.float64 if dtype == "double" else np.float32
    a = np.asfortranarray(x.T) if axis == 1 else x
    r = acd.token_logprob(acd.as_tensor(a, dtype=dtype), acd.as_tensor(tokens, dtype="int64"), axis=axis, scale=scale)
    lse, H = r.logsumexp.as_array().reshape(-1), r.entropy.as_array().reshape(-1)
    g, gH, gl = (rng.uniform(0.5, 1.5, rows).astype(st) for _ in range(3))
    f = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
    far = lse <= FAR[dtype] * max(1.0, scale)
    assert far.sum() == (0 if dtype == "float16" else len(FILLS[dtype]))
    for gHk, glk, inplace in ((None, None, False), (gH, gl, True)):
        got = gradient(acd, x, dtype, axis, tokens, lse, H, g, gHk, glk, scale, stride, inplace)
        exp = O.logprob_grad(x[~far], tokens[~far], f(lse[~far]), f(H[~far]), f(g[~far]),
                             None if gHk is None else f(gHk[~far]), None if glk is None else f(glk[~far]), scale, -np.inf)
        bound = O.logprob_grad_bound(exp, x[~far], f(lse[~far]), f(H[~far]), f(g[~far]),
                                     None if gHk is None else f(gHk[~far]), None if glk is None else f(glk[~far]), scale,
                                     dtype)
        O.assert_within(got[~far], exp, bound, "rows with digits")
        assert not got[far].any(), "masked rows"
    zero = np.zeros(rows, st)
    assert not gradient(acd, x, dtype, axis, tokens, lse, H, zero, zero, zero, scale, stride).any(), "zero gradients"


@pytest.mark.parametrize("dtype", ["float", "float16"])
@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("scale", [1e3, 1e5, 1e6])
def test_ordinary_logits_at_low_temperatures(acd, dtype, axis, scale):
    """A large scale takes lse far down too; the row still has its likeliest token."""
    V, rows = 300, 16
    rng = np.random.default_rng(5)
    x = rng.integers(-60, -31, (rows, V)).astype(NP[dtype])
    best = rng.integers(0, V, rows)
    x[np.arange(rows), best] = -30
    tokens = best + 1
    tokens[::2] = 1 + (best[::2] + 1) % V  # another one
    a = np.asfortranarray(x.T) if axis == 1 else x
    r = acd.token_logprob(acd.as_tensor(a, dtype=dtype), acd.as_tensor(tokens, dtype="int64"), axis=axis, scale=scale)
    lse = r.logsumexp.as_array().reshape(-1)
    g = np.full(rows, 1.0 / scale, np.float32)
    got = gradient(acd, x, dtype, axis, tokens, lse, None, g, None, None, scale).astype(np.float64)
    # p of the likeliest token is 1 to within |lse| 2^-24 (lse's rounding) and as much for scale's
    off = np.expm1(2 * 30 * scale * 2.0 ** -24) + 2.0 ** -10
    want = np.zeros((rows, V))
    want[np.arange(rows), best] -= 1
    want[np.arange(rows), tokens - 1] += 1
    assert np.abs(got - want).max() <= off
    assert np.abs(got[np.arange(rows), tokens - 1][::2] - 1).max() <= 2.0 ** -10


@pytest.mark.parametrize("dtype,top", [("float", 1e9), ("float", 1e30), ("float16", 65504.0), ("double", 1e30)])
@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("scale", [0.7, 1.0, 1.3])
def test_rows_far_up(acd, dtype, top, axis, scale):
    """A probability is never above 1, however lse was rounded; no gradient in, none out."""
    V, rows = 600, 12
    rng = np.random.default_rng(1)
    st = np.float64 if dtype == "double" else np.float32
    x = (rng.standard_normal((rows, V)) * 3).astype(NP[dtype])
    x[1:9] = top
    x[5:9] = top * (1 - rng.uniform(0, 0.5, (4, V)))
    tokens = rng.integers(1, V + 1, rows)
    a = np.asfortranarray(x.T) if axis == 1 else x
    r = acd.token_logprob(acd.as_tensor(a, dtype=dtype), acd.as_tensor(tokens, dtype="int64"), axis=axis, scale=scale)
    lse, H = r.logsumexp.as_array().reshape(-1), r.entropy.as_array().reshape(-1)
    one, zero = np.ones(rows, st), np.zeros(rows, st)
    got = gradient(acd, x, dtype, axis, tokens, lse, H, None, None, one, scale)  # scale * p
    assert (got >= 0).all() and (got <= scale * (1 + 2.0 ** -10)).all()
    got = gradient(acd, x, dtype, axis, tokens, lse, H, one, one, one, scale)
    assert np.isfinite(got).all()
    assert not gradient(acd, x, dtype, axis, tokens, lse, H, zero, zero, zero, scale).any()


@pytest.mark.parametrize("dtype", ["float", "float16"])
@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("shift", [-3e2, -1e4, -6e4, -3e5, 1e4])
def test_rows_on_the_way(acd, dtype, axis, shift):
    """The probabilities are off by what lse's rounding makes of them (half a
    unit in its last place), against the softmax itself in float64."""
    if dtype == "float16" and abs(shift) > 65000:
        pytest.skip("beyond float16")
    V, rows = 700, 16
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((rows, V)) * 3 + shift).astype(NP[dtype])
    tokens = rng.integers(1, V + 1, rows)
    a = np.asfortranarray(x.T) if axis == 1 else x
    r = acd.token_logprob(acd.as_tensor(a, dtype=dtype), acd.as_tensor(tokens, dtype="int64"), axis=axis)
    lse = r.logsumexp.as_array().reshape(-1)
    got = gradient(acd, x, dtype, axis, tokens, lse, None, None, None, np.ones(rows, np.float32), 1.0)
    z = x.astype(np.float64)
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    # lse: its own rounding and that of ln S (a chain of at most V/8 additions); d
    # and d log2 e one rounding each; exp and the product a few u; storage
    u = 2.0 ** -24
    off = u * (np.abs(lse).max() + 100 + V / 8 + 64)
    rs, ss = O.STORE[dtype]
    O.assert_within(got, p, p * (np.expm1(off) + (3 * np.abs(np.log(p)) + 16) * u + rs) + ss + 2e-38, "p")
