"""Scales at the ends of the statistics' range: below the smallest float32 the
distribution is uniform over what is not masked; what has no float32 is refused."""
import numpy as np
import pytest

import acediar._lib as L
import lm_oracle as O

pytestmark = pytest.mark.gpu

NP = {"float": np.float32, "float16": np.float16, "double": np.float64}


@pytest.mark.parametrize("dtype", ["float", "float16", "double"])
@pytest.mark.parametrize("axis,rows,V", [(1, 5, 700), (2, 40, 300), (1, 4, 33)])
@pytest.mark.parametrize("scale", [1e-300, 1e-50, 3e-45, 1e-39, 1e-30])
def test_scales_next_to_zero(acd, dtype, axis, rows, V, scale):
    """scale * x is below 1e-6 for every logit up to 1e24: all that count are alike."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((rows, V)) * (1e24 if dtype == "float" else 100)
    x = x.astype(NP[dtype])
    drop = rng.random((rows, V)) < 0.3
    drop[:, :2] = [True, False]
    x[drop] = -np.inf
    x[rows - 1] = -np.inf
    tokens = np.full(rows, 2)
    tokens[1] = 1  # masked
    a = np.asfortranarray(x.T) if axis == 1 else x
    t, tok = acd.as_tensor(a, dtype=dtype), acd.as_tensor(tokens, dtype="int64")
    r = acd.token_logprob(t, tok, axis=axis, scale=scale, top=2)
    f = lambda v: v.as_array().reshape(-1)  # noqa: E731
    ref = O.logprob(x, tokens, scale, 2)
    u = 2.0 ** -24
    b = (V / 8 + 64) * u * 12 + 2e-6
    O.assert_within(f(r.logprob), ref[0], b, "logprob")
    O.assert_within(f(r.entropy), ref[1], b, "entropy")
    O.assert_within(f(r.logsumexp), ref[2], b, "lse")
    top = r.top_index.as_array()
    assert np.array_equal(top.T if axis == 1 else top, ref[3])
    tl = r.top_logprob.as_array()
    O.assert_within(tl.T if axis == 1 else tl, ref[4], b, "top_logprob")
    sd = "double" if dtype == "double" else "float"
    one = acd.as_tensor(np.ones(rows), dtype=sd)
    g = acd.token_logprob_grad(t, tok, r.logsumexp, r.entropy, one, one, one, axis=axis, scale=scale).as_array()
    # |gradient| <= scale * (1 + p (1 + 1 + small)), rounded to the type's subnormals
    assert np.isfinite(g).all() and np.abs(g.astype(np.float64)).max() <= 4 * scale + 1e-44


@pytest.mark.parametrize("dtype", ["float", "float16"])
def test_large_scales(acd, dtype):
    """1e37 puts everything on the largest logit; beyond float32 a scale is refused."""
    x = np.array([[0.0, 1.0, 0.5], [2.0, -np.inf, 1.0]]).T.astype(NP[dtype])
    t, tok = acd.as_tensor(x, dtype=dtype), acd.as_tensor([2, 1], dtype="int64")
    st = acd.as_tensor([0.0, 0.0], dtype="float")
    r = acd.token_logprob(t, tok, scale=1e37)
    assert np.array_equal(r.logprob.as_array(), [0, 0]) and np.array_equal(r.entropy.as_array(), [0, 0])
    for scale in (3e38, 1e39, 1e300):
        for call in (lambda: acd.token_logprob(t, tok, scale=scale),
                     lambda: acd.token_logprob_grad(t, tok, st, d_logprob=st, scale=scale)):
            with pytest.raises(L.AcdError) as e:
                call()
            assert e.value.status == 1
    d = acd.as_tensor(x.astype(np.float64), dtype="double")
    assert np.array_equal(acd.token_logprob(d, tok, scale=1e300).logprob.as_array(), [0, 0])
