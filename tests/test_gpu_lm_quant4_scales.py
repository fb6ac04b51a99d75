"""quant4_encode: scales, zero points and weights bit for bit, and ranges that the
scales' type does not hold."""
import numpy as np
import pytest

import lm_oracle as O

pytestmark = pytest.mark.gpu

NP = {"float": np.float32, "float16": np.float16, "double": np.float64}


def encode(w, group, zeros, sdt):
    """The definition: float64 throughout, the scale rounded once, and to the type's
    largest value where it is beyond it.  (weights M x K, scales, zeros: groups x M)"""
    M, K = w.shape
    G = -(-K // group)
    w = w.astype(np.float64)
    pad = np.zeros((M, G * group))
    pad[:, :K] = w
    pad = pad.reshape(M, G, group)
    lo, hi = np.minimum(pad.min(2), 0), np.maximum(pad.max(2), 0)
    exact = (hi / 15 - lo / 15) if zeros else np.maximum(hi, -lo) / 7
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        s = exact.astype(NP[sdt]).astype(np.float64)
        big = np.isinf(s)
        s[big] = np.finfo(NP[sdt]).max
        z = np.full((M, G), 8.0)
        if zeros:
            z = np.where(s > 0, np.clip(np.rint(-lo / np.where(big, exact, s)), 0, 15), 0.0)
        g = np.arange(K) // group
        q = np.where(s[:, g] > 0, np.clip(np.rint(w / s[:, g]) + z[:, g], 0, 15), z[:, g])
    return q.astype(int), s.T, z.T


def check(acd, w, group, zeros, sdt, dtype):
    got = acd.quant4_encode(acd.as_tensor(w, dtype=dtype), group, zeros=zeros, scale_dtype=sdt)
    q, s, z = encode(w, group, zeros, sdt)
    assert np.array_equal(got.scales.as_array().astype(np.float64), s)
    if zeros:
        assert np.array_equal(got.zeros.as_array().astype(np.float64), z)
    assert np.array_equal(O.quant4_unpack(got.weights.as_array(), w.shape[1]), q)
    return got, q, s, z


@pytest.mark.parametrize("dtype", ["float", "float16", "double"])
@pytest.mark.parametrize("sdt", ["float", "float16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,K,group", [(700, 256, 32), (33, 1000, 96), (129, 77, 128)])
def test_bit_for_bit(acd, dtype, sdt, zeros, M, K, group):
    rng = np.random.default_rng(M)
    w = rng.standard_normal((M, K)) * rng.choice([1e-3, 1.0, 50.0], (M, 1))
    w[1] = 0
    w[2] = np.abs(w[2])
    w[3] = -np.abs(w[3])
    w[4] = np.rint(w[4]) / 2  # quotients that are ties
    check(acd, w.astype(NP[dtype]), group, zeros, sdt, dtype)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype,sdt,large", [("float", "float16", 4e5), ("float", "float16", 1e6), ("float", "float16", 1e30),
                                             ("float", "float16", 3e38), ("float", "float", 3e38),
                                             ("double", "float16", 1e9), ("double", "float", 1e39),
                                             ("double", "float", 1e300), ("double", "float", 1.7e308)])
def test_finite_weights_stay_finite(acd, dtype, sdt, large, zeros):
    """Scales beyond their type's range are its largest value: weights are cut off,
    never NaN, and their signs stay."""
    rng = np.random.default_rng(7)
    w = rng.uniform(-1, 1, (40, 128))
    w[:, ::32] = 1
    w[:20, 1::32] = -1
    w = (w * large).astype(NP[dtype])
    w[7] = np.abs(w[7])
    w[8] = -np.abs(w[8])
    w[9] = 0.25  # an ordinary row beside
    got, q, s, z = check(acd, w, 32, zeros, sdt, dtype)
    assert np.isfinite(got.scales.as_array()).all()
    x = acd.as_tensor(np.eye(128, 4), dtype="float")
    y = acd.quant4_matvec(got.weights, got.scales, x, 32, zeros=got.zeros).as_array()
    # (products are summed in float32, which weights above its range leave)
    held = (s * 15 <= np.finfo(np.float32).max).all(0)
    assert held[9] and np.isfinite(y[held]).all()
    sign = np.sign(y) * np.sign(w[:, :4])
    assert (sign[held, 0] >= 0).all() and (sign[:20, 1][held[:20]] >= 0).all()


def test_weights_that_are_not_finite(acd):
    """NaN scales for the groups of such weights alone, in every type."""
    for dtype in ("float", "float16", "double"):
        for zeros in (False, True):
            w = np.ones((3, 64), NP[dtype])
            w[0, 3], w[1, 40], w[2, 0] = np.nan, np.inf, -np.inf
            s = acd.quant4_encode(acd.as_tensor(w, dtype=dtype), 32, zeros=zeros).scales.as_array()
            assert np.array_equal(np.isnan(s), [[True, False, True], [False, True, False]])
