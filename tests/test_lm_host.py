"""Language-model operators, what needs no GPU: the plain forms that the kernels
are held to (gradients against differences, a planted mistake is seen), argument
checks, and the packing of descriptors."""
import ctypes

import numpy as np
import pytest
import torch

import lm_oracle as O


@pytest.fixture(scope="module")
def pkg():
    import acediar
    return acediar


def differences(f, x, step=1e-6):
    """Central differences of the scalar f over x (float64, changed in place and back)."""
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        keep = x[i]
        x[i] = keep + step
        up = f()
        x[i] = keep - step
        g[i] = (up - f()) / (2 * step)
        x[i] = keep
    return g


@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_plain_logprob_gradient_against_differences(scale):
    rng = np.random.default_rng(0)
    x, tokens = rng.standard_normal((3, 7)), np.array([2, 7, 0])
    g, gH, gl = rng.standard_normal((3, 3))

    def loss():
        lp, H, lse, _, _ = O.logprob(x, tokens, scale, 0)
        return (g * lp).sum() + (gH * H).sum() + (gl * lse).sum()

    _, H, lse, _, _ = O.logprob(x, tokens, scale, 0)
    got = O.logprob_grad(x, tokens, lse, H, g, gH, gl, scale, -np.inf)
    # the third derivative of the loss is of the order of 10: step^2 of it, and
    # the rounding of the loss over the step
    assert np.abs(got - differences(loss, x)).max() < 1e-11 * 10 + 2 ** -52 * 20 / 1e-6


@pytest.mark.parametrize("post,gates", [(True, 2), (True, 1), (True, 0), (False, 2), (False, 0)])
def test_plain_norm_gradient_against_differences(post, gates):
    rng = np.random.default_rng(1)
    rows, D = 4, 6
    r, b, dh, dy = rng.standard_normal((4, rows, D))
    wp, wo = rng.standard_normal((2, D))
    wo = wo if post else None
    gate = rng.standard_normal((gates, D)) if gates else None
    per, alpha, eps = rows // gates if gates else rows, 0.7, 1e-6

    def loss():
        h, y = O.norm(r, b, wp, wo, gate, alpha, eps, per)[:2]
        return (dh * h).sum() + (dy * y).sum()

    h, _, rh, rb, _ = O.norm(r, b, wp, wo, gate, alpha, eps, per)
    got = O.norm_grad(dh, dy, h, b, rh, rb, wp, wo, gate, alpha, per)
    # as above; the formula leaves out nothing, eps is inside the reciprocal roots
    for g, x in zip(got, (r, b, wp, wo, gate)):
        if x is not None:
            d = differences(loss, x)
            assert np.abs(g - d).max() < 1e-5 * max(1.0, np.abs(d).max())


def test_a_planted_mistake_is_outside_the_bounds():
    """Leaving out one term of the formulas is far more than a float32 kernel may be off by."""
    rng = np.random.default_rng(2)
    x, tokens = rng.standard_normal((4, 1000)), np.array([1, 500, 1000, 3])
    ref = O.logprob(x, tokens, 1.0, 2)
    bound = O.logprob_bounds(ref, 1000, "float")[:3]
    wrong = O.logprob(x[:, :-1], tokens, 1.0, 2)  # a row that ends one logit early
    for k in (1, 2):
        assert (np.abs(wrong[k] - ref[k]) > np.broadcast_to(bound[k], 4)).all()
    w, K = rng.integers(-128, 128, (16 * 3, 5)).astype(np.int8), 90
    s, z = rng.random((3, 5)) + 0.5, rng.integers(0, 16, (3, 5)).astype(float)
    v = rng.standard_normal((K, 2))
    y, b = O.quant4_matvec(w, s, z, v, 32, "float")
    assert (np.abs(O.quant4_matvec(w, s, None, v, 32, "float")[0] - y) > b).all()
    flipped = ((w.view(np.uint8) >> 4) | (w.view(np.uint8) << 4)).astype(np.uint8).view(np.int8)
    assert (np.abs(O.quant4_matvec(flipped, s, z, v, 32, "float")[0] - y) > b).all()


def test_plain_quant4_against_loops():
    rng = np.random.default_rng(3)
    K, M, group = 45, 3, 32
    w = rng.integers(-128, 128, (32, M)).astype(np.int8)
    s, z, x = rng.random((2, M)), rng.random((2, M)) * 15, rng.standard_normal(K)
    y, _ = O.quant4_matvec(w, s, z, x, group, "float")
    for o in range(M):
        e = 0.0
        for k in range(K):
            byte = int(w[k // 2, o]) & 255
            e += ((byte >> 4 if k % 2 else byte & 15) - z[k // group, o]) * s[k // group, o] * x[k]
        assert abs(y[o, 0] - e) < 1e-12 * K * 16


def test_descriptors_are_packed_as_the_structure_lays_them_out(pkg):
    import acediar._lib as L
    from acediar import lm
    for shape, strides, offset, dtype in [((), (), 0, "float"), ((5,), (3,), 2, "float16"),
                                          ((4, 0, 7), (1, 4, 4), 0, "double"),
                                          ((2,) * 8, tuple(2 ** i for i in range(8)), 2 ** 40, "int64")]:
        t = pkg.gpuTensor(torch.empty(1), shape, dtype, strides, offset)
        packed = L.Desc.from_buffer_copy(lm._desc(t))
        made = t.desc()
        assert packed.data == made.data and packed.offset == made.offset
        assert packed.ndim == made.ndim and packed.dtype == made.dtype
        n = len(shape)
        assert list(packed.shape)[:n] == list(shape) and list(packed.stride)[:n] == list(strides)
    assert lm._desc(None) is None


def test_calls_without_a_context_are_refused(pkg):
    lib = pkg.lib()
    for name in ("acd_token_logprob", "acd_token_logprob_grad", "acd_residual_norm", "acd_residual_norm_grad",
                 "acd_quant4_encode", "acd_quant4_matvec"):
        f = getattr(lib, name)
        args = [0.0 if t is ctypes.c_double else 0 if t in (ctypes.c_int32, ctypes.c_int64) else None
                for t in f.argtypes]
        assert f(*args) == 1, name
        assert lib.acd_last_error().decode().startswith(name)


def test_arguments_are_checked_before_any_call(pkg):
    new = lambda shape, dtype="float": pkg.gpuTensor(torch.empty(1), shape, dtype)  # noqa: E731
    x, w = new((8, 4)), new((8,))
    for axis in (0, 3, 1.5, None, "1"):
        with pytest.raises(ValueError):
            pkg.token_logprob(x, None, axis=axis)
        with pytest.raises(ValueError):
            pkg.token_logprob_grad(x, None, w, d_logsumexp=w, axis=axis)
        with pytest.raises(ValueError):
            pkg.residual_norm(x, x, w, axis=axis)
        with pytest.raises(ValueError):
            pkg.residual_norm_grad(None, x, x, x, w, None, w, axis=axis)
    for top in (-1, 2.5, None):
        with pytest.raises(ValueError):
            pkg.token_logprob(x, None, top=top)
    q = new((16, 4), "int8")
    for group in (0, -32, 31, 33.5, None):
        with pytest.raises(ValueError):
            pkg.quant4_encode(x, group=group)
        with pytest.raises(ValueError):
            pkg.quant4_matvec(q, x, w, group=group)
    with pytest.raises(ValueError):
        pkg.quant4_encode(w)
    with pytest.raises(ValueError):
        pkg.quant4_matvec(w, x, w)
    with pytest.raises(ValueError):
        pkg.quant4_matvec(q, x, new((8, 1, 1)))
