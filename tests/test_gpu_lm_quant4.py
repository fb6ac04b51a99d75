"""quant4_matvec and quant4_encode against their formulas."""
import numpy as np
import pytest
import torch

import acediar._lib as L
import lm_oracle as O

pytestmark = pytest.mark.gpu

NP = {"float": np.float32, "float16": np.float16}


def make(rng, M, K, N, group, zeros, xdt="float16", sdt="float16", fractional=False):
    w = rng.integers(-128, 128, (16 * -(-K // 32), M)).astype(np.int8)
    G = -(-K // group)
    s = (rng.uniform(0.5, 1.5, (G, M)) * rng.choice([-1, 1], (G, M)) / 100).astype(NP[sdt])
    z = None
    if zeros:
        z = (rng.uniform(0, 15, (G, M)) if fractional else rng.integers(0, 16, (G, M))).astype(NP[sdt])
    x = rng.standard_normal((K, N) if N else (K,)).astype(NP[xdt])
    return w, s, z, x


def check(acd, M, K, N, group, zeros, xdt="float16", sdt="float16", odt=None, seed=0, fractional=False, x=None):
    w, s, z, x0 = make(np.random.default_rng(seed), M, K, N, group, zeros, xdt, sdt, fractional)
    x = x0 if x is None else x
    wrap = lambda a, d: None if a is None else acd.as_tensor(a, dtype=d)  # noqa: E731
    got = acd.quant4_matvec(wrap(w, "int8"), wrap(s, sdt), wrap(x, xdt), group, zeros=wrap(z, sdt), out_dtype=odt)
    odt = odt or xdt
    assert got.dtype == odt and got.shape == ((M, N) if N else (M,))
    y, bound = O.quant4_matvec(w, s, z, x, group, odt)
    O.assert_within(got.as_array().reshape(M, -1, order="F"), y, bound, "y")
    return got


@pytest.mark.parametrize("xdt", ["float", "float16"])
@pytest.mark.parametrize("M,K,group", [
    (1, 1, 32), (1, 32, 32), (5, 31, 32), (16, 33, 32), (17, 64, 64), (100, 100, 32), (128, 256, 128), (129, 255, 64),
    (300, 1000, 128), (64, 4096, 128), (1000, 513, 96), (257, 2049, 256), (512, 300, 512), (96, 8200, 32),
    (33, 16384, 64), (4096, 128, 32), (2000, 40000, 128)])
def test_products(acd, xdt, M, K, group):
    for N, zeros in ((0, False), (1, True), (3, True)):
        check(acd, M, K, N, group, zeros, xdt, seed=M + K)


@pytest.mark.parametrize("xdt", ["float", "float16"])
@pytest.mark.parametrize("N", [1, 2, 4, 5, 7, 8, 9, 16, 17, 33, 64, 100])
def test_columns(acd, xdt, N):
    check(acd, 200, 700, N, 64, True, xdt, seed=N)
    check(acd, 200, 700, N, 128, False, xdt, seed=N)


@pytest.mark.parametrize("xdt", ["float", "float16"])
@pytest.mark.parametrize("odt", ["float", "float16"])
@pytest.mark.parametrize("sdt", ["float", "float16"])
def test_types(acd, xdt, odt, sdt):
    check(acd, 333, 777, 3, 32, True, xdt, sdt, odt, fractional=True)
    check(acd, 333, 777, 1, 128, False, xdt, sdt, odt)


def test_large_values_in_32_bits(acd):
    """Activations far outside float16's range, and tiny ones, keep float32's accuracy."""
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((512, 3)) * np.array([1e9, 1.0, 1e-20])).astype(np.float32)
    check(acd, 130, 512, 3, 64, True, "float", "float", x=x)


def test_values_that_are_not_finite(acd):
    """An infinite or NaN activation reaches every output it has a weight for, and no other column."""
    for xdt in ("float", "float16"):
        for bad in (np.inf, -np.inf, np.nan):
            w = np.full((16 * 4, 40), 0x5B, np.int8)  # q = 11, 5: weights +3 and -3
            s = np.full((1, 40), 1.0, np.float16)
            x = np.ones((128, 3), NP[xdt])
            x[6, 1] = bad
            got = acd.quant4_matvec(acd.as_tensor(w, dtype="int8"), acd.as_tensor(s, dtype="float16"),
                                    acd.as_tensor(x, dtype=xdt), 128).as_array()
            assert np.array_equal(got[:, [0, 2]], np.zeros((40, 2)))
            want = 3 * bad
            assert np.isnan(got[:, 1]).all() if np.isnan(bad) else np.array_equal(got[:, 1], np.full(40, want)), (xdt, bad)


def test_padding_is_not_used(acd):
    """Bytes beyond the last input change nothing."""
    rng = np.random.default_rng(5)
    for K in (1, 31, 33, 250, 1000):
        w, s, z, x = make(rng, 70, K, 2, 32, True)
        other = w.copy()
        u = other.view(np.uint8)
        u[-(-K // 2):] = 255 - u[-(-K // 2):]
        if K % 2:
            u[K // 2] ^= 0xF0
        t = lambda a, d: acd.as_tensor(a, dtype=d)  # noqa: E731
        args = (t(s, "float16"), t(x, "float16"), 32, t(z, "float16"))
        a = acd.quant4_matvec(t(w, "int8"), *args).as_array()
        assert np.array_equal(a, acd.quant4_matvec(t(other, "int8"), *args).as_array())


@pytest.mark.parametrize("xdt", ["float", "float16"])
def test_views(acd, xdt):
    """x as a row of a matrix, with a column stride, off 16-byte boundaries; a written view."""
    rng = np.random.default_rng(6)
    w, s, z, _ = make(rng, 90, 300, 1, 64, True)
    t = lambda a, d: acd.as_tensor(a, dtype=d)  # noqa: E731
    flat = rng.standard_normal(5000).astype(NP[xdt])
    f = t(flat, xdt)
    for shape, strides, off in (((300,), (1,), 1), ((300,), (7,), 3), ((300, 3), (1, 401), 5), ((300, 4), (4, 1), 2),
                                ((300, 3), (1, 0), 8)):
        v = acd.gpuTensor(f.storage, shape, xdt, strides, off)
        x = v.as_array().reshape(300, -1, order="F")
        got = acd.quant4_matvec(t(w, "int8"), t(s, "float16"), v, 64, t(z, "float16")).as_array()
        y, b = O.quant4_matvec(w, s, z, x, 64, xdt)
        O.assert_within(got.reshape(90, -1, order="F"), y, b)
    import ctypes
    store = acd.as_tensor(np.zeros(1000), dtype="float")
    out = acd.gpuTensor(store.storage, (90, 2), "float", (3, 400), 5)
    x = t(rng.standard_normal((300, 2)), xdt)
    a = [t(w, "int8"), t(s, "float16"), t(z, "float16"), x]
    L.check(L.lib().acd_quant4_matvec(acd.context(), out.desc(), *[v.desc() for v in a], 64,
                                      ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    y, b = O.quant4_matvec(w, s, z, x.as_array(), 64, "float")
    O.assert_within(out.as_array(), y, b)
    after = store.as_array()
    inside = np.zeros(1000, bool)
    for j in range(2):
        inside[5 + 400 * j: 5 + 400 * j + 270: 3] = True
    assert not after[~inside].any(), "wrote outside the view"


def test_empty_products(acd):
    w, s, _, _ = make(np.random.default_rng(1), 8, 64, 1, 64, False)
    t = lambda a, d: acd.as_tensor(a, dtype=d)  # noqa: E731
    r = acd.quant4_matvec(t(w, "int8"), t(s, "float16"), acd.empty_tensor((64, 0), "float"), 64)
    assert r.shape == (8, 0)


def test_same_bits_twice_and_on_another_stream(acd):
    rng = np.random.default_rng(10)
    for M, K, N in ((4096, 4096, 1), (1000, 16000, 6)):
        w, s, z, x = make(rng, M, K, N, 64, True)
        a = [acd.as_tensor(v, dtype=d) for v, d in ((w, "int8"), (s, "float16"), (x, "float16"), (z, "float16"))]
        run = lambda: acd.quant4_matvec(a[0], a[1], a[2], 64, a[3]).as_array()  # noqa: E731
        first = run()
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            again = run()
        torch.cuda.synchronize()
        assert np.array_equal(first, again)


def test_offsets_beyond_32_bits(acd):
    """More than 2^31 bytes of weights; outputs at both ends against the oracle."""
    M, K = (1 << 18) + 3, 1 << 14
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randint(-128, 128, (M * (K // 2),), dtype=torch.int8, device="cuda", generator=g)
    s = torch.rand(M * (K // 128), device="cuda", generator=g).half()
    x = acd.as_tensor(np.random.default_rng(1).standard_normal(K), dtype="float")
    y = acd.quant4_matvec(acd.from_torch(w, (K // 2, M), "int8"), acd.from_torch(s, (K // 128, M), "float16"), x,
                          128).as_array()
    pick = [0, 1, M // 2, M - 1]
    wp = w.view(M, -1)[pick].t().cpu().numpy()
    sp = s.view(M, -1)[pick].t().cpu().numpy()
    ref, b = O.quant4_matvec(np.ascontiguousarray(wp.T).T, sp, None, x.as_array(), 128, "float")
    O.assert_within(y[pick][:, None], ref, b)


@pytest.mark.parametrize("sdt", ["float", "float16"])
@pytest.mark.parametrize("M,K,group", [(1, 1, 32), (40, 300, 32), (65, 256, 128), (3, 1000, 96)])
def test_encode(acd, sdt, M, K, group):
    """Decoded weights are within half a scale of the weights (a scale more
    where rounding the scale or the zero point moves a value past the ends)."""
    rng = np.random.default_rng(2)
    w = rng.standard_normal((M, K)).astype(np.float32)
    if M > 2:
        w[1, :group] = 0
        w[2] = np.abs(w[2])
    G = -(-K // group)
    for zeros in (False, True):
        q = acd.quant4_encode(acd.as_tensor(w, dtype="float"), group, zeros=zeros, scale_dtype=sdt)
        s = q.scales.as_array().astype(np.float64)
        z = q.zeros.as_array().astype(np.float64) if zeros else np.full((G, M), 8.0)
        g = np.arange(K) // group
        back = (O.quant4_unpack(q.weights.as_array(), K) - z.T[:, g]) * s.T[:, g]
        pad = np.zeros((M, G * group))
        pad[:, :K] = w
        pad = pad.reshape(M, G, group)
        lo, hi = np.minimum(pad.min(2), 0), np.maximum(pad.max(2), 0)
        want = ((hi - lo) / 15 if zeros else np.maximum(hi, -lo) / 7).T
        assert np.allclose(s, want, rtol=2.0 ** -10, atol=2.0 ** -24)
        assert np.all(np.abs(back - w) <= s.T[:, g] * ((1.0 if zeros else 0.5) + 0.02) + 1e-30)
        assert np.all((z >= 0) & (z <= 15) & (z == np.rint(z)))
    view = acd.transpose_view(acd.as_tensor(np.ascontiguousarray(w.T), dtype="float"))
    again = acd.quant4_encode(view, group, zeros=True, scale_dtype=sdt)
    assert np.array_equal(again.weights.as_array(), q.weights.as_array())


def test_encode_weights_that_are_not_finite(acd):
    w = np.ones((2, 64), np.float32)
    w[0, 3], w[1, 40] = np.nan, np.inf
    s = acd.quant4_encode(acd.as_tensor(w, dtype="float"), 32).scales.as_array()
    assert np.array_equal(np.isnan(s), [[True, False], [False, True]])


def test_refusals(acd):
    w, s, z, x = make(np.random.default_rng(1), 8, 64, 1, 32, True)
    t = lambda a, d: acd.as_tensor(a, dtype=d)  # noqa: E731
    W, S, Z, X = t(w, "int8"), t(s, "float16"), t(z, "float16"), t(x[:, 0], "float16")

    def status(*a, **k):
        with pytest.raises(L.AcdError) as e:
            acd.quant4_matvec(*a, **k)
        return e.value.status

    for group in (0, -32, 31, 48, 1.5):
        with pytest.raises(ValueError):
            acd.quant4_matvec(W, S, X, group)
    assert status(W, S, t(x[:, 0], "double"), 32, out_dtype="float") == 3
    assert status(W, S, X, 32, out_dtype="int32") == 3
    assert status(W, t(s, "double"), X, 32) == 3
    assert status(W, S, X, 32, zeros=t(z, "float")) == 3
    assert status(t(w, "int32"), S, X, 32) == 3
    assert status(W, S, X, 64) == 2                     # scales of another group
    assert status(W, S, t(np.ones(65), "float16"), 32) == 2
    assert status(W, S, X, 32, zeros=t(z[:1], "float16")) == 2
    off = acd.gpuTensor(W.storage, (32, 7), "int8", None, 4)  # weights off 16 bytes
    assert status(off, t(s[:, :7], "float16"), X, 32) == 8
    with pytest.raises(ValueError):
        acd.quant4_matvec(W, S, t(np.ones((64, 1, 1)), "float16"), 32)
    with pytest.raises(ValueError):
        acd.quant4_encode(X)
    with pytest.raises(ValueError):
        acd.quant4_encode(t(np.ones((4, 4)), "float"), 33)
    with pytest.raises(L.AcdError) as e:
        acd.quant4_encode(t(np.ones((4, 4)), "int32"), 32)
    assert e.value.status == 3
