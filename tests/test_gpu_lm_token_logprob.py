"""token_logprob and token_logprob_grad against their formulas in float64."""
import ctypes

import numpy as np
import pytest
import torch

import acediar._lib as L
import lm_oracle as O

pytestmark = pytest.mark.gpu

NP = {"float": np.float32, "float16": np.float16, "double": np.float64}
LOWEST = {"float": -3.4028234663852886e38, "float16": -3.4028234663852886e38, "double": -1.7976931348623157e308}
NA = np.iinfo(np.int64).min


def make_logits(rng, shape, axis, dtype, spread=3.0):
    off = rng.uniform(-20, 20, [1 if d == axis - 1 else s for d, s in enumerate(shape)])
    return (rng.standard_normal(shape) * spread + off).astype(NP[dtype])


def make_tokens(rng, rows, V):
    t = rng.integers(1, V + 1, rows)
    if rows >= 4:
        t[1] = 0
    return t


def rows_of(t, axis, ndim):
    """A row tensor (or one with `top` on the axis) as rows x entries."""
    a = t.as_array()
    return O.moved(a, axis) if a.ndim == ndim else a.reshape(-1, order="F")


def check_forward(acd, x, dtype, axis, tokens, scale, top, t=None):
    t = acd.as_tensor(x, dtype=dtype) if t is None else t
    xr = O.moved(x, axis)
    shape = tuple(s for d, s in enumerate(x.shape) if d != axis - 1) or (1,)
    tok = acd.as_tensor(tokens.reshape(shape, order="F"), dtype="int64")
    got = acd.token_logprob(t, tok, axis=axis, scale=scale, top=top)
    ref = O.logprob(xr, tokens, scale, top)
    b = O.logprob_bounds(ref, x.shape[axis - 1], dtype)
    flat = lambda v: v.as_array().reshape(-1, order="F")  # noqa: E731
    O.assert_within(flat(got.logprob), ref[0], b[0], "logprob")
    O.assert_within(flat(got.entropy), ref[1], b[1], "entropy")
    O.assert_within(flat(got.logsumexp), ref[2], b[2], "lse")
    if top:
        assert np.array_equal(O.moved(got.top_index.as_array(), axis), ref[3]), "alternatives"
        O.assert_within(O.moved(got.top_logprob.as_array(), axis), ref[4], b[3], "top_logprob")
    else:
        assert got.top_index is None and got.top_logprob is None
    return got


def check_grad(acd, x, dtype, axis, tokens, scale, entropy=True, lse_term=False, inplace=False, seed=0):
    rng = np.random.default_rng(seed)
    xr = O.moved(x, axis)
    rows, V = xr.shape
    st = np.float64 if dtype == "double" else np.float32
    ref = O.logprob(xr, tokens, scale, 0)
    lse, H = ref[2].astype(st), ref[1].astype(st)
    g = -rng.uniform(0.5, 1.5, rows).astype(st)
    gH = rng.uniform(-1, 1, rows).astype(st) if entropy else None
    gl = rng.uniform(-1, 1, rows).astype(st) if lse_term else None
    shape = tuple(s for d, s in enumerate(x.shape) if d != axis - 1) or (1,)
    sd = "double" if dtype == "double" else "float"
    wrap = lambda v: None if v is None else acd.as_tensor(v.reshape(shape, order="F"), dtype=sd)  # noqa: E731
    t = acd.as_tensor(x, dtype=dtype)
    got = acd.token_logprob_grad(t, acd.as_tensor(tokens.reshape(shape, order="F"), dtype="int64"), wrap(lse), wrap(H),
                                 wrap(g), wrap(gH), wrap(gl), axis=axis, scale=scale, inplace=inplace)
    assert (got is t) == inplace
    f = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
    exp = O.logprob_grad(xr, tokens, f(lse), f(H), f(g), f(gH), f(gl), scale, LOWEST[dtype])
    bound = O.logprob_grad_bound(exp, xr, f(lse), f(H), f(g), f(gH), f(gl), scale, dtype)
    bound = np.where(f(lse)[:, None] <= LOWEST[dtype] / 4, 0.0, bound)
    O.assert_within(O.moved(got.as_array(), axis), exp, bound, "grad")


# one row to many, one token to long rows, sizes off every tile and vector
SHAPES = [((1,), 1), ((7,), 1), ((1000,), 1), ((131, 1), 1), ((1, 5), 1), ((2, 3), 2), ((33, 70), 1), ((70, 33), 2),
          ((1024, 40), 1), ((40, 1024), 2), ((4099, 9), 1), ((9, 4099), 2), ((50001, 3), 1), ((65, 3000), 2),
          ((3, 257, 5), 2), ((40, 129, 3), 2), ((129, 5, 3), 1), ((5, 3, 129), 3), ((131072, 2), 1), ((256, 517), 2),
          ((16384, 5), 1), ((33000, 300), 1), ((300, 2050), 2)]


@pytest.mark.parametrize("dtype", ["float", "float16", "double"])
@pytest.mark.parametrize("shape,axis", SHAPES)
def test_forward(acd, dtype, shape, axis):
    rng = np.random.default_rng(abs(hash((shape, axis))) % 1000)
    x = make_logits(rng, shape, axis, dtype)
    V = shape[axis - 1]
    rows = x.size // V
    tokens = make_tokens(rng, rows, V)
    for top, scale in ((0, 1.0), (min(5, V), 0.8), (min(32, V), 1.0)):
        check_forward(acd, x, dtype, axis, tokens, scale, top)


@pytest.mark.parametrize("dtype", ["float", "float16", "double"])
@pytest.mark.parametrize("shape,axis", SHAPES)
def test_grad(acd, dtype, shape, axis):
    rng = np.random.default_rng(abs(hash((shape, axis))) % 1000 + 1)
    x = make_logits(rng, shape, axis, dtype)
    V = shape[axis - 1]
    tokens = make_tokens(rng, x.size // V, V)
    check_grad(acd, x, dtype, axis, tokens, 1.0, entropy=False)
    check_grad(acd, x, dtype, axis, tokens, 0.7, lse_term=True, inplace=True)


@pytest.mark.parametrize("dtype", ["float", "float16", "double"])
@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("V", [3, 600, 5000])
def test_masks_ties_and_odd_values(acd, dtype, axis, V):
    """Rows: empty, one token left, all the type's lowest value, NaN inside,
    +Inf inside, constant (every alternative a tie), two-valued, masked half,
    masked to fewer tokens than alternatives, -0 and +0 mixed."""
    rng = np.random.default_rng(3)
    x = make_logits(rng, (48, V), 2, dtype)
    low = np.finfo(NP[dtype]).min
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, V - 1] = 2.0
    x[2] = low
    x[3, V // 2] = np.nan
    x[4, V // 3] = np.inf
    x[5] = 1.5
    x[6] = np.where(rng.random(V) < 0.5, 1.0, 2.0)
    x[7, rng.random(V) < 0.5] = -np.inf
    x[8] = -np.inf
    x[8, [0, V - 1]] = [3.0, 3.0]
    x[9] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    x[10] = np.nan
    x[11, : V // 2] = low
    tokens = make_tokens(rng, 48, V)
    tokens[:12] = np.minimum(V, [1, 1, 2, 1, 1, 2, 3, 1, 1, V, 1, 1])
    tokens[12:17] = [NA, -3, V + 1, 0, V]
    if axis == 1:
        x = np.asfortranarray(x.T)
    check_forward(acd, x, dtype, axis, tokens, 1.0, min(20, V))
    finite = np.isfinite(np.where(np.isneginf(O.moved(x, axis)), 0, O.moved(x, axis))).all(1)
    keep = np.flatnonzero(finite)  # a NaN row's gradient is NaN: checked below
    xs = O.moved(x, axis)[keep]
    xs = np.asfortranarray(xs.T) if axis == 1 else xs
    check_grad(acd, xs, dtype, axis, tokens[keep], 1.0)


@pytest.mark.parametrize("dtype", ["float", "float16"])
@pytest.mark.parametrize("axis", [1, 2])
@pytest.mark.parametrize("V", [700, 5000, 40000])
def test_ties_of_coarse_logits(acd, dtype, axis, V):
    """Logits of few values: the alternatives hold a few above many equal ones,
    of which the first count, wherever they stand."""
    rng = np.random.default_rng(11)
    x = np.rint(rng.standard_normal((40, V)) * 1.3).astype(NP[dtype])
    x[0] = 0
    x[1] = -np.inf
    x[1, ::7] = 1
    x[2, V // 2:] = 9
    x[3, -3:] = 50
    x[4] = np.arange(V) % 5
    x[5] = np.minimum(np.arange(V), 2000) if dtype == "float" else np.minimum(np.arange(V) // 4, 500)
    x[6] = x[5, ::-1]
    if axis == 1:
        x = np.asfortranarray(x.T)
    tokens = make_tokens(rng, 40, V)
    for top in (1, 7, 20, 32):
        check_forward(acd, x, dtype, axis, tokens, 1.0, top)


@pytest.mark.parametrize("dtype", ["float", "float16"])
@pytest.mark.parametrize("top", [1, 3, 5, 8, 9])
def test_many_rows_across_the_lanes(acd, dtype, top):
    """Rows enough for a thread each: smooth, coarse (ties at the last
    alternative), masked to fewer tokens than alternatives, empty, with NaN."""
    rng = np.random.default_rng(top)
    rows, V = 19001, 270
    x = (rng.standard_normal((rows, V)) * 3).astype(NP[dtype])
    x[:6000] = np.rint(x[:6000])
    x[100:200] = -np.inf
    x[150:200, 17] = 1
    x[160:200, 3] = 1
    x[200:220, ::5] = np.nan
    x[220:240] = 2
    check_forward(acd, x, dtype, 2, make_tokens(rng, rows, V), 1.0, top)


def test_nan_row_has_nan_gradient_and_leaves_its_neighbours(acd):
    x = np.random.default_rng(0).standard_normal((100, 3)).astype(np.float32)
    x[7, 1] = np.nan
    t = acd.as_tensor(x, dtype="float")
    tok = acd.as_tensor([1, 2, 3], dtype="int64")
    r = acd.token_logprob(t, tok)
    g = acd.token_logprob_grad(t, tok, r.logsumexp, d_logprob=acd.as_tensor([1., 1., 1.], dtype="float")).as_array()
    assert np.isnan(g[:, 1]).all() and np.isfinite(g[:, [0, 2]]).all()


@pytest.mark.parametrize("dtype", ["float", "float16"])
def test_views(acd, dtype):
    """Permuted, sliced, offset and strided views; rows off 16-byte boundaries."""
    rng = np.random.default_rng(5)
    big = make_logits(rng, (37, 130, 6), 2, dtype)
    t = acd.as_tensor(big, dtype=dtype)
    tok = make_tokens(rng, 37 * 6, 130)
    check_forward(acd, big, dtype, 2, tok, 1.0, 4, t)
    p = acd.permute_view(t, [3, 1, 2])
    check_forward(acd, np.transpose(big, (2, 0, 1)), dtype, 3, make_tokens(rng, 37 * 6, 130), 1.0, 4, p)
    p = acd.permute_view(t, [2, 3, 1])  # not collapsible: copied
    check_forward(acd, np.transpose(big, (1, 2, 0)), dtype, 1, make_tokens(rng, 37 * 6, 130), 1.0, 4, p)
    flat = make_logits(rng, (20011,), 1, dtype)
    f = acd.as_tensor(flat, dtype=dtype)
    # 9 rows of 1001 elements, row stride 2003, from offset 3
    v = acd.gpuTensor(f.storage, (1001, 9), dtype, (1, 2003), 3)
    host = np.stack([flat[3 + 2003 * k: 3 + 2003 * k + 1001] for k in range(9)], 1)
    check_forward(acd, host, dtype, 1, make_tokens(rng, 9, 1001), 1.0, 7, v)
    # every second element
    v = acd.gpuTensor(f.storage, (5000, 2), dtype, (2, 10001), 1)
    host = np.stack([flat[1 + 10001 * k: 1 + 10001 * k + 10000: 2] for k in range(2)], 1)
    check_forward(acd, host, dtype, 1, make_tokens(rng, 2, 5000), 1.0, 7, v)
    # lanes of odd stride (rows of a matrix with 41 of 43 lanes used)
    v = acd.gpuTensor(f.storage, (41, 400), dtype, (1, 43), 2)
    host = np.stack([flat[2 + 43 * k: 2 + 43 * k + 41] for k in range(400)], 1)
    check_forward(acd, host, dtype, 2, make_tokens(rng, 41, 400), 1.0, 3, v)
    # one row for all: a broadcast view
    v = acd.gpuTensor(f.storage, (1000, 4), dtype, (1, 0), 0)
    check_forward(acd, np.repeat(flat[:1000, None], 4, 1), dtype, 1, make_tokens(rng, 4, 1000), 1.0, 3, v)


def test_grad_into_a_view_in_place(acd):
    rng = np.random.default_rng(6)
    flat = rng.standard_normal(20011).astype(np.float32)
    f = acd.as_tensor(flat, dtype="float")
    v = acd.gpuTensor(f.storage, (1001, 9), "float", (1, 2003), 3)
    tok = acd.as_tensor(rng.integers(1, 1002, 9), dtype="int32")
    r = acd.token_logprob(v, tok)
    g = acd.as_tensor(np.ones(9), dtype="float")
    want = acd.token_logprob_grad(v, tok, r.logsumexp, d_logprob=g).as_array()
    acd.token_logprob_grad(v, tok, r.logsumexp, d_logprob=g, inplace=True)
    after = f.as_array()
    inside = np.zeros(20011, bool)
    for k in range(9):
        s = slice(3 + 2003 * k, 3 + 2003 * k + 1001)
        inside[s] = True
        assert np.array_equal(after[s], want[:, k])
    assert np.array_equal(after[~inside], flat[~inside]), "wrote outside the view"


def test_grad_against_differences(acd):
    """Central differences of the forward call in float64: truncation h^2 and
    rounding 1e-15 / h, both below 1e-8 at h = 1e-5."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((50, 4))
    tok = acd.as_tensor([3, 50, 1, 0], dtype="int64")
    g, gH, gl = rng.standard_normal(4), rng.standard_normal(4), rng.standard_normal(4)
    wrap = lambda v: acd.as_tensor(v, dtype="double")  # noqa: E731

    def loss(a):
        r = acd.token_logprob(wrap(a), tok, scale=1.3)
        return (r.logprob.as_array() * g + r.entropy.as_array() * gH + r.logsumexp.as_array() * gl).sum()

    r = acd.token_logprob(wrap(x), tok, scale=1.3)
    got = acd.token_logprob_grad(wrap(x), tok, r.logsumexp, r.entropy, wrap(g), wrap(gH), wrap(gl),
                                 scale=1.3).as_array()
    h = 1e-5
    for v in (0, 2, 17, 49):
        for row in range(4):
            e = np.zeros_like(x)
            e[v, row] = h
            assert abs((loss(x + e) - loss(x - e)) / (2 * h) - got[v, row]) < 1e-8


def test_parts_alone_and_zero_based(acd):
    """The C call with outputs left out, counted from 0, int32 indices."""
    rng = np.random.default_rng(9)
    x = make_logits(rng, (700, 6), 1, "float")
    t = acd.as_tensor(x, dtype="float")
    full = acd.token_logprob(t, acd.as_tensor([1, 5, 0, 700, 2, 9], dtype="int64"), top=3)
    lib, c = L.lib(), acd.context()
    s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    ent = acd.empty_tensor((6,), "float")
    L.check(lib.acd_token_logprob(c, None, ent.desc(), None, None, None, t.desc(), None, 0, 1.0, 0, s))
    assert np.array_equal(ent.as_array(), full.entropy.as_array())
    lp = acd.empty_tensor((1, 6), "float")
    ix, tl = acd.empty_tensor((3, 6), "int32"), acd.empty_tensor((3, 6), "float")
    tok = acd.as_tensor(np.array([[0, 4, -1, 699, 1, 8]]), dtype="int32")
    L.check(lib.acd_token_logprob(c, lp.desc(), None, None, ix.desc(), tl.desc(), t.desc(), tok.desc(), 0, 1.0, 0, s))
    assert np.array_equal(lp.as_array()[0], full.logprob.as_array())
    assert np.array_equal(ix.as_array(), full.top_index.as_array() - 1)
    assert np.array_equal(tl.as_array(), full.top_logprob.as_array())


def test_no_rows(acd):
    r = acd.token_logprob(acd.empty_tensor((50, 0), "float"), acd.empty_tensor((0,), "int64"), top=2)
    assert r.logprob.shape == (0,) and r.top_index.shape == (2, 0)


@pytest.mark.parametrize("shape,axis", [((131072, 3), 1), ((300, 5000), 2), ((4096, 200), 1)])
def test_same_bits_twice_and_on_another_stream(acd, shape, axis):
    rng = np.random.default_rng(10)
    t = acd.as_tensor(make_logits(rng, shape, axis, "float16"), dtype="float16")
    rows = t.size // shape[axis - 1]
    tok = acd.as_tensor(make_tokens(rng, rows, shape[axis - 1]), dtype="int64")
    first = [v.as_array() for v in acd.token_logprob(t, tok, axis=axis, top=20)]
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        again = [v.as_array() for v in acd.token_logprob(t, tok, axis=axis, top=20)]
    torch.cuda.synchronize()
    for a, b in zip(first, again):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("layout", ["rows", "lanes"])
def test_offsets_beyond_32_bits(acd, layout):
    """More than 2^31 logits: a few rows at both ends against the oracle."""
    V, rows = 1 << 15, (1 << 16) + 40
    g = torch.Generator(device="cuda").manual_seed(1)
    st = torch.empty(V * rows, dtype=torch.float16, device="cuda")
    for part in st.split(1 << 28):
        part.normal_(0, 3, generator=g)
    tokens = torch.randint(1, V + 1, (rows,), device="cuda", generator=g)
    rows_first = layout == "rows"
    t = acd.from_torch(st, (V, rows) if rows_first else (rows, V), "float16")
    tk = acd.from_torch(tokens, (rows,), "int64")
    axis = 1 if rows_first else 2
    r = acd.token_logprob(t, tk, axis=axis, top=2)
    pick = [0, 1, rows // 2, rows - 2, rows - 1]
    x = (st.view(rows, V)[pick] if rows_first else st.view(V, rows)[:, pick].t()).cpu().numpy()
    ref = O.logprob(x, tokens[pick].cpu().numpy(), 1.0, 2)
    b = O.logprob_bounds(ref, V, "float16")
    O.assert_within(r.logprob.as_array()[pick], ref[0], b[0])
    O.assert_within(r.logsumexp.as_array()[pick], ref[2], b[2])
    ix = r.top_index.as_array()
    assert np.array_equal(ix[:, pick].T if rows_first else ix[pick], ref[3])
    ones = acd.from_torch(torch.ones(rows, device="cuda"), (rows,), "float")
    d = acd.token_logprob_grad(t, tk, r.logsumexp, d_logprob=ones, axis=axis, inplace=True)
    got = (d.storage.view(rows, V)[pick] if rows_first else d.storage.view(V, rows)[:, pick].t()).cpu().numpy()
    lse = r.logsumexp.as_array()[pick].astype(np.float64)
    one = np.ones(len(pick))
    exp = O.logprob_grad(x, ref_tokens(tokens, pick), lse, None, one, None, None, 1.0, LOWEST["float16"])
    O.assert_within(got, exp, O.logprob_grad_bound(exp, x, lse, None, one, None, None, 1.0, "float16"))


def ref_tokens(tokens, pick):
    return tokens[pick].cpu().numpy()


def test_refusals(acd):
    t = acd.as_tensor(np.zeros((8, 4)), dtype="float")
    tok = acd.as_tensor([1, 1, 1, 1], dtype="int64")
    st = acd.as_tensor(np.zeros(4), dtype="float")

    def status(f, *a, **k):
        with pytest.raises(L.AcdError) as e:
            f(*a, **k)
        return e.value.status

    F, G = acd.token_logprob, acd.token_logprob_grad
    for axis in (0, 3, 1.5, None):
        with pytest.raises(ValueError):
            F(t, tok, axis=axis)
    with pytest.raises(ValueError):
        F(t, tok, top=-1)
    assert status(F, acd.as_tensor(np.zeros((8, 4)), dtype="int32"), tok) == 3
    assert status(F, t, st) == 3  # tokens of a floating type
    assert status(F, t, acd.as_tensor([1, 1, 1], dtype="int64")) == 2
    assert status(F, t, tok, axis=2) == 2
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert status(F, t, tok, scale=scale) == 1
    assert status(F, t, tok, top=9) == 2      # more than tokens
    assert status(F, acd.as_tensor(np.zeros((64, 4)), dtype="float"), tok, top=33) == 8
    assert status(F, acd.empty_tensor((0, 4), "float"), tok) == 2
    assert status(G, t, tok, st) == 1         # no gradient given
    assert status(G, t, None, st, d_logprob=st) == 1
    assert status(G, t, tok, st, None, None, st) == 1   # entropy missing
    assert status(G, t, tok, acd.as_tensor(np.zeros(4), dtype="double"), d_logprob=st) == 3
    assert status(G, t, tok, acd.as_tensor(np.zeros(5), dtype="float"), d_logprob=st) == 2
    lib, s = L.lib(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    half = acd.empty_tensor((4,), "float")
    assert lib.acd_token_logprob(None, None, half.desc(), None, None, None, t.desc(), None, 0, 1.0, 1, s) == 1
    assert lib.acd_token_logprob(acd.context(), half.desc(), None, None, None, None, t.desc(), None, 0, 1.0, 1, s) == 1
    wide = acd.gpuTensor(half.storage, (2,), "float", (2,))
    two = acd.as_tensor(np.zeros((8, 2)), dtype="float")
    assert lib.acd_token_logprob(acd.context(), None, wide.desc(), None, None, None, two.desc(), None, 0, 1.0, 1, s) == 8
    cube = acd.permute_view(acd.as_tensor(np.zeros((8, 4, 3)), dtype="float"), [1, 3, 2])
    e = acd.empty_tensor((3, 4), "float")
    assert lib.acd_token_logprob(acd.context(), None, e.desc(), None, None, None, cube.desc(), None, 0, 1.0, 1, s) == 8
    assert F(cube, None).entropy.shape == (3, 4)  # the package makes it contiguous
