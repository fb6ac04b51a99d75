"""residual_norm and residual_norm_grad against their formulas in float64."""
import ctypes

import numpy as np
import pytest
import torch

import acediar._lib as L
import lm_oracle as O

pytestmark = pytest.mark.gpu

NP = {"float": np.float32, "float16": np.float16, "double": np.float64}


def make(rng, shape, axis, dtype, post, gshape):
    D = shape[axis - 1]
    n = NP[dtype]
    v = dict(r=rng.standard_normal(shape).astype(n), b=(rng.standard_normal(shape) * rng.uniform(0.1, 3)).astype(n),
             w_pre=rng.uniform(0.5, 1.5, D).astype(n), w_post=rng.uniform(-1.5, 1.5, D).astype(n) if post else None,
             gate=rng.standard_normal(gshape).astype(n) if gshape else None)
    return v


def gate_rows(gate, axis, D):
    return None if gate is None else (gate.reshape(1, -1) if gate.ndim == 1 else O.moved(gate, axis))


def check(acd, shape, axis, dtype, post=True, gshape=None, alpha=1.0, eps=1e-6, seed=0, inplace=False, with_dh=True,
          wrap=None, back=True):
    rng = np.random.default_rng(seed)
    v = make(rng, shape, axis, dtype, post, gshape)
    D = shape[axis - 1]
    dense = lambda a, d=dtype: None if a is None else acd.as_tensor(a, dtype=d)  # noqa: E731
    wrap = wrap or dense
    rows = O.moved(v["r"], axis).shape[0]
    gr = gate_rows(v["gate"], axis, D)
    per = rows // len(gr) if gr is not None else rows
    got = acd.residual_norm(wrap(v["r"]), wrap(v["b"]), dense(v["w_pre"]), dense(v["w_post"]), dense(v["gate"]),
                            axis=axis, alpha=alpha, eps=eps, inplace=inplace)
    ref = O.norm(O.moved(v["r"], axis), O.moved(v["b"], axis), v["w_pre"], v["w_post"], gr, alpha, eps, per)
    bound = O.norm_bounds(ref, v["w_pre"], D, dtype)
    flat = lambda t: t.as_array().reshape(-1, order="F")  # noqa: E731
    O.assert_within(O.moved(got.h.as_array(), axis), ref[0], bound[0], "h")
    O.assert_within(O.moved(got.y.as_array(), axis), ref[1], bound[1], "y")
    O.assert_within(flat(got.rstd_h), ref[2], bound[2], "rstd_h")
    if post:
        O.assert_within(flat(got.rstd_block), ref[3], bound[3], "rstd_block")
    else:
        assert got.rstd_block is None
    if not back:
        return got
    st = np.float64 if dtype == "double" else np.float32
    sd = "double" if dtype == "double" else "float"
    h = ref[0].astype(NP[dtype])
    rh, rb = ref[2].astype(st), ref[3].astype(st) if post else None
    dh = rng.standard_normal(shape).astype(NP[dtype]) if with_dh else None
    dy = rng.standard_normal(shape).astype(NP[dtype])
    rshape = tuple(s for d, s in enumerate(shape) if d != axis - 1) or (1,)
    unmoved = np.moveaxis(h.T.reshape((D,) + tuple(s for d, s in enumerate(shape) if d != axis - 1), order="F"), 0,
                          axis - 1)
    stat = lambda a: None if a is None else acd.as_tensor(a.reshape(rshape, order="F"), dtype=sd)  # noqa: E731
    g = acd.residual_norm_grad(None if dh is None else wrap(dh), wrap(dy), wrap(unmoved), wrap(v["b"]), stat(rh),
                               stat(rb), dense(v["w_pre"]), dense(v["w_post"]), dense(v["gate"]), axis=axis,
                               alpha=alpha)
    mv = lambda a: None if a is None else O.moved(a, axis)  # noqa: E731
    args = (mv(dh), mv(dy), h, mv(v["b"]), rh, rb, v["w_pre"], v["w_post"], gr, alpha, per)
    ref, bound = O.norm_grad(*args), O.norm_grad_bounds(args, dtype)
    O.assert_within(mv(g.d_residual.as_array()), ref[0], bound[0], "d_residual")
    O.assert_within(mv(g.d_block.as_array()), ref[1], bound[1], "d_block")
    O.assert_within(flat(g.d_w_pre), ref[2], bound[2], "d_w_pre")
    assert (g.d_w_post is None) == (not post) and (g.d_gate is None) == (gshape is None)
    if post:
        O.assert_within(flat(g.d_w_post), ref[3], bound[3], "d_w_post")
    if gshape:
        assert g.d_gate.shape == tuple(gshape)
        O.assert_within(gate_rows(g.d_gate.as_array(), axis, D), ref[4], bound[4], "d_gate")
    return got


# width, rows: one element to wide rows, sizes off every tile and vector, one row to many
SIZES = [(1, 1), (1, 40), (2, 3), (7, 5), (8, 1), (33, 9), (64, 100), (255, 17), (256, 300), (1000, 64), (1001, 33),
         (1024, 7), (2048, 150), (2050, 20), (4096, 8), (4096, 700), (4100, 5), (5120, 40), (8192, 30), (8200, 3),
         (16384, 10), (16390, 2), (40000, 3)]


@pytest.mark.parametrize("dtype", ["float", "float16", "double"])
@pytest.mark.parametrize("D,rows", SIZES)
def test_rows_along_the_first_axis(acd, dtype, D, rows):
    check(acd, (D, rows), 1, dtype, post=True, gshape=(D,), alpha=1.0, seed=D + rows)
    check(acd, (D, rows), 1, dtype, post=False, alpha=0.5, seed=D + rows + 1, with_dh=False)


@pytest.mark.parametrize("dtype", ["float", "float16", "double"])
@pytest.mark.parametrize("shape,axis", [((40, 1), 2), ((1, 40), 2), ((3, 50), 2), ((33, 257), 2), ((300, 96), 2),
                                        ((64, 4096), 2), ((5, 129, 3), 2), ((40, 33, 2), 2), ((130, 4, 5), 1),
                                        ((4, 5, 130), 3)])
def test_other_axes(acd, dtype, shape, axis):
    check(acd, shape, axis, dtype, post=True, gshape=(shape[axis - 1],), alpha=1.5, seed=7)
    check(acd, shape, axis, dtype, post=False, seed=8)


@pytest.mark.parametrize("dtype", ["float", "float16"])
@pytest.mark.parametrize("shape,axis,gshape", [
    ((128, 6, 5), 1, (128, 1, 5)), ((128, 6, 5), 1, (128, 6, 5)), ((128, 6, 5), 1, (128, 1, 1)), ((77, 9), 1, (77, 9)),
    ((256, 300, 4), 1, (256, 1, 4)), ((256, 1, 700), 1, (256, 1, 700)), ((1001, 40, 3), 1, (1001, 1, 3)),
    ((9, 77), 2, (1, 77)), ((9, 77), 2, (9, 77)), ((6, 5, 40), 3, (1, 5, 40)), ((4096, 3, 2), 1, (4096, 1, 2))])
def test_gates(acd, dtype, shape, axis, gshape):
    check(acd, shape, axis, dtype, post=True, gshape=gshape, seed=11)
    check(acd, shape, axis, dtype, post=False, gshape=gshape, alpha=0.25, seed=12)


@pytest.mark.parametrize("dtype", ["float", "float16"])
@pytest.mark.parametrize("shape,axis", [((1000, 60), 1), ((1001, 60), 1), ((60, 100), 2), ((50000, 2), 1)])
def test_in_place(acd, dtype, shape, axis):
    rng = np.random.default_rng(2)
    v = make(rng, shape, axis, dtype, True, (shape[axis - 1],))
    t = {k: acd.as_tensor(a, dtype=dtype) for k, a in v.items()}
    want = acd.residual_norm(t["r"], t["b"], t["w_pre"], t["w_post"], t["gate"], axis=axis)
    got = acd.residual_norm(t["r"], t["b"], t["w_pre"], t["w_post"], t["gate"], axis=axis, inplace=True)
    assert got.h is t["r"] and got.y is t["b"]
    for a, b in zip(got, want):
        assert np.array_equal(a.as_array(), b.as_array())


@pytest.mark.parametrize("dtype", ["float", "float16"])
def test_gradients_over_their_sources(acd, dtype):
    """d_residual over d_h and d_block over d_y (the C call allows it)."""
    rng = np.random.default_rng(3)
    for D, rows in ((512, 90), (1001, 40), (20000, 3)):
        v = make(rng, (D, rows), 1, dtype, True, (D,))
        t = {k: acd.as_tensor(a, dtype=dtype) for k, a in v.items()}
        f = acd.residual_norm(t["r"], t["b"], t["w_pre"], t["w_post"], t["gate"])
        dh, dy = (acd.as_tensor(rng.standard_normal((D, rows)), dtype=dtype) for _ in range(2))
        want = acd.residual_norm_grad(dh, dy, f.h, t["b"], f.rstd_h, f.rstd_block, t["w_pre"], t["w_post"], t["gate"])
        sums = [acd.empty_tensor((D,), "float") for _ in range(3)]
        L.check(L.lib().acd_residual_norm_grad(
            acd.context(), dh.desc(), dy.desc(), *[x.desc() for x in sums], dh.desc(), dy.desc(), f.h.desc(),
            t["b"].desc(), f.rstd_h.desc(), f.rstd_block.desc(), t["w_pre"].desc(), t["w_post"].desc(),
            t["gate"].desc(), 0, 1.0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
        for a, b in zip([dh, dy] + sums, want):
            assert np.array_equal(a.as_array(), b.as_array())


@pytest.mark.parametrize("dtype", ["float", "float16"])
def test_views(acd, dtype):
    """Row strides above the width, an offset off 16 bytes, every second element, a permuted tensor."""
    def padded(pitch, offset, step=1):
        def wrap(a):
            D, rows = a.shape
            st = torch.zeros(offset + pitch * rows + 8, dtype=acd.as_tensor([0.0], dtype=dtype).storage.dtype,
                             device="cuda")
            host = np.zeros(st.numel(), NP[dtype])
            for k in range(rows):
                host[offset + pitch * k: offset + pitch * k + step * D: step] = a[:, k]
            st.copy_(torch.from_numpy(host))
            return acd.gpuTensor(st, (D, rows), dtype, (step, pitch), offset)
        return wrap
    for D, pitch, offset, step in ((1000, 1008, 8, 1), (1000, 1003, 3, 1), (1001, 1001, 1, 1), (500, 1200, 0, 2)):
        check(acd, (D, 20), 1, dtype, gshape=(D,), seed=4, wrap=padded(pitch, offset, step))

    def permuted(a):
        return acd.permute_view(acd.as_tensor(np.transpose(a, (2, 0, 1)), dtype=dtype), [2, 3, 1])
    check(acd, (96, 7, 5), 1, dtype, seed=5, wrap=permuted)


@pytest.mark.parametrize("dtype", ["float", "float16"])
@pytest.mark.parametrize("D,pitch,offset", [(2, 2, 0), (6, 6, 0), (98, 98, 2), (98, 99, 0), (130, 132, 1), (634, 640, 4),
                                            (1634, 1636, 2), (1634, 1634, 1), (4098, 4100, 0), (6146, 6146, 0)])
def test_even_widths(acd, dtype, D, pitch, offset):
    """Rows of even width on every second element's boundary, and off it."""
    def wrap(a):
        rows = a.shape[1]
        host = np.zeros(offset + pitch * rows, NP[dtype])
        for k in range(rows):
            host[offset + pitch * k: offset + pitch * k + D] = a[:, k]
        st = torch.from_numpy(host).to("cuda")
        return acd.gpuTensor(st, (D, rows), dtype, (1, pitch), offset)
    check(acd, (D, 21), 1, dtype, gshape=(D,), seed=D, wrap=wrap)
    check(acd, (D, 21), 1, dtype, post=False, gshape=(D, 21), alpha=0.5, seed=D + 1, wrap=wrap, with_dh=False)


def test_zero_rows_and_zero_blocks(acd):
    """A row of zeros: rstd = 1 / sqrt(eps), y = 0; no rows: nothing, sums of 0."""
    z = acd.as_tensor(np.zeros((64, 3)), dtype="float")
    w = acd.as_tensor(np.ones(64), dtype="float")
    r = acd.residual_norm(z, z, w, w)
    assert np.array_equal(r.y.as_array(), np.zeros((64, 3)))
    O.assert_within(r.rstd_h.as_array(), np.full(3, 1e3), 1e3 * 2.0 ** -20)
    e = acd.empty_tensor((64, 0), "float")
    r = acd.residual_norm(e, e, w, w)
    assert r.h.shape == (64, 0)
    g = acd.residual_norm_grad(e, e, e, e, acd.empty_tensor((0,), "float"), acd.empty_tensor((0,), "float"), w, w, w)
    assert not g.d_w_pre.as_array().any() and not g.d_w_post.as_array().any() and not g.d_gate.as_array().any()


def test_nan_stays_in_its_row(acd):
    rng = np.random.default_rng(6)
    b = rng.standard_normal((300, 4)).astype(np.float32)
    b[17, 2] = np.nan
    t = acd.as_tensor(b, dtype="float")
    w = acd.as_tensor(np.ones(300), dtype="float")
    y = acd.residual_norm(acd.as_tensor(np.ones((300, 4)), dtype="float"), t, w, w).y.as_array()
    assert np.isnan(y[:, 2]).all() and np.isfinite(np.delete(y, 2, 1)).all()


def test_grad_against_differences(acd):
    """Central differences of the forward call in float64 (h = 1e-5: below 1e-8)."""
    rng = np.random.default_rng(9)
    D, S, B = 24, 3, 2
    v = dict(r=rng.standard_normal((D, S, B)), b=rng.standard_normal((D, S, B)), w_pre=rng.standard_normal(D),
             w_post=rng.standard_normal(D), gate=rng.standard_normal((D, 1, B)))
    ch, cy = rng.standard_normal((D, S, B)), rng.standard_normal((D, S, B))

    def forward(v):
        return acd.residual_norm(*[acd.as_tensor(v[k], dtype="double") for k in ("r", "b", "w_pre", "w_post", "gate")],
                                 alpha=0.7, eps=1e-3)

    def loss(v):
        f = forward(v)
        return (f.h.as_array() * ch).sum() + (f.y.as_array() * cy).sum()

    f = forward(v)
    t = {k: acd.as_tensor(a, dtype="double") for k, a in v.items()}
    g = acd.residual_norm_grad(acd.as_tensor(ch, dtype="double"), acd.as_tensor(cy, dtype="double"), f.h, t["b"],
                               f.rstd_h, f.rstd_block, t["w_pre"], t["w_post"], t["gate"], alpha=0.7)
    h = 1e-5
    for name, grad in zip(("r", "b", "w_pre", "w_post", "gate"), g):
        grad = grad.as_array()
        for _ in range(8):
            at = tuple(rng.integers(0, s) for s in v[name].shape)
            up, down = dict(v), dict(v)
            up[name], down[name] = v[name].copy(), v[name].copy()
            up[name][at] += h
            down[name][at] -= h
            assert abs((loss(up) - loss(down)) / (2 * h) - grad[at]) < 1e-7 * max(1, abs(grad[at])), name


@pytest.mark.parametrize("D,rows,gates", [(4096, 1000, 4), (1001, 3000, 1), (512, 640, 640)])
def test_same_bits_twice_and_on_another_stream(acd, D, rows, gates):
    rng = np.random.default_rng(10)
    shape = (D, rows // gates, gates)
    t = {k: acd.as_tensor(rng.standard_normal(shape), dtype="float16") for k in ("dh", "dy", "h", "b")}
    w = acd.as_tensor(rng.standard_normal(D), dtype="float16")
    gate = acd.as_tensor(rng.standard_normal((D, 1, gates)), dtype="float16")
    rs = acd.as_tensor(rng.uniform(0.5, 2, shape[1:]), dtype="float")
    run = lambda: [a.as_array() for a in acd.residual_norm_grad(t["dh"], t["dy"], t["h"], t["b"], rs, rs, w, w, gate)]  # noqa: E731
    first = run()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        again = run()
    torch.cuda.synchronize()
    for a, b in zip(first, again):
        assert np.array_equal(a, b)


def test_offsets_beyond_32_bits(acd):
    """More than 2^31 elements a tensor; the last rows against the oracle."""
    D, rows = 1 << 12, (1 << 19) + 5
    g = torch.Generator(device="cuda").manual_seed(2)
    r, b = (torch.empty(D * rows, dtype=torch.float16, device="cuda") for _ in range(2))
    for st in (r, b):
        for part in st.split(1 << 28):
            part.normal_(0, 1, generator=g)
    w = acd.as_tensor(np.linspace(0.5, 1.5, D), dtype="float16")
    wrap = lambda s: acd.from_torch(s, (D, rows), "float16")  # noqa: E731
    pick = [0, rows // 2, rows - 1]
    host = lambda s: s.view(rows, D)[pick].cpu().numpy()  # noqa: E731
    rp, bp = host(r), host(b)
    f = acd.residual_norm(wrap(r), wrap(b), w, w, inplace=True)
    ws = w.as_array()
    ref = O.norm(rp, bp, ws, ws, None, 1.0, 1e-6, 3)
    bound = O.norm_bounds(ref, ws, D, "float16")
    O.assert_within(host(f.h.storage), ref[0], bound[0])
    O.assert_within(host(f.y.storage), ref[1], bound[1])


def test_refusals(acd):
    D, rows = 16, 4
    x = acd.as_tensor(np.ones((D, rows)), dtype="float")
    w = acd.as_tensor(np.ones(D), dtype="float")
    st = acd.as_tensor(np.ones(rows), dtype="float")
    F, G = acd.residual_norm, acd.residual_norm_grad

    def status(f, *a, **k):
        with pytest.raises(L.AcdError) as e:
            f(*a, **k)
        return e.value.status

    for axis in (0, 3, 1.5):
        with pytest.raises(ValueError):
            F(x, x, w, axis=axis)
    i = acd.as_tensor(np.ones((D, rows)), dtype="int32")
    assert status(F, i, i, w) == 3
    assert status(F, acd.as_tensor(np.ones((D, rows)), dtype="double"), x, w) == 3
    assert status(F, acd.as_tensor(np.ones((D, rows + 1)), dtype="float"), x, w) == 2
    assert status(F, x, x, acd.as_tensor(np.ones(D + 1), dtype="float")) == 2
    assert status(F, x, x, acd.as_tensor(np.ones(D), dtype="float16")) == 3
    for gshape in ((D - 1,), (D, 2), (D, 1, 1), (1, rows)):
        assert status(F, x, x, w, gate=acd.as_tensor(np.ones(gshape), dtype="float")) == 2, gshape
    cube = acd.as_tensor(np.ones((D, 3, 2)), dtype="float")
    assert status(F, cube, cube, w, gate=acd.as_tensor(np.ones((D, 3, 1)), dtype="float")) == 2
    for k in (dict(alpha=float("inf")), dict(eps=-1.0), dict(eps=float("nan"))):
        assert status(F, x, x, w, **k) == 1
    e = acd.empty_tensor((0, 4), "float")
    assert status(F, e, e, acd.empty_tensor((0,), "float")) == 2
    assert status(G, x, x, x, x, st, None, w, w) == 1   # rstd_block missing
    assert status(G, x, x, x, x, st, st, w) == 1        # w_post missing
    assert status(G, x, x, x, x, acd.as_tensor(np.ones(rows + 1), dtype="float"), None, w) == 2
    assert status(G, x, x, x, x, acd.as_tensor(np.ones(rows), dtype="double"), None, w) == 3
    assert status(G, x, x, x, x, st, None, w, alpha=float("nan")) == 1
