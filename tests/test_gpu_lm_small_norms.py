"""residual_norm_grad with eps = 0 on rows whose reciprocal norms are far above 1:
no intermediate value leaves float32's range while the gradients are inside it."""
import numpy as np
import pytest

import lm_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,rows", [(5, 3), (64, 40), (1000, 20), (1001, 9), (1002, 9), (2048, 30), (4096, 12), (5003, 3)])
@pytest.mark.parametrize("size", [1e-12, 3e-16, 1e-18, 1e-20])
@pytest.mark.parametrize("post", [False, True])
def test_small_rows(acd, D, rows, size, post):
    rng = np.random.default_rng(D)
    n = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    h = (rng.standard_normal((rows, D)) * size).astype(np.float32)
    b, dy, dh = n(rows, D), n(rows, D), n(rows, D)
    wp, wo, gate = (rng.uniform(0.5, 1.5, D).astype(np.float32) for _ in range(3))
    wo = wo if post else None
    rh = (1 / np.sqrt((h.astype(np.float64) ** 2).mean(1))).astype(np.float32)
    rb = (1 / np.sqrt((b.astype(np.float64) ** 2).mean(1))).astype(np.float32) if post else None
    w = lambda a: None if a is None else acd.as_tensor(a.T if a.ndim == 2 else a, dtype="float")  # noqa: E731
    g = acd.residual_norm_grad(w(dh), w(dy), w(h), w(b), w(rh), w(rb), w(wp), w(wo), w(gate), alpha=0.5)
    args = (dh, dy, h, b, rh, rb, wp, wo, gate[None], 0.5, rows)
    ref, bound = O.norm_grad(*args), O.norm_grad_bounds(args, "float")
    O.assert_within(g.d_residual.as_array().T, ref[0], bound[0], "d_residual")
    O.assert_within(g.d_block.as_array().T, ref[1], bound[1], "d_block")
    O.assert_within(g.d_w_pre.as_array(), ref[2], bound[2], "d_w_pre")
    if post:
        O.assert_within(g.d_w_post.as_array(), ref[3], bound[3], "d_w_post")
    O.assert_within(g.d_gate.as_array(), ref[4][0], bound[4][0], "d_gate")
