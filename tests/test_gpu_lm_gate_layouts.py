"""Which gates residual_norm takes where the axis stands in the middle."""
import numpy as np
import pytest

import acediar._lib as L
import lm_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gshape", [(1, 40, 3), (1, 40, 1), (40,)])
def test_taken(acd, gshape):
    rng = np.random.default_rng(1)
    r, b = (rng.standard_normal((5, 40, 3)).astype(np.float32) for _ in range(2))
    w, gate = np.ones(40, np.float32), rng.standard_normal(gshape).astype(np.float32)
    t = lambda a: acd.as_tensor(a, dtype="float")  # noqa: E731
    got = acd.residual_norm(t(r), t(b), t(w), gate=t(gate), axis=2)
    gr = gate.reshape(1, -1) if gate.ndim == 1 else O.moved(gate, 2)
    ref = O.norm(O.moved(r, 2), O.moved(b, 2), w, None, gr, 1.0, 1e-6, 15 // len(gr))
    bound = O.norm_bounds(ref, w, 40, "float")
    O.assert_within(O.moved(got.h.as_array(), 2), ref[0], bound[0])
    O.assert_within(O.moved(got.y.as_array(), 2), ref[1], bound[1])


def test_one_row_for_each_on_both_sides_is_refused(acd):
    x, w = acd.as_tensor(np.ones((5, 40, 3)), dtype="float"), acd.as_tensor(np.ones(40), dtype="float")
    st = acd.as_tensor(np.ones((5, 3)), dtype="float")
    for call in (lambda: acd.residual_norm(x, x, w, gate=x, axis=2),
                 lambda: acd.residual_norm_grad(None, x, x, x, st, None, w, gate=x, axis=2)):
        with pytest.raises(L.AcdError) as e:
            call()
        assert e.value.status == 8 and "gate" in str(e.value)
