"""The bounds of the peaked rows see one logit that is left out or taken twice, at
the sizes and with the values that the kernels are tested with."""
import numpy as np
import pytest

import lm_peaks as P
from test_gpu_lm_wide_rows import CASES

U = {"float": 2.0 ** -24, "float16": 2.0 ** -24, "double": 2.0 ** -53}
NP = {"float": np.float32, "float16": np.float16, "double": np.float64}


@pytest.mark.parametrize("dtype,layout,V,period,per,top", CASES)
def test_one_peak_less_or_twice_is_outside_the_bounds(dtype, layout, V, period, per, top):
    rng = np.random.default_rng(V)
    first, values = P.peaks(V, period, 3, rng, NP[dtype])
    lse, H = P.statistics(values, 1.0)
    b = P.bounds(values, lse, H, U[dtype])
    for r in range(3):
        v = values[r][~np.isnan(values[r])]
        for changed in (v[:-1], v[1:], np.delete(v, len(v) // 2), np.append(v, v[-1]), np.append(v, v.min())):
            l, h = P.statistics(changed[None], 1.0)
            assert abs(l[0] - lse[r]) > 2 * np.broadcast_to(b[0], 3)[r]
            # the logarithm of the sum moves every log probability as it moves lse
            assert abs(l[0] - lse[r]) > 2 * np.broadcast_to(b[2], 3)[r]
            assert abs(h[0] - H[r]) > np.broadcast_to(b[1], 3)[r]


def test_the_plain_form_agrees():
    """The peaks' statistics are those of the whole rows."""
    import lm_oracle as O
    rng = np.random.default_rng(1)
    for V, period in ((1000, 8), (4099, 64)):
        first, values = P.peaks(V, period, 9, rng, np.float32, 0.8)
        x = P.dense(V, period, first, values, np.float32)
        lse, H = P.statistics(values, 0.8)
        ref = O.logprob(x, np.zeros(9, np.int64), 0.8, 0)
        assert np.abs(ref[2] - lse).max() < 1e-13 and np.abs(ref[1] - H).max() < 1e-12
