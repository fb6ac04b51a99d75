"""The example that trains a model's end and follows it with a 4-bit head: its
first step against the formulas in float64, and what it learns."""
import importlib.util
import os

import numpy as np
import pytest

import lm_oracle as O

pytestmark = pytest.mark.gpu
EXAMPLE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "next_token.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("next_token", EXAMPLE)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_learns_the_table_and_follows_it(example):
    losses, right, follow = example.main()
    assert abs(losses[0] - np.log(500)) < 1e-4  # a head of zeros: every token alike
    assert losses[-1] < 0.1 and right == follow


def test_steps_follow_the_formulas(example):
    """Two steps (the first one's head is zero, so that only the head moves)
    against the same in float64.  Products sum 130 terms at most, in float32 or,
    where the matrix product rounds its operands to 11 bits, in tf32: 2^-10 of
    the head's gradient, and twice that after the second step."""
    m = example.Model(vocabulary=130, width=96, seed=3)
    a = lambda t: example.acd.as_array(t).astype(np.float64)  # noqa: E731
    r, b, pre, post, gate, W = (a(t) for t in (m.stream, m.block, m.w_pre, m.w_post, m.gate, m.head))
    n, rate = 130, 5.0
    for _ in range(2):
        h, y, rh, rb = O.norm(r.T, b.T, pre, post, gate[None], 1.0, 1e-6, n)[:4]
        lp, H, lse, _, _ = O.logprob((W @ y.T).T, m.after + 1, 1.0, 0)
        x = (W @ y.T).T
        dx = O.logprob_grad(x, m.after + 1, lse, H, np.full(n, -1.0 / n), None, None, 1.0, -np.inf)
        g = O.norm_grad(None, dx @ W, h, b.T, rh, rb, pre, post, gate[None], 1.0, n)
        loss = m.step(rate)
        assert abs(loss + lp.mean()) <= 2e-3 * abs(lp.mean())
        W, pre, post, gate = W - rate * dx.T @ y, pre - rate * g[2], post - rate * g[3], gate - rate * g[4][0]
    for t, e in ((m.head, W), (m.w_pre, pre), (m.w_post, post), (m.gate, gate)):
        assert np.linalg.norm(a(t) - e) <= 2.0 ** -9 * np.linalg.norm(e)
