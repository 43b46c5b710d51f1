"""The window oracle against a double loop, and its two forms against each
other."""

import numpy as np
import pytest

from oracle import attention as att
from oracle import windows


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 3), (1, 0), (3, 2), (100, 1)])
def test_window_attention_is_the_loop(window, sinks):
    rng = np.random.default_rng(window + sinks)
    q, k, v = (rng.standard_normal(s) for s in ((7, 4, 8), (11, 2, 8), (11, 2, 8)))
    out, bound, terms = windows.window_attention(q, k, v, window, sinks)
    assert (terms >= np.abs(out)).all() and (bound > 0).all()
    for i in range(7):
        at = 4 + i
        for h in range(4):
            js = [j for j in range(at + 1) if not window or j > at - window or j < sinks]
            s = np.array([q[i, h] @ k[j, h // 2] for j in js]) / np.sqrt(8)
            p = np.exp(s - s.max())
            want = sum(w * v[j, h // 2] for w, j in zip(p / p.sum(), js))
            np.testing.assert_allclose(out[i, h], want, atol=1e-12)


def test_a_token_is_the_last_query_and_masses_sum_to_one():
    rng = np.random.default_rng(3)
    q = rng.standard_normal((1, 4, 8))
    k, v = rng.standard_normal((2, 64, 2, 8))
    for length, window, sinks in ((64, 0, 0), (50, 20, 3), (1, 5, 0)):
        out, mass, _ = windows.paged_token(q[0], k, v, length, np.zeros(64, bool), window, sinks, 16)
        want, _, _ = windows.window_attention(q, k[:length], v[:length], window, sinks)
        np.testing.assert_allclose(out, want[0], atol=1e-12)
        np.testing.assert_allclose(mass.sum(1), 1.0)
    out, mass, _ = windows.paged_token(q[0], k, v, 0, np.zeros(64, bool), 0, 0, 16)
    assert not out.any() and not mass.any()
    full, weights = att.attention64(q, k, v)
    np.testing.assert_allclose(windows.paged_token(q[0], k, v, 64, np.zeros(64, bool), 0, 0, 16)[0],
                               full[0])
