"""Window attention where every score lies hundreds below zero, in one part and
in parts that are joined, rows whose first steps are masked among them."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from test_gpu_kv_pages import mi  # noqa: F401 (the library)
from test_gpu_window import attend, check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seq_q,seq_k,window,sinks", [
    (3, 5000, 0, 0), (200, 700, 90, 5), (1200, 1200, 300, 40), (1, 3000, 1000, 7)])
def test_scores_far_below_zero(seq_q, seq_k, window, sinks, hd):
    rng = np.random.default_rng(seq_q + hd)
    q, k, v = inputs(rng, seq_q, seq_k, 12, 2, hd)
    q[..., 0], k[..., 0] = -200.0, 20.0
    q, k = fp16_exact(q), fp16_exact(k)
    for split in (False, True):
        announce("window low scores", seq_q, seq_k, window, sinks, hd, split)
        check(attend(q, k, v, window, sinks, split), q, k, v, window, sinks, "low scores")
