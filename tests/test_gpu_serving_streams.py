"""The serving operators on two streams at once, each with partials of its own:
the bits of the same calls one after another."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from test_gpu_batch import MIXED, Batch
from test_gpu_int4 import Int4, weight
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu


def test_two_streams_at_once():
    m = mi()
    d = m.device
    rng = np.random.default_rng(0)
    batch = Batch(rng, [3000, 33, 700, 1999], 12, 2, 128, MIXED, 0, 0)
    w = Int4(weight(rng, 1536, 2048), 64)
    bq, seq = put(batch.q), 1500
    q, k, v = (put(fp16_exact(rng.standard_normal((seq, h * 128)))) for h in (12, 2, 2))
    x = put(fp16_exact(rng.standard_normal((40, 2048))))

    class Lane:
        def __init__(self):
            self.batch_parts = d.empty_f32(d.attention_batch_partials(4, batch.max_pages, 12, 2, 128,
                                                                      mass=True))
            self.window_parts = d.empty_f32(65536 * 130)
            self.mass = d.empty_f32(4 * 12 * batch.max_pages)
            self.outs = d.empty(4 * 12 * 128), d.empty(seq * 12 * 128), d.empty(40 * 1536)

        def run(self):
            d.attention_batch(bq, batch.pages, batch.tier_bytes, batch.length_index, self.outs[0], 4,
                              batch.max_pages, 12, 2, 128, mass=self.mass, partials=self.batch_parts)
            d.attention_window(q, k, v, self.outs[1], seq, seq, 12, 2, 128, 300, 4,
                               partials=self.window_parts)
            d.linear_int4(x, *w.on, 64, None, self.outs[2], 40, 2048, 1536)

        def read(self):
            return [t.to_numpy() for t in (*self.outs, self.mass)]

    lanes, streams = [Lane(), Lane()], [m.Stream(), m.Stream()]
    lanes[0].run()
    m.synchronize()
    want = lanes[0].read()
    announce("two streams")
    for _ in range(20):
        for lane, stream in zip(lanes, streams):
            m.set_stream(stream)
            lane.run()
    m.set_stream(None)
    for stream in streams:
        stream.synchronize()
    for lane in lanes:
        for got, one in zip(lane.read(), want):
            np.testing.assert_array_equal(got, one)
