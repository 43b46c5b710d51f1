"""attention_caches captured and replayed, in launches of 32 sequences, while
queries and the tokens' own rows change; and a capture refused while a cache's
page table has entries that are not on the device yet."""

import numpy as np
import pytest

from conftest import announce, assert_attention_close, assert_mass_close, fp16_exact
from oracle import windows
from test_gpu_batch import P, as_read, filled
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128)])
def test_replays_follow_queries_and_own_rows(heads, kv, hd):
    m = mi()
    d = m.device
    rng = np.random.default_rng(hd)
    ends = (70, 33, 150)
    held = [filled(rng, kv, hd, n, True) for n in ends]
    which = [i % 3 for i in range(40)]
    lengths, pages = [ends[i] for i in which], 5
    caches = [held[i][1] for i in which]
    q, own_k, own_v = d.empty(40 * heads * hd), d.empty(40 * kv * hd), d.empty(40 * kv * hd)
    out, mass = d.empty(40 * heads * hd), d.empty_f32(40 * heads * pages)
    parts = d.empty_f32(d.attention_batch_partials(40, pages, heads, kv, hd, 100, 3, mass=True))

    def step():
        d.attention_caches(caches, lengths, 1, q, out, heads, kv, hd, own_k, own_v, 100, 3,
                           mass=mass, partials=parts)

    stream = m.Stream()
    graph = m.Graph(stream)
    m.set_stream(stream)
    step()  # the page tables reach the device
    m.set_stream(None)
    with graph.capture():
        step()
    for i in range(4):
        hq = fp16_exact(rng.standard_normal((40, heads, hd)))
        rows = [fp16_exact(rng.standard_normal((40, kv, hd))) for _ in range(2)]
        for to, host in ((q, hq), (own_k, rows[0]), (own_v, rows[1])):
            m._h2d(to.address, host.astype(np.float16))
        announce("captured caches", heads, kv, hd, i)
        graph.launch()
        stream.synchronize()
        got = out.to_numpy().reshape(40, heads, hd)
        got_mass = mass.to_numpy().reshape(40, heads, pages)
        for b in range(40):
            alloc, cache, k, v = held[which[b]]
            k, v = k.copy(), v.copy()
            k[1, -1], v[1, -1] = rows[0][b], rows[1][b]
            rk, rv, unread = as_read(alloc, cache, 1, k, v, kv, hd, True)
            want, want_mass, bound = windows.paged_token(hq[b], rk, rv, lengths[b], unread, 100, 3, P)
            assert_attention_close(got[b], want, f"replay {i} cache {b}", bound)
            assert_mass_close(got_mass[b, :, :want_mass.shape[1]], want_mass)
        m.synchronize()


def test_a_capture_before_the_page_table_is_on_the_device_is_refused():
    m = mi()
    d = m.device
    rng = np.random.default_rng(1)
    alloc, cache, k, v = filled(rng, 2, 64, 150, True)
    q, out = put(rng.standard_normal((1, 14, 64))), d.empty(14 * 64)
    own = put(k[0, -1]), put(v[0, -1])

    def step():
        d.attention_caches([cache], [150], 0, q, out, 14, 2, 64, *own)

    step()
    m.synchronize()
    before = out.to_numpy()
    stream = m.Stream()
    cache.evict(0, 1)  # an entry that only the host knows
    announce("capture refused")
    with pytest.raises(RuntimeError, match="before they are captured"):
        with m.Graph(stream).capture():
            step()
    step()
    m.synchronize()
    after = out.to_numpy()
    assert (before != after).any()
    graph = m.Graph(stream)
    with graph.capture():
        step()
    for _ in range(3):
        m._h2d(out.address, np.zeros(14 * 64, np.float16))
        announce("captured after all")
        graph.launch()
        stream.synchronize()
        np.testing.assert_array_equal(out.to_numpy(), after)
