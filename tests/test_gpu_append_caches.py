"""Several caches' new rows appended by one call: caches that seal and that do
not, prompts that complete pages, prompts behind a prefix, single tokens, more
caches than a launch holds, layers; then the attention that reads them.

The rows handed back are compared with the formula in float64 (test_gpu_append's
tolerance); what the caches then hold is, to the bit, what a twin cache holds
after a store of those rows, and so are attention_caches' outputs."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from oracle import ragged
from test_gpu_append import LLAMA3, P, close
from test_gpu_batch import LAYERS
from test_gpu_kv_pages import mi, pages_for, put, sealed_pages

pytestmark = pytest.mark.gpu


class Twins:
    """A cache filled by appends and one filled by stores of the rows that came back."""

    def __init__(self, kv, hd, pages, seals, page_tokens=P):
        tier_map = [[(1, 0, 3, 2)[(l + p) % 4] for p in range(pages)] for l in range(LAYERS)]
        self.kv, self.hd, self.seals, self.P, self.end = kv, hd, seals, page_tokens, 0
        self.alloc, self.cache = pages_for(page_tokens, kv, hd, 0, tier_map if seals else None, seals)
        self.twin_alloc, self.twin = pages_for(page_tokens, kv, hd, 0, tier_map if seals else None, seals)

    def pages(self, alloc, layer):
        full = self.end // self.P
        return sealed_pages(alloc, layer, full if self.seals else -(-self.end // self.P))

    def check(self, layer):
        mine, other = self.pages(self.alloc, layer), self.pages(self.twin_alloc, layer)
        assert mine[1] == other[1]
        rows = 2 * self.kv * self.hd  # bytes of a token's keys, or its values
        for p, (a, b) in enumerate(zip(mine[0], other[0])):
            if not self.seals:  # the rows past the end were never written
                n = min(self.P, self.end - p * self.P)
                a, b = (x.view(np.uint8).reshape(2, self.P, rows)[:, :n] for x in (a, b))
            np.testing.assert_array_equal(a, b)


def append(rng, held, counts, heads, rope, freq, magnitude=1.0, interleaved=False, out=True):
    """One call a layer over `held`, then the stores of the twins, then both attentions."""
    d = mi().device
    kv, hd = held[0].kv, held[0].hd
    rows, starts = sum(counts), [h.end for h in held]
    offsets = np.concatenate([[0], np.cumsum(counts)])
    for h, n in zip(held, counts):
        for cache in (h.cache, h.twin):
            cache.reserve(h.end + n)
    for layer in range(LAYERS):
        q, k, v = (fp16_exact(rng.standard_normal((rows, n, hd))) for n in (heads, kv, kv))
        outs = [d.empty(max(1, x.size)) for x in (q, k, v)]
        d.append_caches([h.cache for h in held], starts, counts, layer, put(q), put(k), put(v), outs[0],
                        outs[1] if out else None, outs[2] if out else None, rope, heads, kv, hd,
                        interleaved)
        at = np.concatenate([s + np.arange(n) for s, n in zip(starts, counts)]).astype(int)
        q_out = outs[0].to_numpy().reshape(q.shape).astype(np.float64)
        close(q_out, *ragged.turned(q, at, freq, magnitude, interleaved))
        if out:
            k_out = outs[1].to_numpy().reshape(k.shape)
            close(k_out.astype(np.float64), *ragged.turned(k, at, freq, magnitude, interleaved))
            np.testing.assert_array_equal(outs[2].to_numpy().reshape(v.shape).astype(np.float32), v)
        for i, h in enumerate(held):
            mine = slice(offsets[i], offsets[i + 1])
            if not counts[i]:
                continue
            if out:
                h.twin.store(layer, put(k_out[mine]), put(v[mine]), starts[i], counts[i])
            else:
                alone = d.empty(counts[i] * heads * hd), d.empty(counts[i] * kv * hd)
                d.append_caches([h.twin], [starts[i]], [counts[i]], layer, put(q[mine]), put(k[mine]),
                                put(v[mine]), *alone, None, rope, heads, kv, hd, interleaved)
                close(alone[1].to_numpy().reshape(-1, kv, hd).astype(np.float64),
                      *ragged.turned(k[mine], at[mine], freq, magnitude, interleaved))
        for h, n in zip(held, counts):
            h.end += n
            h.check(layer)
            h.end -= n
        # (A run that completes a page leaves its rows at the page's tier alone:
        # attention_caches refuses its last token in a cache that seals.)
        some = [i for i, n in enumerate(counts)
                if n and not (held[0].seals and n > 1 and (starts[i] + n) % P == 0)]
        if out and some:
            last = [offsets[i + 1] - 1 for i in some]
            lengths = [starts[i] + counts[i] for i in some]
            keys, values = put(k_out[last]), put(v[last])
            got = []
            for which in ("cache", "twin"):
                y = d.empty(len(some) * heads * hd)
                d.attention_caches([getattr(held[i], which) for i in some], lengths, layer, put(q_out[last]),
                                   y, heads, kv, hd, keys if held[0].seals else None,
                                   values if held[0].seals else None)
                got.append(y.to_numpy())
            assert np.isfinite(got[0]).all()
            np.testing.assert_array_equal(*got)
    for h, n in zip(held, counts):
        h.end += n


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128), (32, 8, 64)])
@pytest.mark.parametrize("seals", [True, False])
def test_prompts_prefixes_and_single_tokens(heads, kv, hd, seals):
    """Prompts of no rows, one, a page less one, a page, pages and more; then tokens and runs behind."""
    rng = np.random.default_rng(heads + seals)
    rope = mi().device.RopeTable(hd, 5e5, LLAMA3)
    rope.cover(40 * P)
    freq, magnitude = ragged.frequencies(hd, 5e5, LLAMA3)
    held = [Twins(kv, hd, 40, seals) for _ in range(7)]
    for counts in ([0, 1, 31, 32, 33, 100, 700], [1] * 7, [5, 30, 1, 0, 31, 64, 1], [1] * 7,
                   [0, 0, 1, 65, 0, 0, 330]):
        announce("append caches", heads, kv, hd, seals, counts)
        append(rng, held, counts, heads, rope, freq, magnitude)


def test_more_caches_than_a_launch_holds():
    rng = np.random.default_rng(5)
    rope = mi().device.RopeTable(64, 1e6)
    rope.cover(8 * P)
    for seals in (True, False):
        held = [Twins(2, 64, 8, seals) for _ in range(70)]
        for counts in (rng.integers(0, 70, 70).tolist(), [1] * 70):
            announce("70 caches", seals)
            append(rng, held, counts, 14, rope, ragged.frequencies(64, 1e6, None)[0])


def test_caches_that_do_not_seal_need_no_rows_back():
    rng = np.random.default_rng(6)
    rope = mi().device.RopeTable(48, 1e6)
    rope.cover(8 * P)
    held = [Twins(1, 96, 8, False) for _ in range(3)]
    for counts in ([40, 3, 0], [1, 1, 1]):
        announce("no rows back", counts)
        append(rng, held, counts, 3, rope, ragged.frequencies(48, 1e6, None)[0], interleaved=True, out=False)


@pytest.mark.parametrize("page_tokens", [16, 48])
def test_pages_of_other_sizes(page_tokens):
    """Stored as they are by the caches; (attention_batch's pages hold 32.)"""
    m = mi()
    d = m.device
    rng = np.random.default_rng(page_tokens)
    rope = d.RopeTable(64, 1e4)
    rope.cover(400)
    for seals in (True, False):
        h = Twins(2, 64, 30, seals, page_tokens)
        for n in (page_tokens * 2 + 5, 1, page_tokens - 6, 70):
            announce("pages", page_tokens, seals, n)
            q, k, v = (fp16_exact(rng.standard_normal((n, x, 64))) for x in (4, 2, 2))
            outs = [d.empty(x.size) for x in (q, k, v)]
            for cache in (h.cache, h.twin):
                cache.reserve(h.end + n)
            d.append_caches([h.cache], [h.end], [n], 1, put(q), put(k), put(v), *outs, rope, 4, 2, 64)
            h.twin.store(1, outs[1], outs[2], h.end, n)
            h.end += n
            h.check(1)


def test_refusals():
    """Nothing is written by a call that is refused."""
    m = mi()
    d = m.device
    rope = d.RopeTable(64, 1e4)
    rope.cover(40)
    a, b = Twins(2, 64, 8, True), Twins(2, 64, 8, False)
    for h in (a, b):
        h.cache.reserve(64)
    rows = 64
    q, k, v = (put(np.ones((rows, n, 64), np.float32)) for n in (4, 2, 2))
    outs = [d.empty(rows * n * 64) for n in (4, 2, 2)]
    zero = np.zeros(rows * 2 * 64)
    m._h2d(outs[1].address, zero.astype(np.float16))

    def call(caches, starts, counts, layer=0, kv=2, hd=64, back=True, table=rope):
        d.append_caches([h.cache for h in caches], starts, counts, layer, q, k, v, outs[0],
                        outs[1] if back else None, outs[2] if back else None, table, 4, kv, hd)

    announce("refusals")
    for error, args in ((ValueError, ([b, b], [0, 0], [1, 1])), (ValueError, ([a, a], [0, 0], [1, 0])),
                        (IndexError, ([a], [60], [37])), (KeyError, ([a], [60], [36])), (IndexError, ([b], [65], [0])),
                        (IndexError, ([b], [-1], [2])), (IndexError, ([Twins(2, 64, 8, True)], [0], [1])), (ValueError, ([b], [0], [-1])),
                        (ValueError, ([b], [0], [41])), (ValueError, ([a, b], [0], [1, 1])),
                        (ValueError, ([a, Twins(2, 64, 8, False, 16)], [0, 0], [1, 0]))):
        with pytest.raises(error):
            call(*args)
    with pytest.raises(ValueError):
        call([b, a], [0, 0], [1, 1], back=False)
    with pytest.raises(ValueError):
        call([b], [0], [1], hd=32)
    with pytest.raises(ValueError):
        call([b], [0], [1], kv=1)
    for layer in (-1, LAYERS):
        with pytest.raises((ValueError, IndexError)):
            call([b], [0], [1], layer=layer)
    assert not outs[1].to_numpy()[:zero.size].any()
    call([], [], [])
    call([a, b], [0, 0], [0, 0])
    call([b, a], [0, 3], [40, 0], back=False)


def test_a_completed_page_that_was_evicted_is_refused():
    m = mi()
    d = m.device
    rope = d.RopeTable(64, 1e4)
    rope.cover(4 * P)
    rng = np.random.default_rng(0)
    h = Twins(2, 64, 8, True)
    append(rng, [h], [P + 3], 4, rope, ragged.frequencies(64, 1e4, None)[0])
    h.cache.evict(0, 0)
    announce("evicted")
    rows = [put(np.ones((P, n, 64), np.float32)) for n in (4, 2, 2)]
    outs = [d.empty(P * n * 64) for n in (4, 2, 2)]
    with pytest.raises((KeyError, ValueError, IndexError)):
        d.append_caches([h.cache], [0], [P], 0, *rows, *outs, rope, 4, 2, 64)
