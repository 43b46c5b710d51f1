"""One token of every sequence of a batch on the device: ragged lengths,
windows and sinks, tiers and pages not read, head layouts, with and without
partials, from page tables and from the cache manager, against float64.

Tolerance: the attention outputs' gate (conftest: 1e-3 of the value, or the
fp32 sums' bound where they cancel; the fp16 store's half step is 4.9e-4 of
it) and the masses' 1e-3."""

import numpy as np
import pytest

from conftest import announce, assert_attention_close, assert_mass_close, fp16_exact
from oracle import attention as att
from oracle import quant, windows
from test_gpu_int4 import Bytes
from test_gpu_kv_pages import mi, pages_for, put

pytestmark = pytest.mark.gpu

P, UNREAD = 32, 255


def outliers(k):
    k = k.copy()
    k[..., :2] *= 10
    return fp16_exact(k)


class Batch:
    """Sequences of `lengths` tokens on pages made by the oracle, in one device allocation in a
    shuffled order, and their tables. Rows that no query may see hold NaN where the format lets
    them: past a sequence's end, and (FP16 pages) before its window."""

    def __init__(self, rng, lengths, heads, kv, hd, tiers, window=0, sinks=0, max_pages=None,
                 q_scale=1.0):
        m = mi()
        self.lengths, self.heads, self.kv, self.hd = lengths, heads, kv, hd
        self.window, self.sinks = window, sinks
        n = len(lengths)
        self.max_pages = max_pages or max(1, max(-(-x // P) for x in lengths))
        self.q = fp16_exact(rng.standard_normal((n, heads, hd)) * q_scale)
        raw, self.tiers = {}, np.full((n, self.max_pages), UNREAD, np.uint8)
        self.k = np.zeros((n, self.max_pages * P, kv, hd))
        self.v = np.zeros_like(self.k)
        for b, length in enumerate(lengths):
            for p in range(min(-(-length // P), self.max_pages)):
                tier = tiers(b, p)
                full = (p + 1) * P <= length
                tier = tier if full or tier == UNREAD else 0
                self.tiers[b, p] = tier
                if tier == UNREAD:
                    continue
                k, v = outliers(rng.standard_normal((P, kv, hd))), fp16_exact(
                    rng.standard_normal((P, kv, hd)))
                rows = slice(p * P, (p + 1) * P)
                if tier == 0:
                    held = min(length, self.max_pages * P)  # a longer length is cut to the table
                    seen = windows.visible(held - 1, self.max_pages * P, window, sinks)[rows]
                    raw[b, p] = quant.fp16_page(
                        np.where(seen[:, None, None], k, np.nan).astype(np.float16),
                        np.where(seen[:, None, None], v, np.nan).astype(np.float16))
                    self.k[b, rows], self.v[b, rows] = k, v
                else:
                    raw[b, p] = quant.quantise_page(k.astype(np.float16), v.astype(np.float16), tier, P)
                    self.k[b, rows], self.v[b, rows] = quant.dequantise_page(raw[b, p], tier, kv, hd, P)
        offsets, at = {}, 0
        keys = list(raw)
        for i in rng.permutation(len(keys)):
            offsets[keys[i]] = at
            at += -(-len(raw[keys[i]]) // 64) * 64
        pool = np.zeros(max(at, 64), np.uint8)
        for key, o in offsets.items():
            pool[o:o + len(raw[key])] = np.asarray(raw[key], np.uint8)
        self.pool = m._Storage(pool.size)
        m._h2d(self.pool.ptr, pool)
        table = np.zeros((n, self.max_pages), np.uint64)
        for (b, p), o in offsets.items():
            table[b, p] = self.pool.ptr + o
        self.table = table
        self.upload()

    def upload(self):
        n = len(self.lengths)
        self.pages = Bytes(self.table.reshape(-1).view(np.uint8))
        self.pages.numel = n * self.max_pages
        self.tier_bytes = Bytes(self.tiers.reshape(-1))
        self.tier_bytes.numel = n * self.max_pages
        self.length_index = mi().device.DeviceIndex(np.array(self.lengths, np.int32))

    def want(self, b):
        unread = np.repeat((self.tiers[b] > 3) | (self.table[b] == 0), P)
        length = min(self.lengths[b], self.max_pages * P)
        return windows.paged_token(self.q[b], self.k[b], self.v[b], length, unread, self.window,
                                   self.sinks, P)

    def check(self, got, mass=None, what=""):
        for b in range(len(self.lengths)):
            out, want_mass, bound = self.want(b)
            assert_attention_close(got[b], out, f"{what} sequence {b} of {self.lengths[b]}", bound)
            if mass is not None:
                assert_mass_close(mass[b], want_mass, f"{what} mass {b}")

    def run(self, split, with_mass, q=None, out=None):
        d = mi().device
        n, size = len(self.lengths), (self.heads, self.kv, self.hd)
        q = put(self.q) if q is None else q
        y = Bytes(count=2 * n * self.heads * self.hd) if out is None else out
        y.numel = n * self.heads * self.hd
        mass = d.empty_f32(n * self.heads * self.max_pages) if with_mass else None
        parts = None
        if split or with_mass:
            parts = d.empty_f32(d.attention_batch_partials(
                n, self.max_pages, *size, window=self.window, sinks=self.sinks, mass=with_mass))
        d.attention_batch(q, self.pages, self.tier_bytes, self.length_index, y, n, self.max_pages,
                          *size, window=self.window, sinks=self.sinks, mass=mass, partials=parts)
        got = y.read().view(np.float16).reshape(n, self.heads, self.hd)
        return got, mass.to_numpy().reshape(n, self.heads, -1) if with_mass else None


def cycle(*tiers):
    return lambda b, p: tiers[(b + p) % len(tiers)]


MIXED = cycle(1, 0, 3, 2)
LAYOUTS = [(14, 2, 64), (12, 2, 128), (32, 8, 64), (4, 4, 128), (16, 1, 64), (16, 1, 128),
           (6, 3, 64), (20, 5, 128), (48, 16, 64), (12, 12, 128)]


@pytest.mark.parametrize("heads,kv,hd", LAYOUTS)
def test_head_layouts(heads, kv, hd):
    rng = np.random.default_rng(heads + hd)
    batch = Batch(rng, [1, 0, 31, 32, 33, 64, 65, 300, 129], heads, kv, hd, MIXED)
    for split, mass in ((False, False), (True, False), (True, True)):
        announce("batch layout", heads, kv, hd, split, mass)
        batch.check(*batch.run(split, mass), f"{heads}/{kv}x{hd}")


@pytest.mark.parametrize("tier", [0, 1, 2, 3])
@pytest.mark.parametrize("hd", [64, 128])
def test_each_tier(tier, hd):
    rng = np.random.default_rng(tier + hd)
    batch = Batch(rng, [500, 32, 96], 8, 2, hd, cycle(tier))
    announce("batch tier", tier, hd)
    batch.check(*batch.run(True, True), f"tier {tier}")


@pytest.mark.parametrize("window,sinks", [
    (1, 0), (1, 1), (31, 0), (32, 4), (33, 4), (64, 0), (100, 32), (100, 33), (100, 1000),
    (299, 0), (300, 5), (301, 0), (5000, 7)])
def test_windows_and_sinks(window, sinks):
    rng = np.random.default_rng(window + sinks)
    batch = Batch(rng, [300, 1, 0, 64, 290, 1000, 33, 128], 14, 2, 64, MIXED, window, sinks)
    for split, mass in ((False, False), (True, True)):
        announce("batch window", window, sinks, split)
        batch.check(*batch.run(split, mass), f"window {window} sinks {sinks}")


@pytest.mark.parametrize("hd", [64, 128])
def test_a_long_sequence_among_short_ones_split_and_joined(hd):
    """One sequence of 16K tokens in many runs, others in one or none; the page count past one
    join wave's."""
    rng = np.random.default_rng(hd)
    batch = Batch(rng, [16001, 5, 0, 2049], 4, 2, hd, MIXED)
    for split, mass in ((False, False), (True, True)):
        announce("batch long", hd, split)
        batch.check(*batch.run(split, mass), f"long {hd}")


def test_pages_not_read():
    """Evicted pages (tier 255), a tier that is none, a page with no address, a sequence with every
    page gone, one whose only visible page is gone."""
    rng = np.random.default_rng(5)
    batch = Batch(rng, [200, 64, 96, 320], 12, 2, 128,
                  lambda b, p: UNREAD if b == 1 or p % 3 == 1 else p % 4, window=40, sinks=2)
    batch.tiers[0, 3] = 7
    batch.table[3, 8] = 0
    batch.tiers[2, 1:] = UNREAD
    batch.upload()
    for split in (False, True):
        announce("batch unread", split)
        got, mass = batch.run(split, split)
        batch.check(got, mass, "unread")
        assert not got[1].any()


def test_lengths_past_the_table_and_below_zero():
    rng = np.random.default_rng(6)
    batch = Batch(rng, [1000, 96, -5, 2**31 - 1], 8, 2, 64, cycle(0), max_pages=4)
    announce("batch lengths")
    got, mass = batch.run(True, True)
    batch.check(got, mass, "lengths")
    batch = Batch(rng, [1000, 2**31 - 1], 8, 2, 64, cycle(0), max_pages=4, window=50, sinks=2)
    batch.check(*batch.run(True, True), "lengths behind a window")


def test_scores_far_apart_and_alike():
    """Scores of hundreds (one key takes the softmax), and of zero (every key the same)."""
    rng = np.random.default_rng(7)
    for scale in (60.0, 0.0):
        batch = Batch(rng, [700, 40], 8, 2, 128, MIXED, q_scale=scale)
        announce("batch scores", scale)
        batch.check(*batch.run(True, True), f"scores x {scale}")


def test_values_that_are_not_finite_reach_the_heads_that_see_them():
    rng = np.random.default_rng(8)
    batch = Batch(rng, [70, 70], 8, 2, 64, cycle(0))
    m = mi()
    page = np.empty(2 * P * 2 * 64, np.float16)  # sequence 0's first page
    m._d2h(page, int(batch.table[0, 0]))
    page.reshape(2, P, 2, 64)[1, 3, 0, 5] = np.inf  # a value of KV head 0
    page.reshape(2, P, 2, 64)[0, 4, 1, 6] = np.nan  # a key of KV head 1
    m._h2d(int(batch.table[0, 0]), page)
    announce("batch not finite")
    got, mass = batch.run(True, True)
    assert not np.isfinite(got[0, :4, 5]).any() and np.isfinite(mass[0, :4]).all()
    assert np.isnan(got[0, 4:]).all() and np.isnan(mass[0, 4:]).any()
    out, want_mass, bound = batch.want(1)
    assert_attention_close(got[1], out, "its neighbour", bound)


def test_rows_past_the_batch_stay_and_calls_repeat_to_the_bit():
    rng = np.random.default_rng(9)
    batch = Batch(rng, [500, 33, 128], 12, 2, 128, MIXED)
    d = mi().device
    y = Bytes(count=2 * 5 * 12 * 128)
    y.numel = 5 * 12 * 128
    q = put(batch.q)
    first = None
    for _ in range(3):
        announce("batch repeat")
        parts = d.empty_f32(d.attention_batch_partials(3, batch.max_pages, 12, 2, 128))
        d.attention_batch(q, batch.pages, batch.tier_bytes, batch.length_index, y, 3,
                          batch.max_pages, 12, 2, 128, partials=parts)
        raw = y.read()
        assert (raw[2 * 3 * 12 * 128:] == 0xA5).all()
        first = raw.copy() if first is None else first
        np.testing.assert_array_equal(raw, first)


def test_a_captured_step_follows_the_lengths_on_the_device():
    """Two graphs with partials of their own, replayed in turn while lengths and queries change."""
    m = mi()
    d = m.device
    rng = np.random.default_rng(10)
    batch = Batch(rng, [400, 120, 64], 8, 2, 64, MIXED)
    full = list(batch.lengths)
    stream = m.Stream()
    q = d.empty(3 * 8 * 64)
    graphs = []
    for with_mass in (False, True):
        parts = d.empty_f32(d.attention_batch_partials(3, batch.max_pages, 8, 2, 64, mass=with_mass))
        mass = d.empty_f32(3 * 8 * batch.max_pages) if with_mass else None
        out = d.empty(3 * 8 * 64)
        graph = m.Graph(stream)
        with graph.capture():
            d.attention_batch(q, batch.pages, batch.tier_bytes, batch.length_index, out, 3,
                              batch.max_pages, 8, 2, 64, mass=mass, partials=parts)
        graphs.append((graph, out, mass, parts))
    for lengths in ([400, 120, 64], [32, 0, 1], [399, 64, 33], full):
        batch.lengths = lengths
        batch.q = fp16_exact(rng.standard_normal((3, 8, 64)))
        m._h2d(batch.length_index.address, np.array(lengths, np.int32))
        m._h2d(q.address, batch.q.astype(np.float16))
        for graph, out, mass, _ in graphs:
            announce("batch replay", lengths, mass is not None)
            graph.launch()
            stream.synchronize()
            batch.check(out.to_numpy().reshape(3, 8, 64),
                        mass.to_numpy().reshape(3, 8, -1) if mass else None, f"replay {lengths}")
        m.synchronize()


# -- over the cache manager ---------------------------------------------------------------------

LAYERS = 2


def filled(rng, kv, hd, n, seals):
    """A KVPages with n tokens of LAYERS layers stored (the last by itself, as a decode does)."""
    tier_map = [[(1, 0, 3, 2)[(l + p) % 4] for p in range(n // P + 1)] for l in range(LAYERS)]
    alloc, cache = pages_for(P, kv, hd, 0, tier_map if seals else None, seals)
    k = outliers(rng.standard_normal((LAYERS, n, kv, hd)))
    v = fp16_exact(rng.standard_normal((LAYERS, n, kv, hd)))
    for l in range(LAYERS):
        if n > 1:
            cache.reserve(n - 1)
            cache.store(l, put(k[l, :-1]), put(v[l, :-1]), 0, n - 1)
    if n:
        cache.reserve(n)
    for l in range(LAYERS):
        if n:
            cache.store(l, put(k[l, -1:]), put(v[l, -1:]), n - 1, 1)
    return alloc, cache, k, v


def as_read(alloc, cache, layer, k, v, kv, hd, seals):
    """The rows a token at the end sees: sealed pages as their tiers give them back."""
    n = k.shape[1]
    rows_k, rows_v = k[layer].copy(), v[layer].copy()
    unread = np.zeros(n, bool)
    for p in range((n - 1) // P if seals and n else 0):
        rows = slice(p * P, (p + 1) * P)
        if (layer, p) not in alloc:
            unread[rows] = True
            continue
        tier = int(alloc.locate(layer, p)[0])
        if tier:
            rows_k[rows], rows_v[rows] = quant.dequantise_page(alloc.read(layer, p), tier, kv, hd, P)
    pad = -n % P
    shape = ((0, pad), (0, 0), (0, 0))
    return np.pad(rows_k, shape), np.pad(rows_v, shape), np.pad(unread, (0, pad))


@pytest.mark.parametrize("seals", [True, False])
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128), (32, 8, 64)])
def test_caches_of_the_manager(seals, heads, kv, hd):
    """A page sealed by the token's own row, an open page, the first row; evictions; a cache named
    twice; a slot with no token."""
    m = mi()
    d = m.device
    rng = np.random.default_rng(heads + seals)
    lengths = [1, 31, 32, 33, 64, 97, 200]
    held = [filled(rng, kv, hd, n, seals) for n in lengths]
    if seals:
        held[6][1].evict(0, 2)
        held[6][1].move_pages([(1, 0, 2), (1, 4, 3)])
    held.append(held[5])
    lengths = lengths + [97, 0]
    held.append(held[0])
    n = len(lengths)
    q = fp16_exact(rng.standard_normal((n, heads, hd)))
    for layer in range(LAYERS):
        own = [np.stack([h[i][layer, -1] for h in held]) for i in (2, 3)]
        keys, values = (put(x) for x in own) if seals else (None, None)
        for window, sinks in ((0, 0), (40, 3)):
            pages = -(-max(lengths) // P)
            for with_mass in (False, True):
                announce("caches", seals, heads, kv, hd, layer, window, with_mass)
                out = d.empty(n * heads * hd)
                mass = d.empty_f32(n * heads * pages) if with_mass else None
                parts = d.empty_f32(d.attention_batch_partials(
                    n, pages, heads, kv, hd, window, sinks, with_mass))
                d.attention_caches([h[1] for h in held], lengths, layer, put(q), out, heads, kv, hd,
                                   keys, values, window, sinks, mass=mass, partials=parts)
                got = out.to_numpy().reshape(n, heads, hd)
                for i, (alloc, cache, k, v) in enumerate(held):
                    if lengths[i] == 0:
                        assert not got[i].any()
                        continue
                    rk, rv, unread = as_read(alloc, cache, layer, k, v, kv, hd, seals)
                    want, want_mass, bound = windows.paged_token(q[i], rk, rv, lengths[i], unread,
                                                                 window, sinks, P)
                    assert_attention_close(got[i], want, f"cache {i}", bound)
                    if with_mass:
                        gm = mass.to_numpy().reshape(n, heads, pages)[i]
                        assert_mass_close(gm[:, :want_mass.shape[1]], want_mass, f"mass {i}")
                        assert not gm[:, want_mass.shape[1]:].any()


def test_more_caches_than_a_launch_holds_and_the_single_sequence_s_attention():
    """70 sequences over three caches, in launches of 32; and against KVPages.attention."""
    m = mi()
    d = m.device
    rng = np.random.default_rng(11)
    heads, kv, hd = 12, 2, 128
    held = [filled(rng, kv, hd, n, True) for n in (70, 33, 150)]
    which = [i % 3 for i in range(70)]
    q = fp16_exact(rng.standard_normal((70, heads, hd)))
    keys = put(np.stack([held[i][2][0, -1] for i in which]))
    values = put(np.stack([held[i][3][0, -1] for i in which]))
    lengths = [(70, 33, 150)[i] for i in which]
    out, mass = d.empty(70 * heads * hd), d.empty_f32(70 * heads * 6)
    parts = d.empty_f32(d.attention_batch_partials(70, 6, heads, kv, hd, mass=True))
    announce("70 caches")
    d.attention_caches([held[i][1] for i in which], lengths, 0, put(q), out, heads, kv, hd, keys,
                       values, mass=mass, mass_pages=6, partials=parts)
    got, got_mass = out.to_numpy().reshape(70, heads, hd), mass.to_numpy().reshape(70, heads, 6)
    for i in range(70):
        alloc, cache, k, v = held[which[i]]
        want, want_mass, bound = windows.paged_token(
            q[i], *as_read(alloc, cache, 0, k, v, kv, hd, True)[:2], lengths[i],
            np.zeros(-(-lengths[i] // P) * P, bool), 0, 0, P)
        assert_attention_close(got[i], want, f"cache {i}", bound)
        assert_mass_close(got_mass[i, :, :want_mass.shape[1]], want_mass)
        if i < 3:
            single = d.empty(heads * hd)
            cache.attention(0, put(q[i]), None, None, single, 1, lengths[i], heads, kv, hd,
                            put(k[0, -1]), put(v[0, -1]))
            assert_attention_close(got[i], single.to_numpy().reshape(heads, hd).astype(np.float64),
                                   "the single call", 2 * bound + 2.0**-11 * np.abs(want))
