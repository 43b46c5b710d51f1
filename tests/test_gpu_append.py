"""Rows of a packed batch appended to paged caches with their rotation: ragged
batches, empty sequences, rows of no sequence, pages that are not there, head
layouts and odd sizes, parts of heads, both pairings, scaled angles, strides;
against float64.

Tolerance of a turned channel: cos and sin rounded to fp32 (2^-24 of them), two
products and a sum rounded in fp32, 4 x 2^-24 of |a| + |b| in all, and the
output's half step (2^-11 of it, 2^-25 below fp16's normals). Others are exact."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from oracle import ragged
from test_gpu_int4 import Bytes, halves
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu
P = 32
LLAMA3 = dict(kind="llama3", factor=32.0, low=1.0, high=4.0, original=8192)
YARN = dict(kind="yarn", factor=4.0, original=32768)


def close(got, want, terms):
    limit = 4 * 2.0**-24 * terms + 2.0**-11 * np.abs(want) + 2.0**-25
    assert np.isfinite(got).all()
    err = np.abs(got - want)
    assert (err <= np.where(terms > 0, limit, 0)).all(), (err / limit).max()


class Batch:
    """A packed batch over a pool of FP16 pages in any order."""

    def __init__(self, rng, counts, starts, heads, kv, hd, max_pages, before=0, after=0):
        self.counts, self.starts = np.array(counts), np.array(starts)
        self.heads, self.kv, self.hd, self.max_pages = heads, kv, hd, max_pages
        self.rows = before + int(sum(counts)) + after
        self.offsets = before + np.concatenate([[0], np.cumsum(counts)])
        self.x = [fp16_exact(rng.standard_normal((self.rows, h, hd))) for h in (heads, kv, kv)]
        self.lengths = self.starts + self.counts
        n = len(counts)
        self.tiers = np.full((n, max_pages), 255, np.uint8)
        for i, e in enumerate(self.lengths):
            self.tiers[i, :-(-e // P)] = 0
        self.place = rng.permutation(n * max_pages).reshape(n, max_pages)
        self.page = 4 * P * kv * hd
        self.pool = Bytes(count=n * max_pages * self.page)

    def run(self, rope, interleaved=False, offsets=True, v_out=True, tiers=None, strides=(0, 0, 0),
            views=None):
        d = mi().device
        table = (self.pool.address + self.place.astype(np.int64) * self.page)
        tiers = self.tiers if tiers is None else tiers
        self.q_out, self.k_out, self.v_out = (Bytes(count=2 * x.size) for x in self.x)
        for t in (self.q_out, self.k_out, self.v_out):
            t.numel = t.count // 2
        self.on = views or [put(x) for x in self.x]
        words = np.concatenate([tiers.reshape(-1), np.zeros(-tiers.size % 4, np.uint8)]).view(np.int32)
        d.append_batch(*self.on, self.q_out, self.k_out, d.DeviceIndex(table.view(np.int32)),
                       d.DeviceIndex(words), d.DeviceIndex(self.lengths),
                       d.DeviceIndex(self.offsets) if offsets else None, len(self.counts),
                       self.max_pages, self.rows, rope, self.heads, self.kv, self.hd, interleaved,
                       self.v_out if v_out else None, *strides)
        self.got = [t.read().view(np.float16).reshape(x.shape).astype(np.float64)
                    for t, x in zip((self.q_out, self.k_out, self.v_out), self.x)]
        self.pages = self.pool.read().view(np.float16).reshape(-1, 2, P, self.kv, self.hd)
        return self

    def check(self, freq, magnitude, interleaved=False, tiers=None, v_out=True):
        tiers = self.tiers if tiers is None else tiers
        untouched = np.frombuffer(b"\xa5\xa5", np.float16)[0]
        want_pages = np.full(self.pages.shape, untouched)
        wrote = np.zeros(self.rows, bool)
        for s, (n, start) in enumerate(zip(self.counts, self.starts)):
            mine = slice(self.offsets[s], self.offsets[s] + n)
            wrote[mine] = True
            at = start + np.arange(n)
            for x, got in zip(self.x[:2], self.got[:2]):
                close(got[mine], *ragged.turned(x[mine], at, freq, magnitude, interleaved))
            if v_out:
                np.testing.assert_array_equal(self.got[2][mine], self.x[2][mine])
            for r, p in zip(range(mine.start, mine.stop), at):
                if p // P < self.max_pages and tiers[s, p // P] == 0:
                    page = self.place[s, p // P]
                    want_pages[page, 0, p % P] = self.got[1][r]
                    want_pages[page, 1, p % P] = self.x[2][r]
        np.testing.assert_array_equal(self.pages.view(np.uint16), want_pages.view(np.uint16))
        for got in self.got[:3 if v_out else 2]:  # rows of no sequence
            assert (got[~wrote].astype(np.float16) == untouched).all()


@pytest.mark.parametrize("heads,kv,hd,part", [
    (14, 2, 64, 64), (12, 2, 128, 128), (32, 8, 64, 64), (4, 4, 128, 32), (5, 5, 64, 16),
    (3, 1, 80, 80), (7, 1, 18, 18), (2, 2, 6, 4), (40, 1, 64, 0), (3, 3, 96, 48), (2, 1, 128, 126)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(heads, kv, hd, part, interleaved):
    rng = np.random.default_rng(heads + hd + part)
    b = Batch(rng, [3, 0, 1, 40, 0, 33], [0, 5, 31, 60, 0, 31], heads, kv, hd, 4, before=2, after=3)
    rope = None
    if part:
        rope = mi().device.RopeTable(part, 10000.0)
        rope.cover(4 * P)
    announce("append", heads, kv, hd, part, interleaved)
    b.run(rope, interleaved).check(ragged.frequencies(part, 10000.0, None)[0], 1.0, interleaved)


@pytest.mark.parametrize("scaling", [dict(kind="linear", factor=4.0), LLAMA3, YARN,
                                     dict(kind="yarn", factor=2.0, original=4096, fast=16.0, slow=2.0,
                                          magnitude=1.0)])
def test_scaled_angles_at_far_positions(scaling):
    rng = np.random.default_rng(1)
    b = Batch(rng, [2, 17], [130000, 70001], 4, 2, 128, 4096)
    rope = mi().device.RopeTable(128, 5e5, scaling)
    rope.cover(4096 * P)
    announce("scaled", scaling)
    b.run(rope).check(*ragged.frequencies(128, 5e5, scaling))


def test_one_row_each_without_offsets():
    rng = np.random.default_rng(2)
    rope = mi().device.RopeTable(64, 1e6)
    rope.cover(64 * P)
    for n in (1, 2, 7, 300):
        b = Batch(rng, [1] * n, rng.integers(0, 63 * P, n), 14, 2, 64, 64)
        announce("one row each", n)
        b.run(rope, offsets=False, v_out=False).check(ragged.frequencies(64, 1e6, None)[0], 1.0,
                                                      v_out=False)


@pytest.mark.parametrize("batch", [2047, 2048, 2049, 5000])
def test_more_sequences_than_are_held(batch):
    rng = np.random.default_rng(batch)
    counts = rng.integers(0, 3, batch)
    b = Batch(rng, counts, rng.integers(0, 20, batch), 2, 1, 16, 1)
    rope = mi().device.RopeTable(16, 1e4)
    rope.cover(P)
    announce("sequences", batch)
    b.run(rope).check(ragged.frequencies(16, 1e4, None)[0], 1.0)


def test_long_prompts():
    """Rows past a workgroup's, of sequences that begin and end inside them."""
    rng = np.random.default_rng(4)
    b = Batch(rng, [1, 9000, 0, 777, 2], [40, 100, 7, 0, 9000], 6, 2, 64, 290)
    rope = mi().device.RopeTable(64, 5e5, LLAMA3)
    rope.cover(290 * P)
    announce("long")
    b.run(rope).check(*ragged.frequencies(64, 5e5, LLAMA3))


def test_pages_that_are_not_there():
    """Quantised, unread and address-less pages, and positions past the table, take nothing; the
    rows come out turned all the same."""
    rng = np.random.default_rng(5)
    b = Batch(rng, [64, 40, 5], [0, 100, 10], 4, 2, 64, 4)
    tiers = b.tiers.copy()
    tiers[0, 1], tiers[2, 0] = 2, 255
    rope = mi().device.RopeTable(64, 1e4)
    rope.cover(4 * P)
    freq = ragged.frequencies(64, 1e4, None)[0]
    announce("tiers")
    # Sequence 1 ends at 140, past its 128 positions: those turn as the last does.
    b.run(rope, tiers=tiers)
    b.starts = b.starts.copy()
    got = [g.copy() for g in b.got]
    for i in range(2):
        last = slice(64 + 28, 64 + 40)
        close(got[i][last], *ragged.turned(b.x[i][last], np.full(12, 127), freq, 1.0, False))
        b.got[i][last] = ragged.turned(b.x[i][last], np.arange(128, 140), freq, 1.0, False)[0]
    b.check(freq, 1.0, tiers=tiers)


@pytest.mark.parametrize("hd,pad", [(64, 8), (64, 3), (128, 0)])
def test_views_of_one_projection(hd, pad):
    rng = np.random.default_rng(hd + pad)
    heads, kv = 6, 2
    b = Batch(rng, [70, 3], [0, 44], heads, kv, hd, 3)
    width = (heads + 2 * kv) * hd + pad
    fused = np.zeros((b.rows, width))
    cuts = np.cumsum([0, heads * hd, kv * hd, kv * hd])
    for x, lo, hi in zip(b.x, cuts, cuts[1:]):
        fused[:, lo:hi] = x.reshape(b.rows, -1)
    d = mi().device
    base = put(fused)
    views = [d.view(base, int(lo), b.rows * width - int(lo)) for lo in cuts[:3]]
    rope = d.RopeTable(hd, 1e4)
    rope.cover(3 * P)
    announce("fused", hd, pad)
    b.run(rope, strides=(width,) * 3, views=views).check(ragged.frequencies(hd, 1e4, None)[0], 1.0)


def test_the_rope_kernels_bits():
    m = mi()
    d = m.device
    rng = np.random.default_rng(7)
    b = Batch(rng, [50, 20], [0, 300], 12, 2, 128, 16)
    rope = d.RopeTable(128, 1e6)
    rope.cover(16 * P)
    announce("bits")
    b.run(rope)
    at = d.DeviceIndex(np.concatenate([np.arange(50), np.arange(300, 320)]))
    for x, got in zip(b.x[:2], b.got[:2]):
        out = d.empty(x.size)
        d.rope_from_table(put(x), at, rope, out, b.rows, x.shape[1], 128)
        np.testing.assert_array_equal(out.to_numpy().reshape(x.shape), got)


def test_a_captured_append_follows_its_tables():
    m = mi()
    d = m.device
    rng = np.random.default_rng(8)
    b = Batch(rng, [1] * 6, [0, 5, 31, 32, 63, 90], 4, 2, 64, 4)
    rope = d.RopeTable(64, 1e4)
    rope.cover(4 * P)
    freq = ragged.frequencies(64, 1e4, None)[0]
    b.run(rope)  # eager
    lengths = d.DeviceIndex(b.lengths)
    table = d.DeviceIndex((b.pool.address + b.place.astype(np.int64) * b.page).view(np.int32))
    tiers = np.zeros((6, 4), np.uint8)
    tier_words, offsets = d.DeviceIndex(tiers.view(np.int32)), d.DeviceIndex(b.offsets)
    stream = m.Stream()
    graph = m.Graph(stream)
    with graph.capture():
        d.append_batch(*b.on, b.q_out, b.k_out, table, tier_words, lengths, offsets, 6, 4, 6, rope, 4,
                       2, 64, v_out=b.v_out)
    for i in range(4):
        b.starts = rng.integers(0, 4 * P, 6)
        m._h2d(lengths.address, (b.starts + 1).astype(np.int32))
        m._h2d(b.pool.address, np.full(b.pool.count, 0xA5, np.uint8))
        announce("captured append", i)
        graph.launch()
        stream.synchronize()
        b.got = [t.read().view(np.float16).reshape(x.shape).astype(np.float64)
                 for t, x in zip((b.q_out, b.k_out, b.v_out), b.x)]
        b.pages = b.pool.read().view(np.float16).reshape(-1, 2, P, 2, 64)
        b.check(freq, 1.0, tiers=tiers)
