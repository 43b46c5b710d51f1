"""A layer of a ragged batch as a serving loop runs it: rows in 8-bit codes, one
projection to queries, keys and values, the rows turned into paged caches,
causal attention over the prompts, the output projection into the fp32
residual, logits and a token a sequence; then a token more of each, behind its
cache. Eager, captured and on two streams at once.

Every stage is compared with float64 over what the stage before it left on the
device, with the tolerances of the operators' own tests."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from oracle import ragged
from test_gpu_append import LLAMA3, P, close
from test_gpu_int4 import Bytes
from test_gpu_int8 import floats, quantised
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu

HEADS, KV, HD, VOCAB = 6, 2, 64, 5003
HIDDEN, WIDE = HEADS * HD, (HEADS + 2 * KV) * HD
PROMPTS = [5, 33, 0, 1, 200, 64]


def halves_of(t, *shape):
    return t.read().view(np.float16)[:int(np.prod(shape))].reshape(shape).astype(np.float64)


def within(got, want, off, what):
    limit = off + 2.0**-24 * np.abs(want) * 1.001 + 2.0**-11 * (np.abs(want) + off) + 2.0**-25
    assert (np.abs(got - want) <= limit).all(), f"{what}: {(np.abs(got - want) / limit).max()}"


class Layer:
    """The weights, which runs share."""

    def __init__(self, rng):
        def weight(out, n):
            codes, scales = quantised(fp16_exact(rng.standard_normal((out, n)) / np.sqrt(n)))
            return codes, scales, Bytes(codes.view(np.uint8)), floats(scales)

        self.qkv, self.o, self.head = weight(WIDE, HIDDEN), weight(HIDDEN, HIDDEN), weight(VOCAB, HIDDEN)
        self.bias = fp16_exact(rng.standard_normal(WIDE))
        self.bias_on = put(self.bias)
        self.rope = mi().device.RopeTable(HD, 5e5, LLAMA3)
        self.rope.cover(16 * P)


class Step:
    """A step's buffers, as a program keeps them: `counts` rows a sequence behind `starts`."""

    def __init__(self, counts, starts, pages=None, max_pages=16):
        d = mi().device
        self.counts, self.starts, self.batch = np.array(counts), np.array(starts), len(counts)
        self.offsets = np.concatenate([[0], np.cumsum(counts)])
        n = self.rows = int(self.offsets[-1])
        self.lengths, self.max_pages = self.starts + self.counts, max_pages
        page = 4 * P * KV * HD
        self.pool = pages or Bytes(count=self.batch * max_pages * page)
        table = self.pool.address + np.arange(self.batch * max_pages, dtype=np.int64)[::-1] * page
        tiers = np.where(np.arange(max_pages) * P < self.lengths[:, None], 0, 255).astype(np.uint8)
        self.table = d.DeviceIndex(np.ascontiguousarray(table).view(np.int32))
        self.tiers = d.DeviceIndex(np.ascontiguousarray(tiers.reshape(-1)).view(np.int32))
        self.on_lengths, self.on_offsets = d.DeviceIndex(self.lengths), d.DeviceIndex(self.offsets)

        def half(count):
            t = Bytes(count=2 * count)
            t.numel = count
            return t

        self.x, self.fused, self.y = half(n * HIDDEN), half(n * WIDE), half(n * HIDDEN)
        self.q, self.k, self.v = half(n * HIDDEN), half(n * KV * HD), half(n * KV * HD)
        self.codes, self.scales = Bytes(count=n * HIDDEN), Bytes(count=4 * n)
        self.residual = floats(np.zeros((n, HIDDEN), np.float32))
        self.parts = d.empty_f32(max(1, d.attention_packed_partials(self.batch, n, n, HEADS, KV, HD)))
        self.batch_parts = d.empty_f32(d.attention_batch_partials(self.batch, max_pages, HEADS, KV, HD))
        b = self.batch
        self.last, self.last_codes, self.last_scales = half(b * HIDDEN), Bytes(count=b * HIDDEN), Bytes(count=4 * b)
        self.logits, self.tokens = half(b * VOCAB), Bytes(count=4 * b)
        self.scratch = d.empty_f32(d.sample_scratch(b, VOCAB))
        self.uniforms = floats(np.linspace(0.05, 0.95, b))
        self.settings = dict(temperature=np.linspace(0, 2, b).astype(np.float32),
                             top_k=np.array([0, 40, 5, 1000, 0, 1][:b], np.int32),
                             top_p=np.array([1, 0.9, 0.95, 1, 0.5, 0.7][:b], np.float32))
        self.settings_on = {n: Bytes(v.view(np.uint8)) for n, v in self.settings.items()}

    def views(self):
        """The queries, keys and values in the projection's rows."""
        d = mi().device

        class At:
            def __init__(self, of, first):
                self.address, self.numel = of.address + 2 * first, of.numel - first
                self.nbytes, self.of = 2 * self.numel, of

        return [At(self.fused, first) for first in (0, HIDDEN, HIDDEN + KV * HD)]

    def attend(self, layer, prompts):
        d = mi().device
        n = self.rows
        d.quantise_rows_int8(self.x, self.codes, self.scales, n, HIDDEN)
        d.linear_int8(self.codes, self.scales, *layer.qkv[2:], layer.bias_on, self.fused, n, HIDDEN, WIDE)
        d.append_batch(*self.views(), self.q, self.k, self.table, self.tiers, self.on_lengths,
                       self.on_offsets, self.batch, self.max_pages, n, layer.rope, HEADS, KV, HD,
                       False, self.v, WIDE, WIDE, WIDE)
        if prompts:
            d.attention_packed(self.q, self.k, self.v, self.y, self.on_offsets, None, self.batch, n, n,
                               HEADS, KV, HD, partials=self.parts)
        else:
            d.attention_batch(self.q, self.table, self.tiers, self.on_lengths, self.y, self.batch,
                              self.max_pages, HEADS, KV, HD, partials=self.batch_parts)
        d.quantise_rows_int8(self.y, self.codes, self.scales, n, HIDDEN)
        d.linear_int8_accumulate(self.codes, self.scales, *layer.o[2:], self.residual, n, HIDDEN, HIDDEN)

    def choose(self, layer):
        d, b = mi().device, self.batch
        d.quantise_rows_int8(self.last, self.last_codes, self.last_scales, b, HIDDEN)
        d.linear_int8(self.last_codes, self.last_scales, *layer.head[2:], None, self.logits, b, HIDDEN, VOCAB)
        d.sample(self.logits, self.uniforms, self.tokens, b, VOCAB, scratch=self.scratch, **self.settings_on)

    def give(self, x, residual, last):
        m = mi()
        m._h2d(self.x.address, x.astype(np.float16))
        m._h2d(self.residual.address, residual)
        m._h2d(self.last.address, last.astype(np.float16))

    def read(self):
        return [t.read() for t in (self.fused, self.q, self.k, self.v, self.y, self.residual, self.logits,
                                   self.tokens, self.pool)]

    def check(self, layer, x, residual, last, freq, magnitude, cached=None):
        n = self.rows
        fused = halves_of(self.fused, n, WIDE)
        want, off = ragged.linear_int8(*ragged.quantise_rows(x), *layer.qkv[:2])
        within(fused, want + layer.bias, off, "qkv")
        at = np.concatenate([s + np.arange(c) for s, c in zip(self.starts, self.counts)]).astype(int)
        parts = np.split(fused, [HIDDEN, HIDDEN + KV * HD], 1)
        q, k, v = (halves_of(t, n, h, HD) for t, h in ((self.q, HEADS), (self.k, KV), (self.v, KV)))
        close(q, *ragged.turned(parts[0].reshape(q.shape), at, freq, magnitude, False))
        close(k, *ragged.turned(parts[1].reshape(k.shape), at, freq, magnitude, False))
        np.testing.assert_array_equal(v, parts[2].reshape(v.shape))
        y = halves_of(self.y, n, HEADS, HD)
        keys, values = [], []
        for s in range(self.batch):
            mine = slice(self.offsets[s], self.offsets[s + 1])
            before = cached[s] if cached else (k[:0], v[:0])
            keys.append(np.concatenate([before[0], k[mine]]))
            values.append(np.concatenate([before[1], v[mine]]))
        ok = np.concatenate([[0], np.cumsum([len(r) for r in keys])])
        want, bound, terms = ragged.packed_attention(q, np.concatenate(keys), np.concatenate(values),
                                                     self.offsets, ok)
        limit = bound + (2.0**-11 + 2.0**-20) * terms + 2.0**-11 * np.abs(want) + 2.0**-25
        assert (np.abs(y - want) <= limit).all()
        want, off = ragged.linear_int8(*ragged.quantise_rows(y.reshape(n, HIDDEN)), *layer.o[:2])
        got = self.residual.read().view(np.float32).reshape(n, HIDDEN).astype(np.float64)
        want = want + residual
        assert (np.abs(got - want) <= off + 2.0**-24 * (np.abs(want) + off) + 2.0**-149).all()
        logits = halves_of(self.logits, self.batch, VOCAB)
        within(logits, *ragged.linear_int8(*ragged.quantise_rows(last), *layer.head[:2]), "logits")
        tokens = self.tokens.read().view(np.int32)
        for i in range(self.batch):
            token, border = ragged.sample(logits[i], float(np.float32(np.linspace(0.05, 0.95, self.batch)[i])),
                                          *(v[i].item() for v in self.settings.values()))
            assert border < 1e-9 or tokens[i] == token
        return list(zip(keys, values))


def given(rng, step):
    return (fp16_exact(rng.standard_normal((step.rows, HIDDEN))),
            rng.standard_normal((step.rows, HIDDEN)).astype(np.float32),
            fp16_exact(3 * rng.standard_normal((step.batch, HIDDEN))))


def test_prompts_then_tokens():
    rng = np.random.default_rng(0)
    layer = Layer(rng)
    freq = ragged.frequencies(HD, 5e5, LLAMA3)
    prompts = Step(PROMPTS, [0] * 6)
    x = given(rng, prompts)
    prompts.give(*x)
    announce("prompts")
    prompts.attend(layer, True)
    prompts.choose(layer)
    cached = prompts.check(layer, *x, *freq)
    ends = np.array(PROMPTS)
    for i in range(3):
        tokens = Step([1] * 6, ends, prompts.pool)
        x = given(rng, tokens)
        tokens.give(*x)
        announce("tokens", i)
        tokens.attend(layer, False)
        tokens.choose(layer)
        cached = tokens.check(layer, *x, *freq, cached)
        ends = ends + 1


def test_a_captured_step_and_the_eager_one():
    """One graph, replayed over new rows, with eager steps of another batch between."""
    m = mi()
    rng = np.random.default_rng(1)
    layer = Layer(rng)
    freq = ragged.frequencies(HD, 5e5, LLAMA3)
    captured, eager = Step(PROMPTS, [0] * 6), Step([40, 1, 7], [0] * 3)
    stream = m.Stream()
    graph = m.Graph(stream)
    with graph.capture():
        captured.attend(layer, True)
        captured.choose(layer)
    for i in range(4):
        x = given(rng, captured)
        captured.give(*x)
        announce("replay", i)
        graph.launch()
        stream.synchronize()
        captured.check(layer, *x, *freq)
        x = given(rng, eager)
        eager.give(*x)
        eager.attend(layer, True)
        eager.choose(layer)
        m.synchronize()
        eager.check(layer, *x, *freq)


def test_two_streams_at_once():
    """Each with buffers of its own: the bits of one after another."""
    m = mi()
    rng = np.random.default_rng(2)
    layer = Layer(rng)
    lanes = [Step(PROMPTS, [0] * 6) for _ in range(2)]
    x = given(rng, lanes[0])
    alone = Step(PROMPTS, [0] * 6)
    alone.give(*x)
    alone.attend(layer, True)
    alone.choose(layer)
    m.synchronize()
    want = alone.read()
    streams = [m.Stream(), m.Stream()]
    announce("two streams")
    for lane in lanes:
        lane.give(*x)
    m.synchronize()
    for i in range(10):
        for lane, stream in zip(lanes, streams):
            m.set_stream(stream)
            lane.attend(layer, True)
            lane.choose(layer)
    m.set_stream(None)
    for stream in streams:
        stream.synchronize()
    for lane in lanes:
        got = lane.read()
        for i, (a, b) in enumerate(zip(got, want)):
            if i != 5:  # (the residual, to which ten steps were added)
                np.testing.assert_array_equal(a, b)
    np.testing.assert_array_equal(*(lane.read()[5] for lane in lanes))
