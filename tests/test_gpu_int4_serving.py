"""The 4-bit projections, the prompt's window attention and the batch's token
attention as a server would use them: a stack of layers whose quantised
projections feed window attention and fill the cache manager's pages for each
prompt, then step all sequences a token at a time. Every stage is held against
float64 of what the device gave it, with the tolerances of the stages' own
tests."""

import numpy as np
import pytest

from conftest import announce, assert_attention_close, fp16_exact
from oracle import windows
from test_gpu_batch import LAYERS, P, as_read
from test_gpu_int4 import Bytes, Int4, check_half, weight
from test_gpu_kv_pages import mi, pages_for, put
from test_gpu_window import check as check_window

pytestmark = pytest.mark.gpu

WINDOW, SINKS, GROUP, EPS = 40, 3, 64, 1e-6


class Layer:
    """q, k, v and output projections, quantised on the device."""

    def __init__(self, rng, heads, kv, hd):
        d = mi().device
        hidden = heads * hd
        self.norm = put(fp16_exact(1.0 + 0.1 * rng.standard_normal(hidden)))
        self.parts = {}
        for name, out, n_in in (("q", hidden, hidden), ("k", kv * hd, hidden),
                                ("v", kv * hd, hidden), ("o", hidden, hidden)):
            w = weight(rng, out, n_in)
            want = Int4(w, GROUP)
            groups = out * (n_in // GROUP)
            want.on = (Bytes(count=out * n_in // 2), Bytes(count=2 * groups),
                       Bytes(count=2 * groups))
            d.quantise_int4(put(w), *want.on, GROUP, n_in, out)
            self.parts[name] = (want, out, n_in)
        self.bias = put(fp16_exact(rng.standard_normal(hidden)))

    def project(self, name, x, rows, bias=None):
        """The projection on the device, held against float64 of its input."""
        d = mi().device
        w, out, n_in = self.parts[name]
        y = d.empty(rows * out)
        d.linear_int4(x, *w.on, GROUP, bias, y, rows, n_in, out)
        host = x.to_numpy().astype(np.float64).reshape(rows, n_in)
        full = host @ w.w64.T + (0.0 if bias is None else bias.to_numpy().astype(np.float64))
        check_half(y.to_numpy().astype(np.float64).reshape(rows, out), full,
                   w.bound(host) + (0.0 if bias is None else 2.0**-24 * np.abs(full)))
        return y

    def add_output(self, x, stream, rows):
        d = mi().device
        w, out, n_in = self.parts["o"]
        before = stream.to_numpy().astype(np.float64).reshape(rows, out)
        d.linear_int4_accumulate(x, *w.on, GROUP, stream, rows, n_in, out)
        host = x.to_numpy().astype(np.float64).reshape(rows, n_in)
        want = host @ w.w64.T
        err = np.abs(stream.to_numpy().reshape(rows, out) - (before + want))
        assert (err <= w.bound(host) + 2.0**-23 * (np.abs(before) + np.abs(want))).all()


@pytest.mark.parametrize("seals", [True, False])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (6, 2, 128)])
def test_prompts_then_tokens_of_a_batch(heads, kv, hd, seals):
    m = mi()
    d = m.device
    rng = np.random.default_rng(heads + hd + seals)
    hidden, width = heads * hd, kv * hd
    layers = [Layer(rng, heads, kv, hd) for _ in range(LAYERS)]
    lengths = [1, 45, 96, 31]
    caches, keys, values, last = [], [], [], []

    def normed(layer, stream, rows):
        x = d.empty(rows * hidden)
        d.rmsnorm_f32(stream, layer.norm, x, rows, hidden, EPS)
        return x

    rows_of = lambda t, n: t.to_numpy().astype(np.float64).reshape(n, kv, hd)  # noqa: E731
    for n in lengths:
        tier_map = [[(1, 0, 3, 2)[(l + p) % 4] for p in range(n // P + 2)] for l in range(LAYERS)]
        caches.append(pages_for(P, kv, hd, 0, tier_map if seals else None, seals))
        keys.append([None] * LAYERS)
        values.append([None] * LAYERS)
        stream = d.upload_f32(rng.standard_normal((n, hidden)).astype(np.float32))
        caches[-1][1].reserve(n)
        for l, layer in enumerate(layers):
            announce("prompt", heads, kv, hd, seals, n, l)
            x = normed(layer, stream, n)
            q = layer.project("q", x, n, layer.bias)
            k, v = layer.project("k", x, n), layer.project("v", x, n)
            out = d.empty(n * hidden)
            parts = d.empty_f32(max(1, d.attention_window_partials(n, n, heads, kv, hd, WINDOW,
                                                                   SINKS)))
            d.attention_window(q, k, v, out, n, n, heads, kv, hd, WINDOW, SINKS, partials=parts)
            keys[-1][l], values[-1][l] = rows_of(k, n), rows_of(v, n)
            check_window(out.to_numpy().astype(np.float64).reshape(n, heads, hd),
                         q.to_numpy().astype(np.float64).reshape(n, heads, hd), keys[-1][l],
                         values[-1][l], WINDOW, SINKS, f"prompt of {n}")
            caches[-1][1].store(l, k, v, 0, n)
            layer.add_output(out, stream, n)
        last.append(stream.to_numpy().reshape(n, hidden)[-1])

    batch = len(lengths)
    x0 = np.stack(last)
    for step in range(3):
        stream = d.upload_f32(x0.astype(np.float32))
        lengths = [n + 1 for n in lengths]
        for (_, cache), n in zip(caches, lengths):
            cache.reserve(n)
        pages = -(-max(lengths) // P)
        for l, layer in enumerate(layers):
            announce("token", heads, kv, hd, seals, step, l)
            x = normed(layer, stream, batch)
            q = layer.project("q", x, batch, layer.bias)
            k, v = layer.project("k", x, batch), layer.project("v", x, batch)
            kh, vh = rows_of(k, batch), rows_of(v, batch)
            for i, (_, cache) in enumerate(caches):
                cache.store(l, d.view(k, i * width, width), d.view(v, i * width, width),
                            lengths[i] - 1, 1)
                keys[i][l] = np.concatenate([keys[i][l], kh[i:i + 1]])
                values[i][l] = np.concatenate([values[i][l], vh[i:i + 1]])
            out = d.empty(batch * hidden)
            parts = d.empty_f32(max(1, d.attention_batch_partials(batch, pages, heads, kv, hd,
                                                                  WINDOW, SINKS)))
            own = (k, v) if seals else (None, None)
            d.attention_caches([c for _, c in caches], lengths, l, q, out, heads, kv, hd, *own,
                               WINDOW, SINKS, partials=parts)
            got = out.to_numpy().reshape(batch, heads, hd)
            qh = q.to_numpy().astype(np.float64).reshape(batch, heads, hd)
            for i, (alloc, cache) in enumerate(caches):
                rows = as_read(alloc, cache, l, np.stack([keys[i][l]] * LAYERS),
                               np.stack([values[i][l]] * LAYERS), kv, hd, seals)
                want, _, bound = windows.paged_token(qh[i], *rows[:2], lengths[i], rows[2], WINDOW,
                                                     SINKS, P)
                assert_attention_close(got[i], want, f"sequence {i} step {step}", bound)
            layer.add_output(out, stream, batch)
        x0 = stream.to_numpy().reshape(batch, hidden)
