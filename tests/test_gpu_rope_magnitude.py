"""The key bias turned by a RopeTable whose cos and sin have a magnitude (a YaRN
scaling's): once in every attention that takes a table, the same key for a decode
and a prompt; against float64 over the completed keys."""

import numpy as np
import pytest

from conftest import announce, assert_attention_close, fp16_exact
from oracle import attention as att
from oracle import ragged
from test_gpu_kv_pages import mi, normal, pages_for, put, store_in_runs

pytestmark = pytest.mark.gpu

P = 32
THETA = 1e6
SCALINGS = [dict(kind="yarn", factor=4.0, original=32768),
            dict(kind="yarn", factor=8.0, original=64, magnitude=2.5),
            dict(kind="yarn", factor=4.0, original=32768, magnitude=0.5),
            dict(kind="llama3", factor=32.0, low=1.0, high=4.0, original=8192)]


def inputs(seed, seq, seq_q, heads, kv, hd):
    rng = np.random.default_rng(seed)
    return (normal(rng, seq_q, heads, hd), fp16_exact(0.3 * rng.standard_normal((seq, kv, hd))),
            normal(rng, seq, kv, hd), fp16_exact(2 * rng.standard_normal((kv, hd))))


def completed(k, bias, scaling):
    f, magnitude = ragged.frequencies(k.shape[2], THETA, scaling)
    rows = np.broadcast_to(bias, k.shape)
    return k.astype(np.float64) + ragged.turned(rows, np.arange(len(k)), f, magnitude, False)[0]


def check(got, q, k, v, bias, scaling, what):
    whole = completed(k, bias, scaling)
    want, w = att.attention64(q, whole, v)
    assert_attention_close(got.reshape(q.shape), want, what, att.attention_bound(q, whole, v, w))


def table(hd, scaling, positions):
    rope = mi().device.RopeTable(hd, THETA, scaling)
    rope.cover(positions)
    return rope


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("heads,kv,hd,seq,seq_q", [
    (14, 2, 64, 99, 1), (12, 2, 128, 300, 1), (12, 2, 128, 20, 1), (32, 8, 64, 2081, 1),  # a decode's
    (14, 2, 64, 99, 7), (12, 2, 128, 130, 40), (32, 8, 64, 400, 170),                     # a prompt's
    (6, 2, 48, 70, 1), (6, 2, 48, 70, 3)])                                                # any other
def test_fp16_pages(scaling, heads, kv, hd, seq, seq_q):
    d = mi().device
    q, k, v, bias = inputs(seq + hd, seq, seq_q, heads, kv, hd)
    alloc, cache = pages_for(P, kv, hd, 0)
    store_in_runs(cache, 0, k, v, [seq])
    rope, out = table(hd, scaling, seq), d.empty(q.size)
    announce("magnitude", scaling, heads, kv, hd, seq, seq_q)
    cache.attention(0, put(q), put(bias), rope, out, seq_q, seq, heads, kv, hd, None, None, None, None)
    check(out.to_numpy(), q, k, v, bias, scaling, "FP16 pages")


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128)])
def test_a_sealing_cache_and_a_length_on_the_device(scaling, heads, kv, hd):
    d = mi().device
    seq = 5 * P + 11
    q, k, v, bias = inputs(hd, seq, 1, heads, kv, hd)
    alloc, cache = pages_for(P, kv, hd, 0, always_seal=True)
    store_in_runs(cache, 0, k, v, [seq - 1, 1])
    rope = table(hd, scaling, seq)
    on, own = (put(q), put(bias)), (put(k[-1:]), put(v[-1:]))
    eager, stepped = d.empty(q.size), d.empty(q.size)
    announce("magnitude sealed", scaling, heads, kv, hd)
    cache.attention(0, *on, rope, eager, 1, seq, heads, kv, hd, *own, None, None)
    cache.attention_at(0, *on, rope, stepped, d.DeviceIndex([seq]), seq, heads, kv, hd, *own)
    for out in (eager, stepped):
        check(out.to_numpy(), q, k, v, bias, scaling, "sealed")
