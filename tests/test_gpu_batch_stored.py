"""A batch's token attention over caches whose last store was not one row: a
prompt of several pages at once, a chunk that begins inside a page, earlier
positions of a page that is still being filled, rows stored by steps whose
position is on the device; and the positions whose page's rows a sealing cache
no longer holds as they were stored, which are refused. Against float64, with
the attention outputs' gate."""

import numpy as np
import pytest

from conftest import announce, assert_attention_close, fp16_exact
from oracle import windows
from test_gpu_batch import LAYERS, P, as_read, outliers
from test_gpu_kv_pages import mi, pages_for, put

pytestmark = pytest.mark.gpu


class Stored:
    """A KVPages whose rows come in stores of the given ends."""

    def __init__(self, rng, kv, hd, ends, seals=True):
        n = ends[-1]
        self.kv, self.hd, self.seals = kv, hd, seals
        tier_map = [[(1, 0, 3, 2)[(l + p) % 4] for p in range(n // P + 3)] for l in range(LAYERS)]
        self.alloc, self.cache = pages_for(P, kv, hd, 0, tier_map if seals else None, seals)
        self.k = outliers(rng.standard_normal((LAYERS, n + 2 * P, kv, hd)))
        self.v = fp16_exact(rng.standard_normal((LAYERS, n + 2 * P, kv, hd)))
        self.end = 0
        for end in ends:
            self.store(end)

    def store(self, end):
        self.cache.reserve(end)
        for l in range(LAYERS):
            rows = slice(self.end, end)
            self.cache.store(l, put(self.k[l, rows]), put(self.v[l, rows]), self.end, end - self.end)
        self.end = end

    def want(self, q, layer, seq_k):
        rk, rv, unread = as_read(self.alloc, self.cache, layer, self.k[:, :seq_k],
                                 self.v[:, :seq_k], self.kv, self.hd, self.seals)
        return windows.paged_token(q, rk, rv, seq_k, unread, 0, 0, P)


def attend(held, lengths, q, layer):
    d = mi().device
    heads, hd = q.shape[1:]
    kv, n = held[0].kv, len(held)
    own = [put(np.stack([getattr(h, x)[layer, max(s, 1) - 1] for h, s in zip(held, lengths)]))
           for x in "kv"]
    out = d.empty(n * heads * hd)
    d.attention_caches([h.cache for h in held], lengths, layer, put(q), out, heads, kv, hd, *own)
    return out.to_numpy().reshape(n, heads, hd)


def check(held, lengths, q, layer, what):
    got = attend(held, lengths, q, layer)
    for i, (h, n) in enumerate(zip(held, lengths)):
        out, _, bound = h.want(q[i], layer, n)
        assert_attention_close(got[i], out, f"{what} {n}", bound)


@pytest.mark.parametrize("seals", [True, False])
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128)])
def test_the_last_token_of_a_prompt_stored_at_once(heads, kv, hd, seals):
    rng = np.random.default_rng(heads + seals)
    ends = [(5,), (33,), (63,), (97,), (200,), (20, 90), (20, 31), (64, 65), (10, 130, 131)]
    held = [Stored(rng, kv, hd, e, seals) for e in ends]
    q = fp16_exact(rng.standard_normal((len(held), heads, hd)))
    for layer in range(LAYERS):
        announce("caches after prompts", heads, kv, hd, seals, layer)
        check(held, [e[-1] for e in ends], q, layer, "prompt")


def test_earlier_positions_of_the_page_being_filled():
    """One cache at several positions of its open page, and the row that completes it."""
    rng = np.random.default_rng(3)
    held = Stored(rng, 2, 64, (70, 95))
    q = fp16_exact(rng.standard_normal((4, 14, 64)))
    announce("one cache four times")
    check([held] * 4, [65, 70, 71, 95], q, 0, "position")
    held.store(96)
    announce("the page's last row")
    check([held] * 4, [65, 80, 95, 96], q, 1, "position of a page just sealed")


def test_positions_whose_page_s_rows_are_not_held_are_refused():
    rng = np.random.default_rng(4)
    q = fp16_exact(rng.standard_normal((1, 14, 64)))
    for ends, refused, then in (((64,), 64, 65), ((200,), 100, 201), ((20, 64), 64, 65),
                                ((97,), 96, 98), ((40,), 42, 41)):
        held = Stored(rng, 2, 64, ends)
        if refused > ends[-1]:
            held.cache.reserve(refused)
        announce("refused", ends, refused)
        with pytest.raises(ValueError, match="as they were stored"):
            attend([held], [refused], q, 0)
        held.store(then)
        check([held], [then], q, 0, "after one more row")


def test_rows_stored_by_steps_on_the_device():
    """store_at and stored_on_device, before and after the host is told how far they went."""
    d = mi().device
    rng = np.random.default_rng(5)
    held = Stored(rng, 2, 64, (62,))
    q = fp16_exact(rng.standard_normal((1, 14, 64)))
    for end in range(63, 68):
        held.cache.reserve(end)
        position = d.DeviceIndex(np.array([end - 1], np.int32))
        for l in range(LAYERS):
            held.cache.store_at(l, put(held.k[l, end - 1]), put(held.v[l, end - 1]), position)
        held.end = end
        announce("steps", end)
        check([held], [end], q, 0, "step")
        held.cache.stored_on_device(end)
        check([held], [end], q, 1, "step recorded")
    with pytest.raises(ValueError, match="as they were stored"):
        attend([held], [40], q, 0)


def test_a_page_s_first_token_needs_no_rows_before_it():
    rng = np.random.default_rng(6)
    held = Stored(rng, 2, 64, (200,))
    q = fp16_exact(rng.standard_normal((3, 14, 64)))
    announce("first tokens")
    check([held] * 3, [1, 33, 193], q, 0, "a page's first token")


@pytest.mark.parametrize("offset", [1, 4])
def test_own_rows_on_any_alignment(offset):
    """keys and values as views that begin between 16-byte lines."""
    d = mi().device
    rng = np.random.default_rng(offset)
    heads, kv, hd = 12, 2, 128
    held = [Stored(rng, kv, hd, e) for e in ((70,), (63, 64), (97,))]
    lengths = [70, 64, 97]
    q = fp16_exact(rng.standard_normal((3, heads, hd)))
    rows = [np.stack([getattr(h, x)[0, n - 1] for h, n in zip(held, lengths)]).reshape(-1)
            for x in "kv"]
    buffers = [put(np.concatenate([np.full(offset, np.nan), r])) for r in rows]
    out = d.empty(3 * heads * hd)
    announce("own rows at", offset)
    d.attention_caches([h.cache for h in held], lengths, 0, put(q), out, heads, kv, hd,
                       *(d.view(b, offset, 3 * kv * hd) for b in buffers))
    got = out.to_numpy().reshape(3, heads, hd)
    for i, (h, n) in enumerate(zip(held, lengths)):
        want, _, bound = h.want(q[i], 0, n)
        assert_attention_close(got[i], want, f"offset {offset} {n}", bound)
