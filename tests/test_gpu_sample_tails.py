"""Rows of one logit far above a flat tail that weighs little each and, a hundred
thousand and more of them, something together: borders inside the tail, and tokens
from it.

A token is right where its place by index meets the uniform's share within what is
promised: the tail that top_p keeps to 2^-26 of the weights before it, the share to
2^-26 of those kept. Uniforms are next to one, 2^-24 apart, so that they reach the
tail; a tail of 2^20 logits 26 nats down is 2^-17.5 of the row."""

import numpy as np
import pytest

from conftest import announce
from oracle import ragged
from test_gpu_sample import choose

pytestmark = pytest.mark.gpu

STEP = 2.0**-24


def check(row, token, u, t, top_k, top_p, what):
    l = row.astype(np.float64)
    order = np.argsort(-l, kind="stable")
    if top_k:
        order = order[:top_k]
    w = np.exp((l[order] - l[order[0]]) / t)
    upto = np.cumsum(w)
    slack = 2.0**-26 * upto[-1] if top_p < 1 else 0.0
    least = most = len(w)
    if top_p < 1:
        least = min(len(w), int(np.searchsorted(upto, top_p * upto[-1] - slack)) + 1)
        most = min(len(w), int(np.searchsorted(upto, top_p * upto[-1] + slack)) + 1)
    assert token in order[:most], f"{what}: {token} is not kept"
    kept = order[:most]
    by_index = np.argsort(kept)
    reach = np.cumsum(w[:most][by_index])
    at = int(np.flatnonzero(kept[by_index] == token)[0])
    near = 2.0**-26 * upto[most - 1]
    low, high = u * upto[least - 1] - near, u * upto[most - 1] + 2 * slack + near
    before = reach[at] - w[by_index[at]]
    assert reach[at] >= low and before <= high, (
        f"{what}: token {token} is from {before:.9g} to {reach[at]:.9g}, the share between {low:.9g} and {high:.9g}")


def run(row, t, steps, what, top_k=0, top_p=1.0):
    row = np.asarray(row, np.float32)
    u = (1.0 - STEP * np.asarray(steps)).astype(np.float32)
    announce("tail", what, top_k, top_p)
    settings = dict(temperature=t)
    if top_k:
        settings["top_k"] = top_k
    if top_p < 1:
        settings["top_p"] = top_p
    got = choose(np.repeat(row[None], len(u), 0), u, **settings)
    for token, mine in zip(got, u):
        check(row, token, float(mine), t, top_k, float(np.float32(top_p)), f"{what} {top_k} {top_p} u {mine!r}")


def borders(tail, vocab):
    """top_p's of some of a tail that is `tail` of the row, in steps of STEP."""
    whole = int(tail / STEP)
    return [0, *(j for j in (whole // 4, whole // 2, whole - 1) if j > 0)]


@pytest.mark.parametrize("vocab", [151936, 1 << 20])
@pytest.mark.parametrize("nats", [20.0, 26.0, 26.5, 26.9])
def test_a_flat_tail(vocab, nats):
    rng = np.random.default_rng(vocab + int(10 * nats))
    row = np.zeros(vocab)
    row[rng.integers(0, vocab)] = nats
    tail = vocab * np.exp(-nats)
    steps = np.unique(np.linspace(1, tail / STEP * 0.9, 7).astype(int))
    for top_k in (0, vocab // 2, vocab - 1):
        for j in borders(tail * (top_k or vocab) / vocab, vocab):
            run(row, 1.0, steps, f"flat {vocab} {nats}", top_k, 1.0 - STEP * j)


def test_a_tail_of_different_weights():
    rng = np.random.default_rng(1)
    vocab = 1 << 19
    row = rng.uniform(0, 0.05, vocab)
    row[rng.integers(0, vocab)] = 26.2
    tail = vocab * np.exp(-26.175)
    steps = np.unique(np.linspace(1, tail / STEP * 0.9, 7).astype(int))
    for top_k in (0, vocab // 3):
        for j in borders(tail * (top_k or vocab) / vocab, vocab):
            run(row, 1.0, steps, "different", top_k, 1.0 - STEP * j)


@pytest.mark.parametrize("ulps", [6, 7])
def test_temperatures_that_put_a_row_into_one_bucket(ulps):
    """Logits of 2^26 temperatures: neighbouring values are four nats apart."""
    vocab, t = 1 << 20, 2.0**-20
    row = np.full(vocab, 64.0 - ulps * 2.0**-18)
    row[777777] = 64.0
    tail = vocab * np.exp(-4.0 * ulps)
    steps = np.unique(np.linspace(1, tail / STEP * 0.9, 7).astype(int))
    for top_k in (0, vocab // 2):
        for j in borders(tail * (top_k or vocab) / vocab, vocab):
            run(row, t, steps, f"one bucket {ulps}", top_k, 1.0 - STEP * j)


@pytest.mark.parametrize("t", [1.4e-45, 1e-40])
def test_temperatures_next_to_zero(t):
    """Buckets of a million nats each, whose logits weigh nothing, and of less."""
    rng = np.random.default_rng(2)
    row = rng.uniform(0, 1e-36, 50000).astype(np.float32)
    u = np.array([0.0, 0.3, 0.999], np.float32)
    t32 = float(np.float32(t))
    for settings in (dict(), dict(top_k=25000), dict(top_k=40000, top_p=0.9), dict(top_p=0.5), dict(min_p=0.1)):
        announce("next to zero", t, settings)
        got = choose(np.repeat(row[None], len(u), 0), u, temperature=t, **settings)
        exact = {name: v if name == "top_k" else float(np.float32(v)) for name, v in settings.items()}
        want = [ragged.sample(row, float(mine), temperature=t32, **exact) for mine in u]
        assert all(border > 2.0**-25 or mine == 0 for (_, border), mine in zip(want, u))
        np.testing.assert_array_equal(got, [token for token, _ in want], err_msg=f"{t} {settings}")
