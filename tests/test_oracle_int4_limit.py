"""The projections' limit by steps (oracle.int4.linear_limit): what it must
hold, an fp32 sum in groups, and what it must catch: a lost run or group of
inputs, and a scale or zero of the next group, at inputs of thousands."""

import numpy as np
import pytest

from conftest import fp16_exact
from oracle import int4

SIZES = [(3, 40, 896, 32), (1, 60, 8960, 128), (4, 60, 8960, 128), (1, 33, 24608, 32),
         (5, 40, 24608, 32), (3, 40, 4096, 64)]


def weight(rng, out, n_in):
    w = rng.standard_normal((out, n_in)) * n_in**-0.5
    w[:, rng.random(n_in) < 0.02] *= 8
    return fp16_exact(w)


def parts(rows, out, n_in, group):
    rng = np.random.default_rng(rows + out + n_in)
    codes, scales, zeros = int4.quantise(weight(rng, out, n_in), group)
    x = fp16_exact(rng.standard_normal((rows, n_in)))
    return x, codes, scales, zeros


def allowed(x, codes, scales, zeros, group):
    """The limit with the half step of an fp16 output, as the device's tests have it."""
    want = x @ int4.weight64(codes, scales, zeros, group).T
    return want, int4.linear_limit(x, codes, scales, zeros, group) + 2.0**-11 * np.abs(want) + 2.0**-25


@pytest.mark.parametrize("rows,out,n_in,group", SIZES)
def test_sums_in_fp32_stay_within_it(rows, out, n_in, group):
    """Term by term in fp32, group by group: the longest chains there are."""
    x, codes, scales, zeros = parts(rows, out, n_in, group)
    x32, y = x.astype(np.float32), np.zeros((rows, out), np.float32)
    for g in range(n_in // group):
        dot, total = np.zeros((rows, out), np.float32), np.zeros((rows, 1), np.float32)
        for i in range(g * group, (g + 1) * group):
            dot += x32[:, i:i + 1] * codes[:, i].astype(np.float32)
            total += x32[:, i:i + 1]
        s, z = scales[:, g].astype(np.float32), zeros[:, g].astype(np.float32)
        y += z * total
        y += s * dot
    want, _ = allowed(x, codes, scales, zeros, group)
    limit = int4.linear_limit(x, codes, scales, zeros, group)
    assert (np.abs(y - want) <= limit).all()


@pytest.mark.parametrize("rows,out,n_in,group", SIZES)
def test_what_is_lost_or_misplaced_passes_it(rows, out, n_in, group):
    x, codes, scales, zeros = parts(rows, out, n_in, group)
    want, limit = allowed(x, codes, scales, zeros, group)
    w = int4.weight64(codes, scales, zeros, group)

    def caught(change):
        wrong = w.copy()
        change(wrong)
        return (np.abs(x @ wrong.T - want) > limit).any()

    def lose(run):
        def change(wrong):
            wrong[:, run] = 0.0
        return change

    def next_group_s(array):
        other = array.copy()
        other[:, -2] = array[:, -1]
        return other

    assert caught(lose(slice(n_in - 32, n_in))), "the last 32 inputs"
    assert caught(lose(slice(64, 96))), "32 inputs"
    assert caught(lose(slice(n_in - group, n_in))), "the last group"
    for s, z in ((next_group_s(scales), zeros), (scales, next_group_s(zeros))):
        wrong = int4.weight64(codes, s, z, group)
        assert (np.abs(x @ wrong.T - want) > limit).any(), "the next group's scale or zero"
    flipped = codes.copy()
    flipped[:, -group:] = flipped[:, -group:][:, ::-1]
    wrong = int4.weight64(flipped, scales, zeros, group)
    assert (np.abs(x @ wrong.T - want) > limit).any(), "a group turned around"
