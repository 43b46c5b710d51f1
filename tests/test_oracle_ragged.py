"""The ragged batch's oracle against closed forms, and the library's frequencies
against it."""

import numpy as np
import pytest

from oracle import attention as att
from oracle import ragged

LLAMA3 = dict(kind="llama3", factor=32.0, low=1.0, high=4.0, original=8192)


@pytest.mark.parametrize("scaling", [
    None, dict(kind="linear", factor=4.0), LLAMA3, dict(LLAMA3, factor=8.0, original=500),
    dict(kind="yarn", factor=4.0, original=32768), dict(kind="yarn", factor=16.0, original=300),
    dict(kind="yarn", factor=2.0, original=4096, fast=16.0, slow=2.0, magnitude=1.5)])
@pytest.mark.parametrize("part,theta", [(64, 5e5), (128, 1e6), (16, 1e4), (2, 1e4)])
def test_frequencies(part, theta, scaling):
    from microinfer import _microinfer as m
    got, magnitude = m.device.rope_frequencies(part, theta, scaling)
    want, factor = ragged.frequencies(part, theta, scaling)
    np.testing.assert_allclose(got, want, rtol=1e-13)
    assert magnitude == pytest.approx(factor, rel=1e-15)


def test_llama3_keeps_fast_pairs_and_slows_the_rest():
    f, _ = ragged.frequencies(64, 5e5, None)
    g, _ = ragged.frequencies(64, 5e5, LLAMA3)
    wave = 2 * np.pi / f
    assert (g[wave < 8192 / 4] == f[wave < 8192 / 4]).all()
    assert np.allclose(g[wave > 8192], f[wave > 8192] / 32)
    between = (wave > 8192 / 4) & (wave < 8192)
    assert between.any() and (g[between] < f[between]).all() and (g[between] > f[between] / 32).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_turned(interleaved):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 3, 12))
    f, _ = ragged.frequencies(8, 100.0, None)
    at = np.array([0, 1, 7, 100, 3])
    y, terms = ragged.turned(x, at, f, 1.0, interleaved)
    np.testing.assert_array_equal(y[0], x[0])
    np.testing.assert_array_equal(y[..., 8:], x[..., 8:])
    assert (terms[..., 8:] == 0).all()
    for j in range(4):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + 4)
        z = (x[..., a] + 1j * x[..., b]) * np.exp(1j * at * f[j])[:, None]
        np.testing.assert_allclose(y[..., a] + 1j * y[..., b], z)


def test_packed_attention_is_each_prompt_s():
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((20, h, 8)) for h in (4, 2, 2))
    oq, ok = np.array([1, 6, 6, 9]), np.array([2, 13, 15, 16])
    out, _, _ = ragged.packed_attention(q, k, v, oq, ok)
    assert np.isnan(out[0]).all() and np.isnan(out[9:]).all()
    np.testing.assert_allclose(out[1:6], att.attention64(q[1:6], k[2:13], v[2:13])[0])
    assert (out[6:8] == 0).all()  # three queries of one key
    np.testing.assert_allclose(out[8], np.repeat(v[15], 2, axis=0))


def test_rows_in_bytes():
    x = np.array([[0, 0, 0], [1, -2, 0.5], [127, 0.5, 1.5], [np.inf, 1, 2]], np.float16)
    codes, scale = ragged.quantise_rows(x)
    assert codes.tolist() == [[0, 0, 0], [64, -127, 32], [127, 0, 2], [0, 0, 0]]
    assert scale[0] == 0 and scale[1] == np.float32(2) / np.float32(127) and np.isnan(scale[3])
    y, off = ragged.linear_int8(codes[1:3], scale[1:3], codes[1:3], scale[1:3])
    assert y[1, 1] == 127 * 127 + 4 and (off < 1e-6 * np.abs(y)).all()


def test_sample_by_hand():
    l = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    pick = lambda u, **s: ragged.sample(l, u, **s)[0]  # noqa: E731
    assert [pick(u) for u in (0.0, 0.05, 0.11, 0.49, 0.51, 0.69, 0.71, 0.99)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert pick(0.9, temperature=0.0) == 1 and pick(0.99, top_k=1) == 1
    assert [pick(u, top_k=2) for u in (0.0, 0.56, 0.58)] == [1, 1, 3]
    assert [pick(u, top_p=0.69) for u in (0.5, 0.6)] == [1, 3]
    assert [pick(u, top_p=0.71) for u in (0.43, 0.45, 0.67)] == [1, 2, 3]
    assert [pick(u, min_p=0.6) for u in (0.5, 0.6)] == [1, 3]
    assert ragged.sample(np.zeros(5), 0.5, top_k=2) == (1, pytest.approx(0.0, abs=1e-12))
    assert ragged.sample(np.full(3, -np.inf), 0.5)[0] == 3
    assert [ragged.sample(np.array([0, np.inf, np.nan, np.inf]), u)[0] for u in (0.4, 0.6)] == [1, 3]
