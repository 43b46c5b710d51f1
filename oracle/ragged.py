"""A ragged batch's operators in float64: rows turned to their positions and put
into pages, several prompts' attention, rows in codes of 8 bits and their
products, the choice of a token. Beyond the reference."""

from __future__ import annotations

import math

import numpy as np

from oracle import windows

# -- rotary positions ------------------------------------------------------------------


def frequencies(part: int, theta: float, scaling: dict | None):
    """What a position turns each pair by, and the factor of cos and sin, pair by
    pair."""
    kind = scaling["kind"] if scaling else None
    out, magnitude = [], 1.0
    for j in range(part // 2):
        f = theta ** (-2.0 * j / part)
        if kind == "linear":
            f = f / scaling["factor"]
        elif kind == "llama3":
            turns = scaling["original"] * f / (2 * math.pi)  # over the original context
            if turns < scaling["low"]:
                f = f / scaling["factor"]
            elif turns <= scaling["high"]:
                share = (turns - scaling["low"]) / (scaling["high"] - scaling["low"])
                f = (1 - share) * f / scaling["factor"] + share * f
        elif kind == "yarn":
            magnitude = scaling.get("magnitude", 0.1 * math.log(scaling["factor"]) + 1.0)

            def pair(turns):
                return part * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

            first = max(math.floor(pair(scaling.get("fast", 32.0))), 0)
            last = min(math.ceil(pair(scaling.get("slow", 1.0))), part - 1)
            ramp = min(max((j - first) / max(last - first, 0.001), 0.0), 1.0)
            f = f / scaling["factor"] * ramp + f * (1 - ramp)
        out.append(f)
    return np.array(out), magnitude


def turned(x, positions, freq, magnitude: float, interleaved: bool):
    """Rows (n, heads, hd) turned to positions (n,): the first 2 len(freq)
    channels of a head. Returns (out, terms): terms bounds |a| + |b| of each
    pair, which rounded products err by."""
    x = np.asarray(x, np.float64)
    half = len(freq)
    a, b = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else
            (slice(0, half), slice(half, 2 * half)))
    angle = np.asarray(positions, np.float64)[:, None] * freq
    c, s = (magnitude * f(angle)[:, None] for f in (np.cos, np.sin))
    out, terms = x.copy(), np.zeros(x.shape)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    terms[..., a] = terms[..., b] = magnitude * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return out, terms


# -- several prompts -------------------------------------------------------------------


def packed_attention(q, k, v, offsets_q, offsets_k):
    """q (rows, heads, hd), k and v (keys, kv, hd). Returns (out, bound, terms) as
    windows.window_attention's, NaN in rows of no sequence; zeros where a row
    sees nothing."""
    out, bound, terms = (np.full(np.shape(q), np.nan) for _ in range(3))
    for s in range(len(offsets_q) - 1):
        q0, q1, k0, k1 = (int(x) for x in (offsets_q[s], offsets_q[s + 1], offsets_k[s], offsets_k[s + 1]))
        blind = max(0, (q1 - q0) - (k1 - k0))  # queries before the first key
        for part in (out, bound, terms):
            part[q0:q0 + blind] = 0.0
        if q1 - q0 > blind:
            got = windows.window_attention(q[q0 + blind:q1], k[k0:k1], v[k0:k1], 0, 0)
            for part, x in zip((out, bound, terms), got):
                part[q0 + blind:q1] = x
    return out, bound, terms


# -- 8-bit rows ------------------------------------------------------------------------


def quantise_rows(x):
    """fp16 rows -> codes int8, scales fp32: both divisions in fp32."""
    x = np.asarray(x, np.float16).astype(np.float32)
    top = np.abs(x).max(1)
    fine = np.isfinite(x).all(1)
    with np.errstate(invalid="ignore", over="ignore"):
        scale = np.where(fine, top / np.float32(127), np.float32(np.nan)).astype(np.float32)
        by = np.where(fine & (top > 0), scale, np.float32(1))[:, None]
        code = np.where((fine & (top > 0))[:, None], np.rint(x / by), 0)
    return code.astype(np.int8), scale


def linear_int8(x, x_scale, w, w_scale):
    """What the codes' products stand for, float64 (rows, out), and how far three
    fp32 roundings (of the sum, and of its products by the scales) may take it."""
    y = (x.astype(np.float64) @ w.astype(np.float64).T) * np.outer(
        x_scale.astype(np.float64), w_scale.astype(np.float64))
    return y, 3.001 * 2.0**-24 * np.abs(y)


# -- the choice of a token -------------------------------------------------------------


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row, and the smallest distance, in shares of the kept
    weights, of a decision from its border."""
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    if not (l > -np.inf).any():
        return len(l), 1.0
    if not temperature > 0:
        return int(np.argmax(l)), 1.0
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    top = l[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(l[order] == top, 1.0, np.exp((l[order] - top) / temperature)
                     if np.isfinite(top) else 0.0)
    near = 1.0
    if top_p < 1:
        upto = np.cumsum(w)
        need = max(top_p, 0.0) * upto[-1]
        n = max(1, int(np.searchsorted(upto, need, side="left")) + 1)
        n = min(n, len(w))
        near = min(near, np.abs(upto - need).min() / upto[-1])
        w, order = w[:n], order[:n]
    if min_p > 0:
        n = int((w >= min(min_p, 1.0)).sum())
        w, order = w[:n], order[:n]
    by_index = np.argsort(order)
    upto = np.cumsum(w[by_index])
    share = min(max(u, 0.0), 1.0) * upto[-1]
    near = min(near, np.abs(upto[:-1] - share).min() / upto[-1]) if len(upto) > 1 else near
    i = int(np.searchsorted(upto, share, side="right"))
    if i >= len(upto):  # a share of all of them
        i = int(np.flatnonzero(w[by_index] > 0)[-1])
    return int(order[by_index][i]), float(near)
