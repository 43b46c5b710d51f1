"""Attention through a sliding window with sink tokens, in float64, for a
prompt's queries and for one token of a paged cache. Beyond the reference,
whose attention sees every position; the arithmetic is oracle.attention's."""

from __future__ import annotations

import numpy as np

from oracle import attention as att


def visible(position: int, keys: int, window: int, sinks: int) -> np.ndarray:
    """Which of `keys` keys the query at `position` sees: those up to its own,
    with a window the last `window` of them and the first `sinks`."""
    j = np.arange(keys)
    seen = j <= position
    if window:
        seen &= (j > position - window) | (j < sinks)
    return seen


def window_attention(q, k, v, window: int, sinks: int):
    """q (seq_q, heads, hd), the last of k, v (seq_k, kv, hd)'s positions.
    Returns (out, bound, terms): bound as attention_bound's, terms the sums of
    p |v|, which a relative error of every weight weighs."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    seq_q, heads, hd = q.shape
    seq_k, group = len(k), heads // k.shape[1]
    seen = np.stack([visible(seq_k - seq_q + i, seq_k, window, sinks) for i in range(seq_q)])
    out, bound, terms = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = np.where(seen, q[:, h] @ kh.T / np.sqrt(hd), -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h], terms[:, h] = p @ vh, p @ np.abs(vh)
        size = np.where(seen, np.abs(q[:, h]) @ np.abs(kh).T / np.sqrt(hd), 0.0).max(1)
        bound[:, h] = ((np.sqrt(seen.sum(1)) + np.sqrt(hd) * size)[:, None] *
                       att.FP32_REL_ULP * terms[:, h])
    return out, bound, terms


def paged_token(q, k, v, length: int, unread, window: int, sinks: int, page_tokens: int):
    """One token's attention over its cache's rows k, v (pages * page_tokens,
    kv, hd), `unread` a bool a row. Returns (out (heads, hd), mass (heads,
    pages), bound (heads, hd)); zeros where nothing is seen."""
    heads, hd = q.shape
    pages = len(k) // page_tokens
    seen = visible(length - 1, len(k), window, sinks) & ~np.asarray(unread, bool)
    if length <= 0 or not seen.any():
        return np.zeros((heads, hd)), np.zeros((heads, pages)), np.zeros((heads, hd))
    ki, vi = np.asarray(k, np.float64)[seen], np.asarray(v, np.float64)[seen]
    out, w = att.attention64(q[None], ki, vi)
    bound = att.attention_bound(q[None], ki, vi, w)
    weights = np.zeros((heads, len(k)))
    weights[:, seen] = w[:, -1]
    return out[0], att.page_mass(weights, page_tokens), bound[0]
