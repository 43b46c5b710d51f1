"""Weights at four bits, in NumPy: the page quantiser's rule (oracle.quant) on
groups of a weight's inputs, and projections through such weights in float64.
Beyond the reference, whose weights are fp16."""

from __future__ import annotations

import numpy as np

from oracle import quant


def quantise(weight: np.ndarray, group: int):
    """(out, in) fp16 values -> codes (out, in) 0..15, scales and zeros
    (out, in / group) fp16."""
    w = np.asarray(weight, np.float16)
    out, n_in = w.shape
    g = w.reshape(out, n_in // group, group)
    lo, hi = g.min(2), g.max(2)
    scale = quant.scale_of(lo, hi, 4)
    code = quant.code_of(g, lo[..., None], scale[..., None], 4)
    return code.reshape(out, n_in).astype(np.uint8), scale, lo


def packed(codes: np.ndarray) -> np.ndarray:
    """Codes (out, in) as bytes, the first of two in the low bits."""
    return (codes[:, ::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def weight64(codes, scales, zeros, group: int) -> np.ndarray:
    """What the codes stand for, float64 (out, in)."""
    s = np.repeat(np.asarray(scales, np.float64), group, axis=1)
    z = np.repeat(np.asarray(zeros, np.float64), group, axis=1)
    return codes.astype(np.float64) * s + z


def linear_bound(x, codes, scales, zeros, group: int) -> np.ndarray:
    """How far fp32 sums of s (x . code) + z sum(x) may be from float64's, in
    any order of adding: each of the n terms of a sum errs by at most n 2^-24
    of the terms' magnitudes (products of an 11- and a 4-bit number are
    exact), and the two fmas a group by 2^-24 of theirs; 2^-23 covers an
    adder that truncates."""
    s = np.repeat(np.abs(np.asarray(scales, np.float64)), group, axis=1)
    z = np.repeat(np.abs(np.asarray(zeros, np.float64)), group, axis=1)
    size = np.abs(np.asarray(x, np.float64)) @ (codes * s + z).T
    return (codes.shape[1] + 4) * 2.0**-23 * size
