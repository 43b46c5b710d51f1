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


def linear_limit(x, codes, scales, zeros, group: int) -> np.ndarray:
    """How far the fp32 sums may be from float64's, by the steps they are
    formed in (linear_bound knows the terms alone, which at thousands of inputs
    leaves room for a lost group):

    - within a group: x . code and sum(x), of `group` exact terms each, added in
      any order by an adder that may truncate: at most group 2^-23 of the terms'
      magnitudes;
    - over the groups: two fmas a run of 32 inputs (the finest the sums are
      taken in) and the joins of lanes and waves (fewer than 32), each rounding
      a sum of some runs by 2^-24. Such a sum is at most the runs' own
      |s dot + z sum| and, between the two fmas, one run's |z sum| beside them.
    """
    x = np.asarray(x, np.float64)
    rows, n = x.shape
    s, z = (np.asarray(a, np.float64) for a in (scales, zeros))
    sizes = np.abs(x) @ (codes * np.repeat(s, group, axis=1) + np.repeat(np.abs(z), group, axis=1)).T
    # (runs, rows, out): each run's x . code and sum(x), with its group's scale and zero.
    runs = n // 32
    xr = x.reshape(rows, runs, 32).transpose(1, 0, 2)
    dot = xr @ codes.reshape(len(codes), runs, 32).astype(np.float64).transpose(1, 2, 0)
    of = np.arange(runs) * 32 // group
    zsum = xr.sum(2)[:, :, None] * z.T[of][:, None]
    reach = (np.abs(s.T[of][:, None] * dot + zsum) + np.abs(zsum)).sum(0)
    return group * 2.0**-23 * sizes + (2 * runs + 32) * 2.0**-24 * reach
