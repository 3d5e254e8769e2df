"""A tolerance for chunks over the 4-bit cache that a lost tile or a mask that is off by one exceeds.

The chunk kernel rounds values to fp16 once, and for bf16 queries keys too, which is a function of the
stored bytes: the bound is taken around the answer for the rounded ones, so it does not have to allow for
what that does to the scores. (For fp16 queries it has keys as the sum of two fp16: to 2^-22 of them.) What is left, per output element, with p the row's weights and W = max(|V|, half its group's range):
  e |o|               the output's own rounding, e half a step of its type
  2^-11 sum p W       the weights, rounded to fp16 (in the chunk kernel relative to V, in the streaming
                      kernel relative to the middle of the codes)
  2^-12 sum p W       everything in fp32: exponentials, sums, scores
  2^-30 n max W       what fp16 leaves of weights below its normal range (n tokens)
  2^-25               half a step of fp16 below its normal range (the output)"""
import numpy as np

from oracle import q4 as O


def rounded(x):
    """Values as the chunk kernel's operands."""
    return np.asarray(x, np.float64).astype(np.float16).astype(np.float64)


def bound(q, K, V, scale, G, eps, group, chunk):
    """(the answer, the tolerance) of the last queries q [nq, HQ, d] over K, V [n, H, d] (64 bits, as stored), whose
    type has half a step eps."""
    g = V.reshape(*V.shape[:-1], -1, group)
    half = np.repeat((g.max(-1) - g.min(-1)) / 2, group, -1)
    if chunk:
        K, V = rounded(K) if eps > 2.0 ** -11 else K, rounded(V)
    W = np.maximum(np.abs(V), half)
    want = O.attend(q, K, V, scale, G)
    tol = eps * np.abs(want) + (2.0 ** -11 + 2.0 ** -12) * O.attend(q, K, W, scale, G) + len(K) * 2.0 ** -30 * W.max() + 2.0 ** -25
    return want, tol


def worst(out, want, tol):
    """The largest error over its tolerance (infinite for NaN)."""
    r = np.abs(out - want) / tol
    return float(np.where(np.isnan(r), np.inf, r).max())
