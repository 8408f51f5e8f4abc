"""Beam search's selection from the definition, in 64 bits."""

import math

import numpy as np


def values(x, scores, finished=None, pad=0):
    """[groups, beams, vocabulary] float64: score + log softmax; -inf impossible, NaN undefined."""
    x, s = x.astype(np.float64), scores.astype(np.float64)
    out = np.full(x.shape, -np.inf)
    for g in range(x.shape[0]):
        for b in range(x.shape[1]):
            row, score = x[g, b], s[g, b]
            done = finished is not None and finished[g, b]
            if math.isnan(score) or score == np.inf or \
                    (not done and score > -np.inf and (np.isnan(row).any() or (row == np.inf).any())):
                out[g, b] = np.nan
            elif score == -np.inf:
                continue
            elif done:
                out[g, b, pad] = score
            elif (row > -np.inf).any():
                m = row.max()
                out[g, b] = score + ((row - m) - math.log(np.exp(row - m).sum()))
    return out


def select(x, scores, num, finished=None, pad=0):
    """(scores, parents, tokens): falling, NaN first, equal ones by rising beam and token."""
    v = values(x, scores, finished, pad)
    g, k, n = v.shape
    flat = v.reshape(g, k * n)
    key = np.where(np.isnan(flat), -np.inf, np.where(np.isneginf(flat), np.inf, -flat))
    order = np.argsort(key, axis=1, kind="stable")[:, :num]
    return (np.take_along_axis(flat, order, 1), order // n + k * np.arange(g)[:, None], order % n)
