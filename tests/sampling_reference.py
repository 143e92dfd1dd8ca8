"""Draws and largest log-probabilities of one row at a time in float64 numpy."""

import math

import numpy as np


def order_of(x):
    """Words by falling logit, the first of equals first."""
    return np.lexsort((np.arange(x.size), -x))


def cannot(x):
    return bool(np.isnan(x).any() or x.max() in (math.inf, -math.inf))


def log_softmax(x, t):
    z = (x - x.max()) / t     # before anything else: the largest may be near the type's lowest value
    return z - math.log(np.exp(z).sum())


def top(x, k, t):
    if cannot(x):
        return np.full(k, math.nan), np.full(k, -1)
    ids = order_of(x)[:k]
    return log_softmax(x, t)[ids], ids


def kept(x, t, k, p, m):
    """The kept words, by index, and everyone's weight."""
    order = order_of(x)
    w = np.exp((x - x.max()) / t)
    order = order[:k] if k > 0 else order
    if p < 1:
        before = np.cumsum(w[order]) - w[order]
        inside = before < p * w[order].sum()
        inside[0] = True
        order = order[inside]
    if m > 0:
        inside = w[order] >= m
        inside[0] = True
        order = order[inside]
    return np.sort(order), w


def draw(x, u, t=1.0, k=0, p=1.0, m=0.0):
    if cannot(x):
        return -1, math.nan
    if not t > 0:
        word = int(np.argmax(x))
        return word, log_softmax(x, 1.0)[word]
    words, w = kept(x, t, k, p, m)
    sums = np.cumsum(w[words])
    word = int(words[min(int((sums <= min(max(u, 0.0), 1 - 2.0 ** -24) * sums[-1]).sum()), words.size - 1)])
    return word, log_softmax(x, t)[word]
