"""TEST INFRASTRUCTURE ONLY: keys and values that make every cached position decisive, and what attention over them gives.

A position's value row is 7 at one of the hd values and 0 elsewhere (exact in 4 bits too: scale 1, code 7), its class;
classes are equally often, so value d of an output is 7 times the weight of about n / hd positions.  A position that is
lost or counted twice changes its class by about hd / n of itself, which is many roundings of the output for the lengths
used here; in an attention over random rows it would be lost in the tolerance of the sums.  Two layouts: stripes (p % hd),
and at random, so that a tile taken twice in another one's place shows as well.

A position's key row is 7 at one value too (class (p + head) % hd).  With the query 0 all weights are equal; with a query
that is `LARGE` at one value the positions of that key class weigh 2^16 times the others, which ties each key to its value.
"""
from __future__ import annotations

import numpy as np

SIZE = 7.0
LOG2_WEIGHT = 16
HALF_ULP16 = 2.0**-11  # half a step of fp16, relative
# Equal scores: the weights are powers of two, their sums exact; the quotient and its rounding to fp16 remain.
EVEN = HALF_ULP16 + 2.0**-20
# Chosen scores: probabilities rounded once to fp16; a score of 16 in the exponent off by 2^-19 of itself moves a weight by
# 16 ln 2 2^-19 and the sum of weights by as much (fp32 product, scale and exponential's argument); exponentials 2^-18.
CHOSEN = 2 * HALF_ULP16 + 2 * 16 * 0.6932 * 2.0**-19 + 2.0**-17
# Values below the smallest normal fp16 are rounded by half of its last place.
SMALLEST = 2.0**-25


def value_classes(n, heads, hd, layout, seed=0):
    """[n, heads]"""
    p = np.arange(n)
    if layout == "stripes":
        return np.repeat((p % hd)[:, None], heads, 1)
    rng = np.random.default_rng(seed)
    return np.stack([rng.permutation(p) % hd for _ in range(heads)], 1)


def key_classes(n, heads, hd):
    return (np.arange(n)[:, None] + np.arange(heads)) % hd


def rows(classes, hd):
    """fp16 rows [n, heads, hd] of these classes."""
    out = np.zeros((*classes.shape, hd), np.float16)
    np.put_along_axis(out, classes[..., None], SIZE, -1)
    return out


def large(hd):
    """The query value that lifts its key class by 2^16, as it is held (fp16), and the weight it gives exactly."""
    q = np.float16(LOG2_WEIGHT * np.log(2) * np.sqrt(hd) / SIZE)
    return q, float(np.exp(SIZE * np.float64(q) / np.sqrt(hd)))


def even(classes, counts, hd):
    """Output [heads, hd] under equal weights; counts [n]: how often each position counts (1; 0 for one without a page)."""
    total = counts.sum()
    if total == 0:
        return np.zeros((classes.shape[1], hd))
    return np.stack([np.bincount(classes[:, h], weights=counts, minlength=hd) for h in range(classes.shape[1])]) * SIZE / total


def chosen(classes, keys, counts, hd, wanted):
    """Output [query heads, hd] where query head i asks for key class wanted[i]."""
    rep = len(wanted) // classes.shape[1]
    _, weight = large(hd)
    out = np.zeros((len(wanted), hd))
    for i, c in enumerate(wanted):
        w = np.where(keys[:, i // rep] == c, weight, 1.0) * counts
        if w.sum():
            out[i] = np.bincount(classes[:, i // rep], weights=w, minlength=hd) * SIZE / w.sum()
    return out


def off(got, want, tolerance):
    """The largest error in units of the tolerance."""
    return float(np.max(np.abs(got - want) / (tolerance * np.abs(want) + SMALLEST), initial=0.0))
