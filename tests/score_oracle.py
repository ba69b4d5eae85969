"""Scores of tokens in 64 bits, and how far 32 bits may be from them."""
import numpy as np


def order(row):
    """Ids in the order of alternatives: the greater value first, the lowest id among equals; a NaN
    stands with the negative infinities."""
    return np.argsort(-np.where(np.isnan(row), -np.inf, row), kind="stable")


def scores(x, tokens, top):
    """(log probabilities, entropy, ids, their log probabilities) of rows x [rows, V]."""
    x = np.asarray(x, dtype=np.float64)
    n = len(x)
    lp, h = np.full(n, np.nan), np.full(n, np.nan)
    ids, alt = np.zeros((n, top), dtype=np.int64), np.full((n, top), np.nan)
    for r in range(n):
        ids[r] = order(x[r])[:top]
        if np.isnan(x[r]).any() or np.isposinf(x[r]).any() or np.isneginf(x[r]).all():
            continue
        m = x[r].max()
        logp = x[r] - m - np.log(np.exp(x[r] - m).sum())
        p = np.exp(logp)
        h[r] = -(p[p > 0] * logp[p > 0]).sum()
        if 0 <= tokens[r] < x.shape[1]:
            lp[r] = logp[tokens[r]]
        alt[r] = logp[ids[r]]
    return lp, h, ids, alt


def bounds(x, roundings=96):
    """Per row, how far ln S and the entropy may be off in 32 bits. With p the probabilities and
    d = x - max: the fast exponential is off by 2 + 1.173 |d| units of 2^-23 (its documented bound), so
    S by the mean of that under p, and T = sum e^d d by the mean of |d| times that; each of the (at
    most ``roundings``) additions on a value's way into a sum rounds by 2^-24 of it. The entropy is
    ln S - T / S. Rows without a distribution: 0."""
    x = np.asarray(x, dtype=np.float64)
    ln_s, ent = np.zeros(len(x)), np.zeros(len(x))
    for r, row in enumerate(x):
        if np.isnan(row).any() or np.isposinf(row).any() or np.isneginf(row).all():
            continue
        d = (row - row.max())[np.isfinite(row)]
        p = np.exp(d)
        s = p.sum()
        p /= s
        d = np.abs(d) * (p > 0)
        a1, a2 = (p * d).sum(), (p * d * d).sum()
        ln_s[r] = 2.0 ** -23 * (2 + 1.173 * a1) + 2.0 ** -24 * roundings + 2.0 ** -23 * abs(np.log(s))
        t = 2.0 ** -23 * (2 * a1 + 1.173 * a2) + 2.0 ** -24 * (roundings + 2) * a1
        ent[r] = ln_s[r] * (1 + a1) + t + 2.0 ** -23 * a1
    return ln_s, ent


def check(got, x, tokens, top, moved=0.0):
    """``got``: a ``Scores``; ``x``: the logits in 64 bits; ``moved`` (a number, or one a row): how far
    a logit of the kernel may be from those. Where it is 0 the ids have to be equal, else they have to
    be an order that logits moved so far may have."""
    x = np.asarray(x, dtype=np.float64)
    n = len(x)
    moved = np.broadcast_to(np.asarray(moved, dtype=np.float64), (n,))
    lp, h, ids, alt = scores(x, tokens, top)
    ln_s, ent = bounds(x)
    got_lp, got_h, got_ids, got_alt = (t.cpu().numpy() for t in got.tensors())
    assert got_ids.shape == ids.shape == got_alt.shape and got_lp.shape == got_h.shape == lp.shape
    # two subtractions behind x_t: x_t - max, and that less ln S
    reach = ln_s + 2 * moved
    two = lambda v, s: 2.0 ** -23 * (np.where(np.isfinite(v), np.abs(v), 0.0) + s)
    size = np.log(x.shape[1])
    _close(got_lp, lp, reach + two(lp, size))
    _close(got_h, h, ent + moved * (2 + 2 * size) + two(h, 0.0))
    if top == 0:
        return
    for r in range(n):
        mine = got_ids[r].astype(int)
        assert len(set(mine)) == top and mine.min() >= 0 and mine.max() < x.shape[1]
        if moved[r] == 0.0:
            assert np.array_equal(mine, ids[r]), (r, mine, ids[r])
            continue
        v = x[r][mine]
        assert np.all(v[:-1] - v[1:] >= -2 * moved[r])
        assert v.min() >= x[r][ids[r][-1]] - 2 * moved[r]
        alt[r] += v - x[r][ids[r]]
    _close(got_alt, alt, reach[:, None] + two(alt, size))


def _close(got, want, tol):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    err = np.abs(got - np.where(ok, want, 0.0))[ok]
    tol = np.broadcast_to(tol, want.shape)[ok]
    assert np.all(err <= tol), (err - tol).max()
