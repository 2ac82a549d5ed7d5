"""64-bit definitions of the paged serving operators (numpy, host), and the
error bounds of their f32 / f16 kernels."""
import itertools
import math

import numpy as np

HD, PAGE = 128, 16
EMPTY = 0xFFFFFFFF


def rows_of(pages, n):
    i = np.arange(n)
    return np.asarray(pages, np.int64)[i // PAGE] * PAGE + i % PAGE


def rotate(x, cos, sin):
    """x [..][128] turned by the angles of cos / sin [..][128]; and the sum of the products' magnitudes."""
    x, c, s = x.astype(np.float64), cos.astype(np.float64)[..., :64], sin.astype(np.float64)[..., :64]
    lo, hi = x[..., :64], x[..., 64:]
    y = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
    mag = np.concatenate([abs(lo * c) + abs(hi * s), abs(hi * c) + abs(lo * s)], -1)
    return y, mag


def rotate_bound(y, mag, f16):
    """Two products and a sum, each off by half a step of f32 (2^-24), then the
    cache's rounding: half a step of f16 (2^-11, or 2^-25 below its range)."""
    e = 2.0 ** -24 * (mag + abs(y) + 2.0 ** -20 * mag)
    return e + (2.0 ** -11 * (abs(y) + e) + 2.0 ** -25 if f16 else 0.0)


def attention(q, k, v):
    """o [nh][128] = softmax(q k^T / sqrt(128)) v over k, v [n][nkv][128]; and a
    bound of the kernel's error.

    Scores: q is held to 2^-22 (an f16 hi + lo pair), an f32 key or value too
    (the lo.lo product left out: 2^-22), 24 matrix steps each add to an f32 sum
    with an error of 2^-22 of the magnitudes at most (the tensor core's
    alignment included): A (3 2^-22 + 24 2^-22) < A 2^-17 with A = sum |q k|.
    Weights: the score's error in the exponent (counted twice, sum and
    product), exp2's 2 steps and the hi + lo pair: 2^-20.  Sums over the keys:
    2^-22 for each 16-key step and each merged part."""
    nh, n = q.shape[0], len(k)
    if n == 0:
        return np.zeros((nh, HD)), np.zeros((nh, HD))
    G = nh // k.shape[1]
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    o, bound = np.zeros((nh, HD)), np.zeros((nh, HD))
    for h in range(nh):
        kk, vv = k[:, h // G], v[:, h // G]
        s = kk @ q[h] / math.sqrt(HD)
        A = (abs(kk) @ abs(q[h])).max() / math.sqrt(HD)
        p = np.exp(s - s.max())
        p /= p.sum()
        o[h] = p @ vv
        bound[h] = (2 * A * 2.0 ** -17 + 2.0 ** -20 + (n / 16 + 64) * 2.0 ** -22) * (p @ abs(vv))
    return o, bound + 1e-30


# The relative error (of all outputs together, in the 2-norm) that attention on
# ordinary inputs (q 1.5 and keys 1 in size) may have.  The tensor core's f32 sums
# are cut, not rounded: 2^-24 of the running sum a step on the average, all one
# way.  Scores: 16 steps (24 for an f32 cache) of a sum whose size is 2.2 on the
# average (in powers of 2): 24 2^-24 ln 2 2.2 = 2.2e-6 of a weight.  Outputs: at
# most 48 steps of a part (16 tiles of three products), half of them on the
# average: 1.4e-6.  The hi + lo pairs (2^-22 of a part, its sign random) and the
# roundings of the sums in f32 add a few 2^-24.
LIMIT = 4e-6


def sample(x, t=1.0, k=0, p=1.0, minp=0.0, r=0.5):
    """(id, share of the mass kept) of one row of f32 logits; the parameters in 64 bits."""
    x = np.asarray(x, np.float32)
    t = t if t > 0 else 1.0
    ok = np.flatnonzero(x >= np.float32(-1e30))
    if not len(ok):
        return EMPTY, 0.0
    order = ok[np.argsort(-x[ok].astype(np.float64), kind="stable")]
    order = order[:k] if k > 0 else order
    v = x[order].astype(np.float64)
    w = np.ones(len(v))
    rest = v != v[0]  # an infinite maximum takes all the mass
    w[rest] = np.exp((v[rest] - v[0]) / t)
    c, n = np.cumsum(w), len(w)
    if p < 1:
        n = min(n, int(np.searchsorted(c, max(p, 0.0) * c[-1])) + 1)
    if minp > 0:
        n = min(n, max(1, int((w >= minp).sum())))
    j = min(int(np.searchsorted(c[:n], min(max(r, 0.0), 1.0) * c[n - 1])), n - 1)
    return int(order[j]), w[j] / c[n - 1]


def sample_near(x, got, t=1.0, k=0, p=1.0, minp=0.0, r=0.5):
    """Whether `got` is what the definition gives when p and r are off by 2^-25
    of themselves: a token's weight is held to 2^-26 of it (fixed point), so a
    running mass is off by 2^-26 of itself and its ratio to another by 2^-25."""
    eps = 2.0 ** -25
    for a, b in itertools.product((0, -eps, eps), repeat=2):
        if got == sample(x, t, k, p * (1 + a) if 0 < p < 1 else p, minp, r * (1 + b))[0]:
            return True
    return False
