"""Limits of the paged serving operators that need no GPU."""
import numpy as np
import pytest

import paged_ref as R
from test_paged_ops import sample
from vibethinker_webgpu_lora_b200 import _lib as L


def test_the_longest_row():
    assert sample(n=(1 << 20) + 1, ld=1 << 21) == L.EG_ERR_ARG
    assert sample(rows=0, n=1 << 20, ld=1 << 20) == L.EG_OK


def halves(x):
    """(hi, lo) f16 parts, as the attention kernels split q and the weights."""
    hi = x.astype(np.float16).astype(np.float64)
    return hi, (x - hi).astype(np.float16).astype(np.float64)


@pytest.mark.parametrize("n", [256, 1001, 4096])
def test_the_attention_limit_sees_a_lost_part(n):
    """R.LIMIT is far above what the hi + lo parts leave and far below what is
    left without one: of q, of the weights, or a lo part of q that is not lifted
    (or its row not scaled) under keys of 300."""
    rng = np.random.default_rng(n)
    rows, scale = 64, np.log2(np.e) / np.sqrt(128)
    q = 1.5 * rng.standard_normal((rows, 128)) * scale
    k, v = (rng.standard_normal((n, 128)).astype(np.float16).astype(np.float64) for _ in range(2))

    def out(s, parts=3):
        p = 2.0 ** (s - s.max(1, keepdims=True) + 14)
        hi, lo = halves(p)
        return (hi * (parts & 1) + lo * (parts >> 1)) @ v / p.sum(1, keepdims=True)

    p = 2.0 ** (q @ k.T - (q @ k.T).max(1, keepdims=True))
    want = p @ v / p.sum(1, keepdims=True)
    err = lambda o: np.linalg.norm(o - want) / np.linalg.norm(want)  # noqa: E731
    hi, lo = halves(q)
    assert err(out((hi + lo) @ k.T)) < R.LIMIT / 10
    assert err(out(hi @ k.T)) > 5e-5 and err(out((hi + lo) @ k.T, 1)) > 5e-5
    qs = q / 300
    hs, ls = halves(qs)
    assert err(out((hs + ls) @ (300 * k).T)) > 2 * R.LIMIT
    up = 2.0 ** (14 - np.floor(np.log2(abs(qs).max(1, keepdims=True))))
    hs, ls = halves(qs * up)
    assert err(out((hs + ls) / up @ (300 * k).T)) < R.LIMIT / 10
