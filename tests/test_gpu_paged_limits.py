"""The paged serving operators at the ends of what they take: sizes of q and of
the cache's values, lengths and counts (definitions: paged_ref.py)."""
import numpy as np
import pytest
import torch

import paged_ref as R
from test_gpu_paged_ops import Shared, check_sample, relative, run_sample
from vibethinker_webgpu_lora_b200 import kernels as K

pytestmark = pytest.mark.gpu
HD = R.HD


# ---------------------------------------------------------------- sampling
@pytest.mark.parametrize("rows,n", [(65, 1 << 18), (65, 300000), (33, 1 << 19), (40, (1 << 19) - 1), (13, 1 << 20),
                                    (20, (1 << 20) - 3), (70, 1 << 20)])
@pytest.mark.parametrize("kind", ["equal", "half", "two thirds"])
def test_sample_of_long_rows_of_equal_logits(cuda, rows, n, kind):
    """Vocabularies up to the longest taken, with 2^18 equal logits and more in what
    one CTA holds, alone or above lower ones: every row gets its id."""
    rng = np.random.default_rng(n)
    x = torch.zeros(rows, n, device=cuda)
    if kind != "equal":
        x -= torch.from_numpy((rng.random(n) < (0.5 if kind == "half" else 1 / 3)).astype(np.float32)).to(cuda)
    r = rng.random(rows).astype(np.float32)
    r[0], r[-1] = 0.0, 1.0
    f = lambda v: torch.full((rows,), v, device=cuda)  # noqa: E731
    some = sorted({0, 1, rows // 2, rows - 1})
    host = x[some].cpu().numpy()
    for k, p in ((0, 1.0), (n // 5, 1.0), (n - n // 7, 1.0), (0, 0.75)):
        ids, probs = torch.full((rows,), -7, dtype=torch.int32, device=cuda), f(9.0)
        K.sample_filtered(x, torch.from_numpy(r).to(cuda), ids, top_k=torch.full((rows,), k, dtype=torch.int32, device=cuda),
                          top_p=f(p), probs=probs)
        torch.cuda.synchronize()
        assert ((ids >= 0) & (ids < (k if k and kind == "equal" else n))).all() and (probs < 1e-4).all()
        got, share = ids.cpu().numpy().view(np.uint32), probs.cpu().numpy().astype(np.float64)
        check_sample(host, got[some], share[some], 1.0, k, p, 0.0, r[some])


@pytest.mark.parametrize("t,share", [(1.13e-7, 0.9874), (1e-7, 0.9976), (2.2e-7, 0.1426), (5e-7, 0.0043)])
def test_sample_steps_far_above_the_temperature(cuda, t, share):
    """Temperatures below a step of f32: one best logit of 8 and 3,999 that
    share the value 3 2^-21 below it, whose masses are far from 0 together.
    Each row takes the best token up to its share of the mass, then the others."""
    x = np.full((6, 4000), 8 - 3 * 2.0 ** -21, np.float32)
    for i in range(6):
        x[i, 667 * i] = 8.0
    r = np.array([0.5, 0.9, share - 1e-3, share + 1e-3, 0.9999, 1.0], np.float32)
    for k, p in ((0, 1.0), (2001, 1.0), (0, 0.98)):
        got, probs = run_sample(cuda, x, t, k, p, 0.0, r)
        if not k and p == 1 and share > 0.9:
            assert abs(probs[0] - share) < 1e-4
        check_sample(x, got, probs, t, k, p, 0.0, r)


@pytest.mark.parametrize("value", [-9.5e29, -8.9e29, -1e28, -1e24, -1e22, -3e15, -1.0, -1e-20, 1e-42, 1e15, 6e21, 1e24, 1e30, 3e38])
@pytest.mark.parametrize("n", [1, 41, 9001])
def test_sample_equal_logits_of_any_size(cuda, n, value):
    """A row of one value, and one of it and lower ones, at every size of the value."""
    x = np.full((5, n), value, np.float32)
    x[1, : n // 2] = -np.inf
    x[2, n // 3:] = np.float32(value) - abs(np.float32(value)) / 16  # far below, or the same for the smallest
    x[3, ::2] = np.nan
    x[3, n - 1] = value
    r = np.array([0.3, 0.5, 0.7, 0.9, 1.0], np.float32)
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.05, 7, 1.0, 0.02), (1e-7, 0, 0.9, 0.0), (1e5, 0, 0.5, 0.3)]:
        got, probs = run_sample(cuda, x, t, k, p, m, r)
        check_sample(x, got, probs, t, k, p, m, r)


# ---------------------------------------------------------------- attention
def put(s, **kw):
    """Host arrays of a case, changed, to the device."""
    for name in kw:
        setattr(s, name, kw[name])
    shape = s.d["k_cache"].shape
    s.d["k_cache"].copy_(torch.from_numpy(s.kc.reshape(shape)))
    s.d["v_cache"].copy_(torch.from_numpy(s.vc.reshape(shape)))
    s.d["q"].copy_(torch.from_numpy(s.q[:, :s.nh * HD]))


@pytest.mark.parametrize("size", [0.01, 30.0, 100.0, 300.0, 8000.0])
@pytest.mark.parametrize("n,prefix", [(2, 800), (40, 4000), (130, 1000)])
def test_shared_prefix_f16_keys_of_any_size(cuda, n, prefix, size):
    """Keys of an f16 cache far above 1 under queries as far below it, and the
    other way round: the error is that of ordinary sizes (R.LIMIT)."""
    s = Shared(cuda, prefix, [60] * n, 16, 2, "f16", seed=18)
    put(s, kc=(s.kc.astype(np.float32) * np.float32(size)).astype(np.float16), q=s.q / np.float32(size))
    K.attn_shared_prefix(**s.d)
    err = relative(s, range(0, n, max(1, n // 5)))
    print("relative error", err)
    assert err < R.LIMIT


@pytest.mark.parametrize("kv,n,prefix", [("f16", 2, 800), ("f16", 40, 4000), ("f32", 3, 500), ("f32", 40, 4000)])
def test_shared_prefix_one_large_dimension(cuda, kv, n, prefix):
    """One dimension of the keys 20,000 times the others, one of the queries as far below them."""
    s = Shared(cuda, prefix, [60] * n, 16, 2, kv, seed=19)
    s.kc[..., 7] = (np.sign(s.kc[..., 7]) * 20000).astype(s.kc.dtype)
    q = s.q.reshape(n, 16, HD)
    q[..., 7] *= 1e-4
    put(s, q=q.reshape(n, -1))
    K.attn_shared_prefix(**s.d)
    err = relative(s, range(0, n, max(1, n // 5)))
    print("relative error", err)
    assert err < R.LIMIT


@pytest.mark.parametrize("kv,n,prefix", [("f16", 2, 800), ("f16", 40, 4000), ("f32", 3, 500), ("f32", 40, 4000)])
def test_shared_prefix_largest_queries(cuda, kv, n, prefix):
    """|q| / 8 up to the f16 range's end, 2^19.  What is added to ordinary errors, over
    sqrt(128): an f32 key of 1e-5 is held to 2^-36, evenly spread, which such a query makes
    3.9e-7 of a score; the other queries' lo parts may be held to 2^-39 of the largest
    (2^-23 each, 5.4e-7 of a score)."""
    s = Shared(cuda, prefix, [60] * n, 16, 2, kv, seed=20)
    s.kc[..., 5] = (s.kc[..., 5].astype(np.float32) * np.float32(1e-5)).astype(s.kc.dtype)
    q = s.q.reshape(n, 16, HD)
    q[..., 5] = np.sign(q[..., 5]) * 8 * 65504.0
    put(s, q=q.reshape(n, -1))
    K.attn_shared_prefix(**s.d)
    err = relative(s, range(0, n, max(1, n // 5)))
    print("relative error", err)
    assert err < R.LIMIT + 7e-7


@pytest.mark.parametrize("kv,n,prefix", [("f16", 2, 512), ("f16", 1, 9000), ("f16", 40, 4000), ("f32", 3, 100), ("f32", 9, 4000),
                                         ("f32", 40, 4000), ("f16", 3, 0), ("f32", 70, 0)])
def test_shared_prefix_lengths_where_none_are_allowed(cuda, kv, n, prefix):
    """max_len = 0: a length above it is flagged in every form, and the prefix alone is used."""
    s = Shared(cuda, prefix, [0] * n, 16, 2, kv, seed=21, max_len=0)
    K.attn_shared_prefix(**s.d)
    s.check(range(0, n, max(1, n // 5)))
    assert s.d["err"].item() == 0
    s.d["lens"][n - 1] = 1
    s.d["out"].fill_(5.0)
    K.attn_shared_prefix(**s.d)
    s.check(range(0, n, max(1, n // 5)))
    assert s.d["err"].item() == 1


@pytest.mark.parametrize("kv,n,prefix", [("f16", 2, 300), ("f16", 1, 9000), ("f16", 40, 4000), ("f32", 3, 100), ("f32", 40, 4000)])
@pytest.mark.parametrize("where", ["prefix", "suffix"])
@pytest.mark.parametrize("what", ["k", "v"])
def test_shared_prefix_values_that_are_not_finite(cuda, kv, n, prefix, where, what):
    """An infinity of the cache (an f32 cache: any value past the f16 range): the
    rows that meet it are flagged, all others are right."""
    s = Shared(cuda, prefix, [60] * n, 16, 2, kv, seed=22)
    row = R.rows_of(s.ppages, prefix)[prefix // 3] if where == "prefix" else R.rows_of(s.pages[n - 1], 60)[33]
    c = s.d["k_cache" if what == "k" else "v_cache"].view(-1, 2, HD)
    c[int(row), 1, 3] = float("inf") if kv == "f16" else 1e5
    K.attn_shared_prefix(**s.d)
    torch.cuda.synchronize()
    assert s.d["err"].item() == 1
    met = s.d["out"].view(n, 2, 8 * HD)[:, 1]  # the second KV head's
    assert not torch.isfinite(met[n - 1]).all()
    got = s.d["out"].cpu().numpy().astype(np.float64).reshape(n, 16, HD)
    for b in range(0, n, max(1, n // 5)):
        o, bound = s.want(b)
        heads = slice(0, 16 if where == "suffix" and b < n - 1 else 8)
        assert (abs(got[b] - o) <= bound)[heads].all()


@pytest.mark.parametrize("kv,n,prefix,longest", [
    ("f16", 2, 256, 32), ("f16", 16, 2048, 640), ("f16", 3, 9001, 100), ("f16", 64, 2051, 200), ("f16", 130, 1000, 90),
    ("f16", 300, 257, 30), ("f16", 40, 8192, 1024), ("f32", 2, 300, 60), ("f32", 17, 1001, 333), ("f32", 40, 4000, 200)])
def test_shared_prefix_error_is_that_of_f32(cuda, kv, n, prefix, longest):
    """Ordinary inputs in each form (one launch, warps, tensor cores, f32 in 4
    and 8 warps): the relative error is R.LIMIT at most.  Without one of the lo
    parts it is above 5e-5 (test_paged_limits.py)."""
    s = Shared(cuda, prefix, [(i * 53) % (longest + 1) for i in range(n)], 16, 2, kv, seed=23, max_len=longest)
    K.attn_shared_prefix(**s.d)
    err = relative(s, range(0, n, max(1, n // 6)))
    print("relative error", err)
    assert err < R.LIMIT
