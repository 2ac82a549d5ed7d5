"""Refusals of the paged serving operators (host checks, no GPU), and the
64-bit definitions the GPU tests compare with against worked cases."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from vibethinker_webgpu_lora_b200 import _lib as L
from vibethinker_webgpu_lora_b200 import kernels as K

P = 4096  # a 16-byte aligned address that no refused call touches


def append(**kw):
    a = dict(qkv=P, ld=2560, T=4, pos=P, slot=P, pages=P, n_slots=2, max_pages=4, n_pages=8, prefix_len=0, kc=P, vc=P,
             cos=P, sin=P, table_len=64, nh=16, nkv=2, f16=1, q_out=P, ldq=2048, err=P, stream=None)
    a.update(kw)
    return L.lib().eg_op_kv_append_paged(*a.values())


@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(nkv=0), dict(nh=-1), dict(nh=2000), dict(n_slots=0), dict(max_pages=0), dict(n_pages=0),
    dict(n_pages=(1 << 27) + 1), dict(prefix_len=-1), dict(table_len=0), dict(qkv=None), dict(pos=None),
    dict(slot=None), dict(pages=None), dict(kc=None), dict(vc=None), dict(cos=None), dict(sin=None),
    dict(ld=2556), dict(ld=2562), dict(ldq=2044), dict(ldq=2050), dict(qkv=P + 4), dict(kc=P + 8), dict(vc=P + 2),
    dict(cos=P + 4), dict(sin=P + 4), dict(q_out=P + 4)])
def test_append_refusals(bad):
    assert append(**bad) == L.EG_ERR_ARG
    assert b"kv_append_paged" in L.lib().eg_last_error()


def test_append_of_no_rows_is_nothing():
    assert append(T=0) == L.EG_OK
    assert append(T=0, qkv=None, pos=None) == L.EG_OK


def attn_bytes(*dims):
    n = C.c_uint64(0)
    s = L.lib().eg_op_attn_shared_prefix_bytes(*dims, C.byref(n))
    return s, n.value


def attn(**kw):
    a = dict(q=P, ldq=2048, nseq=4, kc=P, vc=P, n_pages=64, prefix_pages=P, prefix_len=100, pages=P, max_pages=8,
             lens=P, max_len=128, nh=16, nkv=2, f16=1, out=P, ldo=2048, ws=P, ws_bytes=1 << 30, err=P, stream=None)
    a.update(kw)
    return L.lib().eg_op_attn_shared_prefix(*a.values())


@pytest.mark.parametrize("bad", [
    dict(nseq=0), dict(nseq=70000), dict(nh=0), dict(nkv=0), dict(nh=15), dict(nh=2048, nkv=1), dict(prefix_len=-1),
    dict(max_len=-1), dict(max_len=129), dict(prefix_len=1 << 29), dict(q=None), dict(kc=None), dict(vc=None),
    dict(lens=None), dict(out=None), dict(ws=None), dict(prefix_pages=None), dict(pages=None), dict(n_pages=0),
    dict(max_pages=-1), dict(ldq=2046), dict(ldq=2050), dict(ldo=2044), dict(ldo=2049), dict(q=P + 4), dict(kc=P + 8),
    dict(vc=P + 4), dict(out=P + 4), dict(ws=P + 8), dict(ws_bytes=64)])
def test_attention_refusals(bad):
    assert attn(**bad) == L.EG_ERR_ARG
    assert b"attn_shared_prefix" in L.lib().eg_last_error()


def test_attention_workspace_bytes():
    assert attn_bytes(0, 16, 2, 0, 0)[0] == L.EG_ERR_ARG
    assert L.lib().eg_op_attn_shared_prefix_bytes(1, 16, 2, 0, 0, None) == L.EG_ERR_ARG
    s, n = attn_bytes(16, 16, 2, 2048, 640)
    assert s == L.EG_OK and 16 * 16 * 130 * 4 <= n < 1 << 28
    assert attn_bytes(1, 16, 2, 0, 0) [1] >= 16
    # the size passed on is the size asked for
    assert attn(nseq=16, prefix_len=2048, max_len=128, ws_bytes=attn_bytes(16, 16, 2, 2048, 128)[1] - 1) == L.EG_ERR_ARG
    # sizes stay far below what the range of dimensions could overflow
    for dims in [(256, 32, 8, 1 << 20, 1 << 16), (65536, 16, 2, 100, 100)]:
        s, n = attn_bytes(*dims)
        assert s == L.EG_OK and n < 1 << 42


def sample(**kw):
    a = dict(logits=P, ld=100, rows=2, n=100, temp=P, top_k=P, top_p=P, min_p=P, r=P, ids=P, probs=P, stream=None)
    a.update(kw)
    return L.lib().eg_op_sample_filtered(*a.values())


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(n=0), dict(n=(1 << 28) + 1, ld=1 << 30), dict(ld=99),
                                 dict(logits=None), dict(r=None), dict(ids=None), dict(logits=P + 2)])
def test_sample_refusals(bad):
    assert sample(**bad) == L.EG_ERR_ARG
    assert b"sample_filtered" in L.lib().eg_last_error()


def test_sample_of_no_rows_is_nothing():
    assert sample(rows=0, logits=None, r=None, ids=None) == L.EG_OK


def test_wrappers_refuse_wrong_tensors():
    import torch
    f, i = torch.zeros, torch.int32
    cache = f(4, 16, 2, 128, dtype=torch.float16)
    good = dict(qkv=f(3, 2560), pos=f(3, dtype=i), slot=f(3, dtype=i), pages=f(1, 4, dtype=i), k_cache=cache,
                v_cache=cache, cos_t=f(8, 128), sin_t=f(8, 128), nh=16)
    for name, t in [("qkv", f(3, 2559)), ("qkv", f(3, 2560).half()), ("pos", f(3, dtype=torch.int64)),
                    ("slot", f(2, dtype=i)), ("k_cache", cache.float()), ("k_cache", f(4, 8, 2, 128).half()),
                    ("cos_t", f(8, 64)), ("pages", f(4, dtype=i)), ("qkv", f(2560, 3).t())]:
        with pytest.raises(ValueError, match="kv_append_paged"):
            K.kv_append_paged(**{**good, name: t})
    with pytest.raises(ValueError, match="CUDA"):
        K.kv_append_paged(**good)
    good = dict(q=f(2, 2048), k_cache=cache, v_cache=cache, prefix_pages=f(2, dtype=i), prefix_len=20,
                pages=f(2, 1, dtype=i), lens=f(2, dtype=i), max_len=16, out=f(2, 2048), ws=f(16, dtype=torch.uint8))
    for name, t in [("q", f(2, 2000)), ("lens", f(2)), ("pages", f(3, 1, dtype=i)), ("prefix_pages", f(1, dtype=i)),
                    ("out", f(1, 2048)), ("q", f(2, 2048).double()), ("v_cache", cache.float())]:
        with pytest.raises(ValueError, match="attn_shared_prefix"):
            K.attn_shared_prefix(**{**good, name: t})
    with pytest.raises(ValueError, match="CUDA"):
        K.attn_shared_prefix(**good)
    good = dict(logits=f(2, 50), r=f(2), ids=f(2, dtype=i))
    for name, t in [("logits", f(2, 50).half()), ("logits", f(50)), ("r", f(3)), ("ids", f(2)), ("temp", f(1)),
                    ("top_k", f(2)), ("probs", f(2).double())]:
        with pytest.raises(ValueError, match="sample_filtered"):
            K.sample_filtered(**{**good, name: t})


def test_sampling_definition():
    """Worked by hand: weights 4, 2, 1, 1 (logs), ties to the lower id."""
    x = np.log(np.array([1, 4, 2, 1], np.float32))
    ids = lambda **kw: [R.sample(x, r=r, **kw)[0] for r in (0.0, 0.49, 0.51, 0.74, 0.76, 0.87, 0.88, 1.0)]  # noqa: E731
    assert ids() == [1, 1, 2, 2, 0, 0, 3, 3]
    assert ids(k=2) == [1, 1, 1, 2, 2, 2, 2, 2]
    assert ids(p=0.6) == [1, 1, 1, 2, 2, 2, 2, 2]
    assert ids(minp=0.3) == [1, 1, 1, 2, 2, 2, 2, 2]
    assert ids(k=1) == [1] * 8 and ids(p=0.0) == [1] * 8
    assert R.sample(np.array([np.nan, -np.inf, -2e30], np.float32))[0] == R.EMPTY
    assert R.sample(np.array([1, np.inf, np.inf], np.float32), r=0.6) == (2, 0.5)
    assert R.sample(x, r=0.3, k=2)[1] == pytest.approx(4 / 6, rel=1e-6)


def test_attention_definition():
    v = np.arange(2 * 128, dtype=np.float64).reshape(2, 1, 128)
    o, _ = R.attention(np.zeros((2, 128)), np.zeros((2, 1, 128)), v)
    assert np.allclose(o, v.mean(0))
    assert R.attention(np.zeros((2, 128)), np.zeros((0, 1, 128)), np.zeros((0, 1, 128)))[0].tolist() == np.zeros((2, 128)).tolist()
    y, _ = R.rotate(np.eye(128)[:1], np.zeros((1, 128)), np.ones((1, 128)))  # a quarter turn
    assert y[0, 64] == 1 and abs(y).sum() == 1
