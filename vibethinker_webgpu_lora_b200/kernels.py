"""Single-op entry points (the reference's exported WGSL kernels,
src/qwgpu/kernels.js) on device tensors.  Arguments are torch CUDA tensors
(or anything with data_ptr()); calls are asynchronous on `stream`
(torch.cuda.Stream, raw handle, or None for the current torch stream)."""
from __future__ import annotations

from . import _lib as L


def _st(stream):
    if stream is None:
        try:
            import torch
            return torch.cuda.current_stream().cuda_stream
        except Exception:
            return None
    return L.stream_ptr(stream)


def gemv_q4(x, w, scale, N, K, y, bias=None, accumulate=False, group=128, stream=None):
    L.check(L.lib().eg_op_gemv_q4(L.ptr(x), L.ptr(w), L.ptr(scale), L.ptr(bias), N, K, group,
                                  L.ptr(y), int(accumulate), _st(stream)))


def q4_stream_bytes(N, K, R=1):
    """Bytes of the device stream layout of an int4 matrix (R = 2: [gate;up])."""
    import ctypes as C
    n = C.c_uint64(0)
    L.check(L.lib().eg_op_q4_stream_bytes(N, K, R, C.byref(n)))
    return int(n.value)


def q4_to_stream(w, scale, N, K, out, R=1, stream=None):
    """Write the stream layout of a reference-layout int4 matrix into `out`
    (a uint8 device buffer of q4_stream_bytes(N, K, R) bytes), once."""
    L.check(L.lib().eg_op_q4_to_stream(L.ptr(w), L.ptr(scale), N, K, R, L.ptr(out), _st(stream)))


def gemv_q4_stream(x, ws, N, K, y, err, bias=None, pdl=False, stream=None):
    """GEMV4 over a matrix already in the stream layout: no conversion, no
    allocation.  err: int32 device word, zero before the call."""
    L.check(L.lib().eg_op_gemv_q4_stream(L.ptr(x), L.ptr(ws), L.ptr(bias), N, K, L.ptr(y), L.ptr(err),
                                         int(pdl), _st(stream)))


def q4_tc_bytes(N, K, R=1):
    """Bytes of the tensor-core (octet-major) layout of an int4 matrix."""
    import ctypes as C
    n = C.c_uint64(0)
    L.check(L.lib().eg_op_q4_tc_bytes(N, K, R, C.byref(n)))
    return int(n.value)


def q4_stream_to_tc(ws, N, K, out, R=1, stream=None):
    """Regroup a stream-layout matrix into the tensor-core layout, once."""
    L.check(L.lib().eg_op_q4_stream_to_tc(L.ptr(ws), N, K, R, L.ptr(out), _st(stream)))


def gemm_q4_stream(x, T, ws, N, K, y, bias=None, accumulate=False, use_tc=True, stream=None):
    """GEMM4 / GEMM4_ADD_T over a stream-layout matrix: y[t] (+)= W x[t]."""
    L.check(L.lib().eg_op_gemm_q4_stream(L.ptr(x), T, L.ptr(ws), L.ptr(bias), N, K, L.ptr(y),
                                         int(accumulate), int(use_tc), _st(stream)))


def gate_up_silu(x, w, scale, N, K, y, stream=None):
    L.check(L.lib().eg_op_gate_up_silu(L.ptr(x), L.ptr(w), L.ptr(scale), N, K, L.ptr(y), _st(stream)))


def gemv_q8(x, w, scale, N, K, y, stream=None):
    L.check(L.lib().eg_op_gemv_q8(L.ptr(x), L.ptr(w), L.ptr(scale), N, K, L.ptr(y), _st(stream)))


def rmsnorm(x, g, K, eps, f16, y, stream=None):
    L.check(L.lib().eg_op_rmsnorm(L.ptr(x), L.ptr(g), K, eps, int(f16), L.ptr(y), _st(stream)))


def rope_qk(q, k, nq, nkv, pos, cos_t, sin_t, f16, stream=None):
    L.check(L.lib().eg_op_rope_qk(L.ptr(q), L.ptr(k), nq, nkv, pos, L.ptr(cos_t), L.ptr(sin_t),
                                  int(f16), _st(stream)))


def attn_prefill(qkv, T, k_cache, v_cache, cos_t, sin_t, nh, nkv, q_start, max_ctx, kv_f16, out, stream=None):
    """ROPE_T + K/V rows + ATTN_PREFILL_BLOCK of one prefill pass (qkv rotated in place)."""
    L.check(L.lib().eg_op_attn_prefill(L.ptr(qkv), T, L.ptr(k_cache), L.ptr(v_cache), L.ptr(cos_t),
                                       L.ptr(sin_t), nh, nkv, q_start, max_ctx, int(kv_f16), L.ptr(out),
                                       _st(stream)))


def attn_decode(qkv, k_cache, v_cache, cos_t, sin_t, nh, nkv, pos, max_ctx, kv_f16, out, chunk=0,
                stream=None):
    L.check(L.lib().eg_op_attn_decode(L.ptr(qkv), L.ptr(k_cache), L.ptr(v_cache), L.ptr(cos_t),
                                      L.ptr(sin_t), nh, nkv, pos, max_ctx, int(kv_f16), chunk,
                                      L.ptr(out), _st(stream)))


def embed(w, scale, id_dev, H, out, stream=None):
    L.check(L.lib().eg_op_embed(L.ptr(w), L.ptr(scale), L.ptr(id_dev), H, L.ptr(out), _st(stream)))


def lora_a(x, A, K, rank, d, stream=None):
    L.check(L.lib().eg_op_lora_a(L.ptr(x), L.ptr(A), K, rank, L.ptr(d), _st(stream)))


def argmax(logits, n, out, stream=None):
    L.check(L.lib().eg_op_argmax(L.ptr(logits), n, L.ptr(out), _st(stream)))


def topk(logits, n, k, ids, vals, stream=None):
    L.check(L.lib().eg_op_topk(L.ptr(logits), n, k, L.ptr(ids), L.ptr(vals), _st(stream)))


def sample_topk(ids, vals, k, temp, r, out, stream=None):
    L.check(L.lib().eg_op_sample_topk(L.ptr(ids), L.ptr(vals), k, temp, r, L.ptr(out), _st(stream)))


# ---- paged serving ops: tensors carry the sizes and are checked against them
def _need(ok, op, what):
    if not ok:
        raise ValueError(f"{op}: {what}")


def _rows(op, name, t, width):
    """A 2-d f32 tensor whose rows of at least `width` values are contiguous."""
    import torch
    _need(t.dtype is torch.float32 and t.dim() == 2 and t.shape[1] >= width and t.stride(1) == 1, op,
          f"{name} must be f32 rows of {width} contiguous values")
    # a single row's stride says nothing: any multiple of 4 that spans it will do
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 3) // 4 * 4


def _cache(op, k_cache, v_cache):
    import torch
    _need(k_cache.dim() == 4 and k_cache.shape[1] == 16 and k_cache.shape[3] == 128 and
          k_cache.dtype in (torch.float16, torch.float32) and k_cache.is_contiguous(), op,
          "caches must be contiguous [n_pages][16][nkv][128] of f16 or f32")
    _need(v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype and v_cache.is_contiguous(), op,
          "k_cache and v_cache differ in shape or type")
    return k_cache.shape[0], k_cache.shape[2], int(k_cache.dtype is torch.float16)


def _ints(op, name, t, *shape):
    import torch
    _need(t.dtype in (torch.int32, torch.uint32) and tuple(t.shape) == shape and t.is_contiguous(), op,
          f"{name} must be contiguous int32 {list(shape)}")


def _launch(op, stream, first, *others):
    """The stream to launch on, all tensors being on the current device."""
    import torch
    dev = first.device
    _need(dev.type == "cuda", op, "CUDA tensors required")
    for t in others:
        _need(t is None or t.device == dev, op, "tensors are on different devices")
    _need(dev.index == torch.cuda.current_device(), op, f"tensors are on {dev}, which is not the current device")
    return _st(stream)


def kv_append_paged(qkv, pos, slot, pages, k_cache, v_cache, cos_t, sin_t, nh, q_out=None, prefix_len=0, err=None,
                    stream=None):
    """RoPE + paged K/V rows of ragged tokens: row t of qkv [T][(nh + 2 nkv) * 128]
    is the token at position pos[t] of slot slot[t]; k and v go to row pos[t] -
    prefix_len of the slot's pages [n_slots][max_pages], the turned q to q_out.
    pos[t] < 0 pads; err (int32 device word) is set when an index is out of range."""
    import torch
    op = "kv_append_paged"
    n_pages, nkv, f16 = _cache(op, k_cache, v_cache)
    T = qkv.shape[0]
    ld = _rows(op, "qkv", qkv, (nh + 2 * nkv) * 128)
    _ints(op, "pos", pos, T)
    _ints(op, "slot", slot, T)
    _need(pages.dim() == 2, op, "pages must be [n_slots][max_pages]")
    _ints(op, "pages", pages, *pages.shape)
    _need(cos_t.dtype is torch.float32 and cos_t.dim() == 2 and cos_t.shape[1] == 128 and cos_t.is_contiguous() and
          sin_t.dtype is torch.float32 and sin_t.shape == cos_t.shape and sin_t.is_contiguous(), op,
          "cos_t and sin_t must be contiguous f32 [positions][128]")
    ldq = 0
    if q_out is not None:
        ldq = _rows(op, "q_out", q_out, nh * 128)
        _need(q_out.shape[0] == T, op, "q_out must have a row for each of qkv's")
    if err is not None:
        _need(err.dtype is torch.int32 and err.numel() == 1, op, "err must be one int32")
    st = _launch(op, stream, qkv, pos, slot, pages, k_cache, v_cache, cos_t, sin_t, q_out, err)
    L.check(L.lib().eg_op_kv_append_paged(
        qkv.data_ptr(), ld, T, pos.data_ptr(), slot.data_ptr(), pages.data_ptr(), pages.shape[0], pages.shape[1],
        n_pages, prefix_len, k_cache.data_ptr(), v_cache.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(),
        cos_t.shape[0], nh, nkv, f16, L.ptr(q_out), ldq, L.ptr(err), st))


def attn_shared_prefix_bytes(nseq, nh, nkv, prefix_len, max_len):
    """Bytes of attn_shared_prefix's workspace."""
    import ctypes as C
    n = C.c_uint64(0)
    L.check(L.lib().eg_op_attn_shared_prefix_bytes(nseq, nh, nkv, prefix_len, max_len, C.byref(n)))
    return int(n.value)


def attn_shared_prefix(q, k_cache, v_cache, prefix_pages, prefix_len, pages, lens, max_len, out, ws, err=None,
                       stream=None):
    """One decode token of each of nseq sequences over a shared prefix: q
    [nseq][nh * 128] attends over prefix_len rows of prefix_pages, then lens[b]
    (<= max_len) rows of pages[b]; the prefix is computed once for all.  lens[b]
    < 0 pads (out row left as it was).  ws: attn_shared_prefix_bytes(...) bytes
    (uint8), one for each call that may overlap."""
    import torch
    op = "attn_shared_prefix"
    n_pages, nkv, f16 = _cache(op, k_cache, v_cache)
    _need(q.dim() == 2 and q.shape[1] % 128 == 0, op, "q must be [nseq][nh * 128]")
    nseq, width = q.shape
    ldq = _rows(op, "q", q, width)
    ldo = _rows(op, "out", out, width)
    _need(out.shape[0] == nseq, op, "out must have a row for each of q's")
    _ints(op, "lens", lens, nseq)
    _need(pages.dim() == 2, op, "pages must be [nseq][max_pages]")
    _ints(op, "pages", pages, nseq, pages.shape[1])
    if prefix_len > 0:
        _ints(op, "prefix_pages", prefix_pages, *prefix_pages.shape)
        _need(prefix_pages.numel() * 16 >= prefix_len, op, f"prefix_pages do not hold {prefix_len} rows")
    _need(ws.is_contiguous(), op, "ws must be contiguous")
    if err is not None:
        _need(err.dtype is torch.int32 and err.numel() == 1, op, "err must be one int32")
    st = _launch(op, stream, q, k_cache, v_cache, prefix_pages, pages, lens, out, ws, err)
    L.check(L.lib().eg_op_attn_shared_prefix(
        q.data_ptr(), ldq, nseq, k_cache.data_ptr(), v_cache.data_ptr(), n_pages, L.ptr(prefix_pages), prefix_len,
        pages.data_ptr(), pages.shape[1], lens.data_ptr(), max_len, width // 128, nkv, f16, out.data_ptr(), ldo,
        ws.data_ptr(), ws.numel() * ws.element_size(), L.ptr(err), st))


def sample_filtered(logits, r, ids, temp=None, top_k=None, top_p=None, min_p=None, probs=None, stream=None):
    """A token for each row of logits [rows][n] by the random numbers r[rows]:
    temperature, top-k, top-p and min-p (one device value per row each, None:
    1 / off) over the whole row.  ids[rows] int32, probs[rows] the chosen
    token's share of the mass kept.  A row with nothing to take gives id -1."""
    import torch
    op = "sample_filtered"
    _need(logits.dim() == 2 and logits.shape[1] >= 1, op, "logits must be [rows][n]")
    rows, n = logits.shape
    _need(logits.dtype is torch.float32 and logits.stride(1) == 1, op, "logits must be f32, contiguous in a row")
    ld = logits.stride(0) if rows > 1 else n
    _ints(op, "ids", ids, rows)
    for name, t in (("r", r), ("temp", temp), ("top_p", top_p), ("min_p", min_p), ("probs", probs)):
        _need(t is None or (t.dtype is torch.float32 and t.shape == (rows,) and t.is_contiguous()), op,
              f"{name} must be f32 [{rows}]")
    if top_k is not None:
        _ints(op, "top_k", top_k, rows)
    st = _launch(op, stream, logits, r, ids, temp, top_k, top_p, min_p, probs)
    L.check(L.lib().eg_op_sample_filtered(logits.data_ptr(), ld, rows, n, L.ptr(temp), L.ptr(top_k), L.ptr(top_p),
                                          L.ptr(min_p), r.data_ptr(), ids.data_ptr(), L.ptr(probs), st))
