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


# ---- paged serving ops: the tensors carry the sizes and are checked against
# them.  A call's checks are one expression of cheap attribute reads; only when
# it fails are the tensors looked at one by one for the message.  The arguments
# go over as one packed block (eg_packed_*, every value 64 bits wide): ctypes'
# conversion of twenty arguments took 5 us of a call that launches in 3.
_fns = {}


def _packed(op, count):
    if op not in _fns:
        import ctypes as C
        import struct
        f = getattr(L.lib(), "eg_packed_" + op)
        f.restype, f.argtypes = C.c_int, [C.c_char_p]
        pack = struct.Struct(f"{count}q").pack
        _fns[op] = lambda *a: f(pack(*a))
    return _fns[op]


def _need(ok, op, what):
    if not ok:
        raise ValueError(f"{op}: {what}")


def _ld(t, stride):
    """Row stride of a 2-d tensor; a single row's says nothing, any multiple of 4 that spans it will do."""
    return stride[0] if t.shape[0] > 1 else (t.shape[1] + 3) // 4 * 4


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _check_rows(op, name, t, width):
    import torch
    _need(t.dtype is torch.float32 and t.dim() == 2 and t.shape[1] >= width and t.stride(1) == 1, op,
          f"{name} must be f32 rows of {width} contiguous values")


def _check_cache(op, k_cache, v_cache):
    import torch
    _need(k_cache.dim() == 4 and k_cache.shape[1] == 16 and k_cache.shape[3] == 128 and
          k_cache.dtype in (torch.float16, torch.float32) and k_cache.is_contiguous(), op,
          "caches must be contiguous [n_pages][16][nkv][128] of f16 or f32")
    _need(v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype and v_cache.is_contiguous(), op,
          "k_cache and v_cache differ in shape or type")


def _check_ints(op, name, t, *shape):
    import torch
    _need(t.dtype in (torch.int32, torch.uint32) and tuple(t.shape) == shape and t.is_contiguous(), op,
          f"{name} must be contiguous int32 {list(shape)}")


def _check_device(op, first, *others):
    import torch
    _need(first.is_cuda, op, "CUDA tensors required")
    for t in others:
        _need(t is None or t.device == first.device, op, "tensors are on different devices")
    _need(first.get_device() == torch.cuda.current_device(), op,
          f"tensors are on {first.device}, which is not the current device")


def _same_device(*tensors):
    """Whether all are CUDA tensors on the current device (None is skipped)."""
    import torch
    dev = torch.cuda.current_device() if tensors[0].is_cuda else -2
    for t in tensors:
        if t is not None and t.get_device() != dev:
            return False
    return True


def kv_append_paged(qkv, pos, slot, pages, k_cache, v_cache, cos_t, sin_t, nh, q_out=None, prefix_len=0, err=None,
                    stream=None):
    """RoPE + paged K/V rows of ragged tokens: row t of qkv [T][(nh + 2 nkv) * 128]
    is the token at position pos[t] of slot slot[t]; k and v go to row pos[t] -
    prefix_len of the slot's pages [n_slots][max_pages], the turned q to q_out.
    pos[t] < 0 pads; err (int32 device word) is set when an index is out of range."""
    import torch
    f32, i32 = torch.float32, torch.int32
    T, ks, ps, cs = qkv.shape[0], k_cache.shape, pages.shape, cos_t.shape
    st = qkv.stride()
    ldq = 0
    ok = (len(ks) == 4 and len(ps) == 2 and len(st) == 2 and qkv.dtype is f32 and st[1] == 1 and
          ks[1] == 16 and ks[3] == 128 and v_cache.shape == ks and v_cache.dtype is k_cache.dtype and
          (k_cache.dtype is torch.float16 or k_cache.dtype is f32) and k_cache.is_contiguous() and
          v_cache.is_contiguous() and qkv.shape[1] >= (nh + 2 * ks[2]) * 128 and
          pos.dtype is i32 and pos.shape == (T,) and pos.is_contiguous() and
          slot.dtype is i32 and slot.shape == (T,) and slot.is_contiguous() and
          (pages.dtype is i32 or pages.dtype is torch.uint32) and pages.is_contiguous() and
          len(cs) == 2 and cs[1] == 128 and cos_t.dtype is f32 and cos_t.is_contiguous() and
          sin_t.shape == cs and sin_t.dtype is f32 and sin_t.is_contiguous() and
          (err is None or (err.dtype is i32 and err.numel() == 1)))
    if ok and q_out is not None:
        sq = q_out.stride()
        ok = (len(sq) == 2 and sq[1] == 1 and q_out.dtype is f32 and q_out.shape[0] == T and
              q_out.shape[1] >= nh * 128)
        ldq = _ld(q_out, sq) if ok else 0
    if not (ok and _same_device(qkv, pos, slot, pages, k_cache, v_cache, cos_t, sin_t, q_out, err)):
        op = "kv_append_paged"
        _check_cache(op, k_cache, v_cache)
        _check_rows(op, "qkv", qkv, (nh + 2 * ks[2]) * 128)
        _need(len(ps) == 2, op, "pages must be [n_slots][max_pages]")
        for name, t, shape in (("pos", pos, (T,)), ("slot", slot, (T,)), ("pages", pages, ps)):
            _check_ints(op, name, t, *shape)
        for t in (cos_t, sin_t):
            _need(t.dtype is f32 and t.dim() == 2 and t.shape[1] == 128 and t.shape == cs and t.is_contiguous(), op,
                  "cos_t and sin_t must be contiguous f32 [positions][128]")
        if q_out is not None:
            _check_rows(op, "q_out", q_out, nh * 128)
            _need(q_out.shape[0] == T, op, "q_out must have a row for each of qkv's")
        _check_device(op, qkv, pos, slot, pages, k_cache, v_cache, cos_t, sin_t, q_out, err)
        _need(False, op, "pos and slot must be int32, err one int32")
    L.check(_packed("kv_append_paged", 22)(
        qkv.data_ptr(), _ld(qkv, st), T, pos.data_ptr(), slot.data_ptr(), pages.data_ptr(), ps[0], ps[1], ks[0],
        prefix_len, k_cache.data_ptr(), v_cache.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(), cs[0], nh, ks[2],
        k_cache.dtype is torch.float16, _ptr(q_out), ldq, _ptr(err), _st(stream) or 0))


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
    f32, i32 = torch.float32, torch.int32
    qs, ks, ps = q.shape, k_cache.shape, pages.shape
    st, so = q.stride(), out.stride()
    ok = (len(qs) == 2 and len(ks) == 4 and len(ps) == 2 and q.dtype is f32 and st[1] == 1 and qs[1] % 128 == 0 and
          out.dtype is f32 and out.shape == qs and so[1] == 1 and ks[1] == 16 and ks[3] == 128 and
          v_cache.shape == ks and v_cache.dtype is k_cache.dtype and
          (k_cache.dtype is torch.float16 or k_cache.dtype is f32) and k_cache.is_contiguous() and
          v_cache.is_contiguous() and lens.dtype is i32 and lens.shape == (qs[0],) and lens.is_contiguous() and
          (pages.dtype is i32 or pages.dtype is torch.uint32) and ps[0] == qs[0] and pages.is_contiguous() and
          ws.is_contiguous() and (err is None or (err.dtype is i32 and err.numel() == 1)))
    if ok and prefix_len > 0:
        ok = ((prefix_pages.dtype is i32 or prefix_pages.dtype is torch.uint32) and prefix_pages.is_contiguous() and
              prefix_pages.numel() * 16 >= prefix_len)
    if not (ok and _same_device(q, k_cache, v_cache, prefix_pages, pages, lens, out, ws, err)):
        op = "attn_shared_prefix"
        _check_cache(op, k_cache, v_cache)
        _need(q.dim() == 2 and qs[1] % 128 == 0, op, "q must be [nseq][nh * 128]")
        _check_rows(op, "q", q, qs[1])
        _check_rows(op, "out", out, qs[1])
        _need(out.shape == qs, op, "out must have q's shape")
        _check_ints(op, "lens", lens, qs[0])
        _need(len(ps) == 2, op, "pages must be [nseq][max_pages]")
        _check_ints(op, "pages", pages, qs[0], ps[1])
        if prefix_len > 0:
            _check_ints(op, "prefix_pages", prefix_pages, *prefix_pages.shape)
            _need(prefix_pages.numel() * 16 >= prefix_len, op, f"prefix_pages do not hold {prefix_len} rows")
        _need(ws.is_contiguous(), op, "ws must be contiguous")
        _check_device(op, q, k_cache, v_cache, prefix_pages, pages, lens, out, ws, err)
        _need(False, op, "lens must be int32, err one int32")
    L.check(_packed("attn_shared_prefix", 21)(
        q.data_ptr(), _ld(q, st), qs[0], k_cache.data_ptr(), v_cache.data_ptr(), ks[0], _ptr(prefix_pages), prefix_len,
        pages.data_ptr(), ps[1], lens.data_ptr(), max_len, qs[1] // 128, ks[2], k_cache.dtype is torch.float16,
        out.data_ptr(), _ld(out, so), ws.data_ptr(), ws.numel() * ws.element_size(), _ptr(err), _st(stream) or 0))


def sample_filtered(logits, r, ids, temp=None, top_k=None, top_p=None, min_p=None, probs=None, stream=None):
    """A token for each row of logits [rows][n] by the random numbers r[rows]:
    temperature, top-k, top-p and min-p (one device value per row each, None:
    1 / off) over the whole row.  ids[rows] int32, probs[rows] the chosen
    token's share of the mass kept.  A row with nothing to take gives id -1."""
    import torch
    f32, i32 = torch.float32, torch.int32
    ls, st = logits.shape, logits.stride()
    ok = len(ls) == 2 and logits.dtype is f32 and st[1] == 1 and ls[1] >= 1
    for t in (r, temp, top_p, min_p, probs):
        ok = ok and (t is None or (t.dtype is f32 and t.shape == ls[:1] and t.is_contiguous()))
    for t in (ids, top_k):
        ok = ok and (t is None or ((t.dtype is i32 or t.dtype is torch.uint32) and t.shape == ls[:1] and
                                   t.is_contiguous()))
    if not (ok and _same_device(logits, r, ids, temp, top_k, top_p, min_p, probs)):
        op = "sample_filtered"
        _need(len(ls) == 2 and ls[1] >= 1, op, "logits must be [rows][n]")
        _need(logits.dtype is f32 and st[1] == 1, op, "logits must be f32, contiguous in a row")
        for name, t in (("ids", ids), ("top_k", top_k)):
            if t is not None:
                _check_ints(op, name, t, ls[0])
        _check_device(op, logits, r, ids, temp, top_k, top_p, min_p, probs)
        _need(False, op, f"r, temp, top_p, min_p and probs must be contiguous f32 [{ls[0]}]")
    L.check(_packed("sample_filtered", 12)(
        logits.data_ptr(), st[0] if ls[0] > 1 else ls[1], ls[0], ls[1], _ptr(temp), _ptr(top_k), _ptr(top_p),
        _ptr(min_p), r.data_ptr(), ids.data_ptr(), _ptr(probs), _st(stream) or 0))
