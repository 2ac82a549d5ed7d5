// eg_sample.cu -- sampling a token per row of logits with temperature, top-k,
// top-p and min-p filters and given random numbers.
//
// A row's tokens are put in TOPK_SELECT's order (value falling, ties to the
// lower id; NaN and values below -1e30 are never taken, kernels.js:775-776).
// With w_i = exp((x_i - max) / t) (t <= 0 reads as 1, as SAMPLE_TOPK does) each
// filter keeps a leading part of that order: top-k the first k, top-p the
// shortest part whose mass reaches p times the mass left by top-k, min-p the
// tokens with w >= min_p (w = 1 for the best one); one token at least stays.  The sample is
// the first token whose running mass reaches r times the mass kept.
//
// Masses are sums of integers (w in fixed point), so no order of additions
// changes a result.
#include <math.h>

#include "eg_common.cuh"
#include "eg_host.h"
#include "emberglass.h"

namespace eg {
namespace {

constexpr int kThreads = 1024;

struct SampleArgs {
  const float* logits;
  long long ld;
  int rows, n;
  const float* temp;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* r;
  uint32_t* ids;
  float* probs;
};

// Order-preserving integer of a candidate (-0 = +0), 0 for what is never taken.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (!(x >= -1e30f)) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct RowParams {
  double t, p, minp, r;
  int k;  // 0: off
};
__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int row) {
  RowParams q;
  const float t = a.temp ? __ldg(a.temp + row) : 1.f, p = a.top_p ? __ldg(a.top_p + row) : 1.f;
  const float m = a.min_p ? __ldg(a.min_p + row) : 0.f, r = __ldg(a.r + row);
  q.t = t > 0.f ? (double)t : 1.0;        // NaN too
  q.p = p < 1.f ? fmax((double)p, 0.0) : 1.0;
  q.minp = m > 0.f ? (double)m : 0.0;
  q.r = r > 0.f ? fmin((double)r, 1.0) : 0.0;
  q.k = a.top_k ? max(__ldg(a.top_k + row), 0) : 0;
  return q;
}

// w of a candidate; an infinite maximum takes all the mass
__device__ __forceinline__ double weight(float x, float xmax, double t) {
  return x == xmax ? 1.0 : exp(((double)x - (double)xmax) / t);
}

struct Cut {  // a leading part of the order: its size, its mass, its last token's key and place among equal keys
  long long n;
  unsigned long long mass;
  uint32_t key, tie;
};

struct GenericSmem {
  unsigned long long mass[256];
  uint32_t cnt[256];
  uint32_t key, tie;
  long long n;
  unsigned long long m;
  uint32_t red[32];
  unsigned long long red64[32];
};

// The shortest leading part with at least `count` tokens (by_mass = 0) or
// with a mass of at least `target` (by_mass = 1): a descent over the keys' four
// bytes, each level a histogram of the tokens that share the bytes above.
__device__ Cut generic_cut(const float* x, int n, float xmax, double t, double scale, int by_mass, long long count,
                           double target, GenericSmem& S) {
  uint32_t prefix = 0;
  unsigned long long base_m = 0;
  long long base_n = 0;
  for (int level = 0; level < 4; level++) {
    const int shift = 24 - 8 * level;
    for (int i = threadIdx.x; i < 256; i += kThreads) S.mass[i] = 0, S.cnt[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = __ldg(x + i);
      const uint32_t key = order_key(v);
      if (!key || (level && (key >> (shift + 8)) != prefix)) continue;
      const uint32_t b = (key >> shift) & 255;
      atomicAdd(&S.cnt[b], 1u);
      if (by_mass) atomicAdd(&S.mass[b], (unsigned long long)__double2ll_rn(weight(v, xmax, t) * scale));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int at = -1;
      for (int b = 255; b >= 0; b--) {
        if (!S.cnt[b]) continue;
        at = b;
        if (by_mass ? (double)(base_m + S.mass[b]) >= target : base_n + S.cnt[b] >= count) break;
        bool more = false;
        for (int c = b - 1; c >= 0; c--) more |= S.cnt[c] != 0;
        if (!more) break;  // rounding at the very end: the last token there is
        base_m += S.mass[b];
        base_n += S.cnt[b];
      }
      S.key = prefix << 8 | (uint32_t)at;
      S.n = base_n;
      S.m = base_m;
      S.tie = S.cnt[at];
    }
    __syncthreads();
    prefix = S.key;
    base_n = S.n;
    base_m = S.m;
    __syncthreads();
  }
  Cut c;
  c.key = prefix;
  const uint32_t equal = S.tie;
  const unsigned long long w = __double2ll_rn(weight(key_value(prefix), xmax, t) * scale);
  uint32_t j = equal;
  if (!by_mass) {
    j = (uint32_t)min((long long)equal, count - base_n);
  } else {
    uint32_t lo = 1, hi = equal;  // the first j with base + j w >= target
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if ((double)(base_m + mid * w) >= target) hi = mid;
      else lo = mid + 1;
    }
    j = lo;
  }
  c.tie = j;
  c.n = base_n + j;
  c.mass = base_m + j * w;
  return c;
}

// sums of a count and a mass over the CTA
__device__ void block_sums(long long& n, unsigned long long& m, GenericSmem& S) {
  unsigned long long a = (unsigned long long)n, b = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    S.red[threadIdx.x >> 5] = (uint32_t)a;
    S.red64[threadIdx.x >> 5] = b;
  }
  __syncthreads();
  a = b = 0;
  for (int i = 0; i < kThreads / 32; i++) a += S.red[i], b += S.red64[i];
  n = (long long)a;
  m = b;
}

__global__ void __launch_bounds__(kThreads) sample_generic_kernel(SampleArgs a) {
  __shared__ GenericSmem S;
  const int row = blockIdx.x, n = a.n;
  const float* x = a.logits + row * a.ld;
  const RowParams q = row_params(a, row);
  // the maximum and the number of candidates
  uint32_t kmax = 0;
  long long cand = 0;
  unsigned long long total = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) kmax = max(kmax, order_key(__ldg(x + i)));
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  if ((threadIdx.x & 31) == 0) S.red[threadIdx.x >> 5] = kmax;
  __syncthreads();
  for (int i = 0; i < kThreads / 32; i++) kmax = max(kmax, S.red[i]);
  if (!kmax) {  // nothing to take
    if (threadIdx.x == 0) {
      a.ids[row] = 0xffffffffu;
      if (a.probs) a.probs[row] = 0.f;
    }
    return;
  }
  const float xmax = key_value(kmax);
  const double scale = (double)(1ull << (62 - (32 - __clz(n))));  // n tokens of weight 1 stay below 2^62
  long long n_m = 0;  // min-p's part
  unsigned long long mass_m = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float v = __ldg(x + i);
    if (!(v >= -1e30f)) continue;
    const double w = weight(v, xmax, q.t);
    const unsigned long long m = __double2ll_rn(w * scale);
    cand++;
    total += m;
    if (w >= q.minp) n_m++, mass_m += m;
  }
  block_sums(cand, total, S);
  block_sums(n_m, mass_m, S);
  Cut best{cand, total, 0, 0};
  if (q.k > 0 && q.k < cand) best = generic_cut(x, n, xmax, q.t, scale, 0, q.k, 0.0, S);
  if (best.n < cand) {  // the mass of the first k (the descent by count sums none)
    long long nn = 0;
    unsigned long long mm = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = __ldg(x + i);
      if (order_key(v) > best.key) nn++, mm += __double2ll_rn(weight(v, xmax, q.t) * scale);
    }
    block_sums(nn, mm, S);
    best.mass = mm + best.tie * (unsigned long long)__double2ll_rn(weight(key_value(best.key), xmax, q.t) * scale);
  }
  if (q.p < 1.0) {
    const Cut c = generic_cut(x, n, xmax, q.t, scale, 1, 0, q.p * (double)best.mass, S);
    if (c.n < best.n) best = c;
  }
  if (n_m < best.n) best.n = n_m, best.mass = mass_m;
  if (best.n < 1) best.n = 1, best.mass = (unsigned long long)scale;
  const Cut c = generic_cut(x, n, xmax, q.t, scale, 1, 0, q.r * (double)best.mass, S);
  // the c.tie-th token with c.key: each thread counts its stretch of the row
  const int per = (n + kThreads - 1) / kThreads, i0 = min(n, (int)threadIdx.x * per), i1 = min(n, i0 + per);
  uint32_t mine = 0;
  for (int i = i0; i < i1; i++) mine += order_key(__ldg(x + i)) == c.key;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  __syncthreads();
  if (lane == 31) S.red[warp] = incl;
  __syncthreads();
  for (int w = 0; w < warp; w++) incl += S.red[w];
  if (incl >= c.tie && incl - mine < c.tie) {
    uint32_t left = c.tie - (incl - mine);
    for (int i = i0; i < i1; i++)
      if (order_key(__ldg(x + i)) == c.key && --left == 0) {
        a.ids[row] = (uint32_t)i;
        if (a.probs) a.probs[row] = (float)(weight(key_value(c.key), xmax, q.t) * scale / (double)best.mass);
        break;
      }
  }
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" {

EG_API eg_status eg_op_sample_filtered(const float* logits, int64_t ld, int rows, int n, const float* temp,
                                       const int* top_k, const float* top_p, const float* min_p, const float* r,
                                       uint32_t* ids, float* probs, void* stream) {
  if (rows < 0 || n < 1 || n > (1 << 28)) return fail(EG_ERR_ARG, "sample_filtered: need rows >= 0 and 1 <= n <= 2^28");
  if (ld < n) return fail(EG_ERR_ARG, "sample_filtered: row stride %lld below n = %d", (long long)ld, n);
  if (rows == 0) return EG_OK;
  if (!logits || !r || !ids) return fail(EG_ERR_ARG, "sample_filtered: null argument");
  if (reinterpret_cast<uintptr_t>(logits) & 3) return fail(EG_ERR_ARG, "sample_filtered: logits must be 4-byte aligned");
  SampleArgs a = {logits, ld, rows, n, temp, top_k, top_p, min_p, r, ids, probs};
  sample_generic_kernel<<<rows, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(EG_ERR_CUDA, "sample_filtered: %s", cudaGetErrorString(e));
  return EG_OK;
}

}  // extern "C"
