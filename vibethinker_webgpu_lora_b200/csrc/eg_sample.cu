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
#include <cooperative_groups.h>
#include <math.h>
#include <algorithm>

#include "eg_common.cuh"
#include "eg_host.h"
#include "emberglass.h"

namespace eg {
namespace {


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
  double t, p, minp, cut, r;  // cut: how far below the maximum min_p reaches, in x / t
  int k;  // 0: off
};
__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int row) {
  RowParams q;
  const float t = a.temp ? __ldg(a.temp + row) : 1.f, p = a.top_p ? __ldg(a.top_p + row) : 1.f;
  const float m = a.min_p ? __ldg(a.min_p + row) : 0.f, r = __ldg(a.r + row);
  q.t = t > 0.f ? (double)t : 1.0;        // NaN too
  q.p = p < 1.f ? fmax((double)p, 0.0) : 1.0;
  q.minp = m > 0.f ? (double)m : 0.0;
  q.cut = m > 0.f ? -log((double)m) : INFINITY;
  q.r = r > 0.f ? fmin((double)r, 1.0) : 0.0;
  q.k = a.top_k ? max(__ldg(a.top_k + row), 0) : 0;
  return q;
}

// One copy of the 64-bit exponential: inlined at each use it crowds the
// registers of the passes and the instruction cache.
__device__ __noinline__ double exp64(double x) { return exp(x); }

// w of a candidate; an infinite maximum takes all the mass
__device__ __forceinline__ double weight(float x, float xmax, double t) {
  return x == xmax ? 1.0 : exp64(((double)x - (double)xmax) / t);
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
template <int kThreads>
__device__ Cut generic_cut(const float* x, int n, float xmax, double t, double scale, int by_mass, long long count,
                           double target, GenericSmem& S) {
  uint32_t prefix = 0;
  unsigned long long base_m = 0;
  long long base_n = 0;
  for (int level = 0; level < 4; level++) {
    const int shift = 24 - 8 * level;
    for (int i = threadIdx.x; i < 256; i += kThreads) S.mass[i] = 0, S.cnt[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kThreads) {
      const int i = i0 + threadIdx.x;
      const float v = i < n ? __ldg(x + i) : -INFINITY;
      const uint32_t key = order_key(v);
      const bool in = key && (!level || (key >> (shift + 8)) == prefix);
      const uint32_t vote = __ballot_sync(0xffffffffu, in), one = vote & (0u - vote);
      if (!vote) continue;
      // many equal logits: one atomic for the warp
      const uint32_t key1 = __shfl_sync(0xffffffffu, key, __ffs(vote) - 1);
      const bool same = __all_sync(0xffffffffu, !in || key == key1);
      if (!in || (same && !((one >> (threadIdx.x & 31)) & 1))) continue;
      const uint32_t b = (key >> shift) & 255, many = same ? __popc(vote) : 1;
      atomicAdd(&S.cnt[b], many);
      if (by_mass) atomicAdd(&S.mass[b], many * (unsigned long long)__double2ll_rn(weight(v, xmax, t) * scale));
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
template <int kThreads>
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

// The whole row by one CTA, from global memory: right for every row, and the
// path of those that the histogram form below leaves (an infinite maximum,
// more than kList tokens in the bins that decide).
template <int kThreads>
__device__ __noinline__ void sample_generic(const SampleArgs& a, int row, GenericSmem& S) {
  const int n = a.n;
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
  block_sums<kThreads>(cand, total, S);
  block_sums<kThreads>(n_m, mass_m, S);
  Cut best{cand, total, 0, 0};
  if (q.k > 0 && q.k < cand) best = generic_cut<kThreads>(x, n, xmax, q.t, scale, 0, q.k, 0.0, S);
  if (best.n < cand) {  // the mass of the first k (the descent by count sums none)
    long long nn = 0;
    unsigned long long mm = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = __ldg(x + i);
      if (order_key(v) > best.key) nn++, mm += __double2ll_rn(weight(v, xmax, q.t) * scale);
    }
    block_sums<kThreads>(nn, mm, S);
    best.mass = mm + best.tie * (unsigned long long)__double2ll_rn(weight(key_value(best.key), xmax, q.t) * scale);
  }
  if (q.p < 1.0) {
    const Cut c = generic_cut<kThreads>(x, n, xmax, q.t, scale, 1, 0, q.p * (double)best.mass, S);
    if (c.n < best.n) best = c;
  }
  if (n_m < best.n) best.n = n_m, best.mass = mass_m;
  if (best.n < 1) best.n = 1, best.mass = (unsigned long long)scale;
  const Cut c = generic_cut<kThreads>(x, n, xmax, q.t, scale, 1, 0, q.r * (double)best.mass, S);
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

// ======================================================================
// Histogram form: a cluster of CTAs holds one row in shared memory
// ======================================================================
// Bins are equal steps of x below the maximum.  A token's weight is
// 2^-26 q e^(-b step): b its bin, q = 2^26 e^-u an integer, u its distance from
// the bin's middle.  The histogram holds each bin's count and sum of q; in the
// usual form q stays within 2^26 +- 2^22 and two 32-bit shared-memory atomics
// take the count and, modulo 2^32, the bits of kRound + q - 2^26: with the count
// they give the sum of q above 2^26 - 2^22 (below 2^23 each: 512 tokens of a CTA
// in one bin cannot overflow it; rows with more are counted again, and rows with
// steps of x / t above 1/16 at once, with 64-bit atomics: 256 rows of 151,936 118 us
// in the usual form, 210 as bf16 values, 302 with a tenth of the tokens at -1e9).
// The two atomics, 4 cycles of an SM each for a warp, bound the pass (38,000
// tokens a CTA: 5.2 us).  The leader CTA turns the merged bins into running
// counts and masses, which fix each filter's and the sample's bin; only the tokens
// of those few bins are gathered and put in order, in the same integers.
// Tokens past the last bin (64 below the maximum in x / t or more) weigh
// nothing: 2^20 of them are 2^-72 of the best token.
namespace cg = cooperative_groups;

constexpr int kBins = 2048;        // the last one: past the range
constexpr int kList = 2048;        // gathered tokens
constexpr int kCountMost = 384;    // of them put in order by counting
// Most tokens that a CTA stages: with an SM to itself, or as one of two.
constexpr int kSliceAlone = 38912, kSlice = 15872;
constexpr int kHits = 8192, kStagedHits = 4096;  // ids that a pass may pick before they are checked
constexpr int kQBits = 26;
constexpr uint32_t kQBase = (1u << kQBits) - (1u << 22);
constexpr uint32_t kDense = 512;   // tokens of a CTA in one bin, at most, in the usual form
constexpr unsigned long long kCountOne = 1ull << 46;
constexpr int kSliceMost = (1 << 18) - 1;  // tokens of a CTA, at most: what a count above bit 46 holds, and q < 2^28 below it
// Tokens of each of a row's c CTAs, in whole 16-byte pieces.
__host__ __device__ __forceinline__ int slice_of(int n, int c) { return ((n + c - 1) / c + 3) & ~3; }
constexpr float kRound = 12582912.f;  // 1.5 2^23: x + kRound rounds |x| < 2^22 to an integer in the low bits
constexpr uint32_t kRoundBits = 0x4B400000u;
constexpr uint32_t kPartBase = kRoundBits - (1u << 22);  // of a token's part of a sum, what q - kQBase does not hold

struct Ranges {  // bins [lo, hi] of: top-k, top-p, min-p, the sample (lo > hi: none)
  int lo[4], hi[4], redo;
  int n;                // the same as n windows |x - mid| <= half of values, a little wide
  float mid[4], half[4];
};

struct __align__(16) FastSmem {
  union {
    struct {
      uint32_t cnt[kBins], sum[kBins];
    };
    unsigned long long hist[kBins];  // 64-bit form: count << 46 | sum of q, of kSliceMost tokens at most
    double above[kBins];             // then, in the leader, the mass above each bin
  };
  uint32_t count_above[kBins];
  unsigned long long list[kList];    // order key << 32 | ~id: falling is TOPK_SELECT's order
  uint32_t n_list;
  float mx, mn;
  float red[2][32];
  double wsum[32];
  uint32_t wcnt[32];
  unsigned long long lsum[32];
  double unit[4];
  int cross[6], dense;
  Ranges rg;
  // the leader's last reductions
  double z, mass_p, mass_m, mass;
  unsigned long long best;
  uint32_t n_p, n_m;
};

// Bin r's middle is top - r width.  In the usual form top (the maximum, rounded
// up) and width are multiples of 2^-24 of a power of two above every middle, so
// each middle is an f32 without rounding.
struct Bins {
  float xmax, top, width, inv_width, inv_t;
  bool poly;          // steps of x / t up to 1/16: e^z by its series
  double step, lead;  // width / t, (top - xmax) / t
};

// kRound + a candidate's bin, the integer nearest (top - x) / width
__device__ __forceinline__ float bin_place(const Bins& B, float x) { return fmaf(B.top - x, B.inv_width, kRound); }
__device__ __forceinline__ bool in_range(float place) { return place <= kRound + (kBins - 2); }
__device__ __forceinline__ int bin_index(float place) { return __float_as_int(place) - (int)kRoundBits; }
// kRound + 2^26 (e^z - 1), rounded, of a candidate: z = (x - middle) / t, |z| <=
// 1/32 (a little more by place's rounding).  x - middle and z are rounded once
// each, so z is right to 2^-23; z (1 + z (1/2 + z (1/6 + z / 24))) leaves z^5 /
// 120, 0.02 of 2^-26; fused as written, so that every caller gets the same
// integer.
__device__ __forceinline__ float bin_part(const Bins& B, float x, float place) {
  constexpr float kOne = (float)(1 << kQBits);
  const float z = __fmul_rn(__fsub_rn(x, fmaf(kRound - place, B.width, B.top)), B.inv_t);
  float y = fmaf(z, kOne / 24.f, kOne / 6.f);
  y = fmaf(z, y, kOne / 2.f);
  y = fmaf(z, y, kOne);
  return fmaf(z, y, kRound);
}
__device__ __forceinline__ int bin_of(const Bins& B, float x, uint32_t& q) {
  const float p = bin_place(B, x);
  if (!in_range(p)) {
    q = 0;
    return kBins - 1;
  }
  if (B.poly) {
    q = (1u << kQBits) + __float_as_int(bin_part(B, x, p)) - (int)kRoundBits;
  } else {  // |u| up to 1.26: in 64 bits, f32 would leave 2^-23 of the weight; q < 2^27.9
    const double u = ((double)B.top - (double)x - (double)(p - kRound) * B.width) * (B.step / B.width);
    q = (uint32_t)__double2ll_rn(exp64(-u) * (double)(1 << kQBits));
  }
  return bin_index(p);
}

// The weight of q = 1 in bin b; units[j]: of bin j (4 of them).
__device__ __forceinline__ double bin_unit(const Bins& B, const double* units, int b) {
  return exp64(-(double)(b & ~3) * B.step) * units[b & 3];
}
// sums over the warps before this one and over all, of one value a warp in shared memory
template <int kThreads, typename T>
__device__ __forceinline__ void warp_sums(const T* v, T& before, T& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = lane < kThreads / 32 ? v[lane] : T(0), y = lane < warp ? x : T(0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    x += __shfl_xor_sync(0xffffffffu, x, o);
    y += __shfl_xor_sync(0xffffffffu, y, o);
  }
  before = y;
  all = x;
}

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_async16g(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src)
               : "memory");
}

// All CTAs of a row (a cluster of one: its barrier costs 0.3 us more than the CTA's own).
__device__ __forceinline__ void sync_row(cg::cluster_group& cl, int C) {
  if (C > 1) cl.sync();
  else __syncthreads();
}

// list[0 .. np) (np a power of two from 64 to kList) into falling order: 32
// pairs a warp in registers and shuffles, shared memory where a step spans
// more than a warp's 64 values.
template <int kThreads>
__device__ __forceinline__ void bitonic_falling(unsigned long long* list, int np) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto inside = [&](int size, int dmax) {  // the steps of distances dmax <= 32 .. 1 of one size
    for (int base = 64 * warp; base < np; base += 2 * kThreads) {
      unsigned long long x = list[base + lane], y = list[base + 32 + lane];
      for (int d = dmax; d > 0; d /= 2) {
        if (d == 32) {
          const bool fall = ((base + lane) & size) == 0;
          if ((x < y) == fall) {
            const unsigned long long t = x;
            x = y;
            y = t;
          }
        } else {
          const unsigned long long px = __shfl_xor_sync(0xffffffffu, x, d), py = __shfl_xor_sync(0xffffffffu, y, d);
          const bool low = (lane & d) == 0;
          const bool fx = ((base + lane) & size) == 0, fy = ((base + 32 + lane) & size) == 0;
          if ((x < px) == (low == fx)) x = px;  // the pair's larger value where falling, at its lower place
          if ((y < py) == (low == fy)) y = py;
        }
      }
      list[base + lane] = x;
      list[base + 32 + lane] = y;
    }
  };
  for (int size = 2; size <= np; size *= 2) {
    for (int d = size / 2; d > 32; d /= 2) {
      __syncthreads();
      for (int t = threadIdx.x; t < np / 2; t += kThreads) {
        const int i = 2 * t - (t & (d - 1)), k = i + d;
        const unsigned long long x = list[i], y = list[k];
        if ((x < y) == ((i & size) == 0)) {
          list[i] = y;
          list[k] = x;
        }
      }
      __syncthreads();
    }
    inside(size, min(32, size / 2));
    if (size >= 64) __syncthreads();
    else __syncwarp();
  }
  __syncthreads();
}

// The leader's part between the two passes: merged bins to running counts and
// masses (S.above, S.count_above) and the bins that decide (S.rg), or the wish
// for the 64-bit form.
template <int kThreads>
__device__ __forceinline__ void leader_ranges(FastSmem& S, cg::cluster_group& cl, const Bins& B, const RowParams& P, int C,
                                              bool wide, double e4, double cut_pos) {
  constexpr int kPer = kBins / kThreads;  // consecutive bins of a thread: 2 or 4
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned long long q[kPer];
  uint32_t cnt[kPer];
  double m[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j++) q[j] = 0, cnt[j] = 0;
  if (tid < 6) S.cross[tid] = kBins;
  if (wide) {
    for (int c = 0; c < C; c++) {
      const unsigned long long* h = cl.map_shared_rank(&S, c)->hist + tid * kPer;
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        q[j] += h[j] & (kCountOne - 1);
        cnt[j] += (uint32_t)(h[j] >> 46);
      }
    }
  } else {
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < 8; c++) {  // all remote loads in flight
      if (c >= C) break;
      const FastSmem* R = c == 0 ? &S : cl.map_shared_rank(&S, c);  // the leader is rank 0
#pragma unroll
      for (int j = 0; j < kPer; j += 2) {
        const uint2 n = *reinterpret_cast<const uint2*>(R->cnt + tid * kPer + j);
        const uint2 v = *reinterpret_cast<const uint2*>(R->sum + tid * kPer + j);
        cnt[j] += n.x;
        cnt[j + 1] += n.y;
        q[j] += (unsigned long long)n.x * kQBase + (v.x - n.x * kPartBase);
        q[j + 1] += (unsigned long long)n.y * kQBase + (v.y - n.y * kPartBase);
        most = max(most, max(n.x, n.y));
      }
    }
    if (most > kDense) S.dense = 1;
  }
  double ms = 0.0;
  uint32_t cs = 0;
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    m[j] = (double)q[j] * (e4 * S.unit[(tid * kPer + j) & 3]);
    ms += m[j];
    cs += cnt[j];
  }
  double mi = ms;
  uint32_t ci = cs;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, mi, o);
    const uint32_t w = __shfl_up_sync(0xffffffffu, ci, o);
    if (lane >= o) mi += v, ci += w;
  }
  // the last bin with tokens: where a target at the very end falls
  int last = -1;
#pragma unroll
  for (int j = 0; j < kPer; j++)
    if (cnt[j]) last = tid * kPer + j;
  last = __reduce_max_sync(0xffffffffu, last);
  if (lane == 31) S.wsum[warp] = mi, S.wcnt[warp] = ci, S.red[0][warp] = (float)last;
  __syncthreads();  // every thread has read the bins; the sums are there
  if (!wide && S.dense) {
    if (tid == 0) S.rg.redo = 1;
    return;
  }
  double mb, total, ab[kPer];
  uint32_t cb, ncand, ca[kPer];
  warp_sums<kThreads>(S.wsum, mb, total);
  warp_sums<kThreads>(S.wcnt, cb, ncand);
  last = (int)warp_max(lane < kThreads / 32 ? fmaxf(S.red[0][lane], 0.f) : 0.f);
  double am = mb + (mi - ms);
  uint32_t ac = cb + (ci - cs);
  const bool k_on = P.k > 0 && (uint32_t)P.k < ncand;
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    ab[j] = am;
    ca[j] = ac;
    S.above[tid * kPer + j] = am;
    S.count_above[tid * kPer + j] = ac;
    am += m[j];
    ac += cnt[j];
    if (k_on && ca[j] < (uint32_t)P.k && (uint32_t)P.k <= ac) S.cross[0] = tid * kPer + j;
  }
  // the first bin with tokens whose inclusive mass reaches a target
  auto cross_mass = [&](double t, int slot) {
#pragma unroll
    for (int j = 0; j < kPer; j++)
      if (cnt[j] && ab[j] + m[j] >= t) {
        atomicMin(&S.cross[slot], tid * kPer + j);
        break;
      }
  };
  __syncthreads();
  auto mass_above = [&](int b) { return b < kBins ? S.above[b] : total; };
  const int kb = S.cross[0];
  const double z_lo = k_on ? mass_above(kb) : total, z_hi = k_on ? mass_above(kb + 1) : total;
  int p_lo = 1, p_hi = 0, m_lo = 1, m_hi = 0;  // none
  double lo = z_lo, hi = z_hi;
  if (P.p < 1.0) {
    cross_mass(P.p * z_lo * (1.0 - 1e-12), 1);
    cross_mass(P.p * z_hi * (1.0 + 1e-12), 2);
    __syncthreads();
    p_lo = min(S.cross[1], last);
    p_hi = min(S.cross[2], last);
    lo = fmin(lo, mass_above(p_lo));
    hi = fmin(hi, mass_above(p_hi + 1));
  }
  if (P.minp > 0.0) {
    if (cut_pos < kBins - 2) {
      m_lo = max(0, (int)rint(cut_pos - 0.01));
      m_hi = max(0, min(kBins - 2, (int)rint(cut_pos + 0.01)));
      lo = fmin(lo, mass_above(m_lo));
      hi = fmin(hi, mass_above(m_hi + 1));
    }
  }
  hi = fmax(hi, 1.0);  // one token at least
  cross_mass(P.r * lo * (1.0 - 1e-12), 3);
  cross_mass(P.r * hi * (1.0 + 1e-12), 4);
  __syncthreads();
  if (tid < 4) {
    // a bin's tokens lie within half a width of its middle, give or take the rounding of a place
    const int wl = tid == 0 ? min(S.cross[3], last) : tid == 1 ? p_lo : tid == 2 ? (k_on ? kb : 1) : m_lo;
    const int wh = tid == 0 ? min(S.cross[4], last) : tid == 1 ? p_hi : tid == 2 ? (k_on ? kb : 0) : m_hi;
    const double slack = 0.01 * B.width + 0x1p-21 * (fabs((double)B.xmax) + (wh + 1.0) * B.width);
    const uint32_t vote = __ballot_sync(0xfu, wl <= wh);
    const int at = __popc(vote & ((1u << tid) - 1));
    if (wl <= wh) {
      // x - mid is rounded in the pass: so are the ends here, and rounding keeps their order
      const float from = __double2float_rd((double)B.top - (wh + 0.5) * B.width - slack);
      const float to = __double2float_ru((double)B.top - (wl - 0.5) * B.width + slack);
      const float mid = 0.5f * from + 0.5f * to;
      S.rg.mid[at] = mid;
      S.rg.half[at] = fmaxf(mid - from, to - mid);
    }
    if (tid == 0) S.rg.n = __popc(vote);
  }
  if (tid == 32) {
    Ranges& R = S.rg;
    R.lo[0] = k_on ? kb : 1, R.hi[0] = k_on ? kb : 0;
    R.lo[1] = p_lo, R.hi[1] = p_hi;
    R.lo[2] = m_lo, R.hi[2] = m_hi;
    R.lo[3] = min(S.cross[3], last), R.hi[3] = min(S.cross[4], last);
    R.redo = 0;
    S.z = total;
    S.n_p = S.n_m = 0xffffffffu;
    S.best = ~0ull;
  }
}

// The leader's last part: place and running mass of each gathered token (kMine
// consecutive ones a thread), the cuts of the filters, the sample.
template <int kThreads, int kMine>
__device__ __forceinline__ void finish_row(const SampleArgs& a, int row, FastSmem& S, const Bins& B, const RowParams& P,
                                           const unsigned long long* list, int nl, float* xs) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned long long* before = reinterpret_cast<unsigned long long*>(xs);  // sum of q before each; the slice is done with
  int* bins = reinterpret_cast<int*>(before + kList);
  int lb[kMine], start[kMine];
  unsigned long long q[kMine], sum = 0;
#pragma unroll
  for (int j = 0; j < kMine; j++) {
    const int i = tid * kMine + j;
    uint32_t v = 0;
    lb[j] = i < nl ? bin_of(B, key_value((uint32_t)(list[i] >> 32)), v) : kBins;
    bins[i] = lb[j];
    q[j] = v;
    sum += v;
  }
  unsigned long long incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) S.lsum[warp] = incl;
  __syncthreads();
  unsigned long long pre, all;
  warp_sums<kThreads>(S.lsum, pre, all);
  pre += incl - sum;
  int first = 0;
#pragma unroll
  for (int j = 0; j < kMine; j++) {
    const int i = tid * kMine + j;
    before[i] = pre;
    pre += q[j];
    if (i > 0 && bins[i - 1] != lb[j]) first = i;
    start[j] = first;
  }
  int most = first;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, most, o);
    if (lane >= o) most = max(most, v);
  }
  int prev = __shfl_up_sync(0xffffffffu, most, 1);
  if (lane == 0) prev = 0;
  if (lane == 31) S.wcnt[warp] = (uint32_t)most;
  __syncthreads();
  prev = max(prev, __reduce_max_sync(0xffffffffu, lane < warp ? (int)S.wcnt[lane] : 0));
  uint32_t num[kMine];
  double cum[kMine];
#pragma unroll
  for (int j = 0; j < kMine; j++) {
    const int i = tid * kMine + j;
    num[j] = 0xffffffffu;
    cum[j] = 0.0;
    if (i < nl) {
      const int s0 = max(start[j], prev);
      num[j] = S.count_above[lb[j]] + (uint32_t)(i - s0) + 1;
      cum[j] = S.above[lb[j]] + (double)(before[i] - before[s0] + q[j]) * bin_unit(B, S.unit, lb[j]);
      if (P.k > 0 && (uint32_t)P.k == num[j]) S.z = cum[j];
    }
  }
  __syncthreads();
  const Ranges R = S.rg;
  const bool k_in = R.lo[0] <= R.hi[0];
  const double z = S.z;
#pragma unroll
  for (int j = 0; j < kMine; j++) {
    const int i = tid * kMine + j;
    if (i >= nl) continue;
    if (P.p < 1.0 && cum[j] >= P.p * z) atomicMin(&S.n_p, num[j]);
    if (R.lo[2] <= R.hi[2] && lb[j] >= R.lo[2] && lb[j] <= R.hi[2] &&
        weight(key_value((uint32_t)(list[i] >> 32)), B.xmax, P.t) >= P.minp)
      atomicMin(&S.n_m, ~num[j]);  // the largest place
  }
  __syncthreads();
  uint32_t n_keep = k_in ? (uint32_t)P.k : 0xffffffffu;  // 0xffffffff: everything that weighs
  double mass = z;
  const uint32_t n_p = S.n_p;
  uint32_t n_m = 0xffffffffu;
  if (R.lo[2] <= R.hi[2]) n_m = S.n_m == 0xffffffffu ? S.count_above[R.lo[2]] : ~S.n_m;
#pragma unroll
  for (int j = 0; j < kMine; j++) {
    if (num[j] == n_p && n_p != 0xffffffffu) S.mass_p = cum[j];
    if (num[j] == n_m) S.mass_m = cum[j];
  }
  if (tid == 0 && R.lo[2] <= R.hi[2] && S.n_m == 0xffffffffu) S.mass_m = S.above[R.lo[2]];
  __syncthreads();
  if (n_p < n_keep) n_keep = n_p, mass = S.mass_p;
  if (n_m < n_keep) n_keep = n_m, mass = S.mass_m;
  if (n_keep == 0) n_keep = 1, mass = 1.0;  // min_p above 1: the best token stays
  const double target = P.r * mass;
#pragma unroll
  for (int j = 0; j < kMine; j++)
    if (num[j] <= n_keep && num[j] != 0xffffffffu && (cum[j] >= target || num[j] == n_keep))
      atomicMin(&S.best, (unsigned long long)num[j]);
  __syncthreads();
  if (S.best == ~0ull) {  // the target lies past the gathered tokens by a rounding: the last of them
    uint32_t end = 0;
#pragma unroll
    for (int j = 0; j < kMine; j++)
      if (num[j] != 0xffffffffu && num[j] <= n_keep) end = max(end, num[j]);
    end = __reduce_max_sync(0xffffffffu, end);
    if (lane == 0) S.wcnt[warp] = end;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kThreads / 32; w++) end = max(end, S.wcnt[w]);
      S.best = end;
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kMine; j++) {
    const int i = tid * kMine + j;
    if (i < nl && num[j] == (uint32_t)S.best) {
      const unsigned long long me = list[i];
      a.ids[row] = ~(uint32_t)me;
      if (a.probs) a.probs[row] = (float)(weight(key_value((uint32_t)(me >> 32)), B.xmax, P.t) / mass);
    }
  }
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_kernel(const __grid_constant__ SampleArgs a, int staged) {
  extern __shared__ __align__(16) unsigned char dsm[];
  FastSmem& S = *reinterpret_cast<FastSmem*>(dsm);
  float* xs = reinterpret_cast<float*>(dsm + sizeof(FastSmem));  // the slice; the leader's scratch at the end
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* x = a.logits + row * a.ld;
  const int per = slice_of(a.n, C), e0 = min(a.n, rank * per), e1 = min(a.n, e0 + per);
  const RowParams P = row_params(a, row);

  if (staged) {  // 16 bytes a copy where the row allows it
    const int len = e1 - e0, quads = (reinterpret_cast<uintptr_t>(x) & 15) == 0 ? len / 4 : 0;
    for (int i = tid; i < quads; i += kThreads) cp_async16g(xs + 4 * i, x + e0 + 4 * i);
    for (int i = 4 * quads + tid; i < len; i += kThreads) cp_async4(xs + i, x + e0 + i);
    if (tid < (-len & 3)) xs[len + tid] = -INFINITY;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (int i = tid; i < kBins; i += kThreads) S.hist[i] = 0;
  if (tid == 0) S.n_list = 0, S.dense = 0;
  if (staged) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
  }
  // f(four values, id of the first) over the slice, the whole warp at a time (-inf past its end)
  const bool vec = !staged && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  auto each = [&](auto f) {
    const float4 none4 = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (staged) {
#pragma unroll 2
      for (int i0 = e0; i0 < e1; i0 += 4 * kThreads) {
        const int i = i0 + 4 * tid;
        f(i < e1 ? *reinterpret_cast<const float4*>(xs + (i - e0)) : none4, i);
      }
    } else if (vec) {
      // eight tokens a thread, the next eight already on their way; they pass L1 by
      // (256 rows: 119 us, 123 through it)
      const int last = (e1 - e0) & ~3;  // up to here four at a time lie in the row
      const float4* x4 = reinterpret_cast<const float4*>(x + e0);
      auto load = [&](int i) {
        float4 v = none4;
        if (i < last)
          asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                       : "l"(x4 + i / 4));
        return v;
      };
      int i = 4 * tid;
      float4 v0 = load(i), v1 = load(i + 4 * kThreads);
      for (int i0 = 0; i0 < last; i0 += 8 * kThreads, i += 8 * kThreads) {
        const float4 n0 = load(i + 8 * kThreads), n1 = load(i + 12 * kThreads);
        f(v0, e0 + i);
        f(v1, e0 + i + 4 * kThreads);
        v0 = n0;
        v1 = n1;
      }
      if (e0 + last < e1 && warp == 0) {  // and the one to three beyond
        const int k = e0 + last + lane;
        f(make_float4(k < e1 ? __ldg(x + k) : -INFINITY, -INFINITY, -INFINITY, -INFINITY), k);
      }
    } else {
#pragma unroll 4
      for (int i0 = e0; i0 < e1; i0 += kThreads) {
        const int i = i0 + tid;
        f(make_float4(i < e1 ? __ldg(x + i) : -INFINITY, -INFINITY, -INFINITY, -INFINITY), i);
      }
    }
  };
  // ---- the slice's largest and smallest candidate
  float mx = -INFINITY, mn = INFINITY;
  each([&](float4 v, int) {
    const float w[4] = {v.x, v.y, v.z, v.w};
    const float least = fminf(fminf(v.x, v.y), fminf(v.z, v.w));
    if (staged && least >= -1e30f) {  // no masked value among them
      mx = fmaxf(fmaxf(fmaxf(mx, v.x), fmaxf(v.y, v.z)), v.w);
      mn = fminf(mn, least);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        mx = fmaxf(mx, w[j] >= -1e30f ? w[j] : -INFINITY);
        mn = fminf(mn, w[j] >= -1e30f ? w[j] : INFINITY);
      }
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  if (lane == 0) S.red[0][warp] = mx, S.red[1][warp] = mn;
  __syncthreads();
  if (warp == 0) {
    mx = lane < kThreads / 32 ? S.red[0][lane] : -INFINITY;
    mn = lane < kThreads / 32 ? S.red[1][lane] : INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (lane == 0) S.mx = mx, S.mn = mn;
  }
  sync_row(cl, C);
  {
    const FastSmem* R = cl.map_shared_rank(&S, min(lane, C - 1));
    mx = warp_max(R->mx);
    mn = -warp_max(-R->mn);
  }
  // rows of values near -1e30, or of steps that reach there, are left to the byte-wise form
  // (below, what lies in the bins' range is a candidate), and so are temperatures that f32 cannot divide by
  const bool none = mx == -INFINITY, slow0 = mx == INFINITY || (!none && (mx < -9e29f || P.t > 1e27 || P.t < 1e-28));
  Bins B;
  if (!none && !slow0) {
    // the range: all candidates, but at most 64 in x and 64 in x / t (whichever is more, steps of at most 2)
    const double cap = fmax(64.0 * P.t, fmin(64.0, 2.0 * (kBins - 2) * P.t));
    const double range = fmin((double)mx - (double)mn, cap);
    const float w = (float)fmax(range / (kBins - 4), 1e-30);  // equal logits: one bin
    // 2^-24 of the power of two above |mx| + 2044 w and what rounding adds: 2046 width
    // is at most 1.001 of 2044 w and 2^-13 of that power
    const float all = (float)((fabs((double)mx) + (kBins - 4.0) * w) * 1.002);
    const float grid = __uint_as_float((__float_as_uint(all) & 0x7f800000u) - (23u << 23));
    B.xmax = mx;
    B.width = fmaxf(ceilf(w / grid), 1.f) * grid;  // w / grid may underflow
    // a grid far above t (t below a step of f32 at the maximum): steps of w, 2.01 t at
    // most, off the grid, which the 64-bit form takes, but no step that lets q pass 2^28
    const bool on_grid = B.width <= 2.5 * P.t;
    if (!on_grid) B.width = w;
    B.inv_width = 1.f / B.width;
    B.inv_t = (float)(1.0 / P.t);
    B.step = (double)B.width / P.t;
    B.poly = on_grid && B.step <= 0.0625;
    B.top = B.poly ? ceilf(mx / grid) * grid : mx;  // at most grid <= width above: t / 16
    B.lead = ((double)B.top - (double)mx) / P.t;
  }
  FastSmem* L = cl.map_shared_rank(&S, 0);
  bool wide = !none && !slow0 && !B.poly;  // the 64-bit form
  if (!none && !slow0) {
    if (tid < 4) S.unit[tid] = exp64(B.lead - (double)tid * B.step) * (1.0 / (1 << kQBits));
    const uint32_t bins0 = (uint32_t)__cvta_generic_to_shared(S.cnt) - kRoundBits * 4;
    if (!wide)
      each([&](float4 v, int) {
        const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float p = bin_place(B, w[j]);
          if (in_range(p))
            asm volatile("red.shared.add.u32 [%0], 1;\n\tred.shared.add.u32 [%0 + %2], %1;"
                         ::"r"(bins0 + __float_as_uint(p) * 4), "r"(__float_as_uint(bin_part(B, w[j], p))), "n"(4 * kBins)
                         : "memory");  // cnt and sum of the bin
        }
      });
  }
  // bin_unit's factor for the leader's bins, while other CTAs count
  const double e4 = rank == 0 && !none && !slow0 ? exp64(-(double)((tid * (kBins / kThreads)) & ~3) * B.step) : 0.0;
  const double cut_pos = rank == 0 && !none && !slow0 ? (P.cut + B.lead) / B.step : 0.0;
  sync_row(cl, C);
  if (none || slow0) {  // the same in every CTA of the cluster
    if (rank == 0) {
      if (none) {
        if (tid == 0) {
          a.ids[row] = 0xffffffffu;
          if (a.probs) a.probs[row] = 0.f;
        }
      } else {
        sample_generic<kThreads>(a, row, *reinterpret_cast<GenericSmem*>(dsm));
      }
    }
    return;
  }
  for (;;) {
    if (wide) {
      each([&](float4 v, int) {
        const float w[4] = {v.x, v.y, v.z, v.w};
        for (int j = 0; j < 4; j++) {
          const bool in = in_range(bin_place(B, w[j]));
          uint32_t q;
          const int b = bin_of(B, w[j], q);
          const uint32_t vote = __ballot_sync(0xffffffffu, in);
          if (!vote) continue;
          // many equal logits: one atomic for the warp
          const int one = __ffs(vote) - 1;
          const int b1 = __shfl_sync(0xffffffffu, b, one);
          const uint32_t q1 = __shfl_sync(0xffffffffu, q, one);
          const bool same = __all_sync(0xffffffffu, !in || (b == b1 && q == q1));
          if (in && (!same || lane == one)) atomicAdd(&S.hist[b], (kCountOne + q) * (same ? __popc(vote) : 1));
        }
      });
      sync_row(cl, C);
    }
    if (rank == 0) leader_ranges<kThreads>(S, cl, B, P, C, wide, e4, cut_pos);
    sync_row(cl, C);
    if (!L->rg.redo) break;
    wide = true;  // a bin holds too many tokens for the 32-bit sums: once more
    for (int i = tid; i < kBins; i += kThreads) S.hist[i] = 0;
    __syncthreads();
  }
  // ---- the tokens of those bins: gathered in the CTA, then in the leader
  {
    if (rank != 0) {
      if (tid == 0) S.rg = L->rg;
      __syncthreads();
    }
    const int windows = S.rg.n;
    float mid[4], half[4];
#pragma unroll
    for (int j = 0; j < 4; j++) mid[j] = j < windows ? S.rg.mid[j] : 0.f, half[j] = j < windows ? S.rg.half[j] : -1.f;
    // a warp's hits go to its own part of a list of ids: no atomics in the pass
    // (staged: 16-bit offsets; either way a run of kList neighbours finds room)
    const uint32_t room = (staged ? kStagedHits : kHits) / (kThreads / 32);
    unsigned char* hits = dsm + sizeof(FastSmem) + (staged ? per * 4 : 0);
    uint16_t* hits16 = reinterpret_cast<uint16_t*>(hits) + warp * room;
    uint32_t* hits32 = reinterpret_cast<uint32_t*>(hits) + warp * room;
    const uint32_t below = (1u << lane) - 1;
    uint32_t nh = 0;
    each([&](float4 v, int i) {
      const float w[4] = {v.x, v.y, v.z, v.w};
      bool hit[4];
#pragma unroll
      for (int j = 0; j < 4; j++) hit[j] = (fabsf(w[j] - mid[0]) <= half[0]) | (fabsf(w[j] - mid[1]) <= half[1]);
      if (windows > 2)
#pragma unroll
        for (int j = 0; j < 4; j++) hit[j] = hit[j] | (fabsf(w[j] - mid[2]) <= half[2]) | (fabsf(w[j] - mid[3]) <= half[3]);
      if (__any_sync(0xffffffffu, hit[0] | hit[1] | hit[2] | hit[3])) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t vote = __ballot_sync(0xffffffffu, hit[j]);
          const uint32_t to = nh + __popc(vote & below);
          if (hit[j] && to < room) {
            if (staged) hits16[to] = (uint16_t)(i + j - e0);
            else hits32[to] = (uint32_t)(i + j);
          }
          nh += __popc(vote);
        }
      }
    });
    __syncwarp();
    if (nh > room && lane == 0) atomicAdd(&S.n_list, kList + 1u);
    for (uint32_t k0 = 0; k0 < min(nh, room); k0 += 32) {
      bool in = false;
      uint32_t id = 0;
      float v = 0.f;
      if (k0 + lane < min(nh, room)) {
        id = staged ? e0 + hits16[k0 + lane] : hits32[k0 + lane];
        v = staged ? xs[id - e0] : __ldg(x + id);
        const float p = bin_place(B, v);
        const int b = bin_index(p);  // as bin_of, where in_range
#pragma unroll
        for (int j = 0; j < 4; j++) in |= b >= S.rg.lo[j] && b <= S.rg.hi[j];
        in &= in_range(p);
      }
      const uint32_t vote = __ballot_sync(0xffffffffu, in);
      uint32_t to = 0;
      if (lane == 0 && vote) to = atomicAdd(&S.n_list, (uint32_t)__popc(vote));
      to = __shfl_sync(0xffffffffu, to, 0) + __popc(vote & below);
      if (in && to < kList) S.list[to] = (unsigned long long)order_key(v) << 32 | ~id;
    }
    if (C > 1) {
      __syncthreads();
      if (rank != 0) {
        const uint32_t n = S.n_list;
        if (tid == 0) S.wcnt[0] = n ? atomicAdd(&L->n_list, n) : 0u;
        __syncthreads();
        const uint32_t to = S.wcnt[0];
        for (uint32_t i = tid; i < min(n, (uint32_t)kList); i += kThreads)
          if (to + i < kList) L->list[to + i] = S.list[i];
      }
    }
  }
  sync_row(cl, C);
  if (rank != 0) return;

  const int nl = (int)S.n_list;
  if (nl > kList || nl == 0) {  // too many; or, should the bins ever miss a row's tokens, none: every row is written
    __syncthreads();
    sample_generic<kThreads>(a, row, *reinterpret_cast<GenericSmem*>(dsm));
    return;
  }
  // ---- the gathered tokens in falling order
  unsigned long long* list = S.list;
  if (nl <= kCountMost) {
    // a few: each is compared with all, eight threads for every two tokens (a key
    // loaded is compared twice: the loads' bytes bound this)
    list = reinterpret_cast<unsigned long long*>(xs) + kList * 3 / 2;  // behind the two arrays below
    constexpr int kPart = 8, kApart = kThreads / kPart;
    const int part = tid & (kPart - 1);
    for (int e = tid / kPart; e < (nl + 31) / 32 * 32; e += 2 * kApart) {
      const unsigned long long me0 = e < nl ? S.list[e] : 0, me1 = e + kApart < nl ? S.list[e + kApart] : 0;
      int at0 = 0, at1 = 0;
      for (int f = part; f < nl; f += kPart) {
        const unsigned long long u = S.list[f];
        at0 += u > me0;
        at1 += u > me1;
      }
#pragma unroll
      for (int o = 1; o < kPart; o <<= 1) {
        at0 += __shfl_xor_sync(0xffffffffu, at0, o);
        at1 += __shfl_xor_sync(0xffffffffu, at1, o);
      }
      if (part == 0 && e < nl) list[at0] = me0;
      if (part == 0 && e + kApart < nl) list[at1] = me1;
    }
    __syncthreads();
  } else {
    int np = 64;
    while (np < nl) np *= 2;
    for (int i = nl + tid; i < np; i += kThreads) S.list[i] = 0;
    __syncthreads();
    bitonic_falling<kThreads>(S.list, np);
  }
  // one token a thread where that holds them all
  if (nl <= kThreads) finish_row<kThreads, 1>(a, row, S, B, P, list, nl, xs);
  else finish_row<kThreads, kList / kThreads>(a, row, S, B, P, list, nl, xs);
}

// CTAs of a row's cluster: as many as leave every CTA an SM of its own, with
// slices of 4096 tokens or longer, and clusters of 8, which do not fill the GPCs'
// SMs, for up to 12 rows.  us a call for rows of 151,936 (top-p and min-p) by 1 / 2 /
// 4 / 8 CTAs a row: 12 rows 57 / 39 / 31 / 26, 16 rows 57 / 39 / 31 / 42, 32 rows 58 /
// 41 / 33 / 63, 64 rows 65 / 44 / 44 / 106, 256 rows 117 / 127 / 151 / 365; rows of
// 32,000: 12 rows 22 / 21 / 18 / 19, 64 rows 22 / 21 / 24 / 77.  (13 rows would take 27
// by 8 and take 32 by 4, 65 rows 45 by 2 and 65 by 1: clusters find room by GPCs.)
// Slices of 2^18 tokens and more are cut (kSliceMost), and gain: 256 rows of 262,144
// 203 us by 2, 447 by 1; 65 rows of 2^20 281 by 8, 478 by 4, 1197 by 1.
int cluster_size(int rows, int n) {
  int c = 1;
  while (c < 8 && 2LL * rows * c <= (c == 4 ? 96 : 128) && n / (2 * c) >= 4096) c *= 2;
  while (slice_of(n, c) > kSliceMost) c *= 2;  // 8 hold the longest row, 2^20
  return c;
}

template <int kThreads>
cudaError_t launch_sample(const SampleArgs& a, int c, cudaStream_t st) {
  const int per = slice_of(a.n, c);
  const int staged = per <= ((long long)a.rows * c <= 148 ? kSliceAlone : kSlice);
  const size_t smem = sizeof(FastSmem) + std::max<size_t>(staged ? (size_t)per * 4 + kStagedHits * 2 : kHits * 4, kList * 12 + kCountMost * 8);
  static_assert(sizeof(FastSmem) + kSlice * 4 + kStagedHits * 2 <= 113 << 10, "two CTAs an SM");
  static_assert(sizeof(FastSmem) + kSliceAlone * 4 + kStagedHits * 2 <= 227 << 10, "a CTA's shared memory");
  static OncePerDevice once;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && once.first(dev)) {
    e = cudaFuncSetAttribute(sample_kernel<kThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 << 10);
    if (e == cudaSuccess) once.done(dev);
  }
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = c;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<kThreads>, a, staged);
}

// 1024 threads for the few rows that take clusters of 8 (1 row 25.3 us, 25.9 with
// 512), else 512, two CTAs an SM (256 rows 117 us, 121 with 1024).
cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  const int c = cluster_size(a.rows, a.n);
  return c == 8 ? launch_sample<1024>(a, c, st) : launch_sample<512>(a, c, st);
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" {

EG_API eg_status eg_op_sample_filtered(const float* logits, int64_t ld, int rows, int n, const float* temp,
                                       const int* top_k, const float* top_p, const float* min_p, const float* r,
                                       uint32_t* ids, float* probs, void* stream) {
  if (rows < 0 || n < 1 || n > (1 << 20) || rows > (1 << 24)) return fail(EG_ERR_ARG, "sample_filtered: need rows >= 0 and 1 <= n <= 2^20");
  if (ld < n) return fail(EG_ERR_ARG, "sample_filtered: row stride %lld below n = %d", (long long)ld, n);
  if (rows == 0) return EG_OK;
  if (!logits || !r || !ids) return fail(EG_ERR_ARG, "sample_filtered: null argument");
  if (reinterpret_cast<uintptr_t>(logits) & 3) return fail(EG_ERR_ARG, "sample_filtered: logits must be 4-byte aligned");
  SampleArgs a = {logits, ld, rows, n, temp, top_k, top_p, min_p, r, ids, probs};
  const cudaError_t e = launch_sample(a, reinterpret_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(EG_ERR_CUDA, "sample_filtered: %s", cudaGetErrorString(e));
  return EG_OK;
}

}  // extern "C"
