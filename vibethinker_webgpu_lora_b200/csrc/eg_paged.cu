// eg_paged.cu -- operators on a paged K/V cache: the rotated append of ragged
// token rows, and decode attention for a batch that shares a prefix.
//
// The cache is the paged slots' (WRITE_KV_PAGE / ATTN_PARTIAL_PAGED,
// kernels.js:1657-1911): pools [n_pages][16][nkv][128] of f16 or f32, row t of
// a sequence at physical row pages[t / 16] * 16 + t % 16.  Page ids and
// lengths live on the device, so a captured graph serves every step.
#include <cooperative_groups.h>
#include <cuda.h>
#include <math.h>
#include <algorithm>
#include <type_traits>

#include "eg_common.cuh"
#include "eg_device.cuh"
#include "eg_host.h"
#include "eg_tc.cuh"
#include "emberglass.h"

namespace eg {
namespace {

constexpr int kPage = 16;  // rows of a page

// ======================================================================
// Append: RoPE(k) and v of T token rows into the pool, RoPE(q) beside it
// ======================================================================
struct AppendArgs {
  const float* qkv;
  long long ld;
  int T;
  const int* pos;
  const int* slot;
  const uint32_t* pages;
  int n_slots, max_pages, n_pages, prefix_len;
  void* kc;
  void* vc;
  const float* cosT;
  const float* sinT;
  int table_len, nh, nkv;
  float* q_out;
  long long ldq;
  int* err;
};

// A head of a token is 16 lanes: lane l holds dims 4l..4l+3 and their RoPE
// partners 64 + 4l.., so a pair is turned in one thread (rope_pair, f32:
// two rounded products and one sum) and rounded once, to the cache's type.
template <typename KVT>
__device__ __forceinline__ void store4(KVT* d, float4 v);
template <>
__device__ __forceinline__ void store4<float>(float* d, float4 v) {
  *reinterpret_cast<float4*>(d) = v;
}
template <>
__device__ __forceinline__ void store4<__half>(__half* d, float4 v) {
  *reinterpret_cast<uint2*>(d) =
      make_uint2(h2_bits(__floats2half2_rn(v.x, v.y)), h2_bits(__floats2half2_rn(v.z, v.w)));
}

// The bound is bytes, 512 read and 256 or 512 written a head.  U heads a half-
// warp, their loads issued first: at 16384 tokens of 48 heads (743 MB) U = 2
// runs at the copy rate (112 us, U = 1 120), at 512 tokens of 20 the launch and
// three dependent loads are the time (U = 1 3.2 us, U = 2 3.5).  The call takes
// U = 2 from 131,072 heads on (0.94 of U = 1 there); below 36,000 heads it is
// 0.95 to 1.28 of U = 1, from 40,000 to 131,072 0.93 to 0.99.
template <typename KVT, int U>
__global__ void __launch_bounds__(256) kv_append_paged_kernel(AppendArgs a) {
  const int H = a.nh + 2 * a.nkv, l = threadIdx.x & 15;
  const long long first = (long long)blockIdx.x * 16 * U + (threadIdx.x >> 4), n = (long long)a.T * H;
  float4 lo[U], hi[U];
  int t[U], h[U], pos[U], s[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const long long item = first + 16 * u;
    t[u] = item < n ? (int)(item / H) : 0;
    h[u] = (int)(item - (long long)t[u] * H);
    pos[u] = -1;
    if (item < n && (h[u] >= a.nh || a.q_out)) {
      const float* src = a.qkv + t[u] * a.ld + h[u] * kHeadDim + 4 * l;
      lo[u] = __ldcg(reinterpret_cast<const float4*>(src));  // q_out may be these very words
      hi[u] = __ldcg(reinterpret_cast<const float4*>(src + kHeadDim / 2));
      pos[u] = __ldg(a.pos + t[u]);
      s[u] = __ldg(a.slot + t[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    if (pos[u] < 0) continue;  // a padding row
    const int row = pos[u] - a.prefix_len;
    bool ok = pos[u] < a.table_len && row >= 0 && s[u] >= 0 && s[u] < a.n_slots && row / kPage < a.max_pages;
    uint32_t page = 0;
    if (ok) {
      page = __ldg(a.pages + (size_t)s[u] * a.max_pages + row / kPage);
      ok = page < (uint32_t)a.n_pages;
    }
    if (!ok) {
      if (a.err && l == 0) *a.err = 1;
      continue;
    }
    if (h[u] < a.nh + a.nkv) {
      const float4 c = __ldg(reinterpret_cast<const float4*>(a.cosT + (size_t)pos[u] * kHeadDim + 4 * l));
      const float4 d = __ldg(reinterpret_cast<const float4*>(a.sinT + (size_t)pos[u] * kHeadDim + 4 * l));
      rope_pair(lo[u].x, hi[u].x, c.x, d.x, 0);
      rope_pair(lo[u].y, hi[u].y, c.y, d.y, 0);
      rope_pair(lo[u].z, hi[u].z, c.z, d.z, 0);
      rope_pair(lo[u].w, hi[u].w, c.w, d.w, 0);
    }
    if (h[u] < a.nh) {
      float* d = a.q_out + t[u] * a.ldq + h[u] * kHeadDim + 4 * l;
      store4(d, lo[u]);
      store4(d + kHeadDim / 2, hi[u]);
      continue;
    }
    const bool is_k = h[u] < a.nh + a.nkv;
    const int kvh = h[u] - a.nh - (is_k ? 0 : a.nkv);
    KVT* d = static_cast<KVT*>(is_k ? a.kc : a.vc) + (((size_t)page * kPage + row % kPage) * a.nkv + kvh) * kHeadDim + 4 * l;
    store4(d, lo[u]);
    store4(d + kHeadDim / 2, hi[u]);
  }
}

template <typename KVT>
void launch_append(const AppendArgs& a, long long heads, cudaStream_t st) {
  if (heads >= 131072) kv_append_paged_kernel<KVT, 2><<<(unsigned)((heads + 31) / 32), 256, 0, st>>>(a);
  else kv_append_paged_kernel<KVT, 1><<<(unsigned)((heads + 15) / 16), 256, 0, st>>>(a);
}

// ======================================================================
// Decode attention over a shared prefix
// ======================================================================
// Row r = b * G + g of a KV head is query head kvh * G + g of sequence b
// (G = nh / nkv).  o = softmax(q k^T / sqrt(128)) v over the prefix's keys and
// the sequence's own.  The keys are cut into splits; each split of a row
// gives (b, l, o) with p = 2^(s2 - b), s2 = q.k * log2(e)/sqrt(128), l = sum p,
// o = sum p v, and the combine weighs the splits by 2^(b - max b).  The base b
// is the running maximum less kPBits: p reaches up to 2^14, and its f16 hi + lo
// parts keep an absolute error of 2^-39 of the largest weight, so many small
// weights beside one large one are not lost below the f16 range.  Split s has
// its bases and sums at [s][KV head][row] and its o at [s][KV head][row / 8]
// [16-byte piece][row % 8]: a thread a row writes whole sectors, and so does a
// group of 8 rows.
constexpr float kPBits = 14.f;
constexpr int kSoPitch = kHeadDim + 4;  // floats a row of the warps' outputs in shared memory
constexpr int kSms = 148;       // plans are made for the B200's SM count

struct SharedPlan {
  int G, gch;          // query heads per KV head; chunks of 8 of them
  int rows, groups;    // nseq * G rows per KV head, in groups of 8
  int pref_keys, n_pref;  // keys per prefix split, splits
  int tc, row_tiles;   // prefix on the tcgen05 tensor cores, in tiles of 128 rows
  int fused;           // everything in one launch, a cluster of all splits for each 8 rows of a sequence
  int own;             // prefix in a kernel of its own (tc, or f32 in CTAs of 16 rows)
  int lanes;           // of the combine, which take the splits in turns of 8 (one: of 32)
  int many;            // f32: 4 warps a CTA, two CTAs an SM
  int suf_keys, n_suf;                // keys per suffix split, most splits of a sequence
};

struct SharedArgs {
  const float* q;
  long long ldq;
  int nseq, nh, nkv;
  const void* kc;
  const void* vc;
  uint32_t n_pages;
  const uint32_t* prefix_pages;
  int prefix_len;
  const uint32_t* pages;
  int max_pages;
  const int* lens;
  int max_len;
  float* out;
  long long ldo;
  float *pm, *pl;  // [split][KV head][8 groups rows]
  float4* po;      // 32 for each of these
  int* err;
  SharedPlan p;
};

// Where piece c of row r lies in a split's o; its base and sum are at part_row.
__device__ __forceinline__ size_t part_row(const SharedArgs& a, int split, int kvh, int r) {
  return ((size_t)split * a.nkv + kvh) * a.p.groups * 8 + r;
}
__device__ __forceinline__ size_t part_at(size_t row, int c) { return (row >> 3) * 256 + c * 8 + (row & 7); }

int round_up(int x, int m) { return (x + m - 1) / m * m; }

SharedPlan shared_plan(int nseq, int nh, int nkv, int prefix_len, int max_len, int kv_f16) {
  SharedPlan p;
  p.G = nh / nkv;
  p.gch = (p.G + 7) / 8;
  p.rows = nseq * p.G;
  p.groups = (p.rows + 7) / 8;
  p.row_tiles = (p.rows + 127) / 128;
  // What the prefix's scores number decides its kernel: f16 on the tensor cores
  // from 900,000 on (128 shapes of 16/2, 28/4 and 32/8 heads: 1.08 to 1.73 of the
  // warps' time up to 530,000, 0.44 to 0.93 from 1,800,000 on, 0.86 to 1.33 about
  // 900,000 to 1,050,000; 16 heads, 16 sequences x 2048: 15.0 and 10.1 us, x 4096
  // 15.4 and 15.4, x 8192 17.0 and 25.1); f32 in CTAs of 16 rows from 1,000,000 on;
  // below, the prefix and the suffixes share a launch.
  // f32 takes 4 warps a CTA, two CTAs an SM, where there is work for them, else 8
  // warps.  Over 582 shapes (those heads and 8/1, 1 to 64 sequences, prefixes of 128
  // to 32768, own keys of 16 to 1024), 4 warps take of the time of 8, with 16 groups
  // and KV heads or more: 0.84 to 1.13 (median 1.09) below 100,000 scores in all,
  // 0.78 to 1.07 (0.95) to 138,000, 0.59 to 1.08 (0.83) above; with fewer: 0.77 to
  // 1.35 (1.06) up to 1,500,000 of the prefix, 0.74 to 0.95 above (groups > 2: 0.74 to 0.85).
  // The rule is within 0.8 % of the better one on the average, at worst 1.30 of it (1
  // sequence of 32/8 heads, 2048 + 1024 keys).
  const long long scores = (long long)p.rows * nkv * prefix_len;
  p.tc = kv_f16 && prefix_len >= 256 && scores >= 900000;
  p.many = !kv_f16 && ((p.groups * nkv >= 16 && scores + (long long)p.rows * nkv * max_len >= 138000) ||
                       (p.groups > 2 && scores >= 1500000));
  p.own = p.tc || (p.many && p.groups > 2 && scores >= 1000000);
  if (p.tc) {
    // one CTA an SM, about 5.5 us and 1.8 us a block of 128 keys: the number of
    // splits with the shortest rounds
    const int units = p.row_tiles * nkv;
    double best = 1e300;
    for (int n = 1; n <= std::max(1, prefix_len / 256); n++) {
      const int keys = round_up((prefix_len + n - 1) / n, 128), got = (prefix_len + keys - 1) / keys;
      const double t = (double)(((long long)units * got + kSms - 1) / kSms) * (5.5 + 1.8 * (keys / 128)) + 0.1 * got;
      if (t < best) best = t, p.pref_keys = keys;
      if ((long long)units * n > 4 * kSms) break;
    }
  } else {
    // two CTAs an SM (f32 of 8 warps: one): what is resident at once beside the
    // suffixes (16 x 2048 f16 11.2 us so, 13.9 with four an SM); never under 128
    // keys a split and never above 1024: the tensor core's f32 sums lose about
    // 2^-24.5 a step, all one way, so a warp's 16 tiles stay below 2^-20 (256
    // tiles of a 16384-key split: 1e-5)
    const long long units = (long long)(p.own ? (p.groups + 1) / 2 : p.groups) * nkv;
    const long long want = std::max(1LL, (kv_f16 || p.many ? 2LL : 1LL) * kSms / units);
    p.pref_keys = std::min(1024, std::max(128, round_up((int)((prefix_len + want - 1) / want), 64)));
  }
  p.n_pref = (prefix_len + p.pref_keys - 1) / p.pref_keys;
  // suffix: about four CTAs an SM, 128 keys a split at least (64 sequences x up to
  // 1024 keys 12.6 us in splits of 256, 14.9 of 128, 20.2 of 1024), 1024 at most
  // as above
  const int pairs = nseq * nkv * p.gch, want = std::max(1, 4 * kSms / pairs);
  p.suf_keys = std::min(1024, std::max(128, round_up((max_len + want - 1) / want, 64)));
  p.n_suf = (max_len + p.suf_keys - 1) / p.suf_keys;
  // up to 8 splits, few rows: one launch that joins them within a cluster, each
  // sequence reading the prefix for itself (2 sequences x 256 keys 5.6 us, 6.8 with
  // the combine's launch; 16 x (512 + 512) 7.4 and 8.2).  At most as many CTAs as
  // find room at once in clusters of 8: two an SM in f16 (512 CTAs 13.3 us, 7.8 in
  // two launches), three SMs of four in f32 (128 CTAs 13.9 and 8.4).  A single split
  // without a prefix has nothing to join and reads nothing twice: any number (32
  // sequences x 16 heads of their own x 128 keys 9.4 and 11.3).
  const int limit = kv_f16 ? 2 * kSms : kSms * 3 / 4;
  // f16: longer splits where that makes 8 of them, up to 512 keys, 384 with few
  // pairs, which leave SMs to more splits (16 x 2048 + 640 in 384 keys 10.3 us, 12.0
  // in 8 of 256 and 5 of 128 with the combine; 2 x 2048 + 2048 in 512 9.9 and 8.2; f32
  // loses: 2 x 1024 + 1024 in 256 9.8 and 9.0).  Over 350 shapes that it changes, of
  // the time without: 8 query heads a KV head 0.78 to 1.13, 1 to 7 of them, whose
  // CTAs hold empty rows, 0.83 to 1.38 (8 x 3000 + 64 of 4/4 heads 11.0 and 8.0)
  if (kv_f16 && !p.own && p.n_pref + p.n_suf > 8 && pairs * 8 <= limit)
    for (int keys = 64; keys <= (pairs >= 8 ? 512 : 384); keys += 64) {
      const int np = (prefix_len + keys - 1) / keys, ns = (max_len + keys - 1) / keys;
      if (np + ns > 8) continue;
      p.pref_keys = p.suf_keys = keys;
      p.n_pref = np;
      p.n_suf = ns;
      break;
    }
  const int splits = p.n_pref + p.n_suf;
  p.lanes = splits > 16 && nkv * p.groups <= kSms ? 4 : 1;
  p.fused = !p.own && !p.many && splits >= 1 && splits <= 8 &&
            ((splits == 1 && prefix_len == 0) || pairs * splits <= limit);
  return p;
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

// An output: o / l (no key at all: zeros).  What is not finite is flagged: q or a
// key or value that is not, or an f32 cache's value past the f16 range.
__device__ __forceinline__ void store_out(const SharedArgs& a, float* dst, float4 o, float l) {
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const float4 y = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  *reinterpret_cast<float4*>(dst) = y;
  if (!(0.f * y.x + 0.f * y.y + 0.f * y.z + 0.f * y.w == 0.f) && a.err) *a.err = 1;
}

// One warp's walk over the 16-key tiles of a key range, 8 rows at a time.
// S^T = K q^T and O^T = V^T p^T as mma.sync m16n8k16 (16 keys or dims x 8
// rows), so the 8 query heads of a group fill the n side exactly.  q and p are
// f16 hi + lo pairs (two products); with an f32 cache K and V are split too
// (three products, the lo.lo one left out: 2^-22 of the product).  lo parts of
// q, K and V are lifted by 2^11 (split_lifted): an f16 holds them to 2^-36 then,
// not 2^-25, which small values would feel.  The scores sum theirs apart; V's
// meets p hi lowered by 2^-11.
template <typename KVT>
struct WarpTile {
  static constexpr int kRow = kHeadDim * (int)sizeof(KVT);  // bytes of a staged row
  static constexpr int kBytes = 2 * kPage * kRow;           // K and V of one tile
  // warps of a CTA, each with its own tiles, and how many a warp stages: 64 KB for
  // f16 (three CTAs an SM).  f32, whose warps compute longer, gains more by warps
  // than by a second stage: 64 KB in 4 warps, or 128 KB in 8 where there are few
  // CTAs (the plan's choice)
  static constexpr bool kF32 = std::is_same<KVT, float>::value;
  static constexpr int kStages = kF32 ? 1 : 2;
  static constexpr int kChunks = kRow / 16;
};

// 16-byte chunk c of staged row r, XOR-swizzled: 8 rows' chunks of one column
// lie in different banks.
template <typename KVT>
__device__ __forceinline__ int tile_off(int r, int c) {
  return r * WarpTile<KVT>::kRow + ((c ^ (r & 7)) << 4);
}

template <typename KVT>
__device__ __forceinline__ void tile_load(unsigned char* st, const SharedArgs& a, int kvh, uint32_t page, int nv) {
  using W = WarpTile<KVT>;
  const int lane = threadIdx.x & 31;
  const size_t base = ((size_t)page * kPage * a.nkv + kvh) * kHeadDim * sizeof(KVT);
  const char* k = static_cast<const char*>(a.kc) + base;
  const char* v = static_cast<const char*>(a.vc) + base;
  const size_t rs = (size_t)a.nkv * kHeadDim * sizeof(KVT);
#pragma unroll
  for (int i = lane; i < kPage * W::kChunks; i += 32) {
    const int r = i / W::kChunks, c = i % W::kChunks;
    const size_t off = r < nv ? r * rs + c * 16 : 0;  // rows past the end are filled with zeros
    cp_async16(st + tile_off<KVT>(r, c), k + off, r < nv ? 16 : 0);
    cp_async16(st + kPage * W::kRow + tile_off<KVT>(r, c), v + off, r < nv ? 16 : 0);
  }
}

// (x, y) = hi + 2^-11 lo, each an f16 pair
constexpr float kLift = 2048.f;
__device__ __forceinline__ void split_lifted(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = h2_bits(h);
  lo = h2_bits(__floats2half2_rn((x - f.x) * kLift, (y - f.y) * kLift));
}

// (16 keys x 16 dims at dim 16 ks) as A fragments, hi and (f32 cache) lo
__device__ __forceinline__ void k_frag(const unsigned char* st, int ks, uint32_t (&h)[4], uint32_t (&)[4], __half) {
  const int lane = threadIdx.x & 31, i = lane >> 3, r = (lane & 7) + 8 * (i & 1);
  ldsm_x4(smem_addr(st + tile_off<__half>(r, 2 * ks + (i >> 1))), h[0], h[1], h[2], h[3]);
}
__device__ __forceinline__ void k_frag(const unsigned char* st, int ks, uint32_t (&h)[4], uint32_t (&l)[4], float) {
  const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = g + 8 * (i & 1), d = 16 * ks + 8 * (i >> 1) + 2 * tq;
    const float2 x = *reinterpret_cast<const float2*>(st + tile_off<float>(r, d >> 2) + (d & 3) * 4);
    split_lifted(x.x, x.y, h[i], l[i]);
  }
}
// (16 dims at 16 dt x 16 keys) of V^T as A fragments
__device__ __forceinline__ void v_frag(const unsigned char* st, int dt, uint32_t (&h)[4], uint32_t (&)[4], __half) {
  const int lane = threadIdx.x & 31, i = lane >> 3, r = (lane & 7) + 8 * (i >> 1);
  ldsm_x4_t(smem_addr(st + tile_off<__half>(r, 2 * dt + (i & 1))), h[0], h[1], h[2], h[3]);
}
__device__ __forceinline__ void v_frag(const unsigned char* st, int dt, uint32_t (&h)[4], uint32_t (&l)[4], float) {
  const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int d = 16 * dt + g + 8 * (i & 1), r = 8 * (i >> 1) + 2 * tq;
    const float x = *reinterpret_cast<const float*>(st + tile_off<float>(r, d >> 2) + (d & 3) * 4);
    const float y = *reinterpret_cast<const float*>(st + tile_off<float>(r + 1, d >> 2) + (d & 3) * 4);
    split_lifted(x, y, h[i], l[i]);
  }
}

// CTA = one split of the keys for up to 8 NG rows of one KV head.  Blocks
// [0, pref) take the prefix, the others the suffixes (8 rows of a sequence
// each).  NG = 2, for the prefix alone and an f32 cache, halves the reads and
// the splitting of K and V per row.  FUSED: a cluster's CTAs are all splits of 8
// rows of one sequence, the prefix's first, and join their parts through each
// other's shared memory: one launch, for few splits.  Every CTA of a cluster
// reaches both of its barriers; none leaves before the others have read its parts.
template <typename KVT, int NG, int kWarps, bool FUSED>
__global__ void __launch_bounds__(32 * kWarps) attn_shared_kernel(const __grid_constant__ SharedArgs a, int pref) {
  using W = WarpTile<KVT>;
  constexpr bool F32 = W::kF32;
  extern __shared__ __align__(128) unsigned char sm[];
  __shared__ float sm_m[kWarps][8 * NG], sm_l[kWarps][8 * NG];
  __shared__ float part_m[FUSED ? 8 : 1], part_l[FUSED ? 8 : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const SharedPlan& p = a.p;
  const int G = p.G;
  pdl_launch_dependents();  // what follows waits for the end of this kernel before it reads its results

  // the CTA's rows [row0, row0 + nrow) of KV head kvh and its keys [k0, k1)
  int kvh, row0, nrow, k0, k1, split, kmax;
  const uint32_t* table;
  int blk = blockIdx.x;
  if (FUSED) {
    const int c = p.n_pref + p.n_suf;
    split = blk % c;
    blk /= c;
    const int gc = blk % p.gch;
    blk /= p.gch;
    kvh = blk % a.nkv;
    const int b = blk / a.nkv;
    row0 = b * G + 8 * gc;
    nrow = min(8, G - 8 * gc);
    k1 = a.lens[b];
    if (split < p.n_pref) {
      table = a.prefix_pages;
      k0 = split * p.pref_keys;
      kmax = min(a.prefix_len, k0 + p.pref_keys);
    } else {
      table = a.pages + (size_t)b * a.max_pages;
      k0 = (split - p.n_pref) * p.suf_keys;
      kmax = min(a.max_len, k0 + p.suf_keys);
    }
  } else if (blk < pref) {
    const int ng = (p.groups + NG - 1) / NG, rg = blk % ng;
    blk /= ng;
    kvh = blk % a.nkv;
    split = blk / a.nkv;
    row0 = 8 * NG * rg;
    nrow = min(8 * NG, p.rows - row0);
    table = a.prefix_pages;
    k0 = split * p.pref_keys;
    k1 = kmax = min(a.prefix_len, k0 + p.pref_keys);
  } else {
    blk -= pref;
    const int gc = blk % p.gch;
    blk /= p.gch;
    kvh = blk % a.nkv;
    blk /= a.nkv;
    const int b = blk % a.nseq;
    split = blk / a.nseq;
    row0 = b * G + 8 * gc;
    nrow = min(8, G - 8 * gc);
    table = a.pages + (size_t)b * a.max_pages;
    k0 = split * p.suf_keys;
    kmax = min(a.max_len, k0 + p.suf_keys);  // the table holds that many, whatever the length
    k1 = a.lens[b];                          // on its way while the first page ids are read
    split += p.n_pref;
  }
  auto page_at = [&](int t) -> uint32_t { return k0 + t * kPage < kmax ? __ldg(table + k0 / kPage + t) : 0u; };
  const uint32_t page0 = page_at(warp), page1 = page_at(warp + kWarps);
  const int len = k1;  // suffixes: the sequence's own keys
  if (FUSED) {
    if (k1 > a.max_len && a.err && threadIdx.x == 0) *a.err = 1;
    k1 = split < p.n_pref ? kmax : max(k0, min(k1, kmax));
  } else if ((int)blockIdx.x >= pref) {  // a length above max_len is flagged by the combine, which sees every one
    k1 = min(k1, kmax);
    if (k0 >= k1) {
      if (p.own) pdl_wait();
      return;
    }
  }

  unsigned char* st = sm + warp * W::kStages * W::kBytes;
  const int ntile = (k1 - k0 + kPage - 1) / kPage;
  // the warp's tiles: warp, warp + kWarps, ...
  auto issue = [&](int t, uint32_t page, int stage) -> int {
    int nv = t < ntile ? min(kPage, k1 - k0 - t * kPage) : 0;
    if (nv > 0 && page >= a.n_pages) {  // a page outside the pool: its keys are left out
      nv = 0;
      if (a.err && lane == 0) *a.err = 1;
    }
    if (t < ntile) tile_load<KVT>(st + stage * W::kBytes, a, kvh, nv > 0 ? page : 0u, nv);
    cp_async_commit();
    return nv;
  };
  int nv_cur = issue(warp, page0, 0);
  uint32_t page_next = page1;

  // q of the rows as B fragments: lane (g, tq) holds row g's dims 2 tq.. of each k-step
  uint32_t qh[NG][8][2], ql[NG][8][2];
#pragma unroll
  for (int n = 0; n < NG; n++) {
    const int r = row0 + 8 * n + g;
    const bool on = 8 * n + g < nrow;
    const float* q = a.q + (on ? (long long)(r / G) * a.ldq + (kvh * G + r % G) * kHeadDim : 0) + 2 * tq;
    // log2(e) / sqrt(128) / 2: with the half |q| / 8 may fill the f16 range; the scores are doubled again
    const float c = 0.5f * 1.4426950408889634f * 0.08838834764831845f;
#pragma unroll
    for (int ks = 0; ks < 8; ks++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const float2 x = on ? __ldg(reinterpret_cast<const float2*>(q + 16 * ks + 8 * j)) : make_float2(0.f, 0.f);
        split_lifted(x.x * c, x.y * c, qh[n][ks][j], ql[n][ks][j]);
      }
  }
  float O[NG][8][4];
  float m0[NG], m1[NG], l0[NG], l1[NG];  // rows 2 tq and 2 tq + 1
#pragma unroll
  for (int n = 0; n < NG; n++) {
#pragma unroll
    for (int j = 0; j < 8; j++) O[n][j][0] = O[n][j][1] = O[n][j][2] = O[n][j][3] = 0.f;
    m0[n] = m1[n] = -INFINITY;
    l0[n] = l1[n] = 0.f;
  }

  int stage = 0;
  for (int t = warp; t < ntile; t += kWarps) {
    int nv_next = 0;
    if (W::kStages == 2) {
      nv_next = issue(t + kWarps, page_next, stage ^ 1);
      page_next = page_at(t + 2 * kWarps);
    }
    cp_async_wait<W::kStages - 1>();
    __syncwarp();
    const unsigned char* ks_ = st + stage * W::kBytes;
    const unsigned char* vs_ = ks_ + kPage * W::kRow;
    float S[NG][4], S2[NG][4];
    uint32_t fh[4], fl[4];
#pragma unroll
    for (int n = 0; n < NG; n++)
#pragma unroll
      for (int j = 0; j < 4; j++) S[n][j] = S2[n][j] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
      k_frag(ks_, ks, fh, fl, KVT());
#pragma unroll
      for (int n = 0; n < NG; n++) {
        mma16816(S[n], fh, qh[n][ks][0], qh[n][ks][1]);
        mma16816(S2[n], fh, ql[n][ks][0], ql[n][ks][1]);
        if (F32) mma16816(S2[n], fl, qh[n][ks][0], qh[n][ks][1]);
      }
    }
    uint32_t ph[NG][2], pl[NG][2], pd[NG][2];  // p hi, p lo, p hi 2^-11
    float c0[NG], c1[NG];
    const bool v0 = g < nv_cur, v1 = g + 8 < nv_cur;
#pragma unroll
    for (int n = 0; n < NG; n++) {
      // keys g (S[0], S[1]) and g + 8 (S[2], S[3]) for rows 2 tq, 2 tq + 1
      auto score = [&](int j, bool on) { return on ? fmaf(S2[n][j], 2.f / kLift, S[n][j] + S[n][j]) : -INFINITY; };
      const float s0 = score(0, v0), s1 = score(1, v0), s2 = score(2, v1), s3 = score(3, v1);
      float n0 = fmaxf(s0, s2), n1 = fmaxf(s1, s3);
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) {
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
      }
      n0 = fmaxf(n0, m0[n]);
      n1 = fmaxf(n1, m1[n]);
      // no key so far (or every score -inf): a finite base keeps 2^(-inf - base) = 0
      const float b0 = n0 == -INFINITY ? 0.f : n0 - kPBits, b1 = n1 == -INFINITY ? 0.f : n1 - kPBits;
      c0[n] = m0[n] == -INFINITY ? 0.f : exp2f(m0[n] - n0);
      c1[n] = m1[n] == -INFINITY ? 0.f : exp2f(m1[n] - n1);
      m0[n] = n0;
      m1[n] = n1;
      const float p0 = exp2f(s0 - b0), p1 = exp2f(s1 - b1), p2 = exp2f(s2 - b0), p3 = exp2f(s3 - b1);
      l0[n] = l0[n] * c0[n] + (p0 + p2);
      l1[n] = l1[n] * c1[n] + (p1 + p3);
      split2(p0, p1, ph[n][0], pl[n][0]);
      split2(p2, p3, ph[n][1], pl[n][1]);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        ph[n][j] = movmatrix(ph[n][j]);
        pl[n][j] = movmatrix(pl[n][j]);
        if (F32) pd[n][j] = h2_bits(__hmul2(*reinterpret_cast<const __half2*>(&ph[n][j]), __float2half2_rn(1.f / kLift)));
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      v_frag(vs_, j, fh, fl, KVT());
#pragma unroll
      for (int n = 0; n < NG; n++) {
        O[n][j][0] *= c0[n];
        O[n][j][1] *= c1[n];
        O[n][j][2] *= c0[n];
        O[n][j][3] *= c1[n];
        mma16816(O[n][j], fh, ph[n][0], ph[n][1]);
        mma16816(O[n][j], fh, pl[n][0], pl[n][1]);
        if (F32) mma16816(O[n][j], fl, pd[n][0], pd[n][1]);
      }
    }
    __syncwarp();
    if (W::kStages == 1) {
      nv_next = issue(t + kWarps, page_next, stage);
      page_next = page_at(t + 2 * kWarps);
    }
    nv_cur = nv_next;
    stage ^= W::kStages - 1;
  }
  cp_async_wait<0>();
#pragma unroll
  for (int n = 0; n < NG; n++) {
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) {
      l0[n] += __shfl_xor_sync(0xffffffffu, l0[n], o);
      l1[n] += __shfl_xor_sync(0xffffffffu, l1[n], o);
    }
    if (g == 0) {
      sm_m[warp][8 * n + 2 * tq] = m0[n];
      sm_m[warp][8 * n + 2 * tq + 1] = m1[n];
      sm_l[warp][8 * n + 2 * tq] = l0[n];
      sm_l[warp][8 * n + 2 * tq + 1] = l1[n];
    }
  }
  __syncthreads();  // every warp's tiles are consumed: the staging becomes [warp][8 NG][kSoPitch] f32
  float* so = reinterpret_cast<float*>(sm);
#pragma unroll
  for (int n = 0; n < NG; n++)
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float* d = so + (warp * 8 * NG + 8 * n + 2 * tq) * kSoPitch + 16 * j + g;
      d[0] = O[n][j][0];
      d[kSoPitch] = O[n][j][1];
      d[8] = O[n][j][2];
      d[kSoPitch + 8] = O[n][j][3];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NG * 32; i += 32 * kWarps) {
    const int r = (i & 7) + (i >> 8) * 8, c = (i >> 3) & 31;
    if (r >= nrow) continue;  // FUSED: piece c of row r is read and written by this thread alone
    float mm = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; w++) mm = fmaxf(mm, sm_m[w][r]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const float f = sm_m[w][r] == -INFINITY ? 0.f : exp2f(sm_m[w][r] - mm);
      const float4 x = reinterpret_cast<const float4*>(so + (w * 8 * NG + r) * kSoPitch)[c];
      l += f * sm_l[w][r];
      o.x += f * x.x;
      o.y += f * x.y;
      o.z += f * x.z;
      o.w += f * x.w;
    }
    if (FUSED) {
      reinterpret_cast<float4*>(so + r * kSoPitch)[c] = o;
      if (c == 0) part_m[r] = mm, part_l[r] = l;
      continue;
    }
    const size_t at = part_row(a, split, kvh, row0 + r);
    if (c == 0) {
      a.pm[at] = mm - kPBits;
      a.pl[at] = l;
    }
    a.po[part_at(at, c)] = o;
  }
  if (FUSED) {
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    // rows of this CTA: rank, rank + C, ...; 4 rows x 32 pieces at a time
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), c = threadIdx.x & 31;
    for (int r = rank + C * warp; r < nrow && len >= 0; r += C * kWarps) {
      float mm[8], ls[8];
      float4 x[8];
#pragma unroll
      for (int s = 0; s < 8; s++) {
        mm[s] = -INFINITY;
        if (s < C) {
          mm[s] = *cl.map_shared_rank(&part_m[r], s);
          ls[s] = *cl.map_shared_rank(&part_l[r], s);
          x[s] = *cl.map_shared_rank(reinterpret_cast<float4*>(so + r * kSoPitch) + c, s);
        }
      }
      float m = mm[0];
#pragma unroll
      for (int s = 1; s < 8; s++) m = fmaxf(m, mm[s]);
      float l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < 8; s++)
        if (s < C) {
          const float f = mm[s] == -INFINITY ? 0.f : exp2f(mm[s] - m);
          l += f * ls[s];
          o.x += f * x[s].x;
          o.y += f * x[s].y;
          o.z += f * x[s].z;
          o.w += f * x[s].w;
        }
      const int rr = row0 + r;
      store_out(a, a.out + (long long)(rr / G) * a.ldo + (kvh * G + rr % G) * kHeadDim + 4 * c, o, l);
    }
    cl.sync();  // the parts are read
    return;
  }
  // the suffixes, launched beside the prefix's own kernel, whose results they do
  // not need: their end waits for that kernel's, so that the combine, which
  // follows them, finds both
  if (NG == 1 && p.own) pdl_wait();
}

// ======================================================================
// The prefix for many rows on the tcgen05 tensor cores (f16 cache)
// ======================================================================
// A CTA takes 128 rows of one KV head over one split of the prefix, in blocks
// of 128 keys: S = q K^T (M = rows, N = keys; q as f16 hi + lo stacked on the
// same K: 16 MMAs of K = 16), softmax by one thread a row from TMEM, P back to
// TMEM as f16 hi + lo over S's own columns, O = P V (A from TMEM, V^T as the
// key-major tile read MN-major; 16 MMAs).  Two warpgroups take the blocks in
// turn, so one's softmax runs under the other's products.  A block's O is a
// fresh accumulator, added to the row's f32 registers while the next scores are
// made: kept in TMEM over a split it loses about 2^-24.5 a step, all one way
// (2048 keys: 4e-6 of the output, against 1e-6 here).
// Warps: 0-3 and 4-7 softmax, 8 copies K, 9 copies V (TMA: a page of one KV
// head is two boxes of 16 rows x 64 dims, 128-byte swizzle), 10 issues MMAs and
// owns TMEM.
constexpr int kTcThreads = 384, kTcBlock = 128;
constexpr uint32_t kTcTile = 128 * kHeadDim * 2;  // 32 KB: 128 rows or keys of f16
constexpr uint32_t kTcHalf = kTcTile / 2;         // 128 keys x 64 dims, 128-byte rows
constexpr int kTcSmem = 6 * kTcTile;              // q hi, q lo, 2 x (K, V)
constexpr uint32_t kTcCols = 512;                 // per warpgroup 128 of S / P and 128 of O

struct TcSmem {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], v_raw;
  uint32_t tmem;
  int err;
  int nv[2][8];  // valid keys of each page of a stage's block
  float m0[256], m1[256];  // each warpgroup's bases and sums at the end
  float unscale[128];      // of a row's scores
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
// A from tensor memory: 128 lanes x 8 columns of f16 pairs
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Descriptor of a tile of 128-byte rows with the 128-byte swizzle: 8-row groups
// sbo apart; MN-major: 64-element columns lbo apart (K-major: one column, the
// next at another start).
__device__ __forceinline__ uint64_t smem_desc_sw128(const void* p, uint32_t lbo, uint32_t sbo) {
  return smem_desc(p, lbo, sbo) | (2ull << 61);
}
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* map, int dim, int head, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(dim), "r"(head), "r"(row), "r"(smem_addr(bar))
      : "memory");
}

// 16-byte chunk c of row r in a 128-row tile of core matrices (8 rows x 16 bytes)
__device__ __forceinline__ uint32_t core_off(int r, int c) { return c * 2048 + (r >> 3) * 128 + (r & 7) * 16; }

__global__ void __launch_bounds__(kTcThreads, 1) attn_prefix_tc_kernel(const __grid_constant__ SharedArgs a,
                                                                      const __grid_constant__ CUtensorMap kmap,
                                                                      const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ __align__(1024) unsigned char tsm[];
  __shared__ TcSmem S;
  unsigned char* qs = tsm;                  // q hi, then q lo
  unsigned char* kvs = tsm + 2 * kTcTile;   // stage s: K at 2 s tiles, V one further
  // the warp's number through a shuffle: known to be the same in all lanes, so the
  // MMA warp's descriptors stay in uniform registers
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const SharedPlan& p = a.p;
  pdl_launch_dependents();
  int blk = blockIdx.x;
  const int tile = blk % p.row_tiles;
  blk /= p.row_tiles;
  const int kvh = blk % a.nkv, split = blk / a.nkv;
  const int k0 = split * p.pref_keys, k1 = min(a.prefix_len, k0 + p.pref_keys);
  const int nblk = (k1 - k0 + kTcBlock - 1) / kTcBlock;

  if (tid == 0) {
    S.err = 0;
    mbar_init(&S.q_full, 256);
    mbar_init(&S.v_raw, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&S.k_full[i], 1);
      mbar_init(&S.k_empty[i], 1);
      mbar_init(&S.v_full[i], 1);
      mbar_init(&S.v_empty[i], 1);
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i], 128);
      mbar_init(&S.o_full[i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 10) tmem_alloc(&S.tmem, kTcCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  bool dead = false;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp < 10) {
      // ------------------------------------------------ K (warp 8) and V (warp 9) of every block
      const bool is_v = warp == 9;
      const CUtensorMap* map = is_v ? &vmap : &kmap;
      uint32_t raw = 0;
      for (int j = 0; j < nblk; j++) {
        const int st = j & 1, key0 = k0 + j * kTcBlock;
        const int g = lane & 7, half = (lane >> 3) & 1;  // lanes 0-15: one box each
        const int left = k1 - key0 - g * kPage;
        uint32_t page = 0;
        int nv = 0;
        if (left > 0) {
          page = __ldg(a.prefix_pages + key0 / kPage + g);
          nv = min(kPage, left);
          if (page >= a.n_pages) {  // a page outside the pool: its keys are left out
            nv = 0;
            if (a.err) *a.err = 1;
          }
        }
        uint64_t* full = is_v ? &S.v_full[st] : &S.k_full[st];
        if (!dead && !tc_wait(is_v ? &S.v_empty[st] : &S.k_empty[st], ((j >> 1) & 1) ^ 1, &S.err)) dead = true;
        unsigned char* dst = kvs + (2 * st + is_v) * kTcTile;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, nv > 0 && lane < 16)) * (kTcTile / 16);
        const bool whole = __all_sync(0xffffffffu, nv == kPage);
        if (is_v && lane < 8) S.nv[st][lane] = nv;
        // masked rows of V must be zeros (0 x NaN): such a block lands on v_raw, is mended, then is full
        uint64_t* bar = is_v && !whole ? &S.v_raw : full;
        __syncwarp();
        if (lane == 0) mbar_expect_tx(bar, bytes);
        __syncwarp();
        if (lane < 16 && nv > 0)
          tma_page(dst + half * kTcHalf + g * (kPage * 128), map, 64 * half, kvh, (int)(page * kPage), bar);
        if (is_v && !whole) {
          if (!dead && !tc_wait(&S.v_raw, raw, &S.err)) dead = true;
          raw ^= 1;
          for (int i = lane; i < 2 * 128 * 8; i += 32) {  // 16-byte pieces; a row's place is swizzled within itself only
            const int hf = i >> 10, rr = (i >> 3) & 127;
            const int n = __shfl_sync(0xffffffffu, nv, rr >> 4);
            if ((rr & 15) >= n)
              *reinterpret_cast<uint4*>(dst + hf * kTcHalf + rr * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full);
        }
      }
      // every copy has landed before the CTA may end
      for (int j = max(0, nblk - 2); j < nblk; j++)
        tc_wait_bounded(is_v ? &S.v_full[j & 1] : &S.k_full[j & 1], (j >> 1) & 1);
    } else if (warp == 10) {
      // ------------------------------------------------ MMA issue
      // D f32, A and B f16, M = N = 128; for P V the B operand (V) is MN-major
      const uint32_t id_s = (1u << 4) | (16u << 17) | (8u << 24), id_o = id_s | (1u << 16);
      // descriptors of the first MMA of each kind; the others are constants further (units of 16 bytes)
      const uint64_t q_desc = smem_desc(qs, 2048, 128), k_desc = smem_desc_sw128(kvs, 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(kvs + kTcTile, kTcHalf, 1024);  // all dims of a key-major tile
      if (!tc_wait(&S.q_full, 0, &S.err)) dead = true;
      auto issue_s = [&](int j) {
        const uint32_t w = j & 1;
        if (!dead && !tc_wait(&S.k_full[w], (j >> 1) & 1, &S.err)) dead = true;
        tc_fence_after();
        const uint64_t kd = k_desc + w * (2 * kTcTile >> 4);
        const uint32_t d = tmem + w * 256;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < 16; i++)  // q hi, then q lo, against the same K
            mma_f16_ss(d, q_desc + i * (4096 >> 4), kd + ((((i >> 2) & 1) * kTcHalf + (i & 3) * 32) >> 4), id_s, i > 0);
          mma_commit(&S.s_full[w]);
          mma_commit(&S.k_empty[w]);
        }
        __syncwarp();
      };
      issue_s(0);
      if (nblk > 1) issue_s(1);
      for (int j = 0; j < nblk; j++) {
        const uint32_t w = j & 1;
        if (!dead && !tc_wait(&S.v_full[w], (j >> 1) & 1, &S.err)) dead = true;
        if (!dead && !tc_wait(&S.p_full[w], (j >> 1) & 1, &S.err)) dead = true;
        tc_fence_after();
        const uint64_t vd = v_desc + w * (2 * kTcTile >> 4);
        const uint32_t pc = tmem + w * 256, d = pc + 128;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < 8; i++) {  // 16 keys a step: P hi and lo against the same V
            mma_f16_ts(d, pc + 32 * (i >> 1) + 8 * (i & 1), vd + i * (2048 >> 4), id_o, i > 0);
            mma_f16_ts(d, pc + 32 * (i >> 1) + 8 * (i & 1) + 16, vd + i * (2048 >> 4), id_o, true);
          }
          mma_commit(&S.o_full[w]);
          mma_commit(&S.v_empty[w]);
        }
        __syncwarp();
        if (j + 2 < nblk) issue_s(j + 2);  // over P of block j: the tensor core runs these in order
      }
      // every MMA is done before TMEM is freed, also when a wait gave up
      for (int j = max(0, nblk - 2); j < nblk; j++) tc_wait_bounded(&S.o_full[j & 1], (j >> 1) & 1);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // ------------------------------------------------ softmax, one thread a row
    const int w = warp >> 2, r = tid & 127;
    {
      // q times log2(e) / sqrt(128) as f16 hi and lo: 8 rows x 4 float4 a load (full sectors).
      // A row is scaled by the power of two that brings its largest element to [2^14, 2^15),
      // taken out of its scores again, so that its lo parts, of f16's 2^-24 steps, hold it to
      // 2^-39 of that element: large keys under small queries cost no precision, and q has the
      // range of f32.  (Unscaled: keys of 300 and queries of 0.005 gave an error of 4e-5.)
      const float c = 1.4426950408889634f * 0.08838834764831845f;
      float4 qx[16];
#pragma unroll
      for (int g = 0; g < 2; g++) {
        const int gr = tile * 128 + 16 * warp + 8 * g + (lane & 7);
        const float* q = a.q + (gr < p.rows ? (long long)(gr / p.G) * a.ldq + (kvh * p.G + gr % p.G) * kHeadDim : 0);
#pragma unroll
        for (int i = 0; i < 8; i++)
          qx[8 * g + i] = gr < p.rows ? __ldg(reinterpret_cast<const float4*>(q) + 4 * i + (lane >> 3)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float up[2];  // c and the row's scale
#pragma unroll
      for (int g = 0; g < 2; g++) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float4 v = qx[8 * g + i];
          top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));  // the row's other pieces: lanes 8 apart
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        // 2^e, e at most 100: below 2^-86 nothing of q is felt
        const int e = min(100, 14 + 127 - (int)(__float_as_uint(top * c) >> 23));
        up[g] = c * __uint_as_float((uint32_t)(127 + e) << 23);
        if (lane < 8) S.unscale[16 * warp + 8 * g + lane] = __uint_as_float((uint32_t)(127 - e) << 23);
      }
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int rr = 16 * warp + (i & 8) + (lane & 7), f = 4 * (i & 7) + (lane >> 3);  // half a 16-byte chunk
        const float4 v = qx[i];
        const float c = up[i >> 3];
        uint2 h, l;
        split2(v.x * c, v.y * c, h.x, l.x);
        split2(v.z * c, v.w * c, h.y, l.y);
        const uint32_t at = core_off(rr, f >> 1) + (f & 1) * 8;
        *reinterpret_cast<uint2*>(qs + at) = h;
        *reinterpret_cast<uint2*>(qs + kTcTile + at) = l;
      }
      fence_async_smem();
      mbar_arrive(&S.q_full);
    }
    const uint32_t base = tmem + w * 256 + ((uint32_t)(32 * (warp & 3)) << 16);
    float O[kHeadDim];
#pragma unroll
    for (int i = 0; i < kHeadDim; i++) O[i] = 0.f;
    float m = -INFINITY, l = 0.f;  // the base b is m - kPBits
    if (!tc_wait(&S.q_full, 0, &S.err)) dead = true;  // the other warps' S.unscale
    const float us = S.unscale[r];
    for (int j = w; j < nblk; j += 2) {
      if (!dead && !tc_wait(&S.s_full[w], (j >> 1) & 1, &S.err)) dead = true;
      // the block's valid keys: every page whole, but at the end of the prefix (or beside a bad page)
      if (!dead && !tc_wait(&S.v_full[w], (j >> 1) & 1, &S.err)) dead = true;
      bool whole = true;
#pragma unroll
      for (int g = 0; g < 8; g++) whole &= S.nv[w][g] == kPage;
      tc_fence_after();
      // scores 64 at a time, twice: the maximum, then the weights
      auto scores = [&](int half, uint32_t (&v)[2][32]) {
        tmem_ld32(base + 64 * half, v[0]);
        tmem_ld32(base + 64 * half + 32, v[1]);
        tmem_wait_ld();
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 64; i++)
            if (i % kPage >= S.nv[w][4 * half + i / kPage]) v[i / 32][i % 32] = __float_as_uint(-INFINITY);
        }
      };
      float top = m;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        uint32_t v[2][32];
        scores(half, v);
        float mx[2] = {__uint_as_float(v[0][0]), __uint_as_float(v[1][0])};
#pragma unroll
        for (int d = 1; d < 32; d++) {
          mx[0] = fmaxf(mx[0], __uint_as_float(v[0][d]));
          mx[1] = fmaxf(mx[1], __uint_as_float(v[1][d]));
        }
        top = fmaxf(top, us * fmaxf(mx[0], mx[1]));
      }
      const float corr = m == -INFINITY ? 0.f : ex2(m - top), b = top == -INFINITY ? 0.f : top - kPBits;
      m = top;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        uint32_t v[2][32];
        scores(half, v);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          uint32_t o[32];
#pragma unroll
          for (int d = 0; d < 16; d++) {
            const float x = ex2(fmaf(__uint_as_float(v[i][2 * d]), us, -b)), y = ex2(fmaf(__uint_as_float(v[i][2 * d + 1]), us, -b));
            s0 += x;
            s1 += y;
            split2(x, y, o[d], o[16 + d]);
          }
          tmem_st32(base + 64 * half + 32 * i, o);
        }
      }
      l = l * corr + (s0 + s1);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&S.p_full[w]);
      // the block's O, while the next scores are made (p_full of the next block lets O be overwritten)
      if (!dead && !tc_wait(&S.o_full[w], (j >> 1) & 1, &S.err)) dead = true;
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < 2; i++) {
        uint32_t v[2][32];
        tmem_ld32(base + 128 + 64 * i, v[0]);
        tmem_ld32(base + 128 + 64 * i + 32, v[1]);
        tmem_wait_ld();
#pragma unroll
        for (int d = 0; d < 64; d++) O[64 * i + d] = fmaf(O[64 * i + d], corr, __uint_as_float(v[d / 32][d % 32]));
      }
    }
    // ---- the two warpgroups' parts of a row joined: each gives half of its pieces, adds up the other half
    float* mine = w ? S.m1 : S.m0;
    mine[r] = m;
    mine[128 + r] = l;
    asm volatile("bar.sync 2, 256;" ::: "memory");  // both are past their last MMA: K and V are free
    const float mo = (w ? S.m0 : S.m1)[r], lo = (w ? S.m0 : S.m1)[128 + r], mm = fmaxf(m, mo);
    const float f = m == -INFINITY ? 0.f : ex2(m - mm);
    float4* ex = reinterpret_cast<float4*>(kvs) + r;  // [giver][16 pieces][128 rows]
#pragma unroll
    for (int i = 0; i < 16; i++) {
      float4 y;
      if (w) y = make_float4(O[4 * i] * f, O[4 * i + 1] * f, O[4 * i + 2] * f, O[4 * i + 3] * f);
      else y = make_float4(O[64 + 4 * i] * f, O[65 + 4 * i] * f, O[66 + 4 * i] * f, O[67 + 4 * i] * f);
      ex[(16 * w + i) * 128] = y;
    }
    asm volatile("bar.sync 2, 256;" ::: "memory");
    if (tile * 128 + r < p.rows) {
      const size_t at = part_row(a, split, kvh, tile * 128 + r);
      if (w == 0) {
        a.pm[at] = mm - kPBits;
        a.pl[at] = l * f + (mo == -INFINITY ? 0.f : lo * ex2(mo - mm));
      }
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float4 y = ex[(16 * (w ^ 1) + i) * 128];
        if (w) {
          y.x += O[64 + 4 * i] * f;
          y.y += O[65 + 4 * i] * f;
          y.z += O[66 + 4 * i] * f;
          y.w += O[67 + 4 * i] * f;
        } else {
          y.x += O[4 * i] * f;
          y.y += O[4 * i + 1] * f;
          y.z += O[4 * i + 2] * f;
          y.w += O[4 * i + 3] * f;
        }
        a.po[part_at(at, 16 * w + i)] = y;
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (tid == 0 && S.err && a.err) *a.err = 1;  // a bounded wait gave up
  if (warp == 10) tmem_free(tmem, kTcCols);
}

// One CTA per 8 rows of a KV head, a thread per (row, 16-byte piece): 32 splits
// at a time, their weights by thread (row, split) through shared memory, eight
// of a row's parts in flight.
// kLanes groups of 256 threads take the splits in turns and join at the end: few
// rows with many splits wait for one round of loads after the other (1 sequence,
// 8192 keys in 64 splits: 4 lanes 10.8 us, one 13.3; 64 x 8192 28.8 and 30.1).
template <int kLanes>
__global__ void __launch_bounds__(256 * kLanes) attn_shared_combine(const __grid_constant__ SharedArgs a) {
  constexpr int kC = 32 / kLanes;  // splits of a lane's turn
  __shared__ float sb[kLanes][kC][8], sl[kLanes][kC][8];
  const int kvh = blockIdx.x / a.p.groups, row0 = blockIdx.x % a.p.groups * 8;
  const int q = threadIdx.x >> 8, t = threadIdx.x & 255, rr = t & 7, c = t >> 3, r = row0 + rr, G = a.p.G;
  const int b = r / G, len = r < a.p.rows ? __ldg(a.lens + b) : -1;
  const bool on = len >= 0;  // a padding sequence's row stays as it is
  const int ns = on ? a.p.n_pref + (min(len, a.max_len) + a.p.suf_keys - 1) / a.p.suf_keys : 0;
  const size_t row = part_row(a, 0, kvh, r), step = (size_t)a.nkv * a.p.groups * 8;  // rows of a split
  const float4* po = a.po + part_at(row, c);
  if (len > a.max_len && a.err) *a.err = 1;
  pdl_wait();
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = kC * q; __syncthreads_or(s0 < ns); s0 += 32) {
    const int s = s0 + c;
    if (c < kC) {
      sb[q][c][rr] = s < ns ? __ldcg(a.pm + row + s * step) : -INFINITY;
      sl[q][c][rr] = s < ns ? __ldcg(a.pl + row + s * step) : 0.f;
    }
    float4 x[8];
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (s0 + j < ns) x[j] = __ldcg(po + (s0 + j) * step * 32);
    __syncthreads();
    float nm = m;
#pragma unroll 8
    for (int j = 0; j < kC; j++) nm = fmaxf(nm, sb[q][j][rr]);
    __syncthreads();
    if (c < kC) {
      const float mine = sb[q][c][rr];
      sb[q][c][rr] = mine == -INFINITY ? 0.f : exp2f(mine - nm);
    }
    const float f = m == -INFINITY ? 0.f : exp2f(m - nm);
    m = nm;
    l *= f;
    o.x *= f;
    o.y *= f;
    o.z *= f;
    o.w *= f;
    __syncthreads();
    for (int j0 = 0; j0 < kC && s0 + j0 < ns; j0 += 8) {
      if (j0) {
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (s0 + j0 + j < ns) x[j] = __ldcg(po + (s0 + j0 + j) * step * 32);
      }
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (s0 + j0 + j < ns) {
          const float w = sb[q][j0 + j][rr];
          l += w * sl[q][j0 + j][rr];
          o.x += w * x[j].x;
          o.y += w * x[j].y;
          o.z += w * x[j].z;
          o.w += w * x[j].w;
        }
    }
  }
  if (kLanes > 1) {
    __shared__ float4 so[kLanes][256];
    __shared__ float sm[kLanes][256], ss[kLanes][256];
    so[q][t] = o;
    sm[q][t] = m;
    ss[q][t] = l;
    __syncthreads();
    if (q) return;
#pragma unroll
    for (int i = 1; i < kLanes; i++) m = fmaxf(m, sm[i][t]);
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kLanes; i++) {
      const float f = sm[i][t] == -INFINITY ? 0.f : exp2f(sm[i][t] - m);
      const float4 x = so[i][t];
      l += f * ss[i][t];
      o.x += f * x.x;
      o.y += f * x.y;
      o.z += f * x.z;
      o.w += f * x.w;
    }
  }
  if (!on) return;
  store_out(a, a.out + b * a.ldo + (kvh * G + r % G) * kHeadDim + 4 * c, o, l);
}

// The launches of one call: the prefix kernel (tcgen05), the suffix kernel
// beside it, the combine after both.
cudaError_t launch_pdl(const void* fn, OncePerDevice& once, unsigned blocks, int threads, int smem, bool early, void** args,
                       cudaStream_t st, int cluster = 1) {
  int dev = 0;
  cudaError_t e = smem > 48 << 10 ? cudaGetDevice(&dev) : cudaSuccess;
  if (e == cudaSuccess && smem > 48 << 10 && once.first(dev)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) once.done(dev);
  }
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute at = {};
  if (cluster > 1) {
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
  } else {
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = early || cluster > 1 ? 1 : 0;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

// The pool as a tensor of [rows][KV heads][128 dims], read in boxes of 16 rows
// x 1 head x 64 dims with the 128-byte swizzle.
cudaError_t page_map(CUtensorMap* map, const void* pool, const SharedArgs& a) {
  static const auto encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                         const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                         CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill)>(f);
  }();
  if (!encode) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {kHeadDim, (cuuint64_t)a.nkv, (cuuint64_t)a.n_pages * kPage};
  const cuuint64_t strides[2] = {kHeadDim * 2, (cuuint64_t)a.nkv * kHeadDim * 2};
  const cuuint32_t box[3] = {64, 1, kPage}, step[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(pool), dims, strides, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? cudaSuccess
             : cudaErrorInvalidValue;
}

template <typename KVT, int NG, int kWarps, bool FUSED = false>
cudaError_t launch_warps(const SharedArgs& a, long long blocks, int pref, bool early, cudaStream_t st) {
  static OncePerDevice once;
  void* args[2] = {const_cast<SharedArgs*>(&a), &pref};
  using W = WarpTile<KVT>;
  return launch_pdl((const void*)attn_shared_kernel<KVT, NG, kWarps, FUSED>, once, (unsigned)blocks, 32 * kWarps,
                    kWarps * W::kStages * W::kBytes, early, args, st, FUSED ? a.p.n_pref + a.p.n_suf : 1);
}

template <typename KVT>
cudaError_t launch_shared(const SharedArgs& a, cudaStream_t st) {
  static OncePerDevice tc_once, no_smem;
  constexpr bool kF32 = WarpTile<KVT>::kF32;
  cudaError_t e = cudaSuccess;
  if (a.p.fused)
    return launch_warps<KVT, 1, kF32 ? 8 : 4, true>(a, (long long)a.nseq * a.nkv * a.p.gch * (a.p.n_pref + a.p.n_suf), 0, false, st);
  const int pref = a.p.n_pref * a.nkv * (a.p.own ? (a.p.groups + 1) / 2 : a.p.groups);
  if (a.p.tc) {
    CUtensorMap km, vm;
    e = page_map(&km, a.kc, a);
    if (e == cudaSuccess) e = page_map(&vm, a.vc, a);
    void* args[3] = {const_cast<SharedArgs*>(&a), &km, &vm};
    if (e == cudaSuccess)
      e = launch_pdl((const void*)attn_prefix_tc_kernel, tc_once, (unsigned)(a.p.n_pref * a.nkv * a.p.row_tiles), kTcThreads,
                     kTcSmem, false, args, st);
  } else if constexpr (std::is_same<KVT, float>::value) {
    if (a.p.own) e = launch_warps<KVT, 2, 4>(a, pref, pref, false, st);
  }
  const long long blocks = (a.p.own ? 0 : pref) + (long long)a.p.n_suf * a.nseq * a.nkv * a.p.gch;
  if (e == cudaSuccess && blocks > 0)
    e = kF32 && !a.p.many ? launch_warps<KVT, 1, kF32 ? 8 : 4>(a, blocks, a.p.own ? 0 : pref, a.p.own, st)
                          : launch_warps<KVT, 1, 4>(a, blocks, a.p.own ? 0 : pref, a.p.own, st);
  void* args[1] = {const_cast<SharedArgs*>(&a)};
  if (e == cudaSuccess)
    e = launch_pdl(a.p.lanes > 1 ? (const void*)attn_shared_combine<4> : (const void*)attn_shared_combine<1>, no_smem,
                   (unsigned)(a.nkv * a.p.groups), 256 * a.p.lanes, 0, blocks > 0 || a.p.own, args, st);
  return e;
}

bool misaligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) & (to - 1); }

size_t shared_rows(const SharedPlan& p, int nkv) { return (size_t)(p.n_pref + p.n_suf) * nkv * p.groups * 8; }
size_t shared_bytes(const SharedPlan& p, int nkv) { return shared_rows(p, nkv) * (kHeadDim + 2) * sizeof(float); }
// what a call is asked for: enough for either cache type
size_t shared_need(const SharedPlan& p, const SharedPlan& other, int nkv) {
  return std::max<size_t>(16, std::max(shared_bytes(p, nkv), shared_bytes(other, nkv)));
}

const char* shared_dims(int nseq, int nh, int nkv, int prefix_len, int max_len) {
  if (nseq < 1 || nseq > 65536) return "need 1 <= nseq <= 65536";
  if (nkv < 1 || nh < nkv || nh % nkv || nh > 1024) return "need nh a multiple of nkv, at most 1024";
  if (prefix_len < 0 || max_len < 0 || prefix_len > (1 << 28) || max_len > (1 << 28))
    return "need 0 <= prefix_len, max_len <= 2^28";
  return nullptr;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" {

EG_API eg_status eg_op_kv_append_paged(const float* qkv, int64_t ld, int T, const int* pos, const int* slot,
                                       const uint32_t* pages, int n_slots, int max_pages, int n_pages,
                                       int prefix_len, void* k_cache, void* v_cache, const float* cos_t,
                                       const float* sin_t, int table_len, int nh, int nkv, int kv_f16,
                                       float* q_out, int64_t ldq, int* err, void* stream) {
  if (T < 0 || nh < 0 || nkv < 1 || nh > 1024 || nkv > 1024) return fail(EG_ERR_ARG, "kv_append_paged: bad T or heads");
  if (n_slots < 1 || max_pages < 1 || n_pages < 1 || prefix_len < 0 || table_len < 1)
    return fail(EG_ERR_ARG, "kv_append_paged: bad page table, pool or table length");
  if (n_pages > (1 << 27)) return fail(EG_ERR_ARG, "kv_append_paged: more than 2^27 pages");
  if (T == 0) return EG_OK;
  if (!qkv || !pos || !slot || !pages || !k_cache || !v_cache || !cos_t || !sin_t)
    return fail(EG_ERR_ARG, "kv_append_paged: null argument");
  const int H = nh + 2 * nkv;
  if (ld < (int64_t)H * kHeadDim || ld % 4) return fail(EG_ERR_ARG, "kv_append_paged: row stride %lld below %d or not a multiple of 4", (long long)ld, H * kHeadDim);
  if (q_out && (ldq < (int64_t)nh * kHeadDim || ldq % 4))
    return fail(EG_ERR_ARG, "kv_append_paged: q_out row stride %lld below %d or not a multiple of 4", (long long)ldq, nh * kHeadDim);
  if (misaligned(qkv, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(cos_t, 16) ||
      misaligned(sin_t, 16) || misaligned(q_out, 16))
    return fail(EG_ERR_ARG, "kv_append_paged: 16-byte aligned buffers required");
  AppendArgs a = {qkv, ld, T, pos, slot, pages, n_slots, max_pages, n_pages, prefix_len, k_cache, v_cache,
                  cos_t, sin_t, table_len, nh, nkv, q_out, ldq, err};
  const long long heads = (long long)T * H;
  if (heads / 16 >= 0x7fffffffLL) return fail(EG_ERR_ARG, "kv_append_paged: too many rows");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (kv_f16) launch_append<__half>(a, heads, st);
  else launch_append<float>(a, heads, st);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(EG_ERR_CUDA, "kv_append_paged: %s", cudaGetErrorString(e));
  return EG_OK;
}

EG_API eg_status eg_op_attn_shared_prefix_bytes(int nseq, int nh, int nkv, int prefix_len, int max_len,
                                                uint64_t* bytes) {
  if (!bytes) return fail(EG_ERR_ARG, "attn_shared_prefix: null argument");
  if (const char* why = shared_dims(nseq, nh, nkv, prefix_len, max_len)) return fail(EG_ERR_ARG, "attn_shared_prefix: %s", why);
  *bytes = shared_need(shared_plan(nseq, nh, nkv, prefix_len, max_len, 0), shared_plan(nseq, nh, nkv, prefix_len, max_len, 1), nkv);
  return EG_OK;
}

EG_API eg_status eg_op_attn_shared_prefix(const float* q, int64_t ldq, int nseq, const void* k_cache,
                                          const void* v_cache, int n_pages, const uint32_t* prefix_pages,
                                          int prefix_len, const uint32_t* pages, int max_pages, const int* lens,
                                          int max_len, int nh, int nkv, int kv_f16, float* out, int64_t ldo,
                                          void* ws, uint64_t ws_bytes, int* err, void* stream) {
  if (const char* why = shared_dims(nseq, nh, nkv, prefix_len, max_len)) return fail(EG_ERR_ARG, "attn_shared_prefix: %s", why);
  if (!q || !k_cache || !v_cache || !lens || !out || !ws || (prefix_len > 0 && !prefix_pages) || (max_len > 0 && !pages))
    return fail(EG_ERR_ARG, "attn_shared_prefix: null argument");
  if (n_pages < 1 || max_pages < 0 || n_pages > (1 << 27)) return fail(EG_ERR_ARG, "attn_shared_prefix: bad pool or page table");
  if ((long long)max_pages * kPage < max_len)
    return fail(EG_ERR_ARG, "attn_shared_prefix: max_len %d > %d pages of %d", max_len, max_pages, kPage);
  if (ldq < (int64_t)nh * kHeadDim || ldq % 4 || ldo < (int64_t)nh * kHeadDim || ldo % 4)
    return fail(EG_ERR_ARG, "attn_shared_prefix: row strides must be multiples of 4, at least %d", nh * kHeadDim);
  if (misaligned(q, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(out, 16) || misaligned(ws, 16))
    return fail(EG_ERR_ARG, "attn_shared_prefix: 16-byte aligned buffers required");
  SharedArgs a = {};
  a.p = shared_plan(nseq, nh, nkv, prefix_len, max_len, kv_f16);
  const size_t need = shared_need(a.p, shared_plan(nseq, nh, nkv, prefix_len, max_len, !kv_f16), nkv);
  if (ws_bytes < need)
    return fail(EG_ERR_ARG, "attn_shared_prefix: workspace of %llu bytes, %llu needed", (unsigned long long)ws_bytes, (unsigned long long)need);
  a.q = q;
  a.ldq = ldq;
  a.nseq = nseq;
  a.nh = nh;
  a.nkv = nkv;
  a.kc = k_cache;
  a.vc = v_cache;
  a.n_pages = (uint32_t)n_pages;
  a.prefix_pages = prefix_pages;
  a.prefix_len = prefix_len;
  a.pages = pages;
  a.max_pages = max_pages;
  a.lens = lens;
  a.max_len = max_len;
  a.out = out;
  a.ldo = ldo;
  const size_t rows = shared_rows(a.p, nkv);
  a.po = static_cast<float4*>(ws);
  a.pm = reinterpret_cast<float*>(a.po + rows * (kHeadDim / 4));
  a.pl = a.pm + rows;
  a.err = err;
  if (((long long)a.p.n_pref * a.p.groups + (long long)a.p.n_suf * nseq * a.p.gch) * nkv > 0x7fffffffLL)
    return fail(EG_ERR_ARG, "attn_shared_prefix: too many splits");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = kv_f16 ? launch_shared<__half>(a, st) : launch_shared<float>(a, st);
  if (e != cudaSuccess) return fail(EG_ERR_CUDA, "attn_shared_prefix: %s", cudaGetErrorString(e));
  return EG_OK;
}

}  // extern "C"
