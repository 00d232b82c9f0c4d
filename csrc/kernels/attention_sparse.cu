// Attention of one new token per row over pages chosen by a cheap score.
//
// Three kernels over the paged cache ([page][kv_head][16][128] bf16):
//
//   page_bounds    lo[d], hi[d] = min, max over the page's valid keys k[.][d]
//   select_pages   score(p) = max over the KV group's query heads h of
//                             sum_d max(q_hd lo_pd, q_hd hi_pd)
//                  (no logit of the page's tokens is larger); the `first` first
//                  and `last` last pages and the best of the others, ties to
//                  the lowest index
//   decode_sparse  softmax attention over the chosen pages' valid tokens
//
// max(q lo, q hi) = max(q, 0) hi + min(q, 0) lo because lo <= hi, so a page's
// score is a dot product of 256 terms (the bound by a page's smallest and largest keys
// was published by Tang et al., "Query-Aware Sparsity for Efficient Long-Context LLM
// Inference", 2024): tensor-core work with 16 pages as the
// rows and the group's query heads as the columns.  What bounds the selection
// is reading the bounds, 512 bytes per (page, KV head); what bounds the
// attention is reading 8 KB per chosen (page, KV head).
//
// The order of the scores is that of their sums in 64 bits.  bf16 products are exact
// in fp32; their fp32 sums carry an error bound e = kScoreErr * sum|terms|, and
// where the bounds of two pages around the cut overlap, both are summed again
// in fp64.  Where a page or query holds an infinity or a NaN the score counts as
// +infinity, so such a page is taken and shows up in the output as it would without the
// selection; where only the fp32 sums overflow, the error bound is infinite and the
// page compared in fp64.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <stdexcept>

#include "attention_sparse.h"
#include "common.cuh"

namespace lf {
namespace attn {

namespace {

constexpr int D = 128;
constexpr int PAGE = 16;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Streaming 16-byte load: K and V are used once.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ __nv_bfloat162 as_bf2(uint32_t x) { return *reinterpret_cast<__nv_bfloat162*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 x) { return *reinterpret_cast<uint32_t*>(&x); }

__device__ __forceinline__ uint32_t min_nan(uint32_t a, uint32_t b) { return as_u32(__hmin2_nan(as_bf2(a), as_bf2(b))); }
__device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) { return as_u32(__hmax2_nan(as_bf2(a), as_bf2(b))); }

// The physical page of logical page `idx`; a bad table entry is recorded and
// reads the reserved zero page.
__device__ __forceinline__ int table_page(const int32_t* bt, int idx, int num_pages) {
  const int p = bt[idx];
  if (p < 0 || p >= num_pages) {
    set_error(kErrBadIndex, (unsigned long long)idx);
    return 0;
  }
  return p;
}

// A row's KV length; a length beyond the block table is recorded and cut.
__device__ __forceinline__ int row_length(const int32_t* seq_lens, int r, int width) {
  const int L = seq_lens[r];
  if (L > width * PAGE) {
    set_error(kErrBadIndex, (unsigned long long)r);
    return width * PAGE;
  }
  return L > 0 ? L : 0;
}

// ===========================================================================
// page_bounds: one warp per (row, page, KV head).  16 lanes hold the 128
// dimensions, the warp's halves take the even and the odd tokens, all eight
// loads of a lane in flight.
// ===========================================================================
__global__ void __launch_bounds__(128) page_bounds_kernel(const BoundsArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t per_row = (int64_t)a.Hkv * a.max_pages;
  if (unit >= per_row * a.rows) return;
  const int r = (int)(unit / per_row);
  const int rest = (int)(unit % per_row);
  const int kvh = rest % a.Hkv, pi = rest / a.Hkv;
  const int L = row_length(a.seq_lens, r, a.width);
  const int start = a.start[r];
  if (start >= L) return;
  if (start < 0 || L - start > a.max_new) {
    if (lane == 0) set_error(kErrBadIndex, (unsigned long long)r);
    return;
  }
  const int page = start / PAGE + pi;
  const int valid = min(PAGE, L - page * PAGE);
  if (valid <= 0) return;
  const int64_t phys = table_page(a.block_table + (int64_t)r * a.bt_stride, page, a.num_pages);
  const int half = lane >> 4, c = lane & 15;
  const __nv_bfloat16* src = a.kcache + ((phys * a.Hkv + kvh) * PAGE + half) * D + c * 8;
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (2 * i + half < valid) v[i] = *reinterpret_cast<const uint4*>(src + 2 * i * D);
  constexpr uint32_t kPosInf = 0x7f807f80u, kNegInf = 0xff80ff80u;
  uint4 lo = make_uint4(kPosInf, kPosInf, kPosInf, kPosInf), hi = make_uint4(kNegInf, kNegInf, kNegInf, kNegInf);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (2 * i + half < valid) {
      lo.x = min_nan(lo.x, v[i].x), lo.y = min_nan(lo.y, v[i].y);
      lo.z = min_nan(lo.z, v[i].z), lo.w = min_nan(lo.w, v[i].w);
      hi.x = max_nan(hi.x, v[i].x), hi.y = max_nan(hi.y, v[i].y);
      hi.z = max_nan(hi.z, v[i].z), hi.w = max_nan(hi.w, v[i].w);
    }
  }
  lo.x = min_nan(lo.x, __shfl_xor_sync(kFull, lo.x, 16)), lo.y = min_nan(lo.y, __shfl_xor_sync(kFull, lo.y, 16));
  lo.z = min_nan(lo.z, __shfl_xor_sync(kFull, lo.z, 16)), lo.w = min_nan(lo.w, __shfl_xor_sync(kFull, lo.w, 16));
  hi.x = max_nan(hi.x, __shfl_xor_sync(kFull, hi.x, 16)), hi.y = max_nan(hi.y, __shfl_xor_sync(kFull, hi.y, 16));
  hi.z = max_nan(hi.z, __shfl_xor_sync(kFull, hi.z, 16)), hi.w = max_nan(hi.w, __shfl_xor_sync(kFull, hi.w, 16));
  uint4* dst = reinterpret_cast<uint4*>(a.bounds + (phys * a.Hkv + kvh) * 2 * D);
  dst[half * 16 + c] = half ? hi : lo;
}

// ===========================================================================
// Page scores.  A warp takes 16 pages at a time as the 16 rows of m16n8k16; lane
// (g, c) = (lane / 4, lane % 4) loads 16-byte pieces c, c + 4, ... of the bounds
// of pages g and g + 8, sixteen warps per SM with a tile each under way.  A piece is
// eight consecutive dimensions, which serve two k-steps: the order of k is free
// as long as the queries use the same one, so no shared memory is needed.
// Pieces 0..15 (lo) meet min(q, 0) and pieces 16..31 (hi) meet max(q, 0).
//
// Plain loads, because the same pieces by cp.async take 27 cycles per warp
// instruction (19 bytes per clock, where the memory delivers 23), and a bulk copy
// per page 130 cycles of the issuing warp; a second tile in registers halves the
// warps (64 rows x 8 heads x 2048 pages: 92 us so, 97, 97 and 102 the other ways).
//
// Error bound: a k16 step adds 16 exact products to the accumulator with at
// most 17 roundings or truncations at the largest addend, 2^-23 each; four
// chains of four steps over disjoint terms give 68 * 2^-23 = 2^-16.9 of the sum
// of magnitudes, and joining them 2^-22.4 more.  The magnitudes are summed by the
// same instruction on the operands without their signs.
// ===========================================================================
constexpr float kScoreErr = 1.f / 32768.f;   // 2^-15, four times what is derived above
constexpr float kScoreTiny = 0x1p-118f;      // and what 256 products and their sums may lose below 2^-126
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kScoreTile = 16 * kWarps;      // pages of one pass of a CTA
constexpr int kScorePasses = 2;              // most passes of a CTA

template <int NH>   // groups of eight query heads
__global__ void __launch_bounds__(kThreads, NH == 1 ? 4 : 2) page_score_kernel(const SelectArgs a, int passes) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.x % a.Hkv, chunk = blockIdx.x / a.Hkv;
  const int r = blockIdx.y;
  const int G = a.Hq / a.Hkv;
  const int begin = chunk * passes * kScoreTile + warp * 16;   // this warp's first page; the next ones 64 further
  const int32_t* bt = a.block_table + (int64_t)r * a.bt_stride;
  pdl_wait();
  // lane l holds page l % 16 of pass l / 16; fetched before the length is known
  const int lane_page = begin + (lane >> 4) * kScoreTile + (lane & 15);
  int table = (lane >> 4) < passes && lane_page < a.width ? bt[lane_page] : 0;
  const int tok = a.tok_index[r];
  const int L = row_length(a.seq_lens, r, a.width);
  const int n = (L + PAGE - 1) / PAGE;
  const int end = min(n, (chunk + 1) * passes * kScoreTile);
  if (n <= a.budget || begin >= end) return;
  if (tok < 0 || tok >= a.tokens) {
    if (lane == 0) set_error(kErrBadIndex, (unsigned long long)r);
    return;
  }
  const int mine = (end - begin + kScoreTile - 1) / kScoreTile;   // passes of this warp
  if (table < 0 || table >= a.num_pages) {   // recorded; the reserved zero page stands in
    if (lane_page < end) set_error(kErrBadIndex, (unsigned long long)lane_page);
    table = 0;
  }
  const uint4* bounds = reinterpret_cast<const uint4*>(a.bounds) + kvh * (2 * D / 8) + c;
  const int64_t page_pieces = (int64_t)a.Hkv * (2 * D / 8);
  struct Tile {
    uint4 a[8], b[8];
  };
  auto load = [&](int it, Tile& t) {
    const int pa = __shfl_sync(kFull, table, it * 16 + g), pb = __shfl_sync(kFull, table, it * 16 + g + 8);
    // entries past the row's end read page 0 or the table's; their scores are not stored
    const uint4* ra = bounds + pa * page_pieces;
    const uint4* rb = bounds + pb * page_pieces;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      t.a[j] = ld_stream(ra + 4 * j);
      t.b[j] = ld_stream(rb + 4 * j);
    }
  };
  Tile t0;
  load(0, t0);
  uint4 q[NH][4];
#pragma unroll
  for (int t = 0; t < NH; ++t) {
    const __nv_bfloat16* qh = a.q + (int64_t)tok * a.q_ld + (int64_t)(kvh * G + t * 8 + g) * D;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      q[t][j] = t * 8 + g < G ? *reinterpret_cast<const uint4*>(qh + 8 * (c + 4 * j)) : make_uint4(0u, 0u, 0u, 0u);
  }
  float2* ws = a.ws + ((int64_t)r * a.Hkv + kvh) * a.width;
  float odd = 0.f;                        // infinite where a score was not finite
  auto score = [&](int it, const Tile& tile) {
    const int p0 = begin + it * kScoreTile;
    float best_a = -INFINITY, best_b = -INFINITY, err_a = 0.f, err_b = 0.f;
#pragma unroll
    for (int t = 0; t < NH; ++t) {
      float s[4][4], m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = m[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t* pa4 = reinterpret_cast<const uint32_t*>(&tile.a[j]);
        const uint32_t* pb4 = reinterpret_cast<const uint32_t*>(&tile.b[j]);
        const uint32_t* q4 = reinterpret_cast<const uint32_t*>(&q[t][j & 3]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t b0 = j < 4 ? min_nan(q4[2 * h], 0u) : max_nan(q4[2 * h], 0u);
          const uint32_t b1 = j < 4 ? min_nan(q4[2 * h + 1], 0u) : max_nan(q4[2 * h + 1], 0u);
          mma_bf16(s[j & 3], pa4[2 * h], pb4[2 * h], pa4[2 * h + 1], pb4[2 * h + 1], b0, b1);
          constexpr uint32_t kAbs = 0x7fff7fffu;
          mma_bf16(m, pa4[2 * h] & kAbs, pb4[2 * h] & kAbs, pa4[2 * h + 1] & kAbs, pb4[2 * h + 1] & kAbs, b0 & kAbs,
                   b1 & kAbs);
        }
      }
      // columns 2c, 2c + 1 of pages g and g + 8
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = (s[0][i] + s[1][i]) + (s[2][i] + s[3][i]);
        if (t * 8 + 2 * c + (i & 1) < G) {
          const bool fin = isfinite(v) && isfinite(m[i]);
          float& b = i < 2 ? best_a : best_b;
          float& e = i < 2 ? err_a : err_b;
          b = fmaxf(b, fin ? v : 0.f);
          e = fmaxf(e, fin ? fmaf(m[i], kScoreErr, kScoreTiny) : INFINITY);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      best_a = fmaxf(best_a, __shfl_xor_sync(kFull, best_a, o));
      best_b = fmaxf(best_b, __shfl_xor_sync(kFull, best_b, o));
      err_a = fmaxf(err_a, __shfl_xor_sync(kFull, err_a, o));
      err_b = fmaxf(err_b, __shfl_xor_sync(kFull, err_b, o));
    }
    odd = fmaxf(odd, fmaxf(err_a, err_b));
    if (c == 0) {
      if (p0 + g < end) ws[p0 + g] = make_float2(best_a, err_a);
      if (p0 + g + 8 < end) ws[p0 + g + 8] = make_float2(best_b, err_b);
    }
  };
  for (int it = 0; it < mine; ++it) {
    if (it > 0) load(it, t0);
    score(it, t0);
  }
  if (__any_sync(kFull, isinf(odd))) {    // rare: which ones hold an infinity or a NaN, and which only overflow
    auto bad = [](const uint4& x) {
      auto two = [](uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; };
      return two(x.x) || two(x.y) || two(x.z) || two(x.w);
    };
    bool bad_q = false;
#pragma unroll
    for (int t = 0; t < NH; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) bad_q |= bad(q[t][j]);
    bad_q = __any_sync(kFull, bad_q);
#pragma unroll 1
    for (int i = 0; i < mine * 16; i += 8) {   // pages g and g + 8 of every pass
      const uint4* page = bounds + __shfl_sync(kFull, table, i + g) * page_pieces;
      bool bad_p = bad_q;
#pragma unroll 1
      for (int j = 0; j < 8; ++j) bad_p |= bad(page[4 * j]);
      bad_p = __ballot_sync(kFull, bad_p) >> (lane & 28) & 0xfu;
      const int p = begin + (i >> 4) * kScoreTile + (i & 15) + g;
      if (c == 0 && bad_p && p < end) ws[p] = make_float2(INFINITY, 0.f);
    }
  }
  pdl_trigger();
}

// ===========================================================================
// Selection: one CTA per (row, KV head).
//
// With s_k the k-th largest fp32 score of the pages between the first and the
// last ones, at least k pages have an exact score >= lower = min over s >= s_k
// of (s - e), so a page with s + e < lower is out; at most k - 1 pages have
// s > s_k, and of these one with s - e > upper = max over s <= s_k of (s + e) beats
// all others, so it is in.  The pages in between are open and compared exactly
// where they are more than the places left.
//
// The scores stay in registers, a warp holding consecutive pages.  s_k comes from
// a histogram of 1024 equal intervals between the smallest and the largest score
// and a ranking of the pages of the interval it falls into.  Where an interval
// holds too many pages, too many are open or the row is too long for registers,
// a slower general routine takes over.
// ===========================================================================
constexpr int kSelList = 512;                // pages that are ranked in shared memory
constexpr int kSelBins = 1024;

__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long order_key64(double f) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(f);
  return u >> 63 ? ~u : u | (1ull << 63);
}

struct SelectSmem {
  int hist[kSelBins];
  float list_s[kSelList], list_e[kSelList];
  int list_idx[kSelList];
  unsigned long long list_key[kSelList];
  uint32_t red[2][32];
  int count_in[32], count_open[32];
  int cnt[4], totals[4];
  float sk;
};

// One (row, KV head) of a selection.
struct SelectUnit {
  float2* ws;
  int32_t* sel;
  const __nv_bfloat16* q;        // the group's query heads
  const int32_t* bt;
  int kvh, G, n, first, mid1, k;   // pages, first competing, last competing + 1, places for them
};

// Exact score of one page for heads [h0, h1) by one warp: four dimensions per lane, fp64.
__device__ __forceinline__ double exact_score(const SelectArgs& a, const SelectUnit& u, int page, int lane, int h0,
                                              int h1) {
  const __nv_bfloat16* b = a.bounds + ((int64_t)table_page(u.bt, page, a.num_pages) * a.Hkv + u.kvh) * 2 * D + lane * 4;
  const uint2 lo2 = *reinterpret_cast<const uint2*>(b), hi2 = *reinterpret_cast<const uint2*>(b + D);
  const __nv_bfloat16* lo = reinterpret_cast<const __nv_bfloat16*>(&lo2);
  const __nv_bfloat16* hi = reinterpret_cast<const __nv_bfloat16*>(&hi2);
  double best = -INFINITY;
  for (int h = h0; h < h1; ++h) {
    const uint2 q2 = *reinterpret_cast<const uint2*>(u.q + h * D + lane * 4);
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(&q2);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double x = (double)__bfloat162float(q[i]);
      sum += fmax(x * (double)__bfloat162float(lo[i]), x * (double)__bfloat162float(hi[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    best = fmax(best, sum);
  }
  return best + 0.0;   // -0 becomes +0: equal scores have equal keys
}

__device__ __forceinline__ void block_minmax(SelectSmem& sm, uint32_t lo, uint32_t hi, uint32_t& out_lo, uint32_t& out_hi) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
  lo = __reduce_min_sync(kFull, lo);
  hi = __reduce_max_sync(kFull, hi);
  __syncthreads();
  if (lane == 0) sm.red[0][warp] = lo, sm.red[1][warp] = hi;
  __syncthreads();
  out_lo = __reduce_min_sync(kFull, sm.red[0][lane % warps]);
  out_hi = __reduce_max_sync(kFull, sm.red[1][lane % warps]);
}

// The general routine: bisections over the scores' bit patterns, the scores read
// again for every pass, the pages' state in bit masks.
__device__ __noinline__ void select_general(const SelectArgs& a, const SelectUnit& u, SelectSmem& sm, uint32_t* masks) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, NT = blockDim.x, warps = NT / 32;
  const int words = (u.n + 31) / 32;
  uint32_t* in_mask = masks;
  uint32_t* open_mask = masks + words;
  float sk = INFINITY, lower = INFINITY, upper = -INFINITY;
  __syncthreads();
  if (tid < 4) sm.cnt[tid] = 0, sm.totals[tid] = 0;
  __syncthreads();                      // no place to give out (k = 0): nothing below waits before the counts
  if (u.k > 0) {
    uint32_t kmin = 0xffffffffu, kmax = 0u, lo, hi;
    for (int p = u.first + tid; p < u.mid1; p += NT) {
      const uint32_t key = order_key(u.ws[p].x);
      kmin = min(kmin, key), kmax = max(kmax, key);
    }
    block_minmax(sm, kmin, kmax, lo, hi);
    ++hi;                               // count(>= lo) >= k, count(>= hi) < k
    for (int it = 0; hi - lo > 1; ++it) {
      const uint32_t mid = lo + (hi - lo) / 2;
      int mine = 0;
      for (int p = u.first + tid; p < u.mid1; p += NT) mine += order_key(u.ws[p].x) >= mid;
      mine = __reduce_add_sync(kFull, mine);
      if (lane == 0 && mine) atomicAdd(&sm.cnt[it % 3], mine);
      if (tid == 0) sm.cnt[(it + 1) % 3] = 0;   // last read before the previous barrier
      __syncthreads();
      if (sm.cnt[it % 3] >= u.k) lo = mid; else hi = mid;
    }
    sk = key_value(lo);
    uint32_t low_key = 0xffffffffu, up_key = 0u;
    for (int p = u.first + tid; p < u.mid1; p += NT) {
      const float2 v = u.ws[p];
      if (v.x >= sk) low_key = min(low_key, order_key(v.x - v.y));
      if (v.x <= sk) up_key = max(up_key, order_key(v.x + v.y));
    }
    block_minmax(sm, low_key, up_key, lo, hi);
    lower = key_value(lo);
    upper = key_value(hi);
  }
  for (int w = warp; w < words; w += warps) {
    const int p = w * 32 + lane;
    bool in = p < u.n && (p < u.first || p >= u.mid1), open = false;
    if (p >= u.first && p < u.mid1 && u.k > 0) {
      const float2 v = u.ws[p];
      if (v.x > sk) in = v.x - v.y > upper, open = !in;
      else open = v.x + v.y >= lower;
    }
    const uint32_t bi = __ballot_sync(kFull, in), bo = __ballot_sync(kFull, open);
    if (lane == 0) {
      in_mask[w] = bi;
      open_mask[w] = bo;
      if (bi) atomicAdd(&sm.totals[0], __popc(bi));
      if (bo) atomicAdd(&sm.totals[1], __popc(bo));
    }
  }
  __syncthreads();
  const int n_open = sm.totals[1];
  const int need = a.budget - sm.totals[0];   // 0 <= need <= n_open
  if (need == n_open) {
    for (int w = tid; w < words; w += NT) in_mask[w] |= open_mask[w];
  } else {
    // exact scores over the fp32 ones, which are no longer needed; bisection over
    // their 64-bit keys, then ties by index
    double* exact = reinterpret_cast<double*>(u.ws);
    for (int w = warp; w < words; w += warps) {
      uint32_t m = open_mask[w];
      while (m) {
        const int p = w * 32 + __ffs(m) - 1;
        m &= m - 1;
        const bool finite = isfinite(u.ws[p].x);
        __syncwarp();
        const double v = finite ? exact_score(a, u, p, lane, 0, u.G) : INFINITY;
        if (lane == 0) exact[p] = v;
      }
    }
    __syncthreads();
    unsigned long long lo = 0, hi = ~0ull;      // count(>= lo) >= need; no finite or infinite key is ~0
    for (int it = 0; hi - lo > 1; ++it) {
      const unsigned long long mid = lo + (hi - lo) / 2;
      if (tid == 0) sm.cnt[0] = 0;
      __syncthreads();
      int mine = 0;
      for (int p = tid; p < u.n; p += NT)
        mine += (open_mask[p >> 5] >> (p & 31) & 1u) && order_key64(exact[p]) >= mid;
      mine = __reduce_add_sync(kFull, mine);
      if (lane == 0 && mine) atomicAdd(&sm.cnt[0], mine);
      __syncthreads();
      if (sm.cnt[0] >= need) lo = mid; else hi = mid;
      __syncthreads();
    }
    if (tid == 0) sm.cnt[0] = 0;
    __syncthreads();
    for (int w = warp; w < words; w += warps) {
      const int p = w * 32 + lane;
      const bool open = open_mask[w] >> lane & 1u;
      const unsigned long long key = open ? order_key64(exact[p]) : 0ull;
      const uint32_t above = __ballot_sync(kFull, open && key > lo), equal = __ballot_sync(kFull, open && key == lo);
      if (lane == 0) {
        in_mask[w] |= above;
        open_mask[w] = equal;
        if (above) atomicAdd(&sm.cnt[0], __popc(above));
      }
      __syncwarp();
    }
    __syncthreads();
    if (tid == 0) {
      int left = need - sm.cnt[0];
      for (int w = 0; w < words && left > 0; ++w) {
        uint32_t m = open_mask[w];
        while (m && left > 0) {
          in_mask[w] |= m & -m;
          m &= m - 1;
          --left;
        }
      }
    }
  }
  __syncthreads();
  // one warp writes the chosen pages in ascending order
  if (warp == 0) {
    int at = 0;
    for (int w0 = 0; w0 < words; w0 += 32) {
      uint32_t m = w0 + lane < words ? in_mask[w0 + lane] : 0u;
      const int c = __popc(m);
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += v;
      }
      int i = at + incl - c;
      while (m) {
        if (i < a.budget) u.sel[i] = (w0 + lane) * 32 + __ffs(m) - 1;
        ++i;
        m &= m - 1;
      }
      at += __shfl_sync(kFull, incl, 31);
    }
  }
}

// ITEMS: pages per thread (NT * ITEMS >= the block table's width), 0 for rows that
// only the general routine takes.
template <int NT, int ITEMS>
__global__ void __launch_bounds__(NT) page_select_kernel(const SelectArgs a) {
  constexpr int kW = NT / 32, I = ITEMS > 0 ? ITEMS : 1;
  extern __shared__ uint32_t masks[];        // of the general routine: in | open
  __shared__ SelectSmem sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kvh = blockIdx.x, r = blockIdx.y;
  for (int i = tid; i < kSelBins; i += NT) sm.hist[i] = 0;
  if (tid < 4) sm.totals[tid] = 0;
  pdl_wait();
  const int tok = a.tok_index[r];
  const int L = row_length(a.seq_lens, r, a.width);
  const int n = (L + PAGE - 1) / PAGE;
  SelectUnit u;
  u.sel = a.sel + ((int64_t)r * a.Hkv + kvh) * a.budget;
  if (n <= a.budget || tok < 0 || tok >= a.tokens) {
    // everything fits; a row of a bad token (recorded by the score kernel) takes nothing
    const int keep = n <= a.budget ? n : 0;
    for (int i = tid; i < a.budget; i += NT) u.sel[i] = i < keep ? i : -1;
    return;
  }
  u.ws = a.ws + ((int64_t)r * a.Hkv + kvh) * a.width;
  u.G = a.Hq / a.Hkv;
  u.q = a.q + (int64_t)tok * a.q_ld + (int64_t)kvh * u.G * D;
  u.bt = a.block_table + (int64_t)r * a.bt_stride;
  u.kvh = kvh;
  u.n = n;
  u.first = a.first, u.mid1 = n - a.last;                 // pages that compete
  u.k = a.budget - a.first - a.last;                      // for k places; k < mid1 - first
  if (ITEMS == 0) {
    select_general(a, u, sm, masks);
    return;
  }

  // warp w holds pages [w 32 I, (w + 1) 32 I), lane l page 32 i + l of them
  const int page0 = warp * 32 * I + lane;
  float2 v[I];
  uint32_t on = 0;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int p = page0 + i * 32;
    v[i] = make_float2(0.f, 0.f);
    if (p >= u.first && p < u.mid1) on |= 1u << i, v[i] = u.ws[p];
  }
  float sk = INFINITY, lower = INFINITY, upper = -INFINITY;
  if (u.k > 0) {
    uint32_t kmin = 0xffffffffu, kmax = 0u, lo, hi;
#pragma unroll
    for (int i = 0; i < I; ++i)
      if (on >> i & 1u && v[i].x < INFINITY) {
        const uint32_t key = order_key(v[i].x);
        kmin = min(kmin, key), kmax = max(kmax, key);
      }
    block_minmax(sm, kmin, kmax, lo, hi);   // (its barriers publish the zeroed counters)
    // intervals of the finite scores, +infinity in the last one; monotone in the score
    const float vmin = hi >= lo ? key_value(lo) : 0.f;
    const float width = hi >= lo ? key_value(hi) - vmin : 0.f;
    const float scale = width > 0.f && width < INFINITY ? (kSelBins - 1) / width : 0.f;
    auto bin_of = [&](float s) { return s < INFINITY ? min(kSelBins - 2, (int)((s - vmin) * scale)) : kSelBins - 1; };
#pragma unroll
    for (int i = 0; i < I; ++i)
      if (on >> i & 1u) atomicAdd(&sm.hist[bin_of(v[i].x)], 1);
    __syncthreads();
    // the first warp finds the interval of the k-th largest: 32 intervals per lane, from the top
    if (warp == 0) {
      int sum = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) sum += sm.hist[kSelBins - 1 - lane * 32 - (i + lane) % 32];
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += x;
      }
      const int src = __ffs(__ballot_sync(kFull, incl >= u.k)) - 1;
      int above = __shfl_sync(kFull, incl - sum, src);
      const int mine = sm.hist[kSelBins - 1 - src * 32 - lane];
      int in2 = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(kFull, in2, o);
        if (lane >= o) in2 += x;
      }
      const int at = __ffs(__ballot_sync(kFull, above + in2 >= u.k)) - 1;
      above += __shfl_sync(kFull, in2 - mine, at);
      const int members = __shfl_sync(kFull, mine, at);
      if (lane == 0) sm.cnt[0] = kSelBins - 1 - src * 32 - at, sm.cnt[1] = u.k - above, sm.cnt[2] = members;
    }
    __syncthreads();
    const int bin = sm.cnt[0], place = sm.cnt[1], members = sm.cnt[2];
    if (members > kSelList) {
      select_general(a, u, sm, masks);
      return;
    }
    // the interval's pages into a list; the others lie on one side of s_k
    uint32_t low_key = 0xffffffffu, up_key = 0u;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      if (!(on >> i & 1u)) continue;
      const int b = bin_of(v[i].x);
      if (b == bin) {
        const int at = atomicAdd(&sm.totals[0], 1);
        sm.list_s[at] = v[i].x;
        sm.list_e[at] = v[i].y;
      } else if (b > bin) {
        low_key = min(low_key, order_key(v[i].x - v[i].y));
      } else {
        up_key = max(up_key, order_key(v[i].x + v[i].y));
      }
    }
    low_key = __reduce_min_sync(kFull, low_key);
    up_key = __reduce_max_sync(kFull, up_key);
    if (lane == 0) sm.red[0][warp] = low_key, sm.red[1][warp] = up_key;
    __syncthreads();
    for (int i = tid; i < members; i += NT) {
      const float x = sm.list_s[i];
      int rank = 0;
      for (int j = 0; j < members; ++j) rank += sm.list_s[j] > x || (sm.list_s[j] == x && j < i);
      if (rank == place - 1) sm.sk = x;
    }
    __syncthreads();
    sk = sm.sk;
    low_key = sm.red[0][lane % kW], up_key = sm.red[1][lane % kW];
    for (int i = lane; i < members; i += 32) {
      const float x = sm.list_s[i], e = sm.list_e[i];
      if (x >= sk) low_key = min(low_key, order_key(x - e));
      if (x <= sk) up_key = max(up_key, order_key(x + e));
    }
    lower = key_value(__reduce_min_sync(kFull, low_key));
    upper = key_value(__reduce_max_sync(kFull, up_key));
  }
  pdl_trigger();
  uint32_t in = 0, open = 0;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int p = page0 + i * 32;
    if (!(on >> i & 1u)) {
      if (p < n) in |= 1u << i;             // the first and the last pages
    } else if (u.k > 0) {
      if (v[i].x > sk && v[i].x - v[i].y > upper) in |= 1u << i;
      else if (v[i].x > sk || v[i].x + v[i].y >= lower) open |= 1u << i;
    }
  }
  {
    const int ci = __reduce_add_sync(kFull, __popc(in)), co = __reduce_add_sync(kFull, __popc(open));
    if (lane == 0) sm.count_in[warp] = ci, sm.count_open[warp] = co;
  }
  __syncthreads();
  // totals over the warps, and what lies in the warps before this one
  const int ci = lane < kW ? sm.count_in[lane] : 0, co = lane < kW ? sm.count_open[lane] : 0;
  const int n_in = __reduce_add_sync(kFull, ci), n_open = __reduce_add_sync(kFull, co);
  const int need = a.budget - n_in;          // 0 <= need <= n_open
  int at;
  if (need == n_open) {
    in |= open;
    at = __reduce_add_sync(kFull, lane < warp ? ci + co : 0);
  } else if (n_open > kSelList) {
    select_general(a, u, sm, masks);
    return;
  } else {
    int place[I];
#pragma unroll
    for (int i = 0; i < I; ++i) {
      place[i] = 0;
      if (open >> i & 1u) {
        place[i] = atomicAdd(&sm.totals[1], 1);
        sm.list_idx[place[i]] = page0 + i * 32;
        sm.list_key[place[i]] = isfinite(v[i].x) ? 0ull : order_key64(INFINITY);
      }
    }
    __syncthreads();
    // a warp per page and head; the page's score is the heads' largest
    for (int i = warp; i < n_open * u.G; i += kW) {
      const int o = i / u.G, h = i % u.G;
      if (sm.list_key[o] == order_key64(INFINITY)) continue;   // stays so: no finite score reaches it
      const double x = exact_score(a, u, sm.list_idx[o], lane, h, h + 1);
      if (lane == 0) atomicMax(&sm.list_key[o], order_key64(x));
    }
    __syncthreads();
    for (int i = tid; i < n_open; i += NT) {
      const unsigned long long x = sm.list_key[i];
      const int p = sm.list_idx[i];
      int rank = 0;
      for (int j = 0; j < n_open; ++j) rank += sm.list_key[j] > x || (sm.list_key[j] == x && sm.list_idx[j] < p);
      sm.list_e[i] = rank < need ? 1.f : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < I; ++i)
      if (open >> i & 1u && sm.list_e[place[i]] != 0.f) in |= 1u << i;
    const int c = __reduce_add_sync(kFull, __popc(in));
    if (lane == 0) sm.count_in[warp] = c;
    __syncthreads();
    at = __reduce_add_sync(kFull, lane < warp ? sm.count_in[lane] : 0);
  }
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const uint32_t m = __ballot_sync(kFull, in >> i & 1u);
    if (in >> i & 1u) u.sel[at + __popc(m & ((1u << lane) - 1))] = page0 + i * 32;
    at += __popc(m);
  }
}

// ===========================================================================
// decode_sparse: a cluster of CTAs per (row, KV head), every warp a share of the
// chosen pages with its own running maximum and sum; the warps join in shared
// memory, the CTAs by writing into the shared memory of the CTA that owns an
// output, so there is one launch and no workspace.
//
// S^T = K Q^T has the page's 16 tokens as rows and the query heads as columns;
// O^T = V^T P^T has dimensions as rows.  K is read by the lanes in the layout of
// the A operand directly (16 bytes = eight dimensions = two k-steps).  V^T needs
// two tokens side by side: a lane reads the same eight dimensions of two tokens
// and interleaves them with byte permutes; row g of tile t is dimension 8g + t.
// P^T comes from S^T by an 8 x 8 register transpose.  The tensor cores take P as
// two bf16 parts, the upper bits and the rest, which hold each weight to 2^-15; with one
// part (2^-8) the output would be off by up to 2^-8 of sum p |v|, however small the
// mean itself is.  The rest gets 2^-20 of the upper part besides, so that both parts
// have the weight's sign and neither is zero alone: an infinite value stays one.
//
// 16 warps per SM have a page each under way; 64 rows x 8 heads x 128 pages read
// 537 MB in 90 us, 6.0 TB/s (85 with one CTA per row and head).  A page ahead in registers halves the warps, and per-lane
// cp.async delivers less than plain loads: both were slower.
// ===========================================================================
constexpr int kMaxCluster = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t x;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(x));
  return x;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
  return addr;
}
__device__ __forceinline__ void st_cluster4(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ void st_cluster2(uint32_t addr, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}

constexpr int kOLd = D + 4;
template <int NH, int W>
struct SparseSmem {
  float o[W][NH * 8][kOLd];
  float2 ml[W][NH * 8];             // running maximum and sum
  // from every CTA of the cluster, for the outputs this CTA owns: quads of
  // dimensions q with q % cl == this CTA
  float4 in_o[kMaxCluster][NH * 8 * (D / 4) / 2];
  float2 in_ml[kMaxCluster][NH * 8];
};

template <int NH, int W>   // W warps
__global__ void __launch_bounds__(W * 32, (NH == 1 ? 16 : 8) / W) decode_sparse_kernel(const SparseArgs a, int cl) {
  extern __shared__ __align__(128) uint8_t raw[];
  SparseSmem<NH, W>& sm = *reinterpret_cast<SparseSmem<NH, W>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int part = cl > 1 ? (int)cluster_rank() : 0;
  const int unit = blockIdx.x / cl;
  const int kvh = unit % a.Hkv, r = unit / a.Hkv;
  const int G = a.Hq / a.Hkv;
  // this warp's pages: entries w, w + stride, ... of the list; lane j holds the
  // j-th of a window of 32 (first token, physical page), the next window under way
  const int stride = cl * W, w = part * W + warp;
  const int32_t* bt = a.block_table + (int64_t)r * a.bt_stride;
  const int32_t* sel = a.sel + ((int64_t)r * a.Hkv + kvh) * a.budget;
  if (cl > 1) cluster_arrive();         // every CTA of the cluster runs before another one writes to it
  pdl_wait();
  int next_page = w + lane * stride < a.budget ? sel[w + lane * stride] : -1;   // in the same round trip as the length
  const int tok = a.tok_index[r];
  const int L = row_length(a.seq_lens, r, a.width);
  const int n = (L + PAGE - 1) / PAGE;
  const bool tok_ok = tok >= 0 && tok < a.tokens;
  if (!tok_ok && tid == 0) set_error(kErrBadIndex, (unsigned long long)r);
  const int count = tok_ok ? min(n, a.budget) : 0;
  const int mine = count > w ? (count - w + stride - 1) / stride : 0;
  int win_tok = 0, win_phys = 0;
  auto open_window = [&](int i) {
    win_tok = L;                        // nothing valid in the page
    win_phys = 0;
    if (i + lane < mine) {
      if (next_page < 0 || next_page >= n) {
        set_error(kErrBadIndex, (unsigned long long)r);
      } else {
        win_tok = next_page * PAGE;
        win_phys = table_page(bt, next_page, a.num_pages);
      }
    }
    const int j = i + 32 + lane;
    next_page = j < mine ? sel[w + j * stride] : -1;
  };

  // a lane's pieces of a page: K rows g and g + 8, pieces c, c + 4, ...; V rows 2c,
  // 2c + 1, 2c + 8, 2c + 9, piece g of both halves of the dimensions
  const int kl = g * D + c * 8, vl = 2 * c * D + g * 8;
  const int64_t page_elems = (int64_t)a.Hkv * PAGE * D;
  uint4 k0[4], k1[4], v[2][4];          // v[half of the dimensions][token 2c, 2c + 1, 2c + 8, 2c + 9]
  int t0 = L, t0_next = L;
  int64_t at = 0;
  auto locate = [&](int i) {            // page i of this warp
    if ((i & 31) == 0) open_window(i);
    t0_next = __shfl_sync(kFull, win_tok, i & 31);
    at = __shfl_sync(kFull, win_phys, i & 31) * page_elems + kvh * (PAGE * D);
  };
  auto load_k = [&]() {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k0[j] = ld_stream(a.kcache + (at + kl) + j * 32);
      k1[j] = ld_stream(a.kcache + (at + kl) + 8 * D + j * 32);
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int t = (x & 1) + (x >> 1) * 8;
      const bool on = t0_next + 2 * c + t < L;      // zeros past the sequence's end
      v[0][x] = on ? ld_stream(a.vcache + (at + vl) + t * D) : make_uint4(0u, 0u, 0u, 0u);
      v[1][x] = on ? ld_stream(a.vcache + (at + vl) + t * D + 64) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  uint4 q[NH][4];
#pragma unroll
  for (int t = 0; t < NH; ++t) {
    const __nv_bfloat16* qh = a.q + (int64_t)(tok_ok ? tok : 0) * a.q_ld + (int64_t)(kvh * G + t * 8 + g) * D;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      q[t][j] = tok_ok && t * 8 + g < G ? *reinterpret_cast<const uint4*>(qh + 8 * (c + 4 * j))
                                        : make_uint4(0u, 0u, 0u, 0u);
  }
  float o[NH][8][4], m[NH][2], l[NH][2];
#pragma unroll
  for (int t = 0; t < NH; ++t) {
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
  }

  for (int i = 0; i < mine; ++i) {
    locate(i);
    load_k();
    load_v();
    t0 = t0_next;
    float s[NH][2][4];
#pragma unroll
    for (int t = 0; t < NH; ++t) {
#pragma unroll
      for (int x = 0; x < 2; ++x) s[t][x][0] = s[t][x][1] = s[t][x][2] = s[t][x][3] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mma_bf16(s[t][0], k0[j].x, k1[j].x, k0[j].y, k1[j].y, q[t][j].x, q[t][j].y);
        mma_bf16(s[t][1], k0[j].z, k1[j].z, k0[j].w, k1[j].w, q[t][j].z, q[t][j].w);
      }
    }
    uint32_t p[NH][2][2];               // [part][tokens 0 to 7, 8 to 15]
#pragma unroll
    for (int t = 0; t < NH; ++t) {
      // x[0], x[1]: token g, heads 2c, 2c + 1; x[2], x[3]: token g + 8
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = t0 + g + (e >> 1) * 8 < L ? (s[t][0][e] + s[t][1][e]) * a.scale_log2 : -INFINITY;
      float pr[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(x[e], x[e + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
        mx = fmaxf(mx, m[t][e]);
        const float sh = mx == -INFINITY ? 0.f : mx;
        const float al = exp2f(m[t][e] - sh);
        m[t][e] = mx;
        pr[e] = exp2f(x[e] - sh);
        pr[e + 2] = exp2f(x[e + 2] - sh);
        l[t][e] *= al;
#pragma unroll
        for (int i8 = 0; i8 < 8; ++i8) o[t][i8][e] *= al, o[t][i8][e + 2] *= al;
      }
      l[t][0] += pr[0] + pr[2];
      l[t][1] += pr[1] + pr[3];
      float rest[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        rest[e] = fmaf(__uint_as_float(__float_as_uint(pr[e]) & 0xffff0000u), -(1.f - 0x1p-20f), pr[e]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[t][0][e] = movmatrix_trans(__byte_perm(__float_as_uint(pr[2 * e]), __float_as_uint(pr[2 * e + 1]), 0x7632));
        p[t][1][e] = movmatrix_trans(pack_bf16x2(rest[2 * e], rest[2 * e + 1]));
      }
    }
    const uint32_t* vw = reinterpret_cast<const uint32_t*>(v);   // [half][token][word]
#pragma unroll
    for (int i8 = 0; i8 < 8; ++i8) {
      const uint32_t sel2 = i8 & 1 ? 0x7632u : 0x5410u;
      const int wd = i8 >> 1;
      const uint32_t a0 = __byte_perm(vw[0 * 4 + wd], vw[1 * 4 + wd], sel2);
      const uint32_t a1 = __byte_perm(vw[16 + 0 * 4 + wd], vw[16 + 1 * 4 + wd], sel2);
      const uint32_t a2 = __byte_perm(vw[2 * 4 + wd], vw[3 * 4 + wd], sel2);
      const uint32_t a3 = __byte_perm(vw[16 + 2 * 4 + wd], vw[16 + 3 * 4 + wd], sel2);
#pragma unroll
      for (int t = 0; t < NH; ++t) {
        mma_bf16(o[t][i8], a0, a1, a2, a3, p[t][1][0], p[t][1][1]);
        mma_bf16(o[t][i8], a0, a1, a2, a3, p[t][0][0], p[t][0][1]);
      }
    }
  }

  pdl_trigger();
  // the warps' results: o[t][i][0..1] = dim 8g + i, heads 2c, 2c + 1; [2..3] = dim 64 + 8g + i
#pragma unroll
  for (int t = 0; t < NH; ++t) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float s = l[t][e];
      s += __shfl_xor_sync(kFull, s, 4);
      s += __shfl_xor_sync(kFull, s, 8);
      s += __shfl_xor_sync(kFull, s, 16);
      const int h = t * 8 + 2 * c + e;
      if (g == 0) sm.ml[warp][h] = make_float2(m[t][e], s);
      if (h < G) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            *reinterpret_cast<float4*>(&sm.o[warp][h][x * 64 + 8 * g + 4 * y]) =
                make_float4(o[t][4 * y][e + 2 * x], o[t][4 * y + 1][e + 2 * x], o[t][4 * y + 2][e + 2 * x],
                            o[t][4 * y + 3][e + 2 * x]);
      }
    }
  }
  __syncthreads();
  if (cl > 1) cluster_wait();
  __nv_bfloat16* out = a.out + (int64_t)(tok_ok ? tok : 0) * a.out_ld + (int64_t)kvh * G * D;
  auto write = [&](int quad, float4 acc, float sum) {
    // no weight at all: nothing to attend to, or logits of -inf alone, whose softmax is NaN
    const float f = sum > 0.f ? 1.f / sum : count > 0 ? __int_as_float(0x7fffffff) : 0.f;
    if (tok_ok)
      *reinterpret_cast<uint2*>(out + quad * 4) = make_uint2(pack_bf16x2(acc.x * f, acc.y * f), pack_bf16x2(acc.z * f, acc.w * f));
  };
  // quads of four dimensions, head by head: the CTA's warps, then the cluster's CTAs
  for (int quad = tid; quad < G * (D / 4); quad += (W * 32)) {
    const int h = quad / (D / 4), d = quad % (D / 4) * 4;
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < W; ++x) mx = fmaxf(mx, sm.ml[x][h].x);
    const float sh = mx == -INFINITY ? 0.f : mx;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float2 ml = sm.ml[x][h];
      const float f = exp2f(ml.x - sh);
      const float4 y = *reinterpret_cast<const float4*>(&sm.o[x][h][d]);
      acc.x += f * y.x, acc.y += f * y.y, acc.z += f * y.z, acc.w += f * y.w;
      sum += f * ml.y;
    }
    if (cl == 1) {
      write(quad, acc, sum);
    } else {
      st_cluster4(cluster_addr(&sm.in_o[part][quad / cl], quad % cl), acc);
      if (quad % (D / 4) < cl) st_cluster2(cluster_addr(&sm.in_ml[part][h], quad % cl), make_float2(mx, sum));
    }
  }
  if (cl == 1) return;
  cluster_arrive();
  cluster_wait();
  for (int quad = tid * cl + part; quad < G * (D / 4); quad += (W * 32) * cl) {
    const int h = quad / (D / 4);
    float mx = -INFINITY;
    for (int x = 0; x < cl; ++x) mx = fmaxf(mx, sm.in_ml[x][h].x);
    const float sh = mx == -INFINITY ? 0.f : mx;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int x = 0; x < cl; ++x) {
      const float2 ml = sm.in_ml[x][h];
      const float f = exp2f(ml.x - sh);
      const float4 y = sm.in_o[x][quad / cl];
      acc.x += f * y.x, acc.y += f * y.y, acc.z += f * y.z, acc.w += f * y.w;
      sum += f * ml.y;
    }
    write(quad, acc, sum);
  }
}

}  // namespace

void page_bounds(const BoundsArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.max_new <= 0) return;
  BoundsArgs b = a;
  b.max_pages = (a.max_new + PAGE - 2) / PAGE + 1;   // from any offset in a page
  if (b.max_pages > a.width) b.max_pages = a.width;
  const int64_t units = (int64_t)a.rows * a.Hkv * b.max_pages;
  if (units == 0) return;                            // a table without pages
  if (units / 4 >= INT32_MAX) throw std::runtime_error("lunaflux page_bounds: too many pages for one call");
  launch_k(page_bounds_kernel, dim3((unsigned)((units + 3) / 4)), dim3(128), 0, s, 1, b);
}

namespace {
template <int NT, int ITEMS>
void launch_select(const SelectArgs& a, cudaStream_t s) {
  const size_t smem = (size_t)((a.width + 31) / 32) * 2 * sizeof(uint32_t);   // the general routine's masks, at most 16 KB
  launch_k(page_select_kernel<NT, ITEMS>, dim3((unsigned)a.Hkv, (unsigned)a.rows), dim3(NT), smem, s, 1, a);
}
}  // namespace

int select_pages(const SelectArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return 0;
  if (a.width > a.budget) {
    // two passes of 64 pages per CTA where that fills the GPU (64 rows of 2048 pages: 196 us a
    // step, 201 with one; 64 ragged rows 79 and 86; 4 rows of 8192 pages 55.3 and 56.4)
    const int64_t tiles = (int64_t)a.rows * a.Hkv * ((a.width + kScoreTile - 1) / kScoreTile);
    const int passes = tiles > 4 * sm_count() ? kScorePasses : 1;
    const int chunk = passes * kScoreTile;
    const dim3 grid((unsigned)((a.width + chunk - 1) / chunk * a.Hkv), (unsigned)a.rows);
    auto k = a.Hq / a.Hkv <= 8 ? page_score_kernel<1> : page_score_kernel<2>;
    launch_k(k, grid, dim3(kThreads), 0, s, 1, a, passes);
  }
  // As few threads and pages per thread as hold the block table: 8191 tokens 14.0 us
  // a step, 16.0 with <256, 8>, 19.5 with <1024, 8>; 64 rows of 32768 tokens 196 us, 220
  // with <1024, 8>, 311 with the general routine.  Where every CTA has an SM for itself
  // 512 threads for 2048 pages (one row of 32768 tokens 17.5 us, 18.5 with 256; 17 ragged
  // rows 37, 38; 64 rows would take 200, and take 196).
  if (a.width <= 512) launch_select<256, 2>(a, s);
  else if (a.width <= 2048 && (int64_t)a.rows * a.Hkv <= sm_count()) launch_select<512, 4>(a, s);
  else if (a.width <= 2048) launch_select<256, 8>(a, s);
  else if (a.width <= 8192) launch_select<1024, 8>(a, s);
  else launch_select<1024, 0>(a, s);
  return a.width > a.budget ? 2 : 1;
}

namespace {
template <int NH, int W>
void launch_decode(const SparseArgs& a, cudaStream_t s) {
  const int64_t units = (int64_t)a.rows * a.Hkv;
  // CTAs per unit: as many as run at the same time (16 warps per SM, 8 for wide groups)
  // and get two pages per warp; two also where only half of them run at once, because
  // one CTA with a long row would outlast the others of a ragged batch (64 rows of 1 to 32768
  // tokens x 8 heads x 128 pages: a step takes 79 us, 98 with one; all of 32768: 196, 191).
  const int64_t slots = (int64_t)sm_count() * ((NH == 1 ? 16 : 8) / W);
  int cl = 1;
  while (cl < kMaxCluster && units * cl * 2 <= (cl == 1 ? 2 : 1) * slots && a.budget > W * cl) cl *= 2;
  auto k = decode_sparse_kernel<NH, W>;
  static std::atomic<unsigned long long> allowed{0};
  allow_smem(reinterpret_cast<const void*>(k), allowed);
  // Clusters that start while the previous kernel still holds some SMs crowd onto
  // the others; where they would fill the GPU they wait for its end (4 rows x 8
  // heads x 256 pages after a selection: 55 instead of 63 us for the whole step).
  launch_with(cl == 1 || units * cl * W <= sm_count() * 8, k, dim3((unsigned)(units * cl)), dim3(W * 32),
              sizeof(SparseSmem<NH, W>), s, (unsigned)cl, a, cl);
}
}  // namespace

void decode_sparse(const SparseArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  // Eight warps per CTA where clusters of eight CTAs still leave SMs without work (1
  // row x 8 heads x 64 pages: a step takes 14.0 us, 14.4 with four; 8 x 2 x 256 34.2, 38.5)
  // or, with four warps, half of the warps that fit, and each of the eight still gets two
  // pages (4 x 8 x 256 pages 55.3 us, 58.6; 4 x 8 x 128 48.8, 49.8; 4 x 8 x 64 46.2 and 46.0
  // the other way round).  Not good for groups of more than eight heads in between: 8 rows x
  // 4 heads x 256 pages take 73.8 us and would take 57.4 with eight.
  const int64_t ctas = (int64_t)a.rows * a.Hkv * kMaxCluster;
  const bool narrow = a.Hq / a.Hkv <= 8;   // wider groups fit eight warps per SM
  const bool few = ctas <= sm_count() || (narrow && ctas <= 2 * sm_count() && a.budget >= 2 * 8 * kMaxCluster);
  if (narrow) few ? launch_decode<1, 8>(a, s) : launch_decode<1, 4>(a, s);
  else few ? launch_decode<2, 8>(a, s) : launch_decode<2, 4>(a, s);
}

}  // namespace attn
}  // namespace lf
