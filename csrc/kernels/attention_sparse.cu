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
// score is a dot product of 256 terms: tensor-core work with 16 pages as the
// rows and the group's query heads as the columns.  What bounds the selection
// is reading the bounds, 512 bytes per (page, KV head); what bounds the
// attention is reading 8 KB per chosen (page, KV head).
//
// The order of the scores is that of the exact sums.  bf16 products are exact
// in fp32; their fp32 sums carry an error bound e = kScoreErr * sum|terms|, and
// where the bounds of two pages around the cut overlap, both are summed again
// in fp64.  A score that is not finite (a page or query that holds an infinity
// or a NaN) counts as +infinity, so such a page is taken and shows up in the
// output as it would without the selection.
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

// 16-byte copy into shared memory; zeros where `on` is false.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The streaming kernels (scores, attention) run four warps whose lanes copy
// their own operand pieces into their own slots of a ring in shared memory and
// read only those back: 16 pieces of 16 bytes per lane and stage, a pipeline
// without registers and without a barrier.
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = kThreads * 16;
constexpr int kStage = 16 * kUnit;           // 32 KB
constexpr int kStages = 3;                   // 96 KB: two CTAs per SM

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
// Page scores.  A warp takes 16 pages at a time as the 16 rows of m16n8k16;
// lane (g, c) = (lane / 4, lane % 4) loads 16-byte pieces c, c + 4, ... of the
// bounds of pages g and g + 8.  A piece is eight consecutive dimensions, which
// serve two k-steps: the order of k is free as long as the queries use the
// same one, so no shared memory is needed.  lo and hi lie behind one another,
// so pieces 0..15 meet min(q, 0) and pieces 16..31 meet max(q, 0).
//
// Error bound: a k16 step adds 16 exact products to the accumulator with at
// most 17 roundings or truncations at the largest addend, 2^-23 each; four
// chains of four steps over disjoint terms give 68 * 2^-23 = 2^-16.9 of the sum
// of magnitudes, and joining them 2^-22.4 more.  The magnitudes are summed by the
// same instruction on the operands without their signs.
// ===========================================================================
constexpr float kScoreErr = 1.f / 32768.f;   // 2^-15, four times what is derived above
constexpr int kScoreTile = 16 * kWarps;      // pages of one pass of a CTA
constexpr int kScorePasses = 8;              // most passes of a CTA

template <int NH>   // groups of eight query heads
__global__ void __launch_bounds__(kThreads, 2) page_score_kernel(const SelectArgs a, int passes) {
  extern __shared__ __align__(128) uint8_t raw[];
  __shared__ int phys[kScorePasses * kScoreTile];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.x % a.Hkv, chunk = blockIdx.x / a.Hkv;
  const int r = blockIdx.y;
  const int G = a.Hq / a.Hkv;
  const int begin = chunk * passes * kScoreTile;
  const int32_t* bt = a.block_table + (int64_t)r * a.bt_stride;
  const int span = min(passes * kScoreTile, a.width - begin);
  int table[kScorePasses * kScoreTile / kThreads];   // fetched before the length is known
#pragma unroll
  for (int i = 0; i < kScorePasses * kScoreTile / kThreads; ++i) {
    const int p = i * kThreads + tid;
    table[i] = p < span ? bt[begin + p] : 0;
  }
  const int L = row_length(a.seq_lens, r, a.width);
  const int n = (L + PAGE - 1) / PAGE;
  const int end = min(n, begin + passes * kScoreTile);
  if (n <= a.budget || begin >= end) return;
  const int tok = a.tok_index[r];
  if (tok < 0 || tok >= a.tokens) {
    if (tid == 0) set_error(kErrBadIndex, (unsigned long long)r);
    return;
  }
#pragma unroll
  for (int i = 0; i < kScorePasses * kScoreTile / kThreads; ++i) {
    const int p = i * kThreads + tid;
    if (begin + p < end) {
      if (table[i] < 0 || table[i] >= a.num_pages) {   // recorded; the reserved zero page stands in
        set_error(kErrBadIndex, (unsigned long long)(begin + p));
        table[i] = 0;
      }
      phys[p] = table[i];
    }
  }
  __syncthreads();

  const uint32_t ring = smem_u32(raw) + tid * 16;
  const uint4* bounds = reinterpret_cast<const uint4*>(a.bounds);
  const int pieces = 2 * D / 8;              // of one (page, KV head)
  auto issue = [&](int it, uint32_t slot) {
    const int p0 = begin + (it * kWarps + warp) * 16;
    if (it < passes && p0 < end) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int p = p0 + g + 8 * u;
        const bool on = p < end;
        const uint4* src = bounds + ((int64_t)phys[on ? p - begin : 0] * a.Hkv + kvh) * pieces + c;
#pragma unroll
        for (int j = 0; j < 8; ++j) cp_async16(slot + (u * 8 + j) * kUnit, src + 4 * j, on);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) issue(i, ring + i * kStage);

  uint4 q[NH][4];
#pragma unroll
  for (int t = 0; t < NH; ++t) {
    const __nv_bfloat16* qh = a.q + (int64_t)tok * a.q_ld + (int64_t)(kvh * G + t * 8 + g) * D;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      q[t][j] = t * 8 + g < G ? *reinterpret_cast<const uint4*>(qh + 8 * (c + 4 * j)) : make_uint4(0u, 0u, 0u, 0u);
  }
  float2* ws = a.ws + ((int64_t)r * a.Hkv + kvh) * a.width;
  uint32_t slot = ring;
  for (int it = 0; it < passes; ++it) {
    const int p0 = begin + (it * kWarps + warp) * 16;
    if (p0 >= end) break;                    // this warp's later passes lie past the end as well
    cp_async_wait<kStages - 1>();
    float s[NH][4][4], m[NH][4];
#pragma unroll
    for (int t = 0; t < NH; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i][0] = s[t][i][1] = s[t][i][2] = s[t][i][3] = m[t][i] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint4 va = lds16(slot + j * kUnit), vb = lds16(slot + (8 + j) * kUnit);
      const uint32_t* pa4 = reinterpret_cast<const uint32_t*>(&va);
      const uint32_t* pb4 = reinterpret_cast<const uint32_t*>(&vb);
#pragma unroll
      for (int t = 0; t < NH; ++t) {
        const uint32_t* q4 = reinterpret_cast<const uint32_t*>(&q[t][j & 3]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t b0 = j < 4 ? min_nan(q4[2 * h], 0u) : max_nan(q4[2 * h], 0u);
          const uint32_t b1 = j < 4 ? min_nan(q4[2 * h + 1], 0u) : max_nan(q4[2 * h + 1], 0u);
          mma_bf16(s[t][j & 3], pa4[2 * h], pb4[2 * h], pa4[2 * h + 1], pb4[2 * h + 1], b0, b1);
          constexpr uint32_t kAbs = 0x7fff7fffu;
          mma_bf16(m[t], pa4[2 * h] & kAbs, pb4[2 * h] & kAbs, pa4[2 * h + 1] & kAbs, pb4[2 * h + 1] & kAbs,
                   b0 & kAbs, b1 & kAbs);
        }
      }
    }
    issue(it + kStages, slot);
    slot = slot == ring + (kStages - 1) * kStage ? ring : slot + kStage;
    float best_a = -INFINITY, best_b = -INFINITY, err_a = 0.f, err_b = 0.f;
#pragma unroll
    for (int t = 0; t < NH; ++t) {
      // columns 2c, 2c + 1 of pages g and g + 8
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = (s[t][0][i] + s[t][1][i]) + (s[t][2][i] + s[t][3][i]);
        if (t * 8 + 2 * c + (i & 1) < G) {
          const bool fin = isfinite(v) && isfinite(m[t][i]);
          float& b = i < 2 ? best_a : best_b;
          float& e = i < 2 ? err_a : err_b;
          b = fmaxf(b, fin ? v : INFINITY);
          e = fmaxf(e, fin ? m[t][i] * kScoreErr : 0.f);
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
    if (c == 0) {
      if (p0 + g < end) ws[p0 + g] = make_float2(best_a, isinf(best_a) ? 0.f : err_a);
      if (p0 + g + 8 < end) ws[p0 + g + 8] = make_float2(best_b, isinf(best_b) ? 0.f : err_b);
    }
  }
  cp_async_wait<0>();
}

// ===========================================================================
// Selection: one CTA per (row, KV head).
//
// With s_k the k-th largest fp32 score of the pages between the first and the
// last ones, at least k pages have an exact score >= lower = min over s >= s_k
// of (s - e), so a page with s + e < lower is out; at most k - 1 pages have
// s > s_k, and of these one with s - e > upper = max over s <= s_k of (s + e) beats
// all others, so it is in.  The pages in between are compared exactly.
// ===========================================================================
//
// s_k comes from a histogram of 1024 equal intervals between the smallest and the
// largest score and a ranking of the pages of the interval it falls into; where
// one interval holds too many, from a bisection over the scores' bit patterns.
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

// Exact score of one page by one warp: four dimensions per lane, fp64.
__device__ __forceinline__ double exact_score(const SelectArgs& a, const __nv_bfloat16* q, const __nv_bfloat16* b,
                                              int G, int lane) {
  float lo[4], hi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo[i] = __bfloat162float(b[lane * 4 + i]);
    hi[i] = __bfloat162float(b[D + lane * 4 + i]);
  }
  double best = -INFINITY;
  for (int h = 0; h < G; ++h) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double x = (double)__bfloat162float(q[h * D + lane * 4 + i]);
      sum += fmax(x * (double)lo[i], x * (double)hi[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    best = fmax(best, sum);
  }
  return best + 0.0;   // -0 becomes +0: equal scores have equal keys
}

// ITEMS > 0: the row's scores stay in registers (up to ITEMS * NT pages);
// ITEMS = 0: they are read again for every pass.
template <int NT, int ITEMS>
__global__ void __launch_bounds__(NT) page_select_kernel(const SelectArgs a) {
  constexpr int kSelThreads = NT, kSelWarps = NT / 32;
  pdl_trigger();
  pdl_wait();
  extern __shared__ uint32_t masks[];        // in | open | prefix, `words` each
  __shared__ int cnt[3];
  __shared__ uint32_t red[2][kSelWarps];
  __shared__ int totals[4];
  __shared__ int hist[kSelBins];
  __shared__ float found_sk;
  __shared__ int list_idx[kSelList];
  __shared__ double list_val[kSelList];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kvh = blockIdx.x, r = blockIdx.y;
  const int L = row_length(a.seq_lens, r, a.width);
  const int n = (L + PAGE - 1) / PAGE;
  int32_t* sel = a.sel + ((int64_t)r * a.Hkv + kvh) * a.budget;
  const int tok = a.tok_index[r];
  if (n <= a.budget || tok < 0 || tok >= a.tokens) {
    // everything fits; a row of a bad token (recorded by the score kernel) takes nothing
    const int keep = n <= a.budget ? n : 0;
    for (int i = tid; i < a.budget; i += kSelThreads) sel[i] = i < keep ? i : -1;
    return;
  }
  float2* ws = a.ws + ((int64_t)r * a.Hkv + kvh) * a.width;
  const int mid0 = a.first, mid1 = n - a.last;            // pages that compete
  const int k = a.budget - a.first - a.last;              // for k places; k < mid1 - mid0
  const int words = (n + 31) / 32;
  uint32_t* in_mask = masks;
  uint32_t* open_mask = masks + words;
  uint32_t* prefix = masks + 2 * words;
  const int trips = (n + kSelThreads - 1) / kSelThreads;

  float2 sc[ITEMS > 0 ? ITEMS : 1];
  if (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int p = i * kSelThreads + tid;
      sc[i] = p >= mid0 && p < mid1 ? ws[p] : make_float2(-INFINITY, 0.f);
    }
  }
  // f(page, is it a competing page, its score, its error bound) for every page of the thread
  auto each = [&](auto&& f) {
    if (ITEMS > 0) {
#pragma unroll
      for (int i = 0; i < (ITEMS > 0 ? ITEMS : 1); ++i) {
        if (i >= trips) break;
        const int p = i * kSelThreads + tid;
        f(p, p >= mid0 && p < mid1, sc[i].x, sc[i].y);
      }
    } else {
      for (int i = 0; i < trips; ++i) {
        const int p = i * kSelThreads + tid;
        const bool on = p >= mid0 && p < mid1;
        const float2 v = on ? ws[p] : make_float2(-INFINITY, 0.f);
        f(p, on, v.x, v.y);
      }
    }
  };
  auto block_minmax = [&](uint32_t lo, uint32_t hi, uint32_t& out_lo, uint32_t& out_hi) {
    lo = __reduce_min_sync(kFull, lo);
    hi = __reduce_max_sync(kFull, hi);
    __syncthreads();
    if (lane == 0) red[0][warp] = lo, red[1][warp] = hi;
    __syncthreads();
    out_lo = __reduce_min_sync(kFull, red[0][lane % kSelWarps]);
    out_hi = __reduce_max_sync(kFull, red[1][lane % kSelWarps]);
  };

  if (tid < 3) cnt[tid] = 0;
  if (tid < 4) totals[tid] = 0;
  for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
  float lower = INFINITY, upper = -INFINITY, sk = INFINITY;
  if (k > 0) {
    uint32_t kmin = 0xffffffffu, kmax = 0u, fmaxk = 0u;
    each([&](int, bool on, float s, float) {
      if (!on) return;
      const uint32_t key = order_key(s);
      kmin = min(kmin, key), kmax = max(kmax, key);
      if (s < INFINITY) fmaxk = max(fmaxk, key);
    });
    uint32_t lo, hi;
    block_minmax(kmin, fmaxk, lo, hi);  // (its barriers publish the zeroed counters)
    // intervals of the finite scores, +infinity in the last one; monotone in the score
    const float vmin = key_value(lo), vmax = hi >= lo ? key_value(hi) : vmin;
    const float width = vmax - vmin;
    const float scale = width > 0.f && width < INFINITY ? (kSelBins - 1) / width : 0.f;
    auto bin_of = [&](float s) { return s < INFINITY ? min(kSelBins - 2, (int)((s - vmin) * scale)) : kSelBins - 1; };
    each([&](int, bool on, float s, float) {
      if (on) atomicAdd(&hist[bin_of(s)], 1);
    });
    __syncthreads();
    // the first warp finds the interval of the k-th largest: 32 bins per lane, from the top
    if (warp == 0) {
      int sum = 0;
      for (int i = 0; i < 32; ++i) sum += hist[kSelBins - 1 - lane * 32 - (i + lane) % 32];
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += v;
      }
      const uint32_t reach = __ballot_sync(kFull, incl >= k);
      const int src = __ffs(reach) - 1;
      int above = __shfl_sync(kFull, incl - sum, src);
      // the 32 bins of that lane, one per lane
      const int mine = hist[kSelBins - 1 - src * 32 - lane];
      int in2 = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFull, in2, o);
        if (lane >= o) in2 += v;
      }
      const int at = __ffs(__ballot_sync(kFull, above + in2 >= k)) - 1;
      above += __shfl_sync(kFull, in2 - mine, at);
      const int members = __shfl_sync(kFull, mine, at);
      if (lane == 0) cnt[0] = kSelBins - 1 - src * 32 - at, cnt[1] = k - above, cnt[2] = members;
    }
    __syncthreads();
    const int bin = cnt[0], place = cnt[1], members = cnt[2];
    if (members <= kSelList) {
      float* vals = reinterpret_cast<float*>(list_val);
      each([&](int, bool on, float s, float) {
        if (on && bin_of(s) == bin) vals[atomicAdd(&totals[3], 1)] = s;
      });
      __syncthreads();
      for (int i = tid; i < members; i += kSelThreads) {
        const float v = vals[i];
        int rank = 0;
        for (int j = 0; j < members; ++j) rank += vals[j] > v || (vals[j] == v && j < i);
        if (rank == place - 1) found_sk = v;
      }
      __syncthreads();
      sk = found_sk;
    } else {
      // bisection over the order-preserving integer keys
      block_minmax(kmin, kmax, lo, hi);
      if (tid < 3) cnt[tid] = 0;
      __syncthreads();
      ++hi;                             // count(>= lo) >= k, count(>= hi) < k
      for (int it = 0; hi - lo > 1; ++it) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int mine = 0;
        each([&](int, bool on, float s, float) { mine += on && order_key(s) >= mid; });
        mine = __reduce_add_sync(kFull, mine);
        if (lane == 0 && mine) atomicAdd(&cnt[it % 3], mine);
        if (tid == 0) cnt[(it + 1) % 3] = 0;   // last read before the previous barrier
        __syncthreads();
        if (cnt[it % 3] >= k) lo = mid; else hi = mid;
      }
      sk = key_value(lo);
    }
    uint32_t low_key = 0xffffffffu, up_key = 0u;
    each([&](int, bool on, float s, float e) {
      if (!on) return;
      if (s >= sk) low_key = min(low_key, order_key(s - e));
      if (s <= sk) up_key = max(up_key, order_key(s + e));
    });
    block_minmax(low_key, up_key, lo, hi);
    lower = key_value(lo);
    upper = key_value(hi);
  }
  __syncthreads();
  each([&](int p, bool on, float s, float e) {
    bool in = p < n && !on;             // the first and the last pages
    bool open = false;
    if (on && k > 0) {
      if (s > sk) {
        in = s - e > upper;
        open = !in;
      } else {
        open = s + e >= lower;
      }
    }
    const uint32_t bi = __ballot_sync(kFull, in), bo = __ballot_sync(kFull, open);
    if (lane == 0 && p < n) {
      in_mask[p >> 5] = bi;
      open_mask[p >> 5] = bo;
      if (bi) atomicAdd(&totals[0], __popc(bi));
      if (bo) atomicAdd(&totals[1], __popc(bo));
    }
  });
  __syncthreads();
  const int n_open = totals[1];
  const int need = a.budget - totals[0];   // 0 <= need <= n_open
  if (need == n_open) {
    for (int w = tid; w < words; w += kSelThreads) in_mask[w] |= open_mask[w];
  } else {
    const __nv_bfloat16* q = a.q + (int64_t)tok * a.q_ld + (int64_t)kvh * (a.Hq / a.Hkv) * D;
    const int32_t* bt = a.block_table + (int64_t)r * a.bt_stride;
    const int G = a.Hq / a.Hkv;
    const bool small = n_open <= kSelList;
    double* big = reinterpret_cast<double*>(ws);   // the fp32 scores are no longer needed
    // exact scores of the open pages, one warp per page
    for (int w = warp; w < words; w += kSelWarps) {
      uint32_t m = open_mask[w];
      while (m) {
        const int p = w * 32 + __ffs(m) - 1;
        m &= m - 1;
        const bool finite = isfinite(ws[p].x);
        __syncwarp();
        const int64_t phys = table_page(bt, p, a.num_pages);
        const double v = finite ? exact_score(a, q, a.bounds + (phys * a.Hkv + kvh) * 2 * D, G, lane) : INFINITY;
        if (lane == 0) {
          if (small) {
            const int at = atomicAdd(&totals[2], 1);
            list_idx[at] = p;
            list_val[at] = v;
          } else {
            big[p] = v;
          }
        }
      }
    }
    __syncthreads();
    if (small) {
      if (tid < n_open) {
        const double v = list_val[tid];
        const int p = list_idx[tid];
        int rank = 0;
        for (int j = 0; j < n_open; ++j) rank += list_val[j] > v || (list_val[j] == v && list_idx[j] < p);
        if (rank < need) atomicOr(&in_mask[p >> 5], 1u << (p & 31));
      }
    } else {
      // bisection over the 64-bit keys, then ties by index
      unsigned long long lo = 0, hi = ~0ull;      // count(>= lo) >= need; no finite or infinite key is ~0
      for (int it = 0; hi - lo > 1; ++it) {
        const unsigned long long mid = lo + (hi - lo) / 2;
        if (tid == 0) cnt[0] = 0;
        __syncthreads();
        int mine = 0;
        for (int p = tid; p < n; p += kSelThreads)
          mine += (open_mask[p >> 5] >> (p & 31) & 1u) && order_key64(big[p]) >= mid;
        mine = __reduce_add_sync(kFull, mine);
        if (lane == 0 && mine) atomicAdd(&cnt[0], mine);
        __syncthreads();
        if (cnt[0] >= need) lo = mid; else hi = mid;
        __syncthreads();
      }
      if (tid == 0) cnt[0] = 0;
      __syncthreads();
      for (int w = warp; w < words; w += kSelWarps) {
        const int p = w * 32 + lane;
        const bool open = open_mask[w] >> lane & 1u;
        const unsigned long long key = open ? order_key64(big[p]) : 0ull;
        const uint32_t above = __ballot_sync(kFull, open && key > lo), equal = __ballot_sync(kFull, open && key == lo);
        __syncwarp();
        if (lane == 0) {
          in_mask[w] |= above;
          open_mask[w] = equal;
          if (above) atomicAdd(&cnt[0], __popc(above));
        }
      }
      __syncthreads();
      if (tid == 0) {
        int left = need - cnt[0];
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
  }
  __syncthreads();
  // positions of the chosen pages, in ascending order
  const int per = (words + kSelThreads - 1) / kSelThreads;
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int w = tid * per + i;
    if (w < words) mine += __popc(in_mask[w]);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) red[0][warp] = (uint32_t)incl;
  __syncthreads();
  int at = incl - mine;
  for (int w = 0; w < warp; ++w) at += (int)red[0][w];
  for (int i = 0; i < per; ++i) {
    const int w = tid * per + i;
    if (w >= words) break;
    prefix[w] = (uint32_t)at;
    at += __popc(in_mask[w]);
  }
  __syncthreads();
  for (int p = tid; p < n; p += kSelThreads) {
    const uint32_t m = in_mask[p >> 5], bit = 1u << (p & 31);
    if (m & bit) {
      const int i = (int)prefix[p >> 5] + __popc(m & (bit - 1));
      if (i < a.budget) sel[i] = p;
    }
  }
}

// ===========================================================================
// decode_sparse: a cluster of CTAs per (row, KV head), four warps each, every
// warp a share of the chosen pages with its own running maximum and sum; the
// warps join in shared memory, the CTAs through distributed shared memory, so
// there is one launch and no workspace.
//
// S^T = K Q^T has the page's 16 tokens as rows and the query heads as columns;
// O^T = V^T P^T has dimensions as rows.  K is read by the lanes in the layout of
// the A operand directly (16 bytes = eight dimensions = two k-steps).  V^T needs
// two tokens side by side: a lane reads the same eight dimensions of two tokens
// and interleaves them with byte permutes; row g of tile t is dimension 8g + t.
// P^T comes from S^T by an 8 x 8 register transpose.  P is rounded to bf16 for
// the tensor cores, an error of 2^-9 of each weight that averages over the
// tokens; the sum of the weights is kept in fp32 from the same rounded values,
// so the rounding does not scale the output.
// ===========================================================================
constexpr int kSpWarps = kWarps;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t x;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(x));
  return x;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
  uint32_t addr;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int NH>
struct SparseSmem {
  float o[kSpWarps][NH * 8][D];
  float m[kSpWarps][NH * 8];
  float l[kSpWarps][NH * 8];
};

template <int NH>
__global__ void __launch_bounds__(kThreads, 2) decode_sparse_kernel(const SparseArgs a, int cl) {
  extern __shared__ __align__(128) uint8_t raw[];
  SparseSmem<NH>& sm = *reinterpret_cast<SparseSmem<NH>*>(raw);   // over the ring, after the last page
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int part = cl > 1 ? (int)cluster_rank() : 0;
  const int unit = blockIdx.x / cl;
  const int kvh = unit % a.Hkv, r = unit / a.Hkv;
  const int G = a.Hq / a.Hkv;
  const int L = row_length(a.seq_lens, r, a.width);
  const int n = (L + PAGE - 1) / PAGE;
  const int tok = a.tok_index[r];
  const bool tok_ok = tok >= 0 && tok < a.tokens;
  if (!tok_ok && tid == 0) set_error(kErrBadIndex, (unsigned long long)r);
  const int count = tok_ok ? min(n, a.budget) : 0;
  const int32_t* bt = a.block_table + (int64_t)r * a.bt_stride;
  const int32_t* sel = a.sel + ((int64_t)r * a.Hkv + kvh) * a.budget;

  // this warp's pages: entries w, w + stride, ... of the list; lane j holds the
  // j-th of a window of 32 (first token, physical page), the next window under way
  const int stride = cl * kSpWarps, w = part * kSpWarps + warp;
  const int mine = count > w ? (count - w + stride - 1) / stride : 0;
  int win_tok, win_phys, next_page = -1;
  auto fetch_window = [&](int i) { next_page = i + lane < mine ? sel[w + (i + lane) * stride] : -1; };
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
    fetch_window(i + 32);
  };
  fetch_window(0);

  // a lane's pieces of a page: K rows g and g + 8, pieces c, c + 4, ...; V rows 2c,
  // 2c + 1, 2c + 8, 2c + 9, piece g of both halves of the dimensions
  const uint32_t ring = smem_u32(raw) + tid * 16;
  const __nv_bfloat16* kl = a.kcache + (int64_t)kvh * PAGE * D + g * D + c * 8;
  const __nv_bfloat16* vl = a.vcache + (int64_t)kvh * PAGE * D + 2 * c * D + g * 8;
  const int64_t page_elems = (int64_t)a.Hkv * PAGE * D;
  auto issue = [&](int i, uint32_t slot) -> int {   // the page's first token
    int t0 = L;
    if (i < mine) {
      if ((i & 31) == 0) open_window(i);
      t0 = __shfl_sync(kFull, win_tok, i & 31);
      const int64_t at = __shfl_sync(kFull, win_phys, i & 31) * page_elems;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        cp_async16(slot + j * kUnit, kl + at + j * 32, true);
        cp_async16(slot + (4 + j) * kUnit, kl + at + 8 * D + j * 32, true);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int t = (x & 1) + (x >> 1) * 8;
        const bool on = t0 + 2 * c + t < L;         // zeros past the sequence's end
        cp_async16(slot + (8 + x) * kUnit, vl + at + t * D, on);
        cp_async16(slot + (12 + x) * kUnit, vl + at + t * D + 64, on);
      }
    }
    cp_async_commit();
    return t0;
  };
  int first_tok[kStages];
#pragma unroll
  for (int i = 0; i < kStages; ++i) first_tok[i] = issue(i, ring + i * kStage);

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

  uint32_t slot = ring;
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<kStages - 1>();
    const int t0 = first_tok[0];
#pragma unroll
    for (int x = 0; x + 1 < kStages; ++x) first_tok[x] = first_tok[x + 1];
    uint32_t p[NH][2];
    float s[NH][2][4];
#pragma unroll
    for (int t = 0; t < NH; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) s[t][x][0] = s[t][x][1] = s[t][x][2] = s[t][x][3] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 k0 = lds16(slot + j * kUnit), k1 = lds16(slot + (4 + j) * kUnit);
#pragma unroll
      for (int t = 0; t < NH; ++t) {
        mma_bf16(s[t][0], k0.x, k1.x, k0.y, k1.y, q[t][j].x, q[t][j].y);
        mma_bf16(s[t][1], k0.z, k1.z, k0.w, k1.w, q[t][j].z, q[t][j].w);
      }
    }
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
      const uint32_t plo = pack_bf16x2(pr[0], pr[1]), phi = pack_bf16x2(pr[2], pr[3]);
      const float2 f0 = __bfloat1622float2(as_bf2(plo)), f1 = __bfloat1622float2(as_bf2(phi));
      l[t][0] += f0.x + f1.x;
      l[t][1] += f0.y + f1.y;
      p[t][0] = movmatrix_trans(plo);
      p[t][1] = movmatrix_trans(phi);
    }
    uint4 v[2][4];                      // v[half of the dimensions][token 2c, 2c + 1, 2c + 8, 2c + 9]
#pragma unroll
    for (int x = 0; x < 4; ++x) v[0][x] = lds16(slot + (8 + x) * kUnit), v[1][x] = lds16(slot + (12 + x) * kUnit);
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
      for (int t = 0; t < NH; ++t) mma_bf16(o[t][i8], a0, a1, a2, a3, p[t][0], p[t][1]);
    }
    first_tok[kStages - 1] = issue(i + kStages, slot);
    slot = slot == ring + (kStages - 1) * kStage ? ring : slot + kStage;
  }
  cp_async_wait<0>();
  __syncthreads();                      // the ring's memory becomes the warps' results

  // join: o[t][i][0..1] = dim 8g + i, heads 2c, 2c + 1; [2..3] = dim 64 + 8g + i
#pragma unroll
  for (int t = 0; t < NH; ++t) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float s = l[t][e];
      s += __shfl_xor_sync(kFull, s, 4);
      s += __shfl_xor_sync(kFull, s, 8);
      s += __shfl_xor_sync(kFull, s, 16);
      const int h = t * 8 + 2 * c + e;
      if (g == 0) {
        sm.m[warp][h] = m[t][e];
        sm.l[warp][h] = s;
      }
#pragma unroll
      for (int i8 = 0; i8 < 8; ++i8) {
        sm.o[warp][h][8 * g + i8] = o[t][i8][e];
        sm.o[warp][h][64 + 8 * g + i8] = o[t][i8][e + 2];
      }
    }
  }
  __syncthreads();
  // the CTA's warps, into the first warp's place
  const int d = threadIdx.x;
  for (int h = 0; h < G; ++h) {
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < kSpWarps; ++x) mx = fmaxf(mx, sm.m[x][h]);
    const float sh = mx == -INFINITY ? 0.f : mx;
    float acc = 0.f, ls = 0.f;
#pragma unroll
    for (int x = 0; x < kSpWarps; ++x) {
      const float f = exp2f(sm.m[x][h] - sh);
      acc += f * sm.o[x][h][d];
      ls += f * sm.l[x][h];
    }
    if (cl == 1) {
      if (tok_ok)
        a.out[(int64_t)tok * a.out_ld + (int64_t)(kvh * G + h) * D + d] = __float2bfloat16(ls > 0.f ? acc / ls : 0.f);
    } else {
      sm.o[0][h][d] = acc;
      __syncthreads();
      if (d == 0) sm.m[0][h] = mx, sm.l[0][h] = ls;
    }
  }
  if (cl == 1) return;
  cluster_sync_all();
  for (int h = part; h < G; h += cl) {
    float mx = -INFINITY;
    for (int x = 0; x < cl; ++x) mx = fmaxf(mx, ld_cluster(&sm.m[0][h], x));
    const float sh = mx == -INFINITY ? 0.f : mx;
    float acc = 0.f, ls = 0.f;
    for (int x = 0; x < cl; ++x) {
      const float f = exp2f(ld_cluster(&sm.m[0][h], x) - sh);
      acc += f * ld_cluster(&sm.o[0][h][d], x);
      ls += f * ld_cluster(&sm.l[0][h], x);
    }
    if (tok_ok)
      a.out[(int64_t)tok * a.out_ld + (int64_t)(kvh * G + h) * D + d] = __float2bfloat16(ls > 0.f ? acc / ls : 0.f);
  }
  cluster_sync_all();   // no CTA leaves while another reads its shared memory
}

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

}  // namespace

void page_bounds(const BoundsArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.max_new <= 0) return;
  BoundsArgs b = a;
  b.max_pages = (a.max_new + PAGE - 2) / PAGE + 1;   // from any offset in a page
  if (b.max_pages > a.width) b.max_pages = a.width;
  const int64_t units = (int64_t)a.rows * a.Hkv * b.max_pages;
  launch_k(page_bounds_kernel, dim3((unsigned)((units + 3) / 4)), dim3(128), 0, s, 1, b);
}

namespace {
void raise_smem(const void* k, size_t smem) {
  if (smem <= 48 * 1024) return;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) launch_failed(e);
}
}  // namespace

void select_pages(const SelectArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  if (a.width > a.budget) {
    // up to eight passes of 64 pages per CTA, fewer where that leaves SMs without work
    const int64_t tiles = (int64_t)a.rows * a.Hkv * ((a.width + kScoreTile - 1) / kScoreTile);
    const int64_t want = tiles / (4 * sm_count());
    const int passes = want < 1 ? 1 : want > kScorePasses ? kScorePasses : (int)want;
    const int chunk = passes * kScoreTile;
    const dim3 grid((unsigned)((a.width + chunk - 1) / chunk * a.Hkv), (unsigned)a.rows);
    auto k = a.Hq / a.Hkv <= 8 ? page_score_kernel<1> : page_score_kernel<2>;
    raise_smem(reinterpret_cast<const void*>(k), kStages * kStage);
    launch_k(k, grid, dim3(kThreads), kStages * kStage, s, 1, a, passes);
  }
  const size_t smem = (size_t)((a.width + 31) / 32) * 3 * sizeof(uint32_t);   // at most 24 KB
  const dim3 grid((unsigned)a.Hkv, (unsigned)a.rows);
  if (a.width <= 512) launch_k(page_select_kernel<256, 2>, grid, dim3(256), smem, s, 1, a);
  else if (a.width <= 2048) launch_k(page_select_kernel<512, 4>, grid, dim3(512), smem, s, 1, a);
  else if (a.width <= 8192) launch_k(page_select_kernel<1024, 8>, grid, dim3(1024), smem, s, 1, a);
  else launch_k(page_select_kernel<1024, 0>, grid, dim3(1024), smem, s, 1, a);
}

void decode_sparse(const SparseArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  const int64_t units = (int64_t)a.rows * a.Hkv;
  const int64_t slots = (int64_t)sm_count() * 2;
  int cl = 1;
  while (cl < 8 && units * cl * 2 <= slots && a.budget >= kSpWarps * cl * 2) cl *= 2;
  auto k = a.Hq / a.Hkv <= 8 ? decode_sparse_kernel<1> : decode_sparse_kernel<2>;
  raise_smem(reinterpret_cast<const void*>(k), kStages * kStage);   // covers the join's 17 / 33 KB
  launch_k(k, dim3((unsigned)(units * cl)), dim3(kThreads), kStages * kStage, s, (unsigned)cl, a, cl);
}

}  // namespace attn
}  // namespace lf
