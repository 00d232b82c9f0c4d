// Low-rank adapters of many requests beside a shared projection.
//
//   h[t]      = A[a(t)] x[t]                                     (rank values per slice)
//   out[t, c] = base[t, c] + scale[a] * sum_j B[a][c, j] h[t, slice(c) R + j]
//
// for the rows t listed in `rows`, grouped by adapter (`starts` is the CSR
// offset of every adapter of the pool).  Slices are the column ranges of a
// stacked projection (Q, K, V), each with its own A.  Sums are fp32, h is handed
// on as two bf16 parts (three for fp32 outputs), an error of at most 2^-16
// (2^-24) of h, and the output is rounded once.
//
// A cluster of up to eight CTAs owns a tile of up to TM rows of one adapter:
// every CTA multiplies a share of K, the partial h are added through distributed
// shared memory in rank order, and every CTA expands a share of the columns.  So
// the whole operator is one launch without a workspace, x and the weights are
// read by one CTA each, and a result does not depend on the order of arrival.  (The
// large kernel takes one launch per group of slices where slices x rank exceeds an
// accumulator's 256 columns or shared memory.)  The last bits of a row do depend on the
// batch it comes in: on the kernel, the tile and the shares of K.
// Only the adapter's rank is read, of A and of B: inside a tile, h has S * rank
// columns, the rank rounded up to 8 (16 in the large kernel) ("compact" below).
//
// Two kernels.  The small one (TM = 16, mma.sync) is for decode, where reading the
// weights bounds the call; the large one (TM = 64 or 128, tcgen05) is for prefill, where
// x, base and out do, and the weights come from L2 once per tile.  use_large()
// has the rule and both sides' times.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <stdexcept>

#include "common.cuh"
#include "gemm_bf16.h"
#include "lora.h"

namespace lf {
namespace lora {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kCluster = 8;               // largest cluster
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;   // 0 bytes read: the 16 bytes become zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool on) {
  const int n = on ? 8 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
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
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster2(uint32_t addr, uint2 v) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}

// The four values as PARTS bf16 values each that add up to them.  Parts before the last
// one stay finite: a value beyond the largest bf16 is still held, an infinity is the
// last part alone (as the first it would leave inf - inf for the next).
template <int PARTS>
__device__ __forceinline__ void split4(float4 v, uint2 (&p)[PARTS]) {
  constexpr float kMost = 0x1.fep127f;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    float4 w = v;
    if (i + 1 < PARTS)
      w = make_float4(fminf(fmaxf(v.x, -kMost), kMost), fminf(fmaxf(v.y, -kMost), kMost), fminf(fmaxf(v.z, -kMost), kMost),
                      fminf(fmaxf(v.w, -kMost), kMost));
    p[i].x = pack_bf16x2(w.x, w.y);
    p[i].y = pack_bf16x2(w.z, w.w);
    const float2 a = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&p[i].x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&p[i].y));
    v.x -= a.x, v.y -= a.y, v.z -= b.x, v.w -= b.y;
  }
}

// The tile's adapter, by a scan over the tiles of every adapter of the pool.
// Called by whole warps; every warp and CTA that asks finds the same.  The
// ranks and scales are fetched with the offsets, one round trip for all.
struct Tile {
  int adapter;       // -1: past the last tile
  int first, valid;  // its entries of `rows`
  int rank;
  float scale;
};
template <int TM>
__device__ __forceinline__ Tile find_tile(const LoraArgs& a, int tile) {
  const int lane = threadIdx.x & 31;
  Tile t{-1, 0, 0, 0, 0.f};
  int before = 0;
  bool bad = false;
  for (int b0 = 0; b0 < a.pool && t.adapter < 0; b0 += 32) {
    const int ad = b0 + lane;
    int s0 = 0, s1 = 0, rank = 0;
    float scale = 0.f;
    if (ad < a.pool) s0 = a.starts[ad], s1 = a.starts[ad + 1], rank = a.ranks[ad], scale = a.scales[ad];
    if (s0 < 0 || s1 < s0 || s1 > a.L) bad = true, s0 = s1 = 0;
    const int tiles = (s1 - s0 + TM - 1) / TM;
    int incl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, incl, o);
      if (lane >= o) incl += v;
    }
    const uint32_t m = __ballot_sync(kFull, before + incl > tile && before + incl - tiles <= tile);
    if (m) {
      const int src = __ffs(m) - 1;
      const int j = (tile - (before + incl - tiles)) * TM;
      t.adapter = b0 + src;
      t.first = __shfl_sync(kFull, s0 + j, src);
      t.valid = __shfl_sync(kFull, min(TM, s1 - s0 - j), src);
      t.rank = __shfl_sync(kFull, rank, src);
      t.scale = __shfl_sync(kFull, scale, src);
    }
    before += __shfl_sync(kFull, incl, 31);
  }
  if (__any_sync(kFull, bad) && lane == 0) set_error(kErrBadIndex, 0);
  if (t.rank < 0 || t.rank > a.R) {
    if (lane == 0) set_error(kErrBadIndex, (unsigned long long)t.adapter);
    t.rank = 0;
  }
  return t;
}
// Token row i of the tile, -1 where it has none.
__device__ __forceinline__ int tile_row(const LoraArgs& a, const Tile& t, int i) {
  if (i >= t.valid) return -1;
  const int row = a.rows[t.first + i];
  if (row >= 0 && row < a.T) return row;
  set_error(kErrBadIndex, (unsigned long long)(t.first + i));
  return -1;
}

// Streaming 16-byte load (no line kept in L1).
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Eight consecutive output columns of one row: base + scale * d, rounded once.
template <bool F32>
struct BaseCols {
  uint4 v[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* at) {
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) v[i] = ld_stream(reinterpret_cast<const uint4*>(at) + i);
  }
  __device__ __forceinline__ void store(void* at, const float (&d)[8], float scale) const {
    if (F32) {
      float4* p = reinterpret_cast<float4*>(at);
      const float* b = reinterpret_cast<const float*>(v);
      p[0] = make_float4(b[0] + scale * d[0], b[1] + scale * d[1], b[2] + scale * d[2], b[3] + scale * d[3]);
      p[1] = make_float4(b[4] + scale * d[4], b[5] + scale * d[5], b[6] + scale * d[6], b[7] + scale * d[7]);
    } else {
      const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(v);
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(b[i]);
        o[i] = pack_bf16x2(f.x + scale * d[2 * i], f.y + scale * d[2 * i + 1]);
      }
      *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
};

// The idx-th block of W (32 or 128) columns that does not cross a slice: its
// slice (-1 past the last block), first column and the slice's end.
struct Block {
  int slice, c0, end;
};
template <int W>
__device__ __forceinline__ Block column_block(const LoraArgs& a, int idx) {
  const int* first = W == 32 ? a.block32 : a.block128;
  if (idx >= first[kMaxSlices]) return Block{-1, 0, 0};
  int s = 0;
#pragma unroll
  for (int i = 1; i < kMaxSlices; ++i) s += idx >= first[i];   // absent slices begin past the last block
  return Block{s, a.col_begin[s] + (idx - first[s]) * W, a.col_begin[s + 1]};
}

// ===========================================================================
// Small tiles: 16 rows.  Shrink h^T = A x^T: 16 compact columns of h are the
// rows of m16n8k16, the tile's rows its columns; lane (g, c) = (lane / 4,
// lane % 4) needs 16 bytes at k = 32 kb + 8 c of A rows g, g + 8 and of token
// rows g, g + 8: two k-steps whose order of k is the same on both sides.  The
// warps split K further.  Every lane copies its own pieces into its own slots
// of a ring in shared memory (cp.async) and reads only those back: a deep
// pipeline without registers and without a barrier.  Expand: 32 output columns
// per warp, column n of tile t being column 8 (n / 2) + 2 t + n % 2, so that a
// lane ends with eight consecutive columns of two rows; B and base of the next
// columns come through the same ring, the first ones from before the reduction
// of h, on which they do not depend.
// ===========================================================================
constexpr int kSmallRows = 16;

// Two stages of wide slots: more leave too little L1 for one_row()'s loads (64 adapters
// 14.0 us, 14.7 with three).
template <int MT>
constexpr int small_stages() { return MT >= 3 ? 2 : 4; }
// The ring in units of 16 bytes per lane.  The warps' sums take its first 2 MT
// units between the two phases; the expansion's items use the others.
template <bool F32, bool WIDE>
constexpr int item_units() { return (WIDE ? 4 : 2) + (F32 ? 4 : 2); }   // four pieces of B, two of base
template <bool F32, int MT, bool WIDE>
constexpr int small_units() {
  const int k = small_stages<MT>() * (2 * MT + 2), least = 2 * MT + 2 * item_units<F32, WIDE>();
  return k > least ? k : least;
}
template <bool F32, int MT, bool WIDE>
constexpr int small_items() {   // items under way
  const int n = (small_units<F32, MT, WIDE>() - 2 * MT) / item_units<F32, WIDE>();
  return n < 4 ? n : 4;
}

// WIDE: R is a multiple of 32, a lane reads 8 consecutive k of a column (two
// k-steps); else 4 (one k-step).

// Tiles of one row, the usual ones where every request has its own adapter:
// products of the weights with a vector, on the fp32 units.  A warp reads 512
// consecutive bytes of one A row at a time (eight rows under way) against x in
// shared memory, so its sums need no other warp; R / 8 lanes read one column of B.
// R is a power of two.  The loops are kept short: a CTA runs each once or a few
// times, and longer ones would wait for their instructions.
// One request of rank 16 beside the QKV projection takes 6.7 us, 7.5 as a tile of
// 16 rows; 64 requests 14.7 and 15.9.  Rank 64 loses: 64 requests 43 and 39, one of K = 14336
// 12.1 and 11.2.
__device__ __forceinline__ float dot8(const uint4& v, const float4& x0, const float4& x1, float acc) {
  acc += __uint_as_float(v.x << 16) * x0.x;
  acc += __uint_as_float(v.x & 0xffff0000u) * x0.y;
  acc += __uint_as_float(v.y << 16) * x0.z;
  acc += __uint_as_float(v.y & 0xffff0000u) * x0.w;
  acc += __uint_as_float(v.z << 16) * x1.x;
  acc += __uint_as_float(v.z & 0xffff0000u) * x1.y;
  acc += __uint_as_float(v.w << 16) * x1.z;
  acc += __uint_as_float(v.w & 0xffff0000u) * x1.w;
  return acc;
}

template <bool F32>
__device__ __forceinline__ void one_row(const LoraArgs& a, const Tile& tl, int row, int cl, int cta, uint8_t* raw) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = tl.rank, rp = (rank + 7) / 8 * 8, cols = a.S * rp;
  const int kblocks = (a.K + 31) / 32, per_cta = (kblocks + cl - 1) / cl;
  const int kbeg = cta * per_cta * 32, kend = min(a.K, kbeg + per_cta * 32);
  const int span = (per_cta * 32 + 255) / 256 * 256;             // whole steps of a warp
  float* xs = reinterpret_cast<float*>(raw);                     // [span]
  float* part = xs + span;                                       // [cols], this CTA's share of K
  float* h = part + cols;                                        // [cols]
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);

  for (int i = tid * 8; i < span; i += kThreads * 8) {
    const uint4 v = kbeg + i < kend && row >= 0
                        ? *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.x) + (int64_t)row * a.ldx + kbeg + i)
                        : zero;
    float4* d = reinterpret_cast<float4*>(xs + i);
    d[0] = make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
    d[1] = make_float4(__uint_as_float(v.z << 16), __uint_as_float(v.z & 0xffff0000u), __uint_as_float(v.w << 16), __uint_as_float(v.w & 0xffff0000u));
  }
  __syncthreads();

  // h: warp w takes compact columns w, w + 8, ...
  const __nv_bfloat16* A = reinterpret_cast<const __nv_bfloat16*>(a.a) + (int64_t)tl.adapter * a.S * a.R * a.K + kbeg + lane * 8;
#pragma unroll 1
  for (int jg = warp; jg < cols; jg += 8 * kWarps) {
    const __nv_bfloat16* ap[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = jg + u * kWarps, s = j / rp, i = j - s * rp;
      ap[u] = j < cols && i < rank ? A + (int64_t)(s * a.R + i) * a.K : nullptr;
    }
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int c = 0; c < span; c += 256) {
      const bool in = kbeg + c + lane * 8 < kend;
      uint4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = in && ap[u] != nullptr ? ld_stream(ap[u] + c) : zero;
      const float4 x0 = *reinterpret_cast<const float4*>(xs + c + lane * 8), x1 = *reinterpret_cast<const float4*>(xs + c + lane * 8 + 4);
#pragma unroll
      for (int u = 0; u < 8; ++u) acc[u] = dot8(v[u], x0, x1, acc[u]);
    }
    // eight sums over the warp: the lanes halve the set of sums they hold three times
#pragma unroll
    for (int o = 16, n = 4; o >= 4; o >>= 1, n >>= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int u = 0; u < n; ++u) {
        const float keep = up ? acc[u + n] : acc[u], give = up ? acc[u] : acc[u + n];
        acc[u] = keep + __shfl_xor_sync(kFull, give, o);
      }
    }
    acc[0] += __shfl_xor_sync(kFull, acc[0], 2);
    acc[0] += __shfl_xor_sync(kFull, acc[0], 1);
    const int j = jg + ((lane >> 4 & 1) * 4 + (lane >> 3 & 1) * 2 + (lane >> 2 & 1)) * kWarps;
    if ((lane & 3) == 0 && j < cols) part[j] = acc[0];
  }

  // B and base of this warp's next six steps
  constexpr int NB = 6;
  const int per_col = a.R / 8, piece = lane & (per_col - 1), k = piece * 8;   // lanes of a column
  const int cstep = 32 / per_col;         // columns of a step
  const int share = ((a.N + cl - 1) / cl + 31) / 32 * 32;
  const int c_lo = cta * share, c_hi = min(a.N, c_lo + share);
  const __nv_bfloat16* B = reinterpret_cast<const __nv_bfloat16*>(a.b) + (int64_t)tl.adapter * a.N * a.R + k;
  const int64_t base_row = (int64_t)(row >= 0 ? row : 0) * a.ldb, out_row = (int64_t)(row >= 0 ? row : 0) * a.ldo;
  uint4 bv[NB];
  float bs[NB];
  auto fetch = [&](int col0) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int col = col0 + i * (kWarps * cstep);
      bv[i] = col < c_hi && k < rank ? ld_stream(B + (int64_t)col * a.R) : zero;
      bs[i] = 0.f;
      if (col < c_hi && piece == 0)
        bs[i] = F32 ? reinterpret_cast<const float*>(a.base)[base_row + col]
                    : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.base)[base_row + col]);
    }
  };
  int col0 = c_lo + warp * cstep + lane / per_col;
  fetch(col0);
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  for (int i = tid; i < cols; i += kThreads) {
    float v[kCluster], sum = 0.f;
#pragma unroll
    for (int q = 0; q < kCluster; ++q) v[q] = q < cl ? ld_cluster(cluster_addr(part + i, q)) : 0.f;
#pragma unroll
    for (int q = 0; q < kCluster; ++q) sum += v[q];
    h[i] = i % rp < rank ? sum : 0.f;     // past the rank: zero rows of A, times an infinity in x
  }
  cluster_arrive();                       // this CTA has read the others' partials
  __syncthreads();
#pragma unroll 1
  for (; col0 - lane / per_col < c_hi; col0 += NB * kWarps * cstep) {
    float d[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int col = col0 + i * (kWarps * cstep);
      const int s = (a.S > 1 && col >= a.col_begin[1]) + (a.S > 2 && col >= a.col_begin[2]) + (a.S > 3 && col >= a.col_begin[3]);
      d[i] = 0.f;
      if (k < rank && col < c_hi) {
        uint4 v = bv[i];
        if (k + 8 > rank) {               // past the rank nothing counts, not even a NaN
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (k + 2 * e >= rank) w[e] = 0u;
            else if (k + 2 * e + 1 >= rank) w[e] &= 0xffffu;
          }
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        const float4* hr = reinterpret_cast<const float4*>(h + s * rp + k);
        d[i] = dot8(v, hr[0], hr[1], 0.f);
      }
    }
    for (int o = per_col >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < NB; ++i) d[i] += __shfl_xor_sync(kFull, d[i], o);
    }
    if (piece == 0 && row >= 0) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int col = col0 + i * (kWarps * cstep);
        if (col >= c_hi) continue;
        if (F32) reinterpret_cast<float*>(a.out)[out_row + col] = bs[i] + tl.scale * d[i];
        else reinterpret_cast<__nv_bfloat16*>(a.out)[out_row + col] = __float2bfloat16(bs[i] + tl.scale * d[i]);
      }
    }
    fetch(col0 + NB * kWarps * cstep);
  }
  cluster_wait();                         // no CTA leaves while another reads its partial h
}

template <bool F32, int MT, bool WIDE>
__global__ void __launch_bounds__(kThreads, 2) lora_small_kernel(const LoraArgs a, int cols_max, int cl, bool vector) {
  constexpr int TM = kSmallRows;
  constexpr int kParts = F32 ? 3 : 2;
  constexpr int ST = small_stages<MT>();
  constexpr int KB = WIDE ? 32 : 16;      // k of one item of the expansion
  constexpr int kUnit = kThreads * 16;    // a ring unit of all lanes
  constexpr int IU = item_units<F32, WIDE>(), NI = small_items<F32, MT, WIDE>();
  extern __shared__ __align__(128) uint8_t raw[];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int cta = (int)cluster_rank();
  const Tile tl = find_tile<TM>(a, blockIdx.x / cl);
  if (tl.adapter < 0) return;             // the whole cluster
  const int my_row = lane < TM ? tile_row(a, tl, lane) : -1;
  if (vector && tl.valid == 1) {
    one_row<F32>(a, tl, __shfl_sync(kFull, my_row, 0), cl, cta, raw);
    return;
  }
  const int rank = tl.rank;
  const int rb = (rank + 7) / 8;          // 8-row blocks of A per slice
  const int rp = rb * 8;
  const int mtiles = (a.S * rb + 1) / 2;
  float* red = reinterpret_cast<float*>(raw);                      // [kWarps][MT * 16][TM], over the ring
  float* part = reinterpret_cast<float*>(raw + small_units<F32, MT, WIDE>() * kUnit);   // [cols_max][TM]
  __nv_bfloat16* hs = reinterpret_cast<__nv_bfloat16*>(part + cols_max * TM);           // [kParts][TM][hld]
  const int hld = cols_max + 40;          // a 32-wide item may pass the last column
  const uint32_t ring = smem_u32(raw) + tid * 16;

  // The expansion's items: KB values of k of a group of 32 columns; the warp's
  // items run over its groups and, inside, over k.
  const int lcol = (g >> 1) * 8 + (g & 1);                         // this lane's first column of B in a group
  const __nv_bfloat16* B = reinterpret_cast<const __nv_bfloat16*>(a.b) + (int64_t)tl.adapter * a.N * a.R;
  const int gstep = cl * kWarps;
  struct Item {
    int group, kb;
    Block at;
  };
  auto next_item = [&](Item& q) {
    q.kb += KB;
    if (q.kb >= rank) {
      q.kb = 0;
      q.group += gstep;
      q.at = column_block<32>(a, q.group);
    }
  };
  const char *base0 = nullptr, *base1 = nullptr;                   // this lane's columns of base, null without a row
  auto issue_item = [&](const Item& q, uint32_t slot) {
    if (q.at.slice >= 0) {
      const bool kin = q.kb + KB / 4 * c < rank;
      const int left = q.at.end - q.at.c0 - lcol;                  // columns from this lane's first to the slice's end
      const __nv_bfloat16* b = B + (int64_t)(q.at.c0 + lcol) * a.R + q.kb + KB / 4 * c;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool on = kin && 2 * t < left;
        const __nv_bfloat16* src = on ? b + 2 * t * a.R : B;
        if (WIDE) cp_async16(slot + t * kUnit, src, on);
        else cp_async8(slot + (t >> 1) * kUnit + (t & 1) * 8, src, on);
      }
      if (q.kb == 0 && q.at.c0 + 8 * c < q.at.end) {
        const uint32_t ab = slot + (WIDE ? 4 : 2) * kUnit;
        const int64_t off = (int64_t)q.at.c0 * (F32 ? 4 : 2);
        if (base0 != nullptr) {
          cp_async16(ab, base0 + off, true);
          if (F32) cp_async16(ab + kUnit, base0 + off + 16, true);
        }
        if (base1 != nullptr) {
          cp_async16(ab + (F32 ? 2 : 1) * kUnit, base1 + off, true);
          if (F32) cp_async16(ab + 3 * kUnit, base1 + off + 16, true);
        }
      }
    }
    cp_async_commit();
  };
  Item cur{cta * kWarps + warp, 0, column_block<32>(a, cta * kWarps + warp)};
  Item ahead = cur;
  const uint32_t items = ring + 2 * MT * kUnit;
  int r0 = -1, r1 = -1;
  auto start_items = [&]() {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      issue_item(ahead, items + i * IU * kUnit);
      if (ahead.at.slice >= 0) next_item(ahead);
    }
  };
  auto take_rows = [&]() {
    r0 = __shfl_sync(kFull, my_row, g), r1 = __shfl_sync(kFull, my_row, g + 8);
    const int es = F32 ? 4 : 2;
    if (r0 >= 0) base0 = reinterpret_cast<const char*>(a.base) + ((int64_t)r0 * a.ldb + 8 * c) * es;
    if (r1 >= 0) base1 = reinterpret_cast<const char*>(a.base) + ((int64_t)r1 * a.ldb + 8 * c) * es;
  };

  if (mtiles == 0) {                      // rank 0: out = base
    take_rows();
    start_items();
  } else {
    const __nv_bfloat16* A = reinterpret_cast<const __nv_bfloat16*>(a.a) + (int64_t)tl.adapter * a.S * a.R * a.K;
    const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x);
    const int kblocks = (a.K + 31) / 32;
    const int per_cta = (kblocks + cl - 1) / cl;
    const int kb0 = cta * per_cta + warp, kb1 = min(kblocks, (cta + 1) * per_cta);
    const int n = kb1 > kb0 ? (kb1 - kb0 + kWarps - 1) / kWarps : 0;   // this warp's blocks
    const int k0 = kb0 * 32 + c * 8;
    const __nv_bfloat16 *x0 = nullptr, *x1 = nullptr;
    int s = 0, ib = 0;                    // slice and 8-row block of the next rows of A
    for (int m0 = 0; m0 < mtiles; m0 += MT) {
      const __nv_bfloat16* pa[MT][2];     // this lane's rows of A at its first k, null for none
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          pa[m][u] = s < a.S && ib * 8 + g < rank ? A + (int64_t)(s * a.R + ib * 8 + g) * a.K + k0 : nullptr;
          if (++ib == rb) ib = 0, ++s;
        }
      auto issue_a = [&](int it, uint32_t slot) {
        if (it >= n) return;
        const int dk = it * (kWarps * 32);
        const bool in = k0 + dk < a.K;    // K is a multiple of 8
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const bool on = in && pa[m][u] != nullptr;
            cp_async16(slot + (2 * m + u) * kUnit, on ? pa[m][u] + dk : A, on);
          }
      };
      auto issue_x = [&](int it, uint32_t slot) {
        if (it < n) {
          const int dk = it * (kWarps * 32);
          const bool in = k0 + dk < a.K;
          const bool on0 = in && x0 != nullptr, on1 = in && x1 != nullptr;
          cp_async16(slot + 2 * MT * kUnit, on0 ? x0 + dk : x, on0);
          cp_async16(slot + (2 * MT + 1) * kUnit, on1 ? x1 + dk : x, on1);
        }
        cp_async_commit();
      };
      constexpr int kSlot = (2 * MT + 2) * kUnit;
#pragma unroll
      for (int it = 0; it < ST; ++it) issue_a(it, ring + it * kSlot);   // before the token rows have arrived
      if (m0 == 0) {
        take_rows();
        if (r0 >= 0) x0 = x + (int64_t)r0 * a.ldx + k0;
        if (r1 >= 0) x1 = x + (int64_t)r1 * a.ldx + k0;
      }
#pragma unroll
      for (int it = 0; it < ST; ++it) issue_x(it, ring + it * kSlot);
      float acc[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[m][t][0] = acc[m][t][1] = acc[m][t][2] = acc[m][t][3] = 0.f;
      uint32_t slot = ring;
      for (int it = 0; it < n; ++it) {
        cp_async_wait<ST - 1>();
        const uint4 v0 = lds16(slot + 2 * MT * kUnit), v1 = lds16(slot + (2 * MT + 1) * kUnit);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 p = lds16(slot + 2 * m * kUnit), q = lds16(slot + (2 * m + 1) * kUnit);
          mma_bf16(acc[m][0], p.x, q.x, p.y, q.y, v0.x, v0.y);
          mma_bf16(acc[m][0], p.z, q.z, p.w, q.w, v0.z, v0.w);
          mma_bf16(acc[m][1], p.x, q.x, p.y, q.y, v1.x, v1.y);
          mma_bf16(acc[m][1], p.z, q.z, p.w, q.w, v1.z, v1.w);
        }
        issue_a(it + ST, slot);
        issue_x(it + ST, slot);
        slot = slot == ring + (ST - 1) * kSlot ? ring : slot + kSlot;
      }
      cp_async_wait<0>();
      if (m0 + MT >= mtiles) start_items();   // the last pass over K: this lane's slots are free
      __syncthreads();                    // the ring's first units become the warps' sums
      float* rw = red + warp * MT * 16 * TM;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          *reinterpret_cast<float2*>(rw + (m * 16 + g) * TM + t * 8 + 2 * c) = make_float2(acc[m][t][0], acc[m][t][1]);
          *reinterpret_cast<float2*>(rw + (m * 16 + g + 8) * TM + t * 8 + 2 * c) = make_float2(acc[m][t][2], acc[m][t][3]);
        }
      __syncthreads();
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m0 + m >= mtiles) break;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += red[(w * MT + m) * 16 * TM + tid];   // 256 threads = 16 x TM
        part[(m0 + m) * 16 * TM + tid] = v;
      }
      if (m0 + MT < mtiles) __syncthreads();
    }
  }

  cluster_arrive();
  cluster_wait();
  for (int i = tid; i < mtiles * 16 * TM / 4; i += kThreads) {     // four rows of one column
    float4 v[kCluster];
#pragma unroll
    for (int q = 0; q < kCluster; ++q)
      if (q < cl) v[q] = ld_cluster4(cluster_addr(part + i * 4, q));
#pragma unroll
    for (int q = 1; q < kCluster; ++q)
      if (q < cl) v[0].x += v[q].x, v[0].y += v[q].y, v[0].z += v[q].z, v[0].w += v[q].w;
    uint2 p[kParts];
    const int j = i / (TM / 4), row = i % (TM / 4) * 4;
    if (rank < rp && j % rp >= rank) v[0] = make_float4(0.f, 0.f, 0.f, 0.f);   // zero rows of A, times an infinity in x
    split4<kParts>(v[0], p);
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&p[q]);
#pragma unroll
      for (int r = 0; r < 4; ++r) hs[(q * TM + row + r) * hld + j] = e[r];
    }
  }
  cluster_arrive();                       // this CTA has read the others' partials
  pdl_trigger();
  __syncthreads();

  const int es = F32 ? 4 : 2;
  char* out0 = reinterpret_cast<char*>(a.out) + ((int64_t)r0 * a.ldo + 8 * c) * es;   // used where the row exists
  char* out1 = reinterpret_cast<char*>(a.out) + ((int64_t)r1 * a.ldo + 8 * c) * es;
  float acc[4][4];
  BaseCols<F32> bs[2];
  uint32_t slot = items;
  while (cur.at.slice >= 0) {
    cp_async_wait<NI - 1>();
    uint32_t b[4][KB / 8];
    if (WIDE) {
#pragma unroll
      for (int t = 0; t < 4; ++t) *reinterpret_cast<uint4*>(b[t]) = lds16(slot + t * kUnit);
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint4 v = lds16(slot + t * kUnit);
        b[2 * t][0] = v.x, b[2 * t][1] = v.y, b[2 * t + 1][0] = v.z, b[2 * t + 1][1] = v.w;
      }
    }
    if (cur.kb == 0) {
      const uint32_t ab = slot + (WIDE ? 4 : 2) * kUnit;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < (F32 ? 2 : 1); ++v) bs[u].v[v] = lds16(ab + (u * (F32 ? 2 : 1) + v) * kUnit);
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
    }
    const int k = cur.kb + KB / 4 * c;
    if (cur.kb + KB > rank) {             // past the rank nothing counts, not even a NaN
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int x = 0; x < KB / 8; ++x) {
          if (k + 2 * x >= rank) b[t][x] = 0u;
          else if (k + 2 * x + 1 >= rank) b[t][x] &= 0xffffu;
        }
    }
    const __nv_bfloat16* h = hs + g * hld + cur.at.slice * rp + k;
    const bool in = k < rp;               // beyond it lies the next slice's h
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      uint32_t w0[KB / 8], w1[KB / 8];
#pragma unroll
      for (int x = 0; x < KB / 8; ++x) {
        w0[x] = in ? reinterpret_cast<const uint32_t*>(h + q * TM * hld)[x] : 0u;
        w1[x] = in ? reinterpret_cast<const uint32_t*>(h + (q * TM + 8) * hld)[x] : 0u;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int x = 0; x < KB / 16; ++x) mma_bf16(acc[t], w0[2 * x], w1[2 * x], w0[2 * x + 1], w1[2 * x + 1], b[t][2 * x], b[t][2 * x + 1]);
    }
    issue_item(ahead, slot);
    if (ahead.at.slice >= 0) next_item(ahead);
    slot = slot == items + (NI - 1) * IU * kUnit ? items : slot + IU * kUnit;
    if (cur.kb + KB >= rank && cur.at.c0 + 8 * c < cur.at.end) {
      const int64_t off = (int64_t)cur.at.c0 * es;
      float d[8];
      if (r0 >= 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) d[2 * t] = acc[t][0], d[2 * t + 1] = acc[t][1];
        bs[0].store(out0 + off, d, tl.scale);
      }
      if (r1 >= 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) d[2 * t] = acc[t][2], d[2 * t + 1] = acc[t][3];
        bs[1].store(out1 + off, d, tl.scale);
      }
    }
    next_item(cur);
  }
  cluster_wait();                         // no CTA leaves while another reads its partial h
}

// ===========================================================================
// Large tiles: 64 or 128 rows, both products on the fifth-generation tensor cores.
//
// Shrink: h = x A^T accumulates in tensor memory over chunks of 64 k, x rows (gathered,
// cp.async) and the adapter's A rows (TMA, boxes of 16) in a ring of three to six
// stages with the 128-byte swizzle the instruction reads.  Each CTA of the cluster
// has a share of K; the partial h go to shared memory and are reduced in slices: CTA
// q of CL adds rows [q TML / CL, ...) of all CTAs, splits them into bf16 parts and,
// once all partials have been read, stores those in their place into every CTA's
// shared memory, a fraction of the traffic of every CTA reading everything.  Expand:
// blocks of 128 columns of B (two stages) against the parts of h into one of two
// accumulators, read back in the 16 x 256-bit shape, in which a lane holds two
// adjacent columns of rows g and g + 8; B's columns are stored in an order that makes
// them eight consecutive columns over four tiles.
//
// A CTA holds 256 of the SM's 512 columns of tensor memory.  Registers (128 rows) or at
// least 81 KB of shared memory (64 rows) keep it at one or two per SM, so that none
// waits for another one's columns; the other kernels with tensor memory take more
// than half of the shared memory, so that beside one of them at most one of these
// runs.
//
// 8192 rows beside the QKV projection (K = 4096, N = 6144): 76 us, where the bytes that x,
// base, out and the weights must move once take 40.  64-row tiles take 93: the 64-row instruction
// runs at half rate and every tile reads its adapter's weights from L2 again.  Not
// more shared memory than needed, because the loads of base that are under way live
// in what is left of it as L1: with 226 KB instead of 162 the call takes 88 us.
// The same 64-row tiles on mma.sync took 131.
// ===========================================================================
constexpr int kMinStages = 3, kMaxStages = 6;
constexpr int kLargeCols = 256;          // most compact columns (one accumulator)
constexpr int kTmemCols = 256;
constexpr int kBoxRows = 16;             // rows of A per box
constexpr int kBN = 128;                 // columns of a block of the expansion

// Waits of the large kernel.  Unlike mbar_wait() they are not cut short by an error that is
// already recorded: a bad row or rank of one tile must not void the copies and products of
// the others.  A thread whose wait runs out (kErrMbarTimeout) loads nothing more, hardly waits
// again (`gave_up`) and goes on through the barriers; what it has not loaded is not multiplied,
// what is not multiplied is not loaded over, so the CTA comes to rest.  Behind the loops
// it waits for what is under way (drained(): a second at least, whatever the limit is
// set to) before the memory is used again or freed.  Its shares of h become NaN, its
// columns are not written.
__device__ __forceinline__ bool arrived(uint64_t* bar, uint32_t parity, uint32_t where, bool gave_up = false) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  uint32_t spins = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++spins & 255u) == 0 && (gave_up || globaltimer_ns() - t0 > wait_limit_ns())) {
      set_error(kErrMbarTimeout, (unsigned long long)where);
      return false;
    }
  }
}
__device__ __noinline__ void drained(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns(), limit = max(wait_limit_ns(), (uint64_t)1000000000);
  while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 <= limit) {
  }
}

// 16 lanes x 8 groups of 8 columns: r[4 x + 0 / 1] = row g, columns 8 x + 2 c, + 1;
// r[4 x + 2 / 3] = row g + 8.
__device__ __forceinline__ void tmem_ld_16x256b_x8(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// Ring, then partial h, then [parts of h | B stages], one after the other in the same memory.
// What the ring has beyond three stages it uses.
constexpr size_t kLargeSmem = 226 * 1024;
struct LargeSmem {
  size_t b, total;      // offset of the B stages
};
__host__ __device__ inline LargeSmem large_smem(int tm, int cols_max, int R, int parts) {
  const size_t ring = (size_t)kMinStages * 128 * (tm + cols_max);
  const size_t part = (size_t)tm * (cols_max + 4) * 4;
  const size_t hs = (size_t)parts * ((cols_max + 63) / 64) * (tm * 128);
  const size_t b = (size_t)2 * kBN * ((R + 63) / 64 * 128);
  size_t need = hs + b;
  if (need < ring) need = ring;
  if (need < part) need = part;
  need += 1024;                // and the alignment to 1024
  const size_t least = tm == 64 ? 81 * 1024 : 162 * 1024;   // tall tiles: four stages (76 us beside the QKV projection), three take 80
  return {hs, need > least ? need : least};
}

template <bool F32, int TML, int CL>
__global__ void __launch_bounds__(TML * 4, 128 / TML)
    lora_large_kernel(const LoraArgs a, const __grid_constant__ CUtensorMap map_a, int cols_max, int smem_b, int smem_ring) {
  constexpr int kThreads = TML * 4, kWarps = kThreads / 32;
  constexpr int kParts = F32 ? 3 : 2;
  extern __shared__ __align__(128) uint8_t raw_unaligned[];
  __shared__ int tile_rows[TML];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], done[2], rest;
  __shared__ uint32_t tmem_base;
  __shared__ int loaded_most, multiplied_to;
  uint8_t* raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_unaligned) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int cta = (int)cluster_rank();
  if (tid == 0) tma_prefetch_desc(&map_a);
  pdl_wait();
  const Tile tl = find_tile<TML>(a, blockIdx.x / CL);
  if (tl.adapter < 0) return;             // the whole cluster
  const int rank = tl.rank;
  const int rp = (rank + 15) / 16 * 16;   // whole 16-wide steps; what lies past the rank is zero
  const int cols = a.S * rp;
  const int pld = cols_max + 4;
  float* part = reinterpret_cast<float*>(raw);
  uint8_t* hs = raw;                      // [part][64 columns][row][128 bytes]
  const int hpart = (cols_max + 63) / 64 * (TML * 128);
  const uint32_t raw_u = smem_u32(raw);
  if (warp == 0) {
    tmem_alloc(&tmem_base, kTmemCols);
    tmem_relinquish();
  }
  if (tid == 0) {
    // a stage of A is complete when every warp's boxes of it are
    const int box_warps = max(1, min(kWarps, cols / kBoxRows));
    for (int i = 0; i < kMaxStages; ++i) mbar_init(&full[i], box_warps), mbar_init(&empty[i], 1);
    mbar_init(&done[0], 1);
    mbar_init(&done[1], 1);
    mbar_init(&rest, 1);
    fence_barrier_init();
    loaded_most = 0;
  }

  // ---- shrink
  const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x);
  if (tid < TML) tile_rows[tid] = tile_row(a, tl, tid);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  // This warp's 16 rows and 64 of 128 columns of an accumulator.  The 64-row instruction
  // leaves rows 16 i ... in lanes 32 i ..., the 128-row one a row in every lane.
  const int wrow = TML == 64 ? (warp & 3) * 16 : (warp & 3) * 32 + (warp >> 2 & 1) * 16;
  const int half = warp / (kWarps / 2);
  const uint32_t tmem_row = tmem + ((uint32_t)(TML == 64 ? wrow * 2 : wrow) << 16);
  bool ok;                                // no wait of this CTA's has run out, later of this thread's
  {
    const int chunks = (a.K + 63) / 64;
    const int per_cta = (chunks + CL - 1) / CL;
    const int ch0 = cta * per_cta, n = cols > 0 ? max(0, min(chunks, ch0 + per_cta) - ch0) : 0;
    const int stage_bytes = 128 * (TML + cols);
    const int stages = min(kMaxStages, smem_ring / stage_bytes);
    // thread t copies piece t % 8 of token rows t / 8 and t / 8 + TML / 2; a warp's first lane a box of A or two
    const int piece = tid & 7, rfirst = tid >> 3;
    const uint32_t dst0 = raw_u + rfirst * 128 + ((piece ^ (rfirst & 7)) << 4);
    const int row_a = tile_rows[rfirst], row_b = tile_rows[rfirst + TML / 2];
    const __nv_bfloat16* xa = row_a >= 0 ? x + (int64_t)row_a * a.ldx : nullptr;
    const __nv_bfloat16* xb = row_b >= 0 ? x + (int64_t)row_b * a.ldx : nullptr;
    const int first_row = (tl.adapter * a.S_all + a.s0) * a.R;       // of lora_a
    auto box_row = [&](int b) {            // first row of A of box b
      const int j = b * kBoxRows, s = rp > 0 ? j / rp : 0;
      return j < cols ? first_row + s * a.R + j - s * rp : -1;
    };
    const int box0 = box_row(warp), box1 = box_row(warp + kWarps);
    int loads = n, products = n;          // chunks this thread loads and, the one that does, multiplies without a gap
    auto load_stage = [&](int i, int st) {
      if (i < loads) {
        const int k0 = (ch0 + i) * 64, k = k0 + piece * 8;
        if (lane == 0 && box0 >= 0) mbar_arrive_expect_tx(&full[st], (box1 >= 0 ? 2 : 1) * kBoxRows * 128);
        if (lane == 0 && box0 >= 0) tma_load_2d(raw + st * stage_bytes + (TML + warp * kBoxRows) * 128, &map_a, &full[st], k0, box0);
        if (lane == 0 && box1 >= 0)
          tma_load_2d(raw + st * stage_bytes + (TML + (warp + kWarps) * kBoxRows) * 128, &map_a, &full[st], k0, box1);
        const bool in = k < a.K;
        const bool on_a = in && xa != nullptr, on_b = in && xb != nullptr;
        cp_async16(dst0 + st * stage_bytes, on_a ? xa + k : x, on_a);
        cp_async16(dst0 + st * stage_bytes + TML / 2 * 128, on_b ? xb + k : x, on_b);
      }
      cp_async_commit();
    };
    auto wait_stage = [&]() {             // all but the youngest stages - 2 copies have arrived
      if (stages == 3) cp_async_wait<1>();
      else if (stages == 4) cp_async_wait<2>();
      else if (stages == 5) cp_async_wait<3>();
      else cp_async_wait<4>();
    };
    for (int i = 0; i < stages - 1; ++i) load_stage(i, i);
    const uint32_t idesc = idesc_bf16_f32(TML, cols);
    int st = 0, prev = stages - 1;        // slots of chunks i and i - 1, and the parity of their use
    uint32_t use = 0, prev_use = 1;
    for (int i = 0; i < n; ++i) {
      wait_stage();
      fence_proxy_async_smem();
      __syncthreads();
      if (warp == 0 && elect_one()) {     // (a further condition here costs 4 us)
        if (arrived(&full[st], use, 43, products < n)) {
          tc_fence_after();
          const uint32_t at = raw_u + st * stage_bytes;
          const uint64_t xd = sw128_kmajor_desc(at), ad = sw128_kmajor_desc(at + TML * 128);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) umma_f16_ss(tmem, xd + 2 * ks, ad + 2 * ks, idesc, (i | ks) != 0);
          umma_commit(&empty[st]);
        } else {
          products = min(products, i);
          loads = min(loads, i + stages - 1);
        }
      }
      __syncwarp();
      if (i > 0 && i + stages - 1 < loads && !arrived(&empty[prev], prev_use, 40)) loads = i + stages - 1;
      load_stage(i + stages - 1, prev);
      prev = st, prev_use = use;
      if (++st == stages) st = 0, use ^= 1;
    }
    ok = n == 0 || (loads == n && products == n && arrived(&empty[prev], prev_use, 41));
    cp_async_wait<0>();
    ok = __syncthreads_and(ok);           // the ring's memory becomes the partial h
    if (!ok) {
      // Warps that gave up later than others have loaded up to a ring's length more: those stages are
      // completed by plain arrivals.  Then every stage not multiplied, and the products.
      const bool boxes = lane == 0 && box0 >= 0;
      if (boxes) atomicMax(&loaded_most, loads);
      if (warp == 0 && elect_one()) {
        multiplied_to = products;
        umma_commit(&rest);
      }
      __syncthreads();
      if (boxes)
        for (int c = loads; c < loaded_most; ++c) mbar_arrive(&full[c % stages]);
      for (int c = multiplied_to; c < loaded_most; ++c) drained(&full[c % stages], c / stages & 1);
      drained(&rest, 0);
      __syncthreads();
    }
    tc_fence_after();
    for (int c0 = half * 64; c0 < cols; c0 += 128) {
      uint32_t r[32];
      tmem_ld_16x256b_x8(tmem_row + c0, r);
      tmem_wait_ld();
      if (!ok) {
#pragma unroll
        for (int e = 0; e < 32; ++e) r[e] = 0x7fffffffu;
      }
#pragma unroll
      for (int xg = 0; xg < 8; ++xg) {
        const int col = c0 + xg * 8 + 2 * c;
        if (col >= cols) continue;
        float* p = part + (wrow + g) * pld + col;
        // Past the rank h is zero, whatever the boxes brought; a CTA without a share of K adds zero.
        const int left = n > 0 ? rank - col % rp : 0;
        *reinterpret_cast<float2*>(p) =
            make_float2(left > 0 ? __uint_as_float(r[4 * xg]) : 0.f, left > 1 ? __uint_as_float(r[4 * xg + 1]) : 0.f);
        *reinterpret_cast<float2*>(p + 8 * pld) =
            make_float2(left > 0 ? __uint_as_float(r[4 * xg + 2]) : 0.f, left > 1 ? __uint_as_float(r[4 * xg + 3]) : 0.f);
      }
    }
    tc_fence_before();
  }
  cluster_arrive();
  cluster_wait();
  {
    constexpr int kOwn = TML / CL;        // rows this CTA adds up
    uint32_t part_at[CL], hs_at[CL];
#pragma unroll
    for (int q = 0; q < CL; ++q) {
      part_at[q] = cluster_addr(part + cta * kOwn * pld, q);
      hs_at[q] = cluster_addr(hs, q);
    }
    const int quads = cols / 4, items = kOwn * quads;
    constexpr int kIn = kOwn * (kLargeCols / 4) / kThreads;   // items of a thread
    constexpr int kBatch = CL == 2 ? 4 : 2;                   // whose remote loads are under way together
    uint2 p[kIn][kParts];
#pragma unroll
    for (int u0 = 0; u0 < kIn; u0 += kBatch) {
      if (u0 * kThreads >= items) break;
      float4 v[kBatch][CL];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = min(tid + (u0 + u) * kThreads, items - 1);
        const int row = i / quads, j = (i - row * quads) * 4;
#pragma unroll
        for (int q = 0; q < CL; ++q) v[u][q] = ld_cluster4(part_at[q] + (row * pld + j) * 4);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
#pragma unroll
        for (int q = 1; q < CL; ++q)
          v[u][0].x += v[u][q].x, v[u][0].y += v[u][q].y, v[u][0].z += v[u][q].z, v[u][0].w += v[u][q].w;
        split4<kParts>(v[u][0], p[u0 + u]);
      }
    }
    cluster_arrive();                     // all partials have been read: the parts of h take their place
    cluster_wait();
#pragma unroll
    for (int u = 0; u < kIn; ++u) {
      const int i = tid + u * kThreads;
      if (i >= items) break;
      const int row = i / quads, j = (i - row * quads) * 4;
      const int hr = cta * kOwn + row;
      const uint32_t off = (j >> 6) * (TML * 128) + hr * 128 + (((j & 63) >> 3 ^ (hr & 7)) << 4) + (j & 7) * 2;
#pragma unroll
      for (int q = 0; q < CL; ++q)
#pragma unroll
        for (int s = 0; s < kParts; ++s) st_cluster2(hs_at[q] + s * hpart + off, p[u][s]);
    }
  }
  asm volatile("fence.proxy.async;" ::: "memory");   // the tensor cores will read what was just stored
  cluster_arrive();                       // all parts of h are in place
  cluster_wait();
  asm volatile("fence.proxy.async;" ::: "memory");

  // ---- expand
  const __nv_bfloat16* B = reinterpret_cast<const __nv_bfloat16*>(a.b) + (int64_t)tl.adapter * a.N * a.R;
  const int bstage = kBN * ((a.R + 63) / 64 * 128);
  const uint32_t braw_u = raw_u + smem_b;
  const int piece = tid & 7, cfirst = tid >> 3 & 31;
  constexpr int kBi = kWarps / 8;         // groups of 32 columns the threads cover together
  const int ifirst = kBi == 1 ? 0 : tid >> 8;
  auto load_b = [&](const Block& at, int st) {
    if (at.slice >= 0) {
#pragma unroll
      for (int i = ifirst; i < kBN / 32; i += kBi) {
        // column q * 8 + 2 t + e of 32 is stored as row t * 8 + 2 q + e
        const int lc = cfirst, r = i * 32 + (lc >> 1 & 3) * 8 + (lc >> 3) * 2 + (lc & 1);
        const uint32_t dst = braw_u + st * bstage + r * 128 + ((piece ^ (r & 7)) << 4);
        const int col = at.c0 + i * 32 + lc;
        const __nv_bfloat16* src = B + (int64_t)col * a.R;
        for (int kb = 0; kb < rp; kb += 64) {
          const int k = kb + piece * 8;
          const bool on = col < at.end && k < rank;
          if (k < rp) cp_async16(dst + kb * (kBN * 2), on ? src + k : B, on);
        }
      }
    }
    cp_async_commit();
  };
  // past the rank nothing counts, not even a NaN: the piece the rank ends in
  auto trim_b = [&](int st) {
    if ((rank & 7) == 0 || piece != (rank >> 3 & 7)) return;
#pragma unroll
    for (int i = ifirst; i < kBN / 32; i += kBi) {
      const int lc = cfirst, r = i * 32 + (lc >> 1 & 3) * 8 + (lc >> 3) * 2 + (lc & 1);
      uint16_t* p = reinterpret_cast<uint16_t*>(raw + smem_b + st * bstage + (rank >> 6) * (kBN * 128) + r * 128 + ((piece ^ (r & 7)) << 4));
      for (int e = rank & 7; e < 8; ++e) p[e] = 0;
    }
  };
  int row0 = tile_rows[wrow + g], row1 = tile_rows[wrow + g + 8];
  const int es = F32 ? 4 : 2;
  // used where the row exists
  const char* base0 = reinterpret_cast<const char*>(a.base) + ((int64_t)row0 * a.ldb + half * 64 + 8 * c) * es;
  const char* base1 = reinterpret_cast<const char*>(a.base) + ((int64_t)row1 * a.ldb + half * 64 + 8 * c) * es;
  char* out0 = reinterpret_cast<char*>(a.out) + ((int64_t)row0 * a.ldo + half * 64 + 8 * c) * es;
  char* out1 = reinterpret_cast<char*>(a.out) + ((int64_t)row1 * a.ldo + half * 64 + 8 * c) * es;
  const uint32_t idesc = idesc_bf16_f32(TML, kBN);
  const uint32_t hs_u = smem_u32(hs);
  auto load_base = [&](const Block& at, BaseCols<F32> (&bs)[2][2]) {
    if (at.slice < 0) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (at.c0 + half * 64 + h * 32 + 8 * c < at.end) {
        if (row0 >= 0) bs[h][0].load(base0 + (int64_t)(at.c0 + h * 32) * es);
        if (row1 >= 0) bs[h][1].load(base1 + (int64_t)(at.c0 + h * 32) * es);
      }
    }
  };
  // block `it` has been copied by every thread: its product into accumulator it % 2
  auto multiply = [&](const Block& at, int it) {
    trim_b(it & 1);
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (warp == 0 && elect_one()) {
      tc_fence_after();
      const uint32_t bst = braw_u + (it & 1) * bstage;
      uint32_t on = 0;
      for (int q = 0; q < kParts; ++q)
        for (int k = 0; k < rp; k += 16) {
          const int hc = at.slice * rp + k;
          const uint64_t hd = sw128_kmajor_desc(hs_u + q * hpart + (hc >> 6) * (TML * 128)) + ((hc & 63) >> 3);
          const uint64_t bd = sw128_kmajor_desc(bst + (k >> 6) * (kBN * 128)) + ((k & 63) >> 3);
          umma_f16_ss(tmem + (it & 1) * kBN, hd, bd, idesc, on);
          on = 1;
        }
      umma_commit(&done[it & 1]);
    }
    __syncwarp();
  };
  // While block `it` is added to base and written, the product of the next one runs
  // and the copy of the one after it is under way.
  const bool shrunk = ok;
  int block = ok ? cta : a.block128[kMaxSlices];
  Block at = column_block<kBN>(a, block), next = column_block<kBN>(a, block + CL);
  BaseCols<F32> bs[2][2], bs_next[2][2];
  load_b(at, 0);
  load_b(next, 1);
  load_base(at, bs);
  if (at.slice >= 0) {
    cp_async_wait<1>();
    multiply(at, 0);
  }
  for (int it = 0; at.slice >= 0; ++it) {
    load_base(next, bs_next);
    if (next.slice >= 0) {
      cp_async_wait<0>();
      multiply(next, it + 1);             // its accumulator was read before this barrier
    }
    if (!arrived(&done[it & 1], (it >> 1) & 1, 42, !ok)) {
      ok = false;                         // what follows is void and is not written
      row0 = row1 = -1;
    }
    __syncwarp();
    tc_fence_after();
    block += CL;
    const Block after = column_block<kBN>(a, block + CL);
    load_b(after, it & 1);                // block `it` has been multiplied: its stage is free
    uint32_t acc[32];
    tmem_ld_16x256b_x8(tmem_row + (it & 1) * kBN + half * 64, acc);
    tmem_wait_ld();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (at.c0 + half * 64 + h * 32 + 8 * c >= at.end) continue;
      const int64_t off = (int64_t)(at.c0 + h * 32) * es;
      float d[8];
      if (row0 >= 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          d[2 * t] = rp ? __uint_as_float(acc[(h * 4 + t) * 4]) : 0.f, d[2 * t + 1] = rp ? __uint_as_float(acc[(h * 4 + t) * 4 + 1]) : 0.f;
        bs[h][0].store(out0 + off, d, tl.scale);
      }
      if (row1 >= 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          d[2 * t] = rp ? __uint_as_float(acc[(h * 4 + t) * 4 + 2]) : 0.f, d[2 * t + 1] = rp ? __uint_as_float(acc[(h * 4 + t) * 4 + 3]) : 0.f;
        bs[h][1].store(out1 + off, d, tl.scale);
      }
    }
    at = next;
    next = after;
#pragma unroll
    for (int h = 0; h < 2; ++h) bs[h][0] = bs_next[h][0], bs[h][1] = bs_next[h][1];
  }
  cp_async_wait<0>();
  tc_fence_before();
  if (!__syncthreads_and(ok)) {
    if (warp == 0 && elect_one()) umma_commit(&rest);
    drained(&rest, shrunk ? 0 : 1);
    __syncthreads();
  }
  if (warp == 0) tmem_dealloc(tmem, kTmemCols);
}

void set_blocks(LoraArgs& a) {
  a.block32[0] = a.block128[0] = 0;
  for (int i = 0; i < kMaxSlices; ++i) {
    const int width = i < a.S ? a.col_begin[i + 1] - a.col_begin[i] : 0;
    a.block32[i + 1] = a.block32[i] + (width + 31) / 32;
    a.block128[i + 1] = a.block128[i] + (width + 127) / 128;
  }
}

// The small kernel's time grows with the products of its tiles on mma.sync, the
// large one's with the CTAs' trips over K and with the weights that its tiles
// read, whatever the rank.  Tiles are estimated from the number of listed rows and
// of adapters, which is all the host knows.  Over 390 random calls (up to 4096 rows,
// K 512 to 14336, N 768 to 10240, ranks 8 to 128, 1 to 128 adapters) the choice
// costs 1.1 % over the better one in the mean, 50 % at most; large tiles from 768
// rows cost 7.9 % and up to six times.  Small / large, bf16, eight adapters, K = 4096,
// three slices of together 6144 columns: rank 64, 128 rows 19.5 / 25.7 us, 384 rows
// 29.9 / 28.0, 2048 rows 56.9 / 45.4; rank 16, 2048 rows 24.2 / 38.7.
bool use_large(const LoraArgs& a) {
  if ((int64_t)a.pool * a.S * a.R > INT32_MAX) return false;   // rows of A are 32-bit coordinates
  const double small_tiles = (a.L + kSmallRows - 1) / kSmallRows, large_tiles = a.L / 64 + std::min(a.L, a.pool);
  const double work = small_tiles * a.R * ((double)a.S * a.K + (a.f32 ? 3.0 : 2.0) * a.N);
  return work >= 155.0 * (32.0 * a.K + large_tiles * ((double)a.K + a.N));
}

// Clusters of `cl` CTAs of a kernel that run at once.  GPCs hold different
// numbers of SMs, so the device is asked, once per kernel, size and CTAs per SM.
template <typename Kernel>
int clusters_at_once(Kernel kernel, int threads, int cl, size_t smem, std::atomic<int> (&known)[64][2][kCluster + 1]) {
  const int pair = threads == kThreads && 2 * (smem + 2048) <= 228 * 1024 ? 1 : 0;   // two CTAs share an SM
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  if (cl == 1) return (1 + pair) * sm_count();
  if (dev < 64 && (n = known[dev][pair][cl].load(std::memory_order_relaxed)) > 0) return n;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cl;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cl);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
  if (e != cudaSuccess) launch_failed(e);
  n = std::max(n, 1);
  if (dev < 64) known[dev][pair][cl].store(n, std::memory_order_relaxed);
  return n;
}

// CTAs per tile of the small kernel: as many as possible while the tiles still run in
// the fewest waves, a wave costing about 6 us and, per CTA, 24 KB of weights a
// microsecond.  The tiles are those of evenly used adapters.  64 adapters with a row
// each, rank 16: clusters of 8 18.5 us, 6 22.6, 5 23.9, 4 14.7, 2 19.8; 512 rows of 20
// adapters (40 tiles, K = N = 4096): 8 13.8, 6 8.9, 4 10.0, 2 12.3; one tile: 8 8.0, 4 10.0,
// 2 14.0.  Uneven use misleads it: 256 rows of 32 among 48 adapters (36 tiles, taken for 48,
// K = 14336) run in clusters of 5, 24.9 us; 6 would take 22.8, 8 24.7, 4 26.5.
template <typename AtOnce>
int cluster_size(const LoraArgs& a, AtOnce at_once) {
  const int64_t adapters = std::min(a.L, a.pool);
  const int64_t tiles = adapters * ((a.L + kSmallRows * adapters - 1) / (kSmallRows * adapters));
  const int64_t bytes = 2 * (int64_t)a.R * ((int64_t)a.S * a.K + a.N);
  int best = 1;
  int64_t least = INT64_MAX;
  for (int cl = kCluster; cl >= 1; --cl) {
    const int64_t n = at_once(cl), cost = (tiles + n - 1) / n * (144 * 1024 + bytes / cl);
    if (cost < least) least = cost, best = cl;
  }
  return best;
}

template <bool F32, int MT, bool WIDE>
void launch_small(const LoraArgs& a, cudaStream_t s) {
  const int cols = (a.S * a.R + 15) / 16 * 16;
  const int parts = F32 ? 3 : 2;
  const size_t smem = (size_t)small_units<F32, MT, WIDE>() * kThreads * 16 + sizeof(float) * kSmallRows * cols + (size_t)2 * parts * kSmallRows * (cols + 40);
  auto k = lora_small_kernel<F32, MT, WIDE>;
  static std::atomic<unsigned long long> allowed{0};
  allow_smem(reinterpret_cast<const void*>(k), allowed);
  const int tiles = a.L / kSmallRows + std::min(a.L, a.pool);   // at least the sum of ceil(rows / 16) over the adapters
  static std::atomic<int> at_once[64][2][kCluster + 1];
  const int cl = cluster_size(a, [&](int c) { return clusters_at_once(k, kThreads, c, smem, at_once); });
  // one_row() keeps its share of x and h in the same shared memory
  const int64_t span = (((a.K + 31) / 32 + cl - 1) / cl * 32 + 255) / 256 * 256;
  const bool vector = (a.R & (a.R - 1)) == 0 && (span + 2 * cols) * 4 <= (int64_t)smem;
  launch_k(k, dim3((unsigned)(tiles * cl)), dim3(kThreads), smem, s, (unsigned)cl, a, cols, cl, vector);
}

// MT: 16-column tiles of h a warp accumulates at a time, no more than there are
// (256 rows, rank 16 and one slice: 7.5 us, 8.8 with four).  WIDE: steps of 32 along
// the rank, half as many trips over the same bytes (256 rows of rank 64: 23.7 us, 26.2
// with steps of 16), which the rank has to be a multiple of.
template <bool F32>
void small(const LoraArgs& a, cudaStream_t s) {
  const int cols = a.S * a.R;
  if (a.R % 32 == 0) {
    if (cols <= 32) launch_small<F32, 2, true>(a, s);
    else launch_small<F32, 4, true>(a, s);
  } else {
    if (cols <= 16) launch_small<F32, 1, false>(a, s);
    else if (cols <= 48) launch_small<F32, 3, false>(a, s);
    else launch_small<F32, 4, false>(a, s);
  }
}

template <bool F32, int TML, int CL>
struct Large {
  LargeSmem sm;
  int tiles, likely, cols;   // at most and as a rule
  explicit Large(const LoraArgs& a)
      : sm(large_smem(TML, a.S * ((a.R + 15) / 16 * 16), a.R, F32 ? 3 : 2)),
        tiles(a.L / TML + std::min(a.L, a.pool)), likely(a.L / TML + (std::min(a.L, a.pool) + 1) / 2), cols(a.S * ((a.R + 15) / 16 * 16)) {
    static std::atomic<unsigned long long> allowed{0}, allowed_twin{0};
    allow_smem(reinterpret_cast<const void*>(lora_large_kernel<F32, TML, CL>), allowed);
    if (TML == 64) allow_smem(reinterpret_cast<const void*>(kTwin), allowed_twin);
  }
  // The device counts one CTA of a kernel with tensor memory per SM, although two of 64
  // rows do share one: it is asked about a kernel that is alike but for that.
  static constexpr auto kTwin = lora_small_kernel<F32, 4, true>;
  int waves() const {
    static std::atomic<int> at_once[64][2][kCluster + 1];
    const int n = TML == 64 ? clusters_at_once(kTwin, kThreads, CL, sm.total, at_once)
                            : clusters_at_once(lora_large_kernel<F32, TML, CL>, TML * 4, CL, sm.total, at_once);
    return (likely + n - 1) / n;
  }
  void launch(const LoraArgs& a, cudaStream_t s) const {
    const CUtensorMap map_a = gemm::make_tmap_2d(a.a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)a.pool * a.S_all * a.R, a.K,
                                                 a.K, kBoxRows, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    launch_k(lora_large_kernel<F32, TML, CL>, dim3((unsigned)tiles * CL), dim3(TML * 4), sm.total, s, (unsigned)CL, a, map_a, cols,
             (int)sm.b, (int)sm.total - 1024);
  }
};

// Tile and cluster by the number of waves and what one takes (us, ranks up to 64 beside
// the QKV projection, K = 4096, N = 6144): 64 rows in clusters of 8 26, 4 45 (of 2 92, no
// better than two waves of 4); 128 rows in clusters of 4 43, 2 76.  The ratios are taken for
// every K, N and rank; other shapes were not measured.
template <bool F32>
void launch_large(const LoraArgs& a, cudaStream_t s) {
  const Large<F32, 64, 8> a8(a);
  const Large<F32, 64, 4> a4(a);
  const Large<F32, 128, 4> b4(a);
  const Large<F32, 128, 2> b2(a);
  const int64_t us[4] = {26LL * a8.waves(), 45LL * a4.waves(), 43LL * b4.waves(), 76LL * b2.waves()};
  const int best = (int)(std::min_element(us, us + 4) - us);
  if (best == 0) a8.launch(a, s);
  else if (best == 1) a4.launch(a, s);
  else if (best == 2) b4.launch(a, s);
  else b2.launch(a, s);
}

// As many slices per launch as an accumulator (256 columns) and shared memory hold.
template <bool F32>
int large(const LoraArgs& all, cudaStream_t s) {
  int launches = 0;
  const int rp = (all.R + 15) / 16 * 16;
  int step = std::min(all.S, kLargeCols / rp);
  while (step > 1 && large_smem(128, step * rp, all.R, F32 ? 3 : 2).total > kLargeSmem) --step;
  for (int s0 = 0; s0 < all.S; s0 += step) {
    LoraArgs a = all;
    a.s0 = s0;
    a.S = std::min(step, all.S - s0);
    for (int i = 0; i <= kMaxSlices; ++i) a.col_begin[i] = all.col_begin[std::min(s0 + std::min(i, a.S), all.S)];
    set_blocks(a);
    launch_large<F32>(a, s);
    ++launches;
  }
  return launches;
}

}  // namespace

int lora_add(const LoraArgs& args, cudaStream_t s) {
  if (args.L <= 0 || args.N <= 0 || args.pool <= 0) return 0;
  LoraArgs a = args;
  a.s0 = 0;
  a.S_all = a.S;
  set_blocks(a);
  if (use_large(a)) return a.f32 ? large<true>(a, s) : large<false>(a, s);
  a.f32 ? small<true>(a, s) : small<false>(a, s);
  return 1;
}

}  // namespace lora
}  // namespace lf
