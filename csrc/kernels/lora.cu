// Low-rank adapters of many requests beside a shared projection.
//
//   h[t]      = A[a(t)] x[t]                                     (rank values per slice)
//   out[t, c] = base[t, c] + scale[a] * sum_j B[a][c, j] h[t, slice(c) R + j]
//
// for the rows t listed in `rows`, grouped by adapter (`starts` is the CSR
// offset of every adapter of the pool).  Slices are the column ranges of a
// stacked projection (Q, K, V), each with its own A.  Sums are fp32, h is handed
// on as two bf16 parts (three for fp32 outputs), an error of at most 2^-16 (2^-24) of h,
// and the output is rounded once.
//
// A cluster of eight CTAs owns a tile of up to TM rows of one adapter: every
// CTA multiplies an eighth of K, the partial h (TM x S R fp32) are added
// through distributed shared memory in rank order, and every CTA expands an
// eighth of the columns.  So the whole operator is one launch without a
// workspace, x and the weights are read by one CTA each, and a result does not
// depend on the other rows of the call.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <stdexcept>

#include "common.cuh"
#include "lora.h"

namespace lf {
namespace lora {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kCluster = 8;
constexpr int kWarps = 8;
constexpr int TM = 16;                   // rows of a tile

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
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

// Splits v into PARTS bf16 values that add up to it.
template <int PARTS>
__device__ __forceinline__ void split_bf16(float v, __nv_bfloat16 (&p)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    p[i] = __float2bfloat16(v);
    v -= __bfloat162float(p[i]);
  }
}

template <bool F32>
__global__ void __launch_bounds__(kWarps * 32) lora_kernel(const LoraArgs a) {
  constexpr int kParts = F32 ? 3 : 2;
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ int tile_info[3];            // adapter, first entry of rows, valid rows
  __shared__ int tile_rows[TM];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const uint32_t rank_cta = cluster_rank();
  const int tile = blockIdx.x / kCluster;
  const int SR = a.S * a.R;
  const int SRp = (SR + 15) / 16 * 16;    // whole 16-row tiles of A
  float* part = reinterpret_cast<float*>(raw);              // [SRp][TM] this CTA's partial h
  float* red = part + SRp * TM;                             // [kWarps][16][TM]
  __nv_bfloat16* hs = reinterpret_cast<__nv_bfloat16*>(red + kWarps * 16 * TM);   // [kParts][TM][SRp + 8]
  const int hld = SRp + 8;

  // the tile's adapter: a scan over the tiles of every adapter of the pool
  if (warp == 0) {
    int before = 0, found = -1, first = 0, valid = 0;
    bool bad = false;
    for (int b0 = 0; b0 < a.pool && found < 0; b0 += 32) {
      const int ad = b0 + lane;
      int s0 = 0, s1 = 0;
      if (ad < a.pool) s0 = a.starts[ad], s1 = a.starts[ad + 1];
      if (s0 < 0 || s1 < s0 || s1 > a.L) bad = true, s0 = s1 = 0;
      const int tiles = (s1 - s0 + TM - 1) / TM;
      int incl = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += v;
      }
      const bool mine = before + incl > tile && before + incl - tiles <= tile;
      const uint32_t m = __ballot_sync(kFull, mine);
      if (m) {
        const int src = __ffs(m) - 1;
        const int j = tile - (before + incl - tiles);
        found = b0 + src;
        first = __shfl_sync(kFull, s0 + j * TM, src);
        valid = __shfl_sync(kFull, min(TM, s1 - s0 - j * TM), src);
      }
      before += __shfl_sync(kFull, incl, 31);
    }
    if (__any_sync(kFull, bad) && lane == 0) set_error(kErrBadIndex, 0);
    if (lane == 0) tile_info[0] = found, tile_info[1] = first, tile_info[2] = valid;
    if (lane < TM) {
      int row = -1;
      if (found >= 0 && lane < valid) {
        row = a.rows[first + lane];
        if (row < 0 || row >= a.T) {
          set_error(kErrBadIndex, (unsigned long long)(first + lane));
          row = -1;
        }
      }
      tile_rows[lane] = row;
    }
  }
  __syncthreads();
  const int ad = tile_info[0];
  if (ad < 0) return;                     // past the last tile: the whole cluster leaves
  int rank = a.ranks[ad];
  if (rank < 0 || rank > a.R) {
    if (tid == 0) set_error(kErrBadIndex, (unsigned long long)ad);
    rank = 0;
  }
  const float scale = a.scales[ad];

  // shrink: h^T = A x^T over this CTA's eighth of K, the warps splitting it further
  const __nv_bfloat16* A = reinterpret_cast<const __nv_bfloat16*>(a.a) + (int64_t)ad * SR * a.K;
  const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x);
  const int r0 = tile_rows[g], r1 = tile_rows[g + 8];
  const __nv_bfloat16* x0 = r0 >= 0 ? x + (int64_t)r0 * a.ldx : nullptr;
  const __nv_bfloat16* x1 = r1 >= 0 ? x + (int64_t)r1 * a.ldx : nullptr;
  const int kblocks = (a.K + 31) / 32;
  const int per_cta = (kblocks + kCluster - 1) / kCluster;
  const int kb0 = (int)rank_cta * per_cta, kb1 = min(kblocks, kb0 + per_cta);
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int mt = 0; mt < SRp / 16; ++mt) {
    // rows of A past the adapter's rank in their slice count as zero and are not read
    const int j0 = mt * 16 + g, j1 = j0 + 8;
    const bool on0 = j0 < SR && j0 % a.R < rank, on1 = j1 < SR && j1 % a.R < rank;
    const __nv_bfloat16* A0 = A + (int64_t)j0 * a.K;
    const __nv_bfloat16* A1 = A + (int64_t)j1 * a.K;
    float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int kb = kb0 + warp; kb < kb1; kb += kWarps) {
      const int k = kb * 32 + c * 8;
      const bool in = k < a.K;            // K is a multiple of 8
      const uint4 va = in && on0 ? *reinterpret_cast<const uint4*>(A0 + k) : zero;
      const uint4 vb = in && on1 ? *reinterpret_cast<const uint4*>(A1 + k) : zero;
      const uint4 v0 = in && x0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
      const uint4 v1 = in && x1 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
      mma_bf16(acc[0], va.x, vb.x, va.y, vb.y, v0.x, v0.y);
      mma_bf16(acc[0], va.z, vb.z, va.w, vb.w, v0.z, v0.w);
      mma_bf16(acc[1], va.x, vb.x, va.y, vb.y, v1.x, v1.y);
      mma_bf16(acc[1], va.z, vb.z, va.w, vb.w, v1.z, v1.w);
    }
    float* rw = red + warp * 16 * TM;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      rw[g * TM + t * 8 + 2 * c] = acc[t][0];
      rw[g * TM + t * 8 + 2 * c + 1] = acc[t][1];
      rw[(g + 8) * TM + t * 8 + 2 * c] = acc[t][2];
      rw[(g + 8) * TM + t * 8 + 2 * c + 1] = acc[t][3];
    }
    __syncthreads();
    {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s += red[w * 16 * TM + tid];   // 256 threads = 16 x TM
      part[mt * 16 * TM + tid] = s;
    }
    __syncthreads();
  }
  cluster_sync_all();
  for (int i = tid; i < SRp * TM; i += kWarps * 32) {
    float v = 0.f;
    for (int q = 0; q < kCluster; ++q) v += ld_cluster(part + i, q);
    __nv_bfloat16 p[kParts];
    split_bf16<kParts>(v, p);
    const int j = i / TM, row = i % TM;
#pragma unroll
    for (int q = 0; q < kParts; ++q) hs[(q * TM + row) * hld + j] = p[q];
  }
  cluster_sync_all();                     // all partials are read, and hs is complete

  // expand: groups of 32 columns of one slice, dealt over the cluster's warps
  const __nv_bfloat16* B = reinterpret_cast<const __nv_bfloat16*>(a.b) + (int64_t)ad * a.N * a.R;
  const int rows_[2] = {r0, r1};
  int group = 0, begin = 0;
  for (int s = 0; s < a.S; ++s) {
    const int end = a.col_end[s];
    for (int c0 = begin; c0 < end; c0 += 32, ++group) {
      if (group % (kCluster * kWarps) != (int)rank_cta * kWarps + warp) continue;
      float acc[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
      for (int kb = 0; kb < rank; kb += 16) {
        const int k = kb + 4 * c;
        uint2 hv[kParts][2];
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
          // k past R (R a multiple of 8, not of 16) would be the next slice's h
          hv[q][0] = k < a.R ? *reinterpret_cast<const uint2*>(hs + (q * TM + g) * hld + s * a.R + k) : make_uint2(0u, 0u);
          hv[q][1] = k < a.R ? *reinterpret_cast<const uint2*>(hs + (q * TM + g + 8) * hld + s * a.R + k) : make_uint2(0u, 0u);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          // column n = g of tile t is column 8 (g / 2) + 2 t + g % 2 of the group:
          // a lane then ends up with eight consecutive columns
          const int col = c0 + (g >> 1) * 8 + 2 * t + (g & 1);
          uint2 bv = make_uint2(0u, 0u);
          if (col < end && k < rank) {
            bv = *reinterpret_cast<const uint2*>(B + (int64_t)col * a.R + k);
            if (k + 1 >= rank) bv.x &= 0xffffu;
            if (k + 2 >= rank) bv.y = 0u;
            else if (k + 3 >= rank) bv.y &= 0xffffu;
          }
#pragma unroll
          for (int q = 0; q < kParts; ++q) mma_bf16(acc[t], hv[q][0].x, hv[q][1].x, hv[q][0].y, hv[q][1].y, bv.x, bv.y);
        }
      }
      const int col = c0 + 8 * c;
      if (col >= end) continue;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (rows_[u] < 0) continue;
        float d[8];
#pragma unroll
        for (int t = 0; t < 4; ++t) d[2 * t] = scale * acc[t][2 * u], d[2 * t + 1] = scale * acc[t][2 * u + 1];
        if (F32) {
          const float4* bp = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.base) + (int64_t)rows_[u] * a.ldb + col);
          float4* op = reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + (int64_t)rows_[u] * a.ldo + col);
          const float4 b0 = bp[0], b1 = bp[1];
          op[0] = make_float4(b0.x + d[0], b0.y + d[1], b0.z + d[2], b0.w + d[3]);
          op[1] = make_float4(b1.x + d[4], b1.y + d[5], b1.z + d[6], b1.w + d[7]);
        } else {
          const uint4 bv = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.base) + (int64_t)rows_[u] * a.ldb + col);
          const __nv_bfloat162* b2 = reinterpret_cast<const __nv_bfloat162*>(&bv);
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(b2[i]);
            o[i] = pack_bf16x2(f.x + d[2 * i], f.y + d[2 * i + 1]);
          }
          *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.out) + (int64_t)rows_[u] * a.ldo + col) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    }
    begin = end;
  }
}

}  // namespace

void lora_add(const LoraArgs& a, cudaStream_t s) {
  if (a.L <= 0 || a.N <= 0 || a.pool <= 0) return;
  const int SRp = (a.S * a.R + 15) / 16 * 16;
  const int parts = a.f32 ? 3 : 2;
  const size_t smem = sizeof(float) * (SRp * TM + kWarps * 16 * TM) + (size_t)2 * parts * TM * (SRp + 8);
  const int tiles = a.L / TM + (a.L < a.pool ? a.L : a.pool);   // sum of ceil(rows / TM) over the adapters
  auto k = a.f32 ? lora_kernel<true> : lora_kernel<false>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) launch_failed(e);
  }
  launch_k(k, dim3((unsigned)tiles * kCluster), dim3(kWarps * 32), smem, s, (unsigned)kCluster, a);
}

}  // namespace lora
}  // namespace lf
