// RMS norm of every query and key head, split-half rotation and the paged
// K / V write in one pass over the QKV projection's output.
//
//   y = x * rsqrt(mean_d(x^2) + eps) * w        (w: one [D] weight for Q, one for K)
//   o[i]       = y[i] cos_i - y[i + D/2] sin_i
//   o[i + D/2] = y[i + D/2] cos_i + y[i] sin_i   (i < D/2, angles of the token's position)
//
// V heads are copied.  All arithmetic is fp32 with one rounding to bf16 at the
// store; the sum of squares of a head stays in registers.
//
// Bound by memory: every head is read once and written once.  D / 16 lanes own
// one head, each 16 bytes of its first half and the 16 bytes D / 2 further on, so
// both elements of a rotation pair lie in one lane and the sum of squares takes
// three shuffles for 16 elements: no shared memory and no barrier.  A CTA owns one
// token; its lanes load the token's (cos, sin) row and the two weights once and
// keep them while they walk the heads.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <stdexcept>

#include "common.cuh"
#include "qk_norm_rope.h"

namespace lf {
namespace ew {

namespace {

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(p[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}

// Heads whose loads are in flight together per lane group.
constexpr int kBatch = 3;

template <int D, int NT>
__global__ void __launch_bounds__(NT) qk_norm_rope_kernel(const QkNormRopeArgs a) {
  constexpr int kLanes = D / 16;         // lanes of one head
  constexpr int kHalf = D / 16;          // 16-byte pieces of half a head
  constexpr int kGroups = NT / kLanes;   // heads a CTA works on at a time
  pdl_wait();
  const int t = blockIdx.x;
  const int group = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
  const int heads = a.Hq + 2 * a.Hkv;
  const uint4* row = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.qkv) + (int64_t)t * a.ld) + l;
  uint4 v[kBatch][2];
  auto load = [&](int h0) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * kGroups;
      if (h < heads) {
        v[b][0] = row[h * 2 * kHalf];
        v[b][1] = row[h * 2 * kHalf + kHalf];
      } else {
        v[b][0] = v[b][1] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  const int pos = a.positions[t];
  const int slot = a.slots[t];
  load(group);                           // under way before the position is known
  const uint4* wq = reinterpret_cast<const uint4*>(a.q_weight) + l;
  const uint4* wk = reinterpret_cast<const uint4*>(a.k_weight) + l;
  const uint4 wq0 = wq[0], wq1 = wq[kHalf], wk0 = wk[0], wk1 = wk[kHalf];
  const bool pos_ok = pos >= 0 && pos < a.max_pos;
  const bool slot_ok = slot >= 0 && (int64_t)slot < a.num_slots;

  float cs[8], sn[8];
  {
    // a position outside the table is recorded and not rotated
    const float4* tab = reinterpret_cast<const float4*>(a.cos_sin) + ((int64_t)(pos_ok ? pos : 0) * (D / 2) + l * 8) / 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = pos_ok ? tab[i] : make_float4(1.f, 0.f, 1.f, 0.f);
      cs[2 * i] = x.x;
      sn[2 * i] = x.y;
      cs[2 * i + 1] = x.z;
      sn[2 * i + 1] = x.w;
    }
  }
  if (threadIdx.x == 0 && (!pos_ok || (slot >= 0 && !slot_ok))) set_error(kErrBadIndex, (unsigned long long)t);

  const int64_t pg = slot_ok ? slot / a.page : 0;
  const int off = slot_ok ? slot % a.page : 0;
  uint4* qrow = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.q_out) + (int64_t)t * a.q_ld) + l;
  uint4* krow = reinterpret_cast<uint4*>(a.kcache) + (pg * a.Hkv * a.page + off) * 2 * kHalf + l;
  uint4* vrow = reinterpret_cast<uint4*>(a.vcache) + (pg * a.Hkv * a.page + off) * 2 * kHalf + l;

  for (int h0 = group; h0 - group < heads; h0 += kBatch * kGroups) {   // uniform trip count over the CTA
    if (h0 != group) load(h0);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * kGroups;
      if (h - group >= heads) break;     // uniform: no lane group of this CTA has such a head
      if (__all_sync(0xffffffffu, h >= a.Hq + a.Hkv)) {   // V heads only (or none)
        if (h < heads && slot_ok) {
          uint4* dst = vrow + (int64_t)(h - a.Hq - a.Hkv) * a.page * 2 * kHalf;
          dst[0] = v[b][0];
          dst[kHalf] = v[b][1];
        }
        continue;
      }
      float x[8], y[8], w[8];
      unpack8(v[b][0], x);
      unpack8(v[b][1], y);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
      for (int m = kLanes / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
      const float inv = rsqrtf(ss * (1.f / D) + a.eps);
      unpack8(h < a.Hq ? wq0 : wk0, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i];
      unpack8(h < a.Hq ? wq1 : wk1, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * w[i];
      float o[8], p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o[i] = x[i] * cs[i] - y[i] * sn[i];
        p[i] = y[i] * cs[i] + x[i] * sn[i];
      }
      if (h < a.Hq) {
        qrow[h * 2 * kHalf] = pack8(o);
        qrow[h * 2 * kHalf + kHalf] = pack8(p);
      } else if (h < heads && slot_ok) {
        const bool is_k = h < a.Hq + a.Hkv;
        uint4* dst = (is_k ? krow : vrow) + (int64_t)(h - a.Hq - (is_k ? 0 : a.Hkv)) * a.page * 2 * kHalf;
        dst[0] = is_k ? pack8(o) : v[b][0];
        dst[kHalf] = is_k ? pack8(p) : v[b][1];
      }
    }
  }
}

// Few tokens (two per SM at most) are bound by latency: 256 threads each, so that a
// head group has one or two heads.  Many are bound by memory: 64 threads, whose 1 KB
// rounds of loads and stores interleave best.  In between 128 threads would be better;
// the rule ignores that.  us, head_dim 128, 64 / 128 / 256 threads:
//
//   tokens        256               300               600                1023               2000                8192
//   32 + 8 heads  3.2 / 2.7 / 2.8   3.5 / 3.1 / 3.7   5.0 / 4.2 / 6.3    7.5 / 8.2 / 11.1   12.4 / 12.5 / 18.7  36.9 / 40.6 / 67.2
//   64 + 8 heads  5.2 / 4.0 / 3.4   6.2 / 4.4 / 4.8   9.3 / 7.4 / 8.8   11.2 / 11.7 / 13.6  19.3 / 18.2 / 23.0
template <int D>
void launch_d(const QkNormRopeArgs& a, cudaStream_t s) {
  if (a.T <= 2 * sm_count()) launch_k(qk_norm_rope_kernel<D, 256>, dim3(a.T), dim3(256), 0, s, 1, a);
  else launch_k(qk_norm_rope_kernel<D, 64>, dim3(a.T), dim3(64), 0, s, 1, a);
}

}  // namespace

bool qk_norm_rope_supported(int D) { return D == 64 || D == 128 || D == 256; }

void qk_norm_rope_kv_write(const QkNormRopeArgs& a, cudaStream_t s) {
  if (a.T <= 0) return;
  if (a.D == 64) launch_d<64>(a, s);
  else if (a.D == 128) launch_d<128>(a, s);
  else if (a.D == 256) launch_d<256>(a, s);
  else throw std::runtime_error("lunaflux qk_norm_rope: head_dim 64, 128 or 256");
}

}  // namespace ew
}  // namespace lf
