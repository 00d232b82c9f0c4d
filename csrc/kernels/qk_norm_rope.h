#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace lf {
namespace ew {

struct QkNormRopeArgs {
  const void* qkv;            // [T, (Hq + 2 Hkv) * D] bf16, row stride ld
  int64_t ld;
  void* q_out;                // [T, Hq * D] bf16, row stride q_ld; may be the Q columns of qkv themselves
  int64_t q_ld;
  const void* q_weight;       // [D] bf16
  const void* k_weight;       // [D] bf16
  const int32_t* positions;   // [T]
  const int32_t* slots;       // [T]; negative: no K / V write
  const void* cos_sin;        // [max_pos, D / 2] float2
  void* kcache;               // [pages][Hkv][page][D] bf16
  void* vcache;
  int T, Hq, Hkv, D, page, max_pos;
  int64_t num_slots;
  float eps;
};

bool qk_norm_rope_supported(int D);   // head sizes with a compiled kernel
void qk_norm_rope_kv_write(const QkNormRopeArgs& a, cudaStream_t s);

}  // namespace ew
}  // namespace lf
