#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace lf {
namespace lora {

constexpr int kMaxSlices = 4;
constexpr int kMaxRank = 128;

struct LoraArgs {
  const void* x;              // [T, K] bf16, row stride ldx
  int64_t ldx;
  const void* a;              // [pool, S * R, K] bf16
  const void* b;              // [pool, N, R] bf16
  const float* scales;        // [pool]
  const int32_t* ranks;       // [pool], <= R
  const int32_t* rows;        // [L] token rows grouped by adapter, each at most once
  const int32_t* starts;      // [pool + 1] offsets into rows
  const void* base;           // [T, N] bf16 or fp32, row stride ldb; may be out itself
  int64_t ldb;
  void* out;                  // [T, N], row stride ldo
  int64_t ldo;
  int T, K, N, R, pool, L, S;
  int col_begin[kMaxSlices + 1];   // first column of every slice, then N
  // set at the launch: first slice and slices of lora_a (a launch may take some of
  // them), blocks of 32 / 128 columns before every slice
  int s0, S_all;
  int block32[kMaxSlices + 1];
  int block128[kMaxSlices + 1];
  bool f32;                   // base and out are fp32
};

int lora_add(const LoraArgs& a, cudaStream_t s);   // kernels launched

}  // namespace lora
}  // namespace lf
