#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace lf {
namespace attn {

constexpr int kSparseMaxPages = 65536;   // pages of one row (1 Mi tokens): the selection's bit mask in shared memory

struct BoundsArgs {
  const __nv_bfloat16* kcache;   // [pages, Hkv, 16, 128]
  __nv_bfloat16* bounds;         // [pages, Hkv, 2, 128]: smallest, largest key per dimension
  const int32_t* block_table;    // [rows, bt_stride]
  int64_t bt_stride;
  const int32_t* start;          // [rows] first new token
  const int32_t* seq_lens;       // [rows] tokens with the new ones
  int rows, Hkv, width, num_pages;
  int max_new;                   // most new tokens of a row
  int max_pages;                 // pages they can touch (set at the launch)
};

struct SelectArgs {
  const __nv_bfloat16* q;        // token rows, Q heads first; row stride q_ld
  int64_t q_ld;
  const int32_t* tok_index;      // [rows]
  const int32_t* seq_lens;       // [rows]
  const int32_t* block_table;    // [rows, bt_stride]
  int64_t bt_stride;
  const __nv_bfloat16* bounds;   // [pages, Hkv, 2, 128]
  int32_t* sel;                  // [rows, Hkv, budget] logical pages, ascending, then -1
  float2* ws;                    // [rows, Hkv, width] (score, error bound) of every page
  int rows, Hq, Hkv, width, num_pages, tokens, budget, first, last;
};

struct SparseArgs {
  const __nv_bfloat16* q;
  int64_t q_ld;
  __nv_bfloat16* out;            // [T, Hq * 128]; row stride out_ld
  int64_t out_ld;
  const int32_t* tok_index;
  const int32_t* seq_lens;
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* sel;            // [rows, Hkv, budget]
  const __nv_bfloat16* kcache;
  const __nv_bfloat16* vcache;
  int rows, Hq, Hkv, width, num_pages, tokens, budget;
  float scale_log2;
};

void page_bounds(const BoundsArgs& a, cudaStream_t s);
int select_pages(const SelectArgs& a, cudaStream_t s);   // kernels launched
void decode_sparse(const SparseArgs& a, cudaStream_t s);

}  // namespace attn
}  // namespace lf
