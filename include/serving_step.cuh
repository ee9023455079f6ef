// C++ launchers of the serving-step operators around the paged decode, in the style of
// paged_attention.cuh: thin, typed forms of the C entries of flash_engine_c.h, which state
// the operators' contracts. New: the reference has none of these.
#pragma once

#include <cuda_runtime.h>

#include "flash_engine_c.h"

namespace flash_engine {
namespace serving {

// Element types and cache layouts as the C entries number them.
enum class DType : int { kBf16 = 0, kFp16 = 1, kFp32 = 2 };
enum class KvLayout : int { kFlat = 0, kVllm = 1 };

struct StepPlanConfig {
  int num_seqs, max_num_blocks_per_seq, num_blocks, block_size, max_tokens;
};

// A paged cache: [num_blocks, num_kv_heads, block_size, head_dim] (flat).
struct CacheConfig {
  int num_blocks, num_kv_heads, head_dim, block_size;
  DType dtype = DType::kBf16;
  KvLayout layout = KvLayout::kFlat;
};

struct RopeTables {
  const float* cos = nullptr;  // [max_pos, rotary_dim / 2]; nullptr = no rotation
  const float* sin = nullptr;
  int rotary_dim = 0, max_pos = 0;
  bool interleaved = true;
};

inline cudaError_t launch_plan_paged_step(
    const int* d_context_lens, const int* d_new_lens, const unsigned char* d_finished,
    int* d_block_tables, int* d_free_blocks, const int* d_free_state, int* d_context_lens_out,
    int* d_cu_seqlens, int* d_positions, long long* d_slots, int* d_free_state_out,
    const StepPlanConfig& c, cudaStream_t stream = nullptr) {
  return static_cast<cudaError_t>(fe_plan_paged_step(
      d_context_lens, d_new_lens, d_finished, d_block_tables, d_free_blocks, d_free_state,
      d_context_lens_out, d_cu_seqlens, d_positions, d_slots, d_free_state_out, c.num_seqs,
      c.max_num_blocks_per_seq, c.num_blocks, c.block_size, c.max_tokens, stream));
}

// weights_fp32: the norm weights are fp32, not the cache's type; nullptr weights = no norm.
inline cudaError_t launch_paged_qkv_append(const void* d_qkv, long long row_stride, void* d_q_out,
                                           void* d_key_cache, void* d_value_cache,
                                           const int* d_positions, const long long* d_slots,
                                           const void* d_q_weight, const void* d_k_weight,
                                           bool weights_fp32, float eps, const RopeTables& rope,
                                           int num_tokens, int num_heads, const CacheConfig& c,
                                           cudaStream_t stream = nullptr) {
  return static_cast<cudaError_t>(fe_paged_qkv_append(
      d_qkv, row_stride, d_q_out, d_key_cache, d_value_cache, d_positions, d_slots, d_q_weight,
      d_k_weight, weights_fp32 ? 1 : 0, eps, rope.cos, rope.sin, rope.rotary_dim, rope.max_pos,
      rope.interleaved ? 1 : 0, num_tokens, num_heads, c.num_kv_heads, c.head_dim, c.block_size,
      c.num_blocks, static_cast<int>(c.dtype), static_cast<int>(c.layout), stream));
}

inline cudaError_t launch_update_page_bounds(const void* d_key_cache, signed char* d_values,
                                             float* d_scales, const long long* d_slots,
                                             int num_tokens, const CacheConfig& c,
                                             cudaStream_t stream = nullptr) {
  return static_cast<cudaError_t>(fe_update_page_bounds(
      d_key_cache, d_values, d_scales, d_slots, num_tokens, c.num_kv_heads, c.head_dim,
      c.block_size, c.num_blocks, static_cast<int>(c.dtype), static_cast<int>(c.layout), stream));
}

// d_scratch: fe_sparse_paged_attention_scratch_ints(...) ints. scale <= 0: 1 / sqrt(head_dim).
inline cudaError_t launch_sparse_paged_attention(
    const void* d_query, const void* d_key_cache, const void* d_value_cache, void* d_output,
    const signed char* d_values, const float* d_scales, const int* d_block_tables,
    const int* d_context_lens, int* d_selected, int* d_scratch, int num_seqs, int num_heads,
    int max_num_blocks_per_seq, int num_pages, int keep_first, int keep_last, float scale,
    const CacheConfig& c, float* d_workspace = nullptr,
    size_t workspace_floats = FE_WORKSPACE_LIBRARY, cudaStream_t stream = nullptr) {
  return static_cast<cudaError_t>(fe_sparse_paged_attention(
      d_query, d_key_cache, d_value_cache, d_output, d_values, d_scales, d_block_tables,
      d_context_lens, d_selected, d_scratch, num_seqs, num_heads, c.num_kv_heads, c.head_dim,
      c.block_size, max_num_blocks_per_seq, c.num_blocks, num_pages, keep_first, keep_last, scale,
      static_cast<int>(c.dtype), static_cast<int>(c.layout), d_workspace, workspace_floats,
      stream));
}

}  // namespace serving
}  // namespace flash_engine
