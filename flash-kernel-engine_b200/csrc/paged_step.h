// Internal interface of the serving-step kernels around the paged decode: the step plan
// (paged_plan.cu), the QKV append (qkv_append.cu), the page boxes (page_bounds.cu) and the
// sparse decode (sparse_decode.cu). Element types are numbered as in
// paged_decode.h (DecodeType), cache layouts as KvLayout.
#pragma once

#include <cuda_runtime.h>

namespace fe {
namespace step {

// Largest request count of one plan (its prefix sums stay in shared memory) and the
// largest token / block count (32-bit saturating sums).
constexpr int kMaxPlanSeqs = 16384;
constexpr int kMaxPlanCount = 1 << 30;

struct PlanParams {
  const int* context_lens;        // [S] tokens each request holds
  const int* new_lens;            // [S] tokens it adds in this step
  const unsigned char* finished;  // [S] or null: requests whose blocks go back first
  int* block_tables;              // [S, width], extended in place
  int* free_blocks;               // ring [num_blocks]
  const int* state;               // (head, count) of the ring
  int* context_lens_out;          // [S]
  int* cu_seqlens;                // [S + 1]
  int* positions;                 // [max_tokens], -1 past the step's tokens
  long long* slots;               // [max_tokens], -1 past the step's tokens
  int* state_out;                 // (head, count, requests served, tokens)
  int num_seqs, width, num_blocks, block_size, max_tokens;
  unsigned* err;
};
cudaError_t launch_plan(const PlanParams& p, cudaStream_t stream);

struct QkvParams {
  const void* qkv;  // [T, (H + 2 Hkv) d], rows row_stride elements apart
  void* q_out;      // [T, H, d]
  void* k_cache;
  void* v_cache;
  const int* positions;
  const long long* slots;
  const void* q_weight;  // [d] or null (no norm); fp32 if weight_f32, else the data's type
  const void* k_weight;
  const float* rope_cos;  // [rope_max_pos, rotary_dim / 2] or null
  const float* rope_sin;
  long long row_stride;
  float eps;
  int tokens, heads, kv_heads, head_dim, block_size, num_blocks;
  int rotary_dim, rope_max_pos, interleaved, weight_f32, kv_layout;
  unsigned* err;
};
cudaError_t launch_qkv_append(const QkvParams& p, int dtype, cudaStream_t stream);

struct BoundsParams {
  const void* k_cache;
  signed char* values;     // [num_blocks, Hkv, 2, d]: largest, then smallest, per channel
  float* scales;           // [num_blocks, Hkv]
  const long long* slots;  // [T]
  int tokens, kv_heads, num_blocks, kv_layout;
  unsigned* err;
};
cudaError_t launch_page_bounds(const BoundsParams& p, int head_dim, int block_size, int dtype,
                               cudaStream_t stream);

struct SelectParams {
  const void* q;             // [S, H, d]
  const void* k_cache;
  const void* v_cache;
  void* out;                 // [S, H, d]
  const signed char* values;
  const float* scales;
  const int* block_tables;   // [S, width]
  const int* context_lens;   // [S]
  int* selected;             // [S, Hkv, num_pages] page indices, ascending, -1 past the count
  int* sel_blocks;           // [S * Hkv, num_pages] block * Hkv + head of each chosen page
  int* sel_lens;             // [S * Hkv] tokens in the chosen pages
  unsigned* keys;            // sparse_key_ints(...) of scratch
  unsigned* maxima;          // maxima and key_stride: set by the launch
  long long key_stride;
  int num_seqs, heads, kv_heads, width, num_blocks, block_size;
  int num_pages, keep_first, keep_last;
  float scale_log2;
  unsigned* err;
};
// Ints of scratch for the scores.
long long sparse_key_ints(long long rows, int width);
// Whether launch_sparse(fused = true) runs the attention too; otherwise it fills sel_blocks
// and sel_lens for the paged decode.
bool sparse_fused(const SelectParams& p, int dtype, int kv_layout);
cudaError_t launch_sparse(SelectParams p, int head_dim, int dtype, bool fused, cudaStream_t stream);

}  // namespace step
}  // namespace fe
