// Arguments of the calls on pages held in 8 bits, as one block of bytes: passing some forty of them one by one costs the caller 4 us a call, packing them 0.7.
// Pointers, then ints, then floats, in the order of the formats in ops/kv8.py; a block of another length is refused.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

namespace eredu {

struct Kv8StoreArgs {
  const void *q, *k, *v;                  // bf16 [M, heads, D], rows of ld_q, ld_k, ld_v elements
  void* q_out;                            // optional [M, n_q, D], bf16 or fp32
  void *k_codes, *v_codes;
  float *k_scales, *v_scales;
  const int* positions;
  const long long* slots;
  const float *inv_freq, *q_norm_w, *k_norm_w;
  int* status;
  cudaStream_t stream;
  int M, ld_q, ld_k, ld_v, n_q, n_kv, D, rot, interleaved, num_pages, q_out_fp32;
  float attn_factor, norm_eps, norm_w_off;
};

struct Kv8ValuesArgs {
  const void *k_codes, *v_codes;
  const float *k_scales, *v_scales;
  void *k_out, *v_out;
  const int *pages, *seq_lens, *cu_q;
  int* table_out;
  int* status;
  cudaStream_t stream;
  int rows, pitch, table_wide, wide, n_kv, D, num_pages, window, chunk;
  int entries;                            // with seq_lens: room of k_out and v_out where the rows follow one another; 0: rows of `wide`
};

struct Kv8AttentionArgs {
  const void* q;                          // queries, or (step) the projection's output, rows of ld elements
  float* q32;                             // step: [batch * q_per_seq, n_q, D] where the rows are written by a kernel in front
  void *k_codes, *v_codes;
  float *k_scales, *v_scales;
  void* out;
  const int *block_table, *seq_lens;
  const float* sinks;
  float *part_o, *part_ml;                // even shares
  void* joins;
  const int* positions;                   // step: this and what follows
  const long long* slots;
  const float *inv_freq, *q_norm_w, *k_norm_w;
  int* status;
  cudaStream_t stream;
  int ld, batch, q_per_seq, max_pages, pitch, num_pages, n_q, n_kv, D, rot, interleaved, splits, ctas, window, chunk, settled;
  float scale, attn_factor, norm_eps, norm_w_off;
};

template <typename Args>
inline bool kv8_args(Args& a, const void* bytes, int n) {
  if (bytes == nullptr || n != static_cast<int>(sizeof(Args))) return false;
  memcpy(&a, bytes, sizeof(Args));
  return true;
}
// Rows into blocks, as eredu_kv8_store does.
int kv8_store(const Kv8StoreArgs& a);

}  // namespace eredu
