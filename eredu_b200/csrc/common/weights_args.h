// Arguments of the calls that add up the weights of cached tokens and evict by them, as one block of bytes (see kv8_args.h for why): pointers, then ints,
// then floats, in the order of the formats in ops/eviction.py; a block of another length is refused.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

namespace eredu {

struct EvictArgs {
  void *k, *v;                            // [layers, pages, n_kv, 16] rows of k_row, v_row bytes
  float* weights;                         // [layers, pages, n_kv, 16]
  const int *block_table, *seq_lens;
  int* left;                              // [batch]: tokens that every sequence has left
  int* list;                              // scratch [layers, batch, n_kv, keep] of long sequences: the tokens that stay, in order
  int* status;
  cudaStream_t stream;
  int layers, batch, n_kv, num_pages, pitch, max_tokens, keep, recent, first, k_row, v_row, sm_count;
};

struct WeighedDecodeArgs {
  const void *q, *k, *v;
  void* out;
  const int *block_table, *seq_lens;
  const float* sinks;
  float* weights;                         // [pages, n_kv, 16]
  float* scores;                          // scratch [batch, n_kv, room, pad]
  float *part_o, *part_ml;                // scratch of more splits than a cluster holds: [batch, n_kv, splits, rows, D] and [.., 2]
  int* status;
  cudaStream_t stream;
  int batch, q_per_seq, pitch, max_tokens, room, num_pages, n_q, n_kv, D, splits, window;
  float scale;
};

struct WeighedPrefillArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;                             // scratch [total_q, n_q]: log2 of the sum of 2^(score log2 e)
  const int *block_table, *seq_lens, *cu_q;
  const float* sinks;
  float* weights;
  int* status;
  cudaStream_t stream;
  int batch, total_q, max_q_len, max_kv_len, wide, num_pages, n_q, n_kv, D, window, observed, ranks, sm_count;
  float scale;
};

template <typename Args>
inline bool weights_args(Args& a, const void* bytes, int n) {
  if (bytes == nullptr || n != static_cast<int>(sizeof(Args))) return false;
  memcpy(&a, bytes, sizeof(Args));
  return true;
}

}  // namespace eredu
