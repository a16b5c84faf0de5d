// Eviction from a paged cache by the weight that attention has given its tokens: sequences longer than `keep` tokens are brought down to it,
// for every layer and key / value head by itself. The first `first` and the last `recent` tokens stay; of those between them the
// keep - first - recent with the largest weights (the earlier one of equal weights, and what is no number behind all numbers). What stays moves to the
// front in its order: keys, values and weights.
//
// Two launches. The first finds who stays: the border of the weights digit by digit (8 bits a round, from the highest) over an order-preserving map
// to unsigned numbers, then the places by a running count; it moves the weights and writes the list of the tokens that stay. The second moves keys and values by that list.
// Rows move within the same pages, so a row must have been read before another one takes its place: a token never moves
// back, so that what is read for places >= i lies at >= i, and walking the places upwards, with a barrier between the reads of a stretch and its writes, is
// enough. Columns do not meet: 128 bytes of a row are a CTA's own.
#include <cuda_runtime.h>

#include <algorithm>

#include "../common/launch.h"
#include "../common/launch_count.h"
#include "../common/ptx.cuh"
#include "../common/weights_args.h"

namespace eredu {

constexpr int kEvictPage = 16;
constexpr int kSelectThreads = 512;
constexpr int kSelectPer = 4;                       // tokens of a thread in a tile of the running count
constexpr int kSelectHeld = 48 * 1024;              // weights that find room in shared memory; longer sequences are read again for every digit
constexpr int kMoveThreads = 256;
constexpr int kMoveBytes = 128;                     // columns of a CTA: four whole sectors of a row
constexpr int kMoveDeep = 8;                        // rows a thread has on their way

// Larger numbers of the order are larger unsigned ones, both zeros the same; 0: no number.
__device__ __forceinline__ uint32_t weight_order(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  return w != w ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A page that the table must not name is not touched.
__device__ __forceinline__ int evict_page(const EvictArgs& p, int b, int entry) {
  const int page = p.block_table[static_cast<size_t>(b) * p.pitch + entry];
  if (page >= 0 && page < p.num_pages) return page;
  report_status(p.status, kStatusBadArgument);
  return -1;
}

// Tokens of a sequence, no more than its row of the table holds.
__device__ __forceinline__ int evict_length(const EvictArgs& p, int b) {
  const int n = p.seq_lens[b], most = p.max_tokens;
  if (n > most) report_status(p.status, kStatusBadArgument);
  return min(n, most);
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictArgs p, const int held) {
  extern __shared__ float kept[];
  __shared__ int hist[256];
  __shared__ int s_digit, s_left;
  __shared__ int warp_sum[kSelectThreads / 32];
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = evict_length(p, b);
  if (h == 0 && layer == 0 && tid == 0) p.left[b] = min(p.seq_lens[b], p.keep);
  if (n <= p.keep) return;
  float* w = p.weights + static_cast<size_t>(layer) * p.num_pages * p.n_kv * kEvictPage;
  auto cell = [&](int t) -> float* {
    const int page = evict_page(p, b, t / kEvictPage);
    return page < 0 ? nullptr : w + (static_cast<size_t>(page) * p.n_kv + h) * kEvictPage + t % kEvictPage;
  };
  auto value = [&](int t) -> float {
    if (t < held) return kept[t];
    const float* at = cell(t);
    return at == nullptr ? 0.f : *at;
  };
  for (int t = tid; t < min(n, held); t += kSelectThreads) {
    const float* at = cell(t);
    kept[t] = at == nullptr ? 0.f : *at;
  }
  // ---- the border: the quota-th largest of the tokens [first, last)
  const int first = p.first, last = n - p.recent, quota = p.keep - p.first - p.recent;
  uint32_t border = 0;
  int left = quota;                                  // of those that agree with the border so far, how many stay
  for (int shift = 24; shift >= 0 && quota > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t0 = first; t0 < last; t0 += kSelectThreads) {
      const int t = t0 + tid;
      const uint32_t u = t < last ? weight_order(value(t)) : 0u;
      const bool in = t < last && (shift == 24 || (u >> (shift + 8)) == (border >> (shift + 8)));
      const int digit = in ? static_cast<int>((u >> shift) & 255u) : 256;
      const unsigned same = __match_any_sync(0xffffffffu, digit);
      if (in && lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
    }
    __syncthreads();
    if (warp == 0) {
      // lane l has the digits 255 - 8 l down to 248 - 8 l
      int own = 0;
      for (int i = 0; i < 8; ++i) own += hist[255 - 8 * lane - i];
      int before = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += other;
      }
      before -= own;
      if (before < left && before + own >= left) {
        for (int i = 0; i < 8; ++i) {
          const int d = 255 - 8 * lane - i;
          if (before + hist[d] >= left) {
            s_digit = d;
            s_left = left - before;
            break;
          }
          before += hist[d];
        }
      }
    }
    __syncthreads();
    border |= static_cast<uint32_t>(s_digit) << shift;
    left = s_left;
  }
  // ---- places: those above the border and the protected ones, and the first `left` at it
  int* list = p.list + ((static_cast<size_t>(layer) * p.batch + b) * p.n_kv + h) * p.keep;
  int above_before = 0, equal_before = 0;
  __syncthreads();
  for (int t0 = 0; t0 < n; t0 += kSelectThreads * kSelectPer) {
    float x[kSelectPer];
    int above = 0, equal = 0;                        // bits
#pragma unroll
    for (int i = 0; i < kSelectPer; ++i) {
      const int t = t0 + tid * kSelectPer + i;
      x[i] = t < n ? value(t) : 0.f;
      const uint32_t u = weight_order(x[i]);
      const bool stays = t < n && (t < first || t >= last), open = t < n && !stays && quota > 0;
      if (stays || (open && u > border)) above |= 1 << i;
      if (open && u == border) equal |= 1 << i;
    }
    const int own = __popc(above) | __popc(equal) << 16;
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += other;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int in_front = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSelectThreads / 32; ++i) {
      const int s = warp_sum[i];
      if (i < warp) in_front += s;
      all += s;
    }
    in_front += sum - own;
    int a = above_before + (in_front & 0xffff), e = equal_before + (in_front >> 16);
#pragma unroll
    for (int i = 0; i < kSelectPer; ++i) {
      const bool is_above = (above >> i) & 1, is_equal = (equal >> i) & 1;
      const int to = a + min(e, left);
      if (is_above || (is_equal && e < left)) {
        const int t = t0 + tid * kSelectPer + i;
        list[to] = t;
        if (to != t) {
          float* at = cell(to);
          if (at != nullptr) *at = x[i];
        }
      }
      a += is_above;
      e += is_equal;
    }
    above_before += all & 0xffff;
    equal_before += all >> 16;
    __syncthreads();                                 // warp_sum is used again; the next tile's weights are read behind these writes
  }
}

// grid (column slices of keys, then of values; heads of all sequences; layers)
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs p, const int k_slices) {
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const bool keys = static_cast<int>(blockIdx.x) < k_slices;
  const int slice = keys ? blockIdx.x : blockIdx.x - k_slices;
  const int b = blockIdx.y / p.n_kv, h = blockIdx.y % p.n_kv, layer = blockIdx.z;
  const int n = evict_length(p, b);
  if (n <= p.keep) return;
  const int row = keys ? p.k_row : p.v_row;          // bytes
  const int at = slice * kMoveBytes + (threadIdx.x & 7) * 16;
  const bool in = at < row;
  char* base = static_cast<char*>(keys ? p.k : p.v) + static_cast<size_t>(layer) * p.num_pages * p.n_kv * kEvictPage * row + at;
  const int* list = p.list + ((static_cast<size_t>(layer) * p.batch + b) * p.n_kv + h) * p.keep;
  constexpr int LANES = kMoveThreads / 8, STRETCH = LANES * kMoveDeep;
  const int mine = threadIdx.x >> 3;
  auto cell = [&](int t) -> char* {
    const int page = evict_page(p, b, t / kEvictPage);
    return page < 0 ? nullptr : base + ((static_cast<size_t>(page) * p.n_kv + h) * kEvictPage + t % kEvictPage) * row;
  };
  for (int j0 = 0; j0 < p.keep; j0 += STRETCH) {
    uint4 x[kMoveDeep];
    int from[kMoveDeep];
#pragma unroll
    for (int i = 0; i < kMoveDeep; ++i) {
      const int j = j0 + i * LANES + mine;
      from[i] = j < p.keep && in ? list[j] : j;
      if (from[i] != j) {
        const char* src = cell(from[i]);
        if (src == nullptr) from[i] = j;
        else x[i] = *reinterpret_cast<const uint4*>(src);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMoveDeep; ++i) {
      const int j = j0 + i * LANES + mine;
      if (from[i] == j) continue;
      char* dst = cell(j);
      if (dst != nullptr) *reinterpret_cast<uint4*>(dst) = x[i];
    }
  }
}

}  // namespace eredu

using namespace eredu;

extern "C" int eredu_evict_tokens(const void* args, int bytes) {
  EvictArgs a;
  if (!weights_args(a, args, bytes)) return -2;
  if (a.layers <= 0 || a.batch <= 0) return 0;
  if (a.n_kv <= 0 || a.num_pages <= 0 || a.keep <= 0 || a.first < 0 || a.recent < 0 || a.first + a.recent > a.keep || a.k_row <= 0 || a.v_row <= 0 ||
      (a.k_row | a.v_row) % 16 != 0 || a.layers > 65535 || a.batch > 65535 / a.n_kv || a.max_tokens < 0)
    return -2;
  const int held = std::min(a.max_tokens, kSelectHeld);
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    if (cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelectHeld * 4) != cudaSuccess) return -1;
    configured[dev] = true;
  }
  cudaError_t e = launch_pdl(evict_select_kernel, dim3(a.n_kv, a.batch, a.layers), dim3(kSelectThreads), static_cast<size_t>(held) * 4, a.stream, a, held);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int k_slices = (a.k_row + kMoveBytes - 1) / kMoveBytes, v_slices = (a.v_row + kMoveBytes - 1) / kMoveBytes;
  e = launch_pdl(evict_move_kernel, dim3(k_slices + v_slices, a.n_kv * a.batch, a.layers), dim3(kMoveThreads), 0, a.stream, a, k_slices);
  eredu_count_launches(2);
  return static_cast<int>(e);
}
