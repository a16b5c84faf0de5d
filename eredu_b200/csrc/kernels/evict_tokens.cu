// Eviction from a paged cache by the weight that attention has given its tokens: sequences longer than `keep` tokens are brought down to it,
// for every layer and key / value head by itself. The first `first` and the last `recent` tokens stay; of those between them the
// keep - first - recent with the largest weights (the earlier one of equal weights, and what is no number behind all numbers). What stays moves to the
// front in its order: keys, values and weights.
//
// Who stays: the border of the weights digit by digit (11, 11 and 10 bits, from the highest) over an order-preserving map to unsigned numbers, counted in shared memory;
// then the places by a running count. Rows move within the same pages, so a row must have been read before another one takes its place: a token never moves
// back, so that what is read for places >= i lies at >= i, and walking the places upwards, with a barrier between the reads of a stretch and its writes, is
// enough. Columns do not meet.
//
// One launch where the weights of a sequence and head find room in shared memory (48 k tokens): a CTA selects, keeps the list of what stays over the weights
// that it has looked at - a token's place is never behind the token -, and moves. The selections of some CTAs run under the moves of others. Few sequences and heads are
// shared by the CTAs of a cluster, which select alike and move some columns each. Longer sequences: one launch that writes the list to memory, another one that moves by it.
//
// Measured (floor: sums of all tokens, and rows that stay read and written, at 6.54 TB/s; first evictions, memory flushed in between): 8 sequences of 1008 to 1152 tokens to 1024, 8 heads
// of 128 in 32 layers, 289 us (floor 330, which counts rows that are where they belong; bound by memory); one of 32768 to 2048, 8 heads of 64 in 16 layers, 66 us (23: the selection, by one
// CTA a head and layer, and reads of single rows); one of 600 to 513, 4 heads of 128 in 4 layers, 16 us, latencies; one of 100000 to 4096, 8 heads of 128 in 8 layers, 244 us (45: four
// reads of the sums by 64 CTAs).
#include <cuda_runtime.h>

#include <algorithm>

#include "../common/launch.h"
#include "../common/launch_count.h"
#include "../common/ptx.cuh"
#include "../common/weights_args.h"

namespace eredu {

constexpr int kEvictPage = 16;
constexpr int kEvictHeld = 48 * 1024;               // weights that find room in shared memory
constexpr int kEvictThreads = 1024;                 // at most
constexpr int kEvictBins = 2048;
constexpr int kMoveBytes = 128;                     // columns that threads take together: four whole sectors of a row
constexpr int kMoveDeep = 4;                        // rows a thread has on their way, twice

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

// The pages of a sequence: its row of the table, or (HELD) a copy in shared memory in which -1 stands for what the table must not name.
template <bool HELD>
struct EvictTable {
  const EvictArgs& p;
  const int* held;
  int b;
  __device__ __forceinline__ int operator[](int entry) const { return HELD ? held[entry] : evict_page(p, b, entry); }
};

// Tokens of a sequence, no more than its row of the table holds.
__device__ __forceinline__ int evict_length(const EvictArgs& p, int b) {
  const int n = p.seq_lens[b];
  if (n > p.max_tokens) report_status(p.status, kStatusBadArgument);
  return min(n, p.max_tokens);
}

// Rows to their places list[begin .. keep), by all threads of the CTA: columns of the slices mine, mine + step, ..
template <typename Table>
__device__ __forceinline__ void evict_move(const EvictArgs& p, const Table& table, int layer, int h, const int* list, int begin, int mine, int step) {
  const int k_slices = (p.k_row + kMoveBytes - 1) / kMoveBytes, slices = k_slices + (p.v_row + kMoveBytes - 1) / kMoveBytes;
  const int wide = min((slices - mine + step - 1) / step, static_cast<int>(blockDim.x) / 8);     // slices side by side
  const int group = wide * 8, rows = blockDim.x / group, r = threadIdx.x / group, lane = threadIdx.x % group;
  for (int s0 = mine; s0 < slices; s0 += wide * step) {
    const int slice = s0 + lane / 8 * step;
    const bool keys = slice < k_slices;
    const int row = keys ? p.k_row : p.v_row, at = (keys ? slice : slice - k_slices) * kMoveBytes + (lane & 7) * 16;
    const bool in = slice < slices && at < row && r < rows;
    char* base = static_cast<char*>(keys ? p.k : p.v) + static_cast<size_t>(layer) * p.num_pages * p.n_kv * kEvictPage * row + at;
    auto cell = [&](int t) -> char* {
      const int page = table[t / kEvictPage];
      return page < 0 ? nullptr : base + ((static_cast<size_t>(page) * p.n_kv + h) * kEvictPage + t % kEvictPage) * row;
    };
    uint4 x[kMoveDeep], next[kMoveDeep];
    uint32_t moves = 0, next_moves = 0;              // bits
    auto read = [&](int j0) {
      next_moves = 0;
#pragma unroll
      for (int i = 0; i < kMoveDeep; ++i) {
        const int j = j0 + i * rows + r;
        if (!in || j >= p.keep) continue;
        const int from = list[j];
        const char* src = from != j ? cell(from) : nullptr;
        if (src == nullptr) continue;
        next[i] = *reinterpret_cast<const uint4*>(src);
        next_moves |= 1u << i;
      }
    };
    read(begin);
    for (int j0 = begin; j0 < p.keep; j0 += rows * kMoveDeep) {
#pragma unroll
      for (int i = 0; i < kMoveDeep; ++i) x[i] = next[i];
      moves = next_moves;
      read(j0 + rows * kMoveDeep);                   // (lies behind all that this stretch writes)
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMoveDeep; ++i) {
        if (!(moves >> i & 1)) continue;
        char* dst = cell(j0 + i * rows + r);
        if (dst != nullptr) *reinterpret_cast<uint4*>(dst) = x[i];
      }
    }
  }
}

// grid (CTAs of a cluster, heads of all sequences, layers). HELD: the weights are held in shared memory, and the rows are moved here.
template <bool HELD>
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const EvictArgs p, const int ranks) {
  extern __shared__ float4 evict_raw[];
  float* kept = reinterpret_cast<float*>(evict_raw);
  __shared__ int hist[kEvictBins];
  __shared__ int s_digit, s_left, s_first;
  __shared__ int warp_sum[32];
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int rank = blockIdx.x, b = blockIdx.y / p.n_kv, h = blockIdx.y % p.n_kv, layer = blockIdx.z;
  const int threads = blockDim.x, warps = threads >> 5, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = evict_length(p, b);
  if (rank == 0 && h == 0 && layer == 0 && tid == 0) p.left[b] = min(p.seq_lens[b], p.keep);
  if (n <= p.keep) return;
  float* w = p.weights + static_cast<size_t>(layer) * p.num_pages * p.n_kv * kEvictPage;
  int* pages = reinterpret_cast<int*>(kept + (p.max_tokens + 3) / 4 * 4);
  const EvictTable<HELD> table{p, pages, b};
  if (HELD)
    for (int i = tid; i * kEvictPage < n; i += threads) pages[i] = evict_page(p, b, i);
  for (int i = tid; i < kEvictBins; i += threads) hist[i] = 0;
  if (tid == 0) s_first = n;
  __syncthreads();
  auto page_cell = [&](int t) -> float* {
    const int page = table[t / kEvictPage];
    return page < 0 ? nullptr : w + (static_cast<size_t>(page) * p.n_kv + h) * kEvictPage + t % kEvictPage;
  };
  // four tokens of a page from memory
  auto quad = [&](int t) -> float4 {
    const float* at = t < n ? page_cell(t) : nullptr;
    return at == nullptr ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(at);
  };
  // ---- the border: the quota-th largest of the tokens [first, last)
  const int first = p.first, last = n - p.recent, quota = p.keep - p.first - p.recent;
  uint32_t border = 0;
  int left = quota;                                  // of those that agree with the border so far, how many stay
  int shift = 21, bins = kEvictBins;                 // the digit that is counted
  uint32_t above = 0;                                // bits in front of it
  // Lanes that all have the same digit (weights that are equal) count as one. Behind the first round few weights agree with the border.
  auto count = [&](int t, const float4& q) {
    const float x[4] = {q.x, q.y, q.z, q.w};
    uint32_t u[4];
    bool in[4], any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = weight_order(x[i]);
      in[i] = t + i >= first && t + i < last && (u[i] & above) == border;
      any = any || in[i];
    }
    if (above != 0 && !__any_sync(0xffffffffu, any)) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int digit = in[i] ? static_cast<int>(u[i] >> shift) & (bins - 1) : -1;
      if (__all_sync(0xffffffffu, digit == __shfl_sync(0xffffffffu, digit, 0))) {
        if (lane == 0 && digit >= 0) atomicAdd(&hist[digit], 32);
      } else if (digit >= 0) {
        atomicAdd(&hist[digit], 1);
      }
    }
  };
  // (HELD: the first digits are counted as the weights come in)
  auto from_memory = [&](bool counted) {
    for (int t0 = 0; t0 < n; t0 += 16 * threads) {
      float4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = quad(t0 + 4 * (i * threads + tid));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (t0 + 4 * i * threads >= n) break;
        const int t = t0 + 4 * (i * threads + tid);
        if (HELD && t < n) *reinterpret_cast<float4*>(kept + t) = x[i];
        __syncwarp();
        if (counted) count(t, x[i]);
      }
    }
  };
  if (HELD) from_memory(quota > 0);
  if (ranks > 1) {
    __syncwarp();
    cluster_arrive_release();                        // this CTA has read the weights, which the first one moves
  }
  for (int round = 0; round < 3 && quota > 0; ++round) {
    if (round > 0) {
      shift = round == 1 ? 10 : 0;
      bins = round == 1 ? 2048 : 1024;
      above = ~0u << (shift + (round == 1 ? 11 : 10));
      for (int i = tid; i < bins; i += threads) hist[i] = 0;
      __syncthreads();
    }
    if (!HELD) {
      from_memory(true);
    } else if (round > 0) {
      for (int t0 = 0; t0 < n; t0 += 4 * threads) {
        const int t = t0 + 4 * tid;
        count(t, t < n ? *reinterpret_cast<const float4*>(kept + t) : make_float4(0.f, 0.f, 0.f, 0.f));
      }
    }
    __syncthreads();
    // thread i has the bins from the top down, `per` each
    const int per = (bins + threads - 1) / threads, top = bins - 1 - tid * per;
    int own = 0;
    for (int i = 0; i < per; ++i)
      if (top - i >= 0) own += hist[top - i];
    int before = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += other;
    }
    if (lane == 31) warp_sum[warp] = before;
    __syncthreads();
    before -= own;
    for (int i = 0; i < warp; ++i) before += warp_sum[i];
    if (before < left && before + own >= left) {     // one thread
      for (int i = 0; i < per; ++i) {
        const int c = hist[top - i];
        if (before + c >= left) {
          s_digit = top - i;
          s_left = left - before;
          break;
        }
        before += c;
      }
    }
    __syncthreads();
    border |= static_cast<uint32_t>(s_digit) << shift;
    left = s_left;
  }
  // ---- places: those above the border and the protected ones, and the first `left` at it
  if (ranks > 1) {
    __syncwarp();
    cluster_wait_acquire();
  }
  int* list = HELD ? reinterpret_cast<int*>(kept) : p.list + ((static_cast<size_t>(layer) * p.batch + b) * p.n_kv + h) * p.keep;
  int above_before = 0, equal_before = 0;
  __syncthreads();
  for (int t0 = 0; t0 < n; t0 += 4 * threads) {
    const int t = t0 + 4 * tid;
    const float4 q = !HELD ? quad(t) : t < n ? *reinterpret_cast<const float4*>(kept + t) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float x[4] = {q.x, q.y, q.z, q.w};
    int above = 0, equal = 0;                        // bits
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = weight_order(x[i]);
      const bool stays = t + i < n && (t + i < first || t + i >= last), open = t + i < n && !stays && quota > 0;
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
    int in_front = lane < warp ? warp_sum[lane] : 0, all = lane < warps ? warp_sum[lane] : 0;
    in_front = __reduce_add_sync(0xffffffffu, in_front) + sum - own;
    all = __reduce_add_sync(0xffffffffu, all);
    int a = above_before + (in_front & 0xffff), e = equal_before + (in_front >> 16);
    int gone = n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool is_above = (above >> i) & 1, is_equal = (equal >> i) & 1;
      const int to = a + min(e, left);
      if (is_above || (is_equal && e < left)) {
        list[to] = t + i;
        if (to != t + i && rank == 0) {
          float* at = page_cell(to);
          if (at != nullptr) *at = x[i];
        }
      } else if (t + i < n) {
        gone = min(gone, t + i);
      }
      a += is_above;
      e += is_equal;
    }
    if (above_before + min(equal_before, left) == t0) {   // nobody has gone in front of this tile
      gone = __reduce_min_sync(0xffffffffu, gone);
      if (lane == 0 && gone < n) atomicMin(&s_first, gone);
    }
    above_before += all & 0xffff;
    equal_before += all >> 16;
    __syncthreads();                                 // warp_sum is used again; the next tile's weights are read behind these writes
  }
  if (HELD) evict_move(p, table, layer, h, list, min(s_first, p.keep), rank, ranks);
}

// grid (column slices of keys and values, heads of all sequences, layers)
constexpr int kMoveThreads = 256;
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs p) {
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.y / p.n_kv, h = blockIdx.y % p.n_kv, layer = blockIdx.z;
  if (evict_length(p, b) <= p.keep) return;
  evict_move(p, EvictTable<false>{p, nullptr, b}, layer, h, p.list + ((static_cast<size_t>(layer) * p.batch + b) * p.n_kv + h) * p.keep, 0, blockIdx.x, gridDim.x);
}

// Weights, and pages, of one sequence.
static int evict_smem(int tokens) { return (tokens + 3) / 4 * 16 + (tokens + kEvictPage - 1) / kEvictPage * 4; }

template <bool HELD>
static cudaError_t launch_evict(const EvictArgs& a, int threads, int ranks, size_t smem) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (HELD && dev >= 0 && dev < 64 && !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(evict_kernel<HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, evict_smem(kEvictHeld));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, a.n_kv * a.batch, a.layers);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  eredu_count_launches(1);
  return cudaLaunchKernelEx(&cfg, evict_kernel<HELD>, a, ranks);
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
  const int slices = (a.k_row + kMoveBytes - 1) / kMoveBytes + (a.v_row + kMoveBytes - 1) / kMoveBytes;
  if (a.max_tokens > kEvictHeld) {
    if (a.list == nullptr) return -2;
    const cudaError_t e = launch_evict<false>(a, kEvictThreads, 1, 0);
    if (e != cudaSuccess) return static_cast<int>(e);
    eredu_count_launches(1);
    return static_cast<int>(launch_pdl(evict_move_kernel, dim3(slices, a.n_kv * a.batch, a.layers), dim3(kMoveThreads), 0, a.stream, a));
  }
  const long long heads = static_cast<long long>(a.layers) * a.batch * a.n_kv;
  int ranks = 1;
  while (ranks < 8 && ranks * 2 <= slices && heads * ranks * 2 <= (a.max_tokens > 16384 ? 1 : 2) * a.sm_count) ranks *= 2;
  // (us with 256 / 512 / 1024 threads: 64 heads of 1152 tokens in 32 layers 353 / 347 / 420; one sequence of 32768, 128 heads 113 / 74 / 58)
  const int threads = a.max_tokens > 8192 ? 1024 : 512;
  return static_cast<int>(launch_evict<true>(a, threads, ranks, evict_smem(a.max_tokens)));
}
