// Pages of a cache held in 8 bits (common/kv8.cuh): rows are written, values read back, and pages of any cache copied.
#include <algorithm>

#include "../common/kv8_store.cuh"
#include "../common/launch.h"
#include "../common/launch_count.h"
#include "../common/ptx.cuh"
#include "../common/trace.cuh"

namespace eredu {

// ============================================================================ rows into their blocks
// q, k rotated by their positions (optional RMSNorm per head in front), k and v rounded into their blocks, q stored as it is.
//
// A run is a stretch of rows that follow one another in one page; its rows share a scale per head. Four warps have the run's keys in registers and four its
// values (16 x 128 / 128 values a thread), find the largest together and store the codes: one read. A lane has four neighbouring values of a row; the
// partner of a rotation sits `rot / 8` lanes further. The angles of a tile of rows are computed once for the head's keys and its query heads.
// 4096 rows, 32 heads of 128 over 8: a warp to a run's keys, in 128 registers, 92 us.
constexpr int kStoreThreads = 256, kStoreShare = kStoreThreads / 64;   // half of the warps for keys, half for values
constexpr int kStoreRows = 32;      // a tile of 16 rows and what the last run of it has behind them

// grid (tiles of rows, n_kv)
template <int D, bool WHOLE>
__global__ void __launch_bounds__(kStoreThreads) kv8_store_kernel(Kv8StoreParams p) {
  using Rows = Kv8Rows<D, WHOLE>;
  extern __shared__ __align__(16) float turns[];          // [rows of the tile and the last run][rot / 2 cosines, rot / 2 sines]
  __shared__ int run_row[kKv8Page], run_len[kKv8Page];
  __shared__ long long run_slot[kKv8Page];
  __shared__ uint32_t tops[kStoreThreads / 32];
  __shared__ int runs, behind;
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = blockIdx.x * p.tile, rows = min(p.tile, p.M - row0), h0 = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rot = WHOLE ? D : p.rot, half = rot / 2;
  if (warp == 0) {
    // lane r has the slots of rows r - 1 and r of the tile and the 16 behind it: a row continues the one in front where its slot is the next of the same page
    const int r = row0 + lane;
    const bool known = r < p.M && lane < rows + kKv8Page;
    const long long slot = known ? p.slots[r] : -1, front = known && r > 0 ? p.slots[r - 1] : -1;
    const bool follows = slot >= 0 && (slot & 15) != 0 && front == slot - 1;
    bool begins = lane < rows && slot >= 0 && !follows;
    if (begins && (slot >> 4) >= p.num_pages) {
      report_status(p.status, kStatusBadArgument);
      begins = false;
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, begins), more = __ballot_sync(0xffffffffu, follows);
    // (a tile of 16 rows and 15 more at most: what follows the last row of the warp's 32 cannot belong to a run of this tile)
    const int n = begins ? 1 + __ffs(~(more >> lane >> 1)) - 1 : 0;
    if (begins) {
      const int i = __popc(mask & ((1u << lane) - 1));
      run_row[i] = lane;
      run_len[i] = n;
      run_slot[i] = slot;
    }
    const int end = __reduce_max_sync(0xffffffffu, begins ? lane + n : 0);
    if (lane == 0) {
      runs = __popc(mask);
      behind = max(rows, end);
    }
  }
  __syncthreads();
  for (int r = threadIdx.x / (D / 2), i = threadIdx.x % (D / 2); r < behind; r += kStoreThreads / (D / 2))
    if (i < half) turn_of(p.positions[row0 + r], p.inv_freq[i], p.attn_factor, turns[r * rot + i], turns[r * rot + half + i]);
  __syncthreads();
  for (int i = 0; i < runs; ++i) {
    const int at = run_row[i];
    const long long cell = (run_slot[i] >> 4) * p.n_kv + h0;
    const int first = static_cast<int>(run_slot[i] & 15);
    if (warp < kStoreShare) store_block<D, true, kStoreShare, WHOLE>(p, row0 + at, run_len[i], first, cell, h0, turns + at * rot, lane, warp, tops);
    else store_block<D, false, kStoreShare, WHOLE>(p, row0 + at, run_len[i], first, cell, h0, turns, lane, warp - kStoreShare, tops + kStoreShare);
  }
  // ---- query rows of this head, four at a time on their way
  constexpr int DEEP = 4, STRIDE = kStoreThreads / 32 * Rows::ROWS;
  const int mine = p.q_out == nullptr ? 1 : p.n_q / p.n_kv, items = p.q_out == nullptr ? 0 : rows * mine, sub = Rows::row(lane);
  const uint32_t per_mine = ((1u << 20) + mine - 1) / mine;     // item / mine by a product: exact below 2^20 / mine, and there are 16 mine of them at most
  for (int i0 = warp * Rows::ROWS; i0 < items; i0 += STRIDE * DEEP) {
    Rows query[DEEP];
#pragma unroll
    for (int j = 0; j < DEEP; ++j) {
      const int item = min(i0 + j * STRIDE + sub, items - 1), r = static_cast<int>(item * per_mine >> 20);
      query[j].load(p.q + static_cast<size_t>(row0 + r) * p.ld_q + (h0 * mine + item - r * mine) * D, lane);
    }
#pragma unroll
    for (int j = 0; j < DEEP; ++j) {
      const int item = i0 + j * STRIDE + sub, r = static_cast<int>(min(item, items - 1) * per_mine >> 20), head = h0 * mine + min(item, items - 1) - r * mine;
      if (i0 + j * STRIDE >= items) break;
      query[j].prepare(p, p.q_norm_w, turns + r * rot, lane);
      if (item >= items) continue;
      const size_t at = (static_cast<size_t>(row0 + r) * p.n_q + head) * D;
#pragma unroll
      for (int i = 0; i < Rows::PER; ++i) {
        const float4 x = query[j].x[i];
        if (p.q_out_fp32) *reinterpret_cast<float4*>(static_cast<float*>(p.q_out) + at + Rows::channel(lane, i)) = x;
        else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.q_out) + at + Rows::channel(lane, i)) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
      }
    }
  }
}

// ============================================================================ values of pages
// Codes times scale as bf16 (exact: 8 significant bits): [entries, n_kv, 16, D] for keys and for values. The pages are a list, or (seq_lens given)
// the rows of a block table: then entries that no query of the sequence sees are left out, and `table_out` [rows, wide] says where each one is - those left out
// lie behind the last one, where a tensor map reads zeros.
struct Kv8ValuesParams {
  const int8_t *k_codes, *v_codes;
  const float *k_scales, *v_scales;
  __nv_bfloat16 *k_out, *v_out;
  const int* pages;        // [rows of `pitch`]
  const int* seq_lens;     // optional [rows]
  const int* cu_q;         // with seq_lens: query offsets
  int* table_out;          // with seq_lens: [rows, wide]
  int pitch, table_wide, wide, n_kv, num_pages, window, chunk;   // table_wide: entries of a row of `pages`; wide: of a row of the output
  int* status;
};
constexpr int kValuesThreads = 256;
template <int D>
__global__ void __launch_bounds__(kValuesThreads) kv8_values_kernel(Kv8ValuesParams p) {
  constexpr int BLOCK = kKv8Page * D, DEEP = 4;   // codes of a block; pieces of eight codes a thread has on their way
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, i = blockIdx.x;
  const size_t entry = static_cast<size_t>(row) * p.wide + i;
  if (p.seq_lens != nullptr) {
    const int len = p.seq_lens[row], first = len - (p.cu_q[row + 1] - p.cu_q[row]);
    const int low = p.window > 0 ? first - p.window + 1 : p.chunk > 0 && first > 0 ? first - first % p.chunk : 0;
    const bool seen = i * kKv8Page < len && i * kKv8Page + kKv8Page > low && first < len && i < p.table_wide;
    if (threadIdx.x == 0 && blockIdx.z == 0) p.table_out[entry] = static_cast<int>(seen ? entry : static_cast<size_t>(gridDim.y) * p.wide);
    if (!seen) return;
  }
  int page = p.pages[static_cast<size_t>(row) * p.pitch + i];
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) report_status(p.status, kStatusBadArgument);
    page = 0;
  }
  const size_t all = static_cast<size_t>(p.n_kv) * BLOCK;
  const int8_t* codes = (blockIdx.z == 0 ? p.k_codes : p.v_codes) + page * all;
  const float* scales = (blockIdx.z == 0 ? p.k_scales : p.v_scales) + static_cast<size_t>(page) * p.n_kv;
  __nv_bfloat16* out = (blockIdx.z == 0 ? p.k_out : p.v_out) + entry * all;
  for (int c0 = threadIdx.x * 8; c0 < p.n_kv * BLOCK; c0 += kValuesThreads * 8 * DEEP) {
    uint2 u[DEEP];
    float s[DEEP];
#pragma unroll
    for (int j = 0; j < DEEP; ++j) {
      const int c = min(c0 + j * kValuesThreads * 8, p.n_kv * BLOCK - 8);
      u[j] = *reinterpret_cast<const uint2*>(codes + c);
      s[j] = scales[c / BLOCK];
    }
#pragma unroll
    for (int j = 0; j < DEEP; ++j) {
      const int c = c0 + j * kValuesThreads * 8;
      if (c < p.n_kv * BLOCK)
        *reinterpret_cast<uint4*>(out + c) =
            make_uint4(pack_bf16x2(kv8_code(u[j].x, 0) * s[j], kv8_code(u[j].x, 1) * s[j]), pack_bf16x2(kv8_code(u[j].x, 2) * s[j], kv8_code(u[j].x, 3) * s[j]),
                       pack_bf16x2(kv8_code(u[j].y, 0) * s[j], kv8_code(u[j].y, 1) * s[j]), pack_bf16x2(kv8_code(u[j].y, 2) * s[j], kv8_code(u[j].y, 3) * s[j]));
    }
  }
}

// ============================================================================ pages copied
struct PageCopyParams {
  char* base[8];                 // [layers, pages, bytes]
  long long layer_stride[8];
  int bytes[8], layers[8];       // of a page; a multiple of 4
  const int *src, *dst;
  int num_pages;
  int* status;
};
template <typename T>
__device__ __forceinline__ void copy_page(char* to, const char* from, int bytes) {
  const int n = bytes / static_cast<int>(sizeof(T));
  for (int i = threadIdx.x; i < n; i += blockDim.x) reinterpret_cast<T*>(to)[i] = reinterpret_cast<const T*>(from)[i];
}
// grid (pairs, layers, tensors)
__global__ void __launch_bounds__(256) copy_pages_kernel(PageCopyParams p) {
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.z, layer = blockIdx.y;
  if (layer >= p.layers[t]) return;
  const int src = p.src[blockIdx.x], dst = p.dst[blockIdx.x];
  if (src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages) {
    if (threadIdx.x == 0) report_status(p.status, kStatusBadArgument);
    return;
  }
  char* base = p.base[t] + layer * p.layer_stride[t];
  const char* from = base + static_cast<long long>(src) * p.bytes[t];
  char* to = base + static_cast<long long>(dst) * p.bytes[t];
  if (p.bytes[t] % 16 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0) copy_page<uint4>(to, from, p.bytes[t]);
  else copy_page<uint32_t>(to, from, p.bytes[t]);
}

}  // namespace eredu

using namespace eredu;

extern "C" int eredu_kv8_store(const void* q, const void* k, const void* v, void* q_out, void* k_codes, void* v_codes, float* k_scales, float* v_scales,
                               const int* positions, const long long* slots, const float* inv_freq, const float* q_norm_w, const float* k_norm_w, int M,
                               int ld_q, int ld_k, int ld_v, int n_q, int n_kv, int D, int rot, int interleaved, int num_pages, int q_out_fp32,
                               float attn_factor, float norm_eps, float norm_w_off, int* status, cudaStream_t stream) {
  if (M <= 0) return 0;
  if ((D != 64 && D != 128) || n_kv <= 0 || num_pages <= 0 || rot < 0 || rot > D || rot % 8 != 0 || ld_q % 4 != 0 || ld_k % 4 != 0 || ld_v % 4 != 0 ||
      (q_out != nullptr && (n_q <= 0 || n_q % n_kv != 0 || n_q / n_kv > 256)))
    return -2;
  Kv8StoreParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_out = q_out;
  p.q_out_fp32 = q_out_fp32;
  p.k_codes = static_cast<int8_t*>(k_codes);
  p.v_codes = static_cast<int8_t*>(v_codes);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.positions = positions;
  p.slots = slots;
  p.inv_freq = inv_freq;
  p.q_norm_w = q_norm_w;
  p.k_norm_w = k_norm_w;
  p.M = M;
  p.ld_q = ld_q;
  p.ld_k = ld_k;
  p.ld_v = ld_v;
  p.n_q = n_q;
  p.n_kv = n_kv;
  p.rot = rot;
  p.interleaved = interleaved;
  p.num_pages = num_pages;
  p.attn_factor = attn_factor;
  p.norm_eps = norm_eps;
  p.norm_w_off = norm_w_off;
  p.status = status;
  // a key / value head with its query heads per CTA, and a row or, where there are many, 16, in which most runs are whole
  p.tile = M <= 256 ? 1 : 16;
  const dim3 grid((M + p.tile - 1) / p.tile, n_kv);
  const size_t smem = static_cast<size_t>(kStoreRows) * rot * sizeof(float);
  const bool whole = rot == D && interleaved == 0;
  const cudaError_t e = D == 128 ? (whole ? launch_pdl(kv8_store_kernel<128, true>, grid, dim3(kStoreThreads), smem, stream, p)
                                          : launch_pdl(kv8_store_kernel<128, false>, grid, dim3(kStoreThreads), smem, stream, p))
                                 : (whole ? launch_pdl(kv8_store_kernel<64, true>, grid, dim3(kStoreThreads), smem, stream, p)
                                          : launch_pdl(kv8_store_kernel<64, false>, grid, dim3(kStoreThreads), smem, stream, p));
  eredu_count_launches(1);
  return static_cast<int>(e);
}

extern "C" int eredu_kv8_values(const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales, void* k_out, void* v_out,
                                const int* pages, const int* seq_lens, const int* cu_q, int* table_out, int rows, int pitch, int table_wide, int wide, int n_kv, int D,
                                int num_pages, int window, int chunk, int* status, cudaStream_t stream) {
  if (rows <= 0 || wide <= 0) return 0;
  if ((D != 64 && D != 128) || n_kv <= 0 || rows > 65535 || num_pages <= 0) return -2;
  Kv8ValuesParams p = {};
  p.k_codes = static_cast<const int8_t*>(k_codes);
  p.v_codes = static_cast<const int8_t*>(v_codes);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.pages = pages;
  p.seq_lens = seq_lens;
  p.cu_q = cu_q;
  p.table_out = table_out;
  p.pitch = pitch;
  p.wide = wide;
  p.table_wide = table_wide;
  p.n_kv = n_kv;
  p.num_pages = num_pages;
  p.window = window;
  p.chunk = chunk;
  p.status = status;
  const cudaError_t e = D == 128 ? launch_pdl(kv8_values_kernel<128>, dim3(wide, rows, 2), dim3(kValuesThreads), 0, stream, p)
                                 : launch_pdl(kv8_values_kernel<64>, dim3(wide, rows, 2), dim3(kValuesThreads), 0, stream, p);
  eredu_count_launches(1);
  return static_cast<int>(e);
}

// tensors: `count` <= 8 descriptions of {address, bytes between layers, bytes of a page, layers}
extern "C" int eredu_copy_pages(const long long* tensors, int count, const int* src, const int* dst, int pairs, int num_pages, int* status,
                                cudaStream_t stream) {
  if (pairs <= 0 || count <= 0) return 0;
  if (count > 8) return -2;
  PageCopyParams p = {};
  int layers = 0;
  for (int i = 0; i < count; ++i) {
    const long long* t = tensors + 4 * i;
    if (t[2] <= 0 || t[2] % 4 != 0 || t[2] > (1 << 30) || t[0] % 4 != 0 || t[1] % 4 != 0 || t[3] > 65535) return -2;
    p.base[i] = reinterpret_cast<char*>(t[0]);
    p.layer_stride[i] = t[1];
    p.bytes[i] = static_cast<int>(t[2]);
    p.layers[i] = static_cast<int>(t[3]);
    layers = std::max(layers, p.layers[i]);
  }
  if (layers <= 0) return 0;
  p.src = src;
  p.dst = dst;
  p.num_pages = num_pages;
  p.status = status;
  const cudaError_t e = launch_pdl(copy_pages_kernel, dim3(pairs, layers, count), dim3(256), 0, stream, p);
  eredu_count_launches(1);
  return static_cast<int>(e);
}
