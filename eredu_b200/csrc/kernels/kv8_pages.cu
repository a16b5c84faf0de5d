// Pages of a cache held in 8 bits (common/kv8.cuh): rows are written, values read back, and pages of any cache copied.
#include <algorithm>

#include "../common/kv8_args.h"
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
// values (16 x 128 / 128 values a thread), find the largest together and store the codes: one read. The angles of a tile of rows are computed once for
// the head's keys and its query heads. Short chains of dependent reads and few instructions a row decide the time: queries and rows of the first run are asked for ahead of
// the angles, those of the next run ahead of this one's codes, and a lane has both halves of a rotation.
// 4096 rows, 32 heads of 128 over 8 (92 MB): 19.8 us, 4.7 TB/s (into bf16 pages, 100 MB, 17.0); a warp to a run's keys, in 128 registers, 92; partners of a rotation by
// shuffles 26.2; queries and runs not ahead 24.4; three CTAs an SM 22.9 before the runs were. Five runs of 39 to 77 rows, head size 64: 5.1.
constexpr int kStoreThreads = 256, kStoreShare = kStoreThreads / 64;   // half of the warps for keys, half for values
constexpr int kStoreRoom = 3 * 148;  // CTAs beyond which tiles of more rows are taken (256 rows over 8 heads: 4.1 us with tiles of 8, of 4 5.3, of 1 9.4)
constexpr int kStoreRows = 32;      // a tile of 16 rows and what the last run of it has behind them

// grid (tiles of rows, n_kv)
template <int D, bool WHOLE>
__global__ void __launch_bounds__(kStoreThreads, 4) kv8_store_kernel(Kv8StoreParams p) {
  using Rows = Kv8Rows<D, WHOLE>;
  constexpr int PER = Rows::PER, SHARED = Rows::ROWS * kStoreShare, STEPS = kKv8Page / SHARED;   // rows that the warps of a run hold at once, and how often
  extern __shared__ __align__(16) float turns[];          // [rows of the tile and the last run][rot / 2 cosines, rot / 2 sines]
  __shared__ uint32_t tops[2][kStoreShare];
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = blockIdx.x * p.tile, rows = min(p.tile, p.M - row0), h0 = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rot = WHOLE ? D : p.rot, half = rot / 2;
  // lane r has the slots of rows r - 1 and r of the tile and the 16 behind it: a row continues the one in front where its slot is the next of the same page
  const bool known = row0 + lane < p.M && lane < rows + kKv8Page;
  const long long slot = known ? p.slots[row0 + lane] : -1, front = known && row0 + lane > 0 ? p.slots[row0 + lane - 1] : -1;
  // ---- query rows of this head, a warp has DEEP (times as many as it holds at once) on their way
  constexpr int DEEP = 4, STRIDE = kStoreThreads / 32 * Rows::ROWS;
  const int mine = p.q_out == nullptr ? 1 : p.n_q / p.n_kv, items = p.q_out == nullptr ? 0 : rows * mine, sub = Rows::row(lane);
  const uint32_t per_mine = ((1u << 20) + mine - 1) / mine;     // item / mine by a product: exact below 2^20 / mine, and there are 16 mine of them at most
  uint2 query[DEEP][PER];
  auto load_queries = [&](int i0) {
#pragma unroll
    for (int j = 0; j < DEEP; ++j) {
      const int item = min(i0 + j * STRIDE + sub, items - 1), r = static_cast<int>(item * per_mine >> 20);
      const __nv_bfloat16* from = p.q + static_cast<size_t>(row0 + r) * p.ld_q + (h0 * mine + item - r * mine) * D;
#pragma unroll
      for (int i = 0; i < PER; ++i) query[j][i] = *reinterpret_cast<const uint2*>(from + Rows::channel(lane, i));
    }
  };
  if (warp * Rows::ROWS < items) load_queries(warp * Rows::ROWS);
  // ---- the tile's runs, by every warp for itself: bits of `begin`; their first lanes have length and slot
  const bool follows = slot >= 0 && (slot & 15) != 0 && front == slot - 1;
  bool begins = lane < rows && slot >= 0 && !follows;
  if (begins && (slot >> 4) >= p.num_pages) {
    report_status(p.status, kStatusBadArgument);
    begins = false;
  }
  uint32_t begin = __ballot_sync(0xffffffffu, begins);
  const uint32_t more = __ballot_sync(0xffffffffu, follows);
  // (a tile of 16 rows and 15 more at most: what follows the last row of the warp's 32 cannot belong to a run of this tile)
  const int length = begins ? __ffs(~(more >> lane >> 1)) : 0;
  const int behind = max(rows, __reduce_max_sync(0xffffffffu, begins ? lane + length : 0));
  // ---- a run: half of the warps have its keys, half its values
  const bool keys = warp < kStoreShare;
  const int part = keys ? warp : warp - kStoreShare, mine0 = sub + part * Rows::ROWS, ld = keys ? p.ld_k : p.ld_v;
  const __nv_bfloat16* src = (keys ? p.k : p.v) + static_cast<size_t>(row0) * ld + h0 * D;
  uint2 raw[STEPS][PER];
  int at = 0, n = 0, first = 0;
  size_t cell = 0;
  float before = 0.f;
  auto next_run = [&]() {
    at = __ffs(begin) - 1;
    begin &= begin - 1;
    n = __shfl_sync(0xffffffffu, length, at);
    const long long to = __shfl_sync(0xffffffffu, slot, at);
    first = static_cast<int>(to & 15);
    cell = static_cast<size_t>(to >> 4) * p.n_kv + h0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int r = i * SHARED + mine0;
#pragma unroll
      for (int j = 0; j < PER; ++j) raw[i][j] = r < n ? *reinterpret_cast<const uint2*>(src + static_cast<size_t>(at + r) * ld + Rows::channel(lane, j)) : make_uint2(0, 0);
    }
    before = first > 0 ? (keys ? p.k_scales : p.v_scales)[cell] : 0.f;
  };
  bool left = begin != 0;
  if (left) next_run();
  for (int r = threadIdx.x / (D / 2), i = threadIdx.x % (D / 2); r < behind; r += kStoreThreads / (D / 2))
    if (i < half) turn_of(p.positions[row0 + r], p.inv_freq[i], p.attn_factor, turns[r * rot + i], turns[r * rot + half + i]);
  __syncthreads();
  while (left) {
    const int at_now = at, n_now = n, first_now = first;
    const float before_now = before;
    int8_t* codes = (keys ? p.k_codes : p.v_codes) + cell * (kKv8Page * D);
    float* scale_at = (keys ? p.k_scales : p.v_scales) + cell;
    Rows held[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) held[i].take(raw[i]);
    left = begin != 0;
    if (left) next_run();
    uint32_t top = 0;   // as bits, so that what is no number wins
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (i * SHARED + part * Rows::ROWS >= n_now) break;
      if (keys) held[i].prepare(p, p.k_norm_w, turns + (at_now + min(i * SHARED + mine0, n_now - 1)) * rot, lane);   // (rows behind the last are zero: they stay so)
#pragma unroll
      for (int j = 0; j < PER; ++j) top = kv8_top(top, held[i].x[j]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[keys ? 0 : 1][part] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kStoreShare; ++i) top = max(top, tops[keys ? 0 : 1][i]);
    const float scale = kv8_raised(top, first_now, before_now), inv = kv8_inverse(scale);
    if (first_now > 0 && scale != before_now) {
      const float ratio = before_now * inv;
      for (int r = mine0; r < first_now; r += SHARED) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          uint32_t* w = reinterpret_cast<uint32_t*>(codes + r * D + Rows::channel(lane, j));
          const uint32_t u = *w;
          *w = kv8_pack(kv8_code(u, 0), kv8_code(u, 1), kv8_code(u, 2), kv8_code(u, 3), ratio);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int r = i * SHARED + mine0;
      if (r >= n_now) continue;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float4 x = held[i].x[j];
        *reinterpret_cast<uint32_t*>(codes + (first_now + r) * D + Rows::channel(lane, j)) = kv8_pack(x.x, x.y, x.z, x.w, inv);
      }
    }
    if (lane == 0 && part == 0) *scale_at = scale;
    if (left) __syncthreads();   // the next run's words
  }
  for (int i0 = warp * Rows::ROWS; i0 < items; i0 += STRIDE * DEEP) {
    if (i0 >= STRIDE * DEEP) load_queries(i0);
#pragma unroll
    for (int j = 0; j < DEEP; ++j) {
      const int item = i0 + j * STRIDE + sub, r = static_cast<int>(min(item, items - 1) * per_mine >> 20), head = h0 * mine + min(item, items - 1) - r * mine;
      if (i0 + j * STRIDE >= items) break;
      Rows x;
      x.take(query[j]);
      x.prepare(p, p.q_norm_w, turns + r * rot, lane);
      if (item >= items) continue;
      const size_t at = (static_cast<size_t>(row0 + r) * p.n_q + head) * D;
#pragma unroll
      for (int i = 0; i < Rows::PER; ++i) {
        const float4 y = x.x[i];
        if (p.q_out_fp32) *reinterpret_cast<float4*>(static_cast<float*>(p.q_out) + at + Rows::channel(lane, i)) = y;
        else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.q_out) + at + Rows::channel(lane, i)) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
      }
    }
  }
}

// ============================================================================ values of pages
// Codes times scale as bf16 (exact: 8 significant bits): [entries, n_kv, 16, D] for keys and for values. The pages are a list, or (seq_lens given)
// the rows of a block table: then entries that no query of the sequence sees are left out, and `table_out` [rows, wide] says where each one is - those left out
// lie behind the last one, where a tensor map reads zeros. With `entries` the rows of the table follow one another without what is left out: the memory is the
// sum of what sequences see, not as many times the longest as there are sequences, and every CTA adds up the rows in front of its own (two numbers each, 256 at once).
// One byte in, two out, bound by memory: 8192 tokens of 8 heads of 128, 7.6 us (50 MB, 6.6 TB/s).
struct Kv8ValuesParams {
  const int8_t *k_codes, *v_codes;
  const float *k_scales, *v_scales;
  __nv_bfloat16 *k_out, *v_out;
  const int* pages;        // [rows of `pitch`]
  const int* seq_lens;     // optional [rows]
  const int* cu_q;         // with seq_lens: query offsets
  int* table_out;          // with seq_lens: [rows, wide]
  int pitch, table_wide, wide, n_kv, num_pages, window, chunk;   // table_wide: entries of a row of `pages`; wide: of a row of the output
  int entries;             // with seq_lens: entries that the output has room for, where rows follow one another; 0: rows of `wide`
  int* status;
};
constexpr int kValuesThreads = 256;
// Entries [first, end) of a row that one of its sequence's queries sees.
__device__ __forceinline__ int2 seen_entries(const Kv8ValuesParams& p, int row) {
  const int len = p.seq_lens[row], first = len - (p.cu_q[row + 1] - p.cu_q[row]);
  if (first >= len || len <= 0) return make_int2(0, 0);
  const int low = p.window > 0 ? max(0, first - p.window + 1) : p.chunk > 0 && first > 0 ? first - first % p.chunk : 0;
  const int end = min(min((len - 1) / kKv8Page + 1, p.wide), p.table_wide);
  return make_int2(min(low / kKv8Page, end), end);
}
template <int D>
__global__ void __launch_bounds__(kValuesThreads) kv8_values_kernel(Kv8ValuesParams p) {
  constexpr int BLOCK = kKv8Page * D, DEEP = 4;   // codes of a block; pieces of eight codes a thread has on their way
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, i = blockIdx.x;
  size_t entry = static_cast<size_t>(row) * p.wide + i;
  if (p.seq_lens != nullptr) {
    const size_t place = entry;
    const int2 mine = seen_entries(p, row);
    bool seen = i >= mine.x && i < mine.y;      // (for all of the CTA)
    if (seen && p.entries > 0) {
      __shared__ int parts[kValuesThreads / 32];
      int front = 0;
      for (int r = threadIdx.x; r < row; r += kValuesThreads) {
        const int2 other = seen_entries(p, r);
        front += other.y - other.x;
      }
      front = __reduce_add_sync(0xffffffffu, front);
      if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = front;
      __syncthreads();
      entry = i - mine.x;
#pragma unroll
      for (int w = 0; w < kValuesThreads / 32; ++w) entry += parts[w];
      if (entry >= static_cast<size_t>(p.entries)) {      // sequences are longer than the caller has said
        if (threadIdx.x == 0) report_status(p.status, kStatusBadArgument);
        seen = false;
      }
    }
    if (threadIdx.x == 0 && blockIdx.z == 0) p.table_out[place] = static_cast<int>(seen ? entry : p.entries > 0 ? static_cast<size_t>(p.entries) : static_cast<size_t>(gridDim.y) * p.wide);
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
// A CTA copies a page of one layer and tensor, 16 bytes a thread at a time. 2000 pages of 16 layers, 2.1 GB read and written: 318 us, the rate of a copy (6.6 TB/s).
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

int eredu::kv8_store(const Kv8StoreArgs& a) {
  const int M = a.M, n_kv = a.n_kv, rot = a.rot;
  if (M <= 0) return 0;
  if ((a.D != 64 && a.D != 128) || n_kv <= 0 || a.num_pages <= 0 || rot < 0 || rot > a.D || rot % 8 != 0 || a.ld_q % 4 != 0 || a.ld_k % 4 != 0 || a.ld_v % 4 != 0 ||
      (a.q_out != nullptr && (a.n_q <= 0 || a.n_q % n_kv != 0 || a.n_q / n_kv > 256)))
    return -2;
  Kv8StoreParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.k = static_cast<const __nv_bfloat16*>(a.k);
  p.v = static_cast<const __nv_bfloat16*>(a.v);
  p.q_out = a.q_out;
  p.q_out_fp32 = a.q_out_fp32;
  p.k_codes = static_cast<int8_t*>(a.k_codes);
  p.v_codes = static_cast<int8_t*>(a.v_codes);
  p.k_scales = a.k_scales;
  p.v_scales = a.v_scales;
  p.positions = a.positions;
  p.slots = a.slots;
  p.inv_freq = a.inv_freq;
  p.q_norm_w = a.q_norm_w;
  p.k_norm_w = a.k_norm_w;
  p.M = M;
  p.ld_q = a.ld_q;
  p.ld_k = a.ld_k;
  p.ld_v = a.ld_v;
  p.n_q = a.n_q;
  p.n_kv = n_kv;
  p.rot = rot;
  p.interleaved = a.interleaved;
  p.num_pages = a.num_pages;
  p.attn_factor = a.attn_factor;
  p.norm_eps = a.norm_eps;
  p.norm_w_off = a.norm_w_off;
  p.status = a.status;
  // a key / value head with its query heads per CTA, and as few rows as find room at once
  p.tile = 1;
  while (p.tile < kKv8Page && static_cast<long long>((M + p.tile - 1) / p.tile) * n_kv > kStoreRoom) p.tile *= 2;
  const dim3 grid((M + p.tile - 1) / p.tile, n_kv);
  const size_t smem = static_cast<size_t>(kStoreRows) * rot * sizeof(float);
  const bool whole = rot == a.D && a.interleaved == 0;
  const cudaError_t e = a.D == 128 ? (whole ? launch_pdl(kv8_store_kernel<128, true>, grid, dim3(kStoreThreads), smem, a.stream, p)
                                            : launch_pdl(kv8_store_kernel<128, false>, grid, dim3(kStoreThreads), smem, a.stream, p))
                                   : (whole ? launch_pdl(kv8_store_kernel<64, true>, grid, dim3(kStoreThreads), smem, a.stream, p)
                                            : launch_pdl(kv8_store_kernel<64, false>, grid, dim3(kStoreThreads), smem, a.stream, p));
  eredu_count_launches(1);
  return static_cast<int>(e);
}

extern "C" int eredu_kv8_store(const void* args, int bytes) {
  Kv8StoreArgs a;
  return kv8_args(a, args, bytes) ? kv8_store(a) : -2;
}

extern "C" int eredu_kv8_values(const void* args, int bytes) {
  Kv8ValuesArgs a;
  if (!kv8_args(a, args, bytes)) return -2;
  if (a.rows <= 0 || a.wide <= 0) return 0;
  if ((a.D != 64 && a.D != 128) || a.n_kv <= 0 || a.rows > 65535 || a.num_pages <= 0 || a.entries < 0) return -2;
  Kv8ValuesParams p = {};
  p.k_codes = static_cast<const int8_t*>(a.k_codes);
  p.v_codes = static_cast<const int8_t*>(a.v_codes);
  p.k_scales = a.k_scales;
  p.v_scales = a.v_scales;
  p.k_out = static_cast<__nv_bfloat16*>(a.k_out);
  p.v_out = static_cast<__nv_bfloat16*>(a.v_out);
  p.pages = a.pages;
  p.seq_lens = a.seq_lens;
  p.cu_q = a.cu_q;
  p.table_out = a.table_out;
  p.pitch = a.pitch;
  p.wide = a.wide;
  p.table_wide = a.table_wide;
  p.n_kv = a.n_kv;
  p.num_pages = a.num_pages;
  p.window = a.window;
  p.chunk = a.chunk;
  p.entries = a.entries;
  p.status = a.status;
  const cudaError_t e = a.D == 128 ? launch_pdl(kv8_values_kernel<128>, dim3(a.wide, a.rows, 2), dim3(kValuesThreads), 0, a.stream, p)
                                   : launch_pdl(kv8_values_kernel<64>, dim3(a.wide, a.rows, 2), dim3(kValuesThreads), 0, a.stream, p);
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
