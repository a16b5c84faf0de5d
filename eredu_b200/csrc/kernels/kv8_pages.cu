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
// A run is a stretch of rows that follow one another in one page; its rows share a scale per head, so one warp holds all of a run's rows of a
// head in registers (16 x 128 / 32 values a lane), finds the largest and stores the codes: one read, no shared memory. A lane has four
// neighbouring values of a row; the partner of a rotation sits `rot / 8` lanes further. The angles of a tile of rows are computed once for all heads.
constexpr int kStoreThreads = 256;
constexpr int kStoreRows = 32;      // a tile of 16 rows and what the last run of it has behind them

// grid (tiles of rows, groups of key / value heads)
template <int D>
__global__ void __launch_bounds__(kStoreThreads) kv8_store_kernel(Kv8StoreParams p, int heads) {
  constexpr int RPI = 128 / D;
  extern __shared__ float2 turns[];          // [rows of the tile and the last run][rot / 2]
  __shared__ int run_row[kKv8Page], run_len[kKv8Page];
  __shared__ int runs, behind;
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = blockIdx.x * p.tile, rows = min(p.tile, p.M - row0);
  const int h0 = blockIdx.y * heads, hn = min(heads, p.n_kv - h0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = p.rot / 2;
  if (warp == 0) {
    // lane r < 16: row r of the tile; its run, where it begins one
    const int r = row0 + lane;
    const bool in = lane < rows;
    const long long slot = in ? p.slots[r] : -1;
    bool begins = in && slot >= 0 && (r == 0 || (slot & 15) == 0 || p.slots[r - 1] != slot - 1);
    if (begins && (slot >> 4) >= p.num_pages) {
      report_status(p.status, kStatusBadArgument);
      begins = false;
    }
    int n = begins ? 1 : 0;
    if (begins)
      while (n < kKv8Page - static_cast<int>(slot & 15) && r + n < p.M && p.slots[r + n] == slot + n) ++n;
    const uint32_t mask = __ballot_sync(0xffffffffu, begins);
    if (begins) {
      const int i = __popc(mask & ((1u << lane) - 1));
      run_row[i] = lane;
      run_len[i] = n;
    }
    const int end = __reduce_max_sync(0xffffffffu, begins ? lane + n : 0);
    if (lane == 0) {
      runs = __popc(mask);
      behind = max(rows, end);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < behind * half; i += kStoreThreads)
    turns[i] = turn_of(p.positions[row0 + i / half], p.inv_freq[i % half], p.attn_factor);
  __syncthreads();
  for (int i = warp; i < runs * hn * 2; i += kStoreThreads / 32) {
    const int run = i / (2 * hn), h = h0 + (i >> 1) % hn;
    const int at = run_row[run], row = row0 + at, n = run_len[run];
    const long long slot = p.slots[row], cell = (slot >> 4) * p.n_kv + h;
    if ((i & 1) == 0) store_block<D, true>(p, row, n, static_cast<int>(slot & 15), cell, h, turns + at * half, lane);
    else store_block<D, false>(p, row, n, static_cast<int>(slot & 15), cell, h, turns, lane);
  }
  if (p.q_out == nullptr) return;
  const int group = p.n_q / p.n_kv, mine = hn * group;     // query heads of this CTA
  const int sub = RPI == 1 ? 0 : lane >> 4;
  for (int i = warp * RPI; i < rows * mine; i += kStoreThreads / 32 * RPI) {
    const int item = min(i + sub, rows * mine - 1), r = item / mine, head = h0 * group + item % mine;
    const size_t row = row0 + r;
    const float4 x = prepared<D>(p, load_row4<D>(p.q + row * p.ld_q + head * D, lane), p.q_norm_w, turns + r * half, lane);
    if (i + sub < rows * mine)
      *reinterpret_cast<uint2*>(p.q_out + (row * p.n_q + head) * D + 4 * (lane & (D / 4 - 1))) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
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
  int pitch, wide, n_kv, block, num_pages, window, chunk;   // block = 16 D
  int* status;
};
__global__ void __launch_bounds__(256) kv8_values_kernel(Kv8ValuesParams p) {
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, i = blockIdx.x;
  const size_t entry = static_cast<size_t>(row) * p.wide + i;
  if (p.seq_lens != nullptr) {
    const int len = p.seq_lens[row], first = len - (p.cu_q[row + 1] - p.cu_q[row]);
    const int low = p.window > 0 ? first - p.window + 1 : p.chunk > 0 && first > 0 ? first - first % p.chunk : 0;
    const bool seen = i * kKv8Page < len && i * kKv8Page + kKv8Page > low && first < len && i < p.pitch;
    if (threadIdx.x == 0 && blockIdx.z == 0) p.table_out[entry] = static_cast<int>(seen ? entry : static_cast<size_t>(gridDim.y) * p.wide);
    if (!seen) return;
  }
  int page = p.pages[static_cast<size_t>(row) * p.pitch + i];
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) report_status(p.status, kStatusBadArgument);
    page = 0;
  }
  const int8_t* codes = (blockIdx.z == 0 ? p.k_codes : p.v_codes) + static_cast<size_t>(page) * p.n_kv * p.block;
  const float* scales = (blockIdx.z == 0 ? p.k_scales : p.v_scales) + static_cast<size_t>(page) * p.n_kv;
  __nv_bfloat16* out = (blockIdx.z == 0 ? p.k_out : p.v_out) + entry * p.n_kv * p.block;
  for (int c = threadIdx.x * 16; c < p.n_kv * p.block; c += 256 * 16) {
    const uint4 u = *reinterpret_cast<const uint4*>(codes + c);
    const float s = scales[c / p.block];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[2 * j] = pack_bf16x2(kv8_code(w[j], 0) * s, kv8_code(w[j], 1) * s);
      o[2 * j + 1] = pack_bf16x2(kv8_code(w[j], 2) * s, kv8_code(w[j], 3) * s);
    }
    *reinterpret_cast<uint4*>(out + c) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(o[4], o[5], o[6], o[7]);
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
                               int ld_q, int ld_k, int ld_v, int n_q, int n_kv, int D, int rot, int interleaved, int num_pages, float attn_factor,
                               float norm_eps, float norm_w_off, int* status, cudaStream_t stream) {
  if (M <= 0) return 0;
  if ((D != 64 && D != 128) || n_kv <= 0 || num_pages <= 0 || rot < 0 || rot > D || rot % 8 != 0 || ld_q % 4 != 0 || ld_k % 4 != 0 || ld_v % 4 != 0 ||
      (q_out != nullptr && (n_q <= 0 || n_q % n_kv != 0)))
    return -2;
  Kv8StoreParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
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
  // few rows: a row and a head per CTA; many: a tile of 16 rows, in which most runs are whole, and all heads
  const bool few = M <= 256;
  p.tile = few ? 1 : 16;
  const int heads = few ? 1 : n_kv;
  const dim3 grid((M + p.tile - 1) / p.tile, (n_kv + heads - 1) / heads);
  const size_t smem = static_cast<size_t>(kStoreRows) * (rot / 2) * sizeof(float2);
  const cudaError_t e = D == 128 ? launch_pdl(kv8_store_kernel<128>, grid, dim3(kStoreThreads), smem, stream, p, heads)
                                 : launch_pdl(kv8_store_kernel<64>, grid, dim3(kStoreThreads), smem, stream, p, heads);
  eredu_count_launches(1);
  return static_cast<int>(e);
}

extern "C" int eredu_kv8_values(const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales, void* k_out, void* v_out,
                                const int* pages, const int* seq_lens, const int* cu_q, int* table_out, int rows, int pitch, int wide, int n_kv, int D,
                                int num_pages, int window, int chunk, int* status, cudaStream_t stream) {
  if (rows <= 0 || wide <= 0) return 0;
  if (D % 16 != 0 || n_kv <= 0 || rows > 65535 || num_pages <= 0) return -2;
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
  p.n_kv = n_kv;
  p.block = kKv8Page * D;
  p.num_pages = num_pages;
  p.window = window;
  p.chunk = chunk;
  p.status = status;
  const cudaError_t e = launch_pdl(kv8_values_kernel, dim3(wide, rows, 2), dim3(256), 0, stream, p);
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
