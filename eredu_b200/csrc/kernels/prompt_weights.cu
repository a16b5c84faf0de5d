// The weight that the rows of a prompt, or of a portion of one, give to every cached token: for each key / value head the sum over rows and over the
// query heads that share it of 2^(s - lse), where s is a score in powers of two and lse the logarithm of its row's sum, which the attention kernel
// (attention_tc.cu) has left. Tokens of the call's own rows are set, older ones added to.
//
// The sum runs over the rows of a column, so the scores are taken as S^T = K Q^T: a tensor-memory lane is a key, and a thread adds up what lies in its
// lane without any exchange. A CTA has 256 keys of one head (two tiles of 128, resident), and the rows that see them come by in tiles of 128:
// 128 / 2^gshift tokens of 2^gshift query heads, so that few tokens of many heads fill a tile as well.
//   warp 0      : TMA producer - both key tiles once (sixteen pages), then tiles of query rows through a ring, and beside them the rows' -lse (-inf where a row
//                 does not count) as three bf16 pieces of 24 bits in all
//   warp 1      : MMA issuer - two accumulators for each key tile, so that the tensor core runs ahead. One step more along K, ones by those pieces, takes lse off the scores:
//                 read from shared memory it cost every thread 512 bytes a tile
//   warps 2..5  : sums of key tile a, warps 6..9 of tile b: a score row comes to registers in halves, the next one asked for while one is added up: a product and an
//                 exponential for each score (products of two at once were slower: 4096 tokens 254 -> 244 us), one addition for two
// The CTAs of a cluster share the rows of the same keys; their sums are added up in the order of their ranks.
//
// Bound by exponentials, 2048 cycles of the special-function unit for a pair of tiles (the tensor core needs 1050), and by what each tile costs beside them: 4096 tokens, 32 heads
// of 128 over 8, 101 us of the 240 that the call takes, 61 at the unit's rate. Left out in a copy for the time's sake, the exponentials take 32 us of it, the products of the tensor core 6;
// 60 are tiles without arithmetic - accumulators read, barriers - and 12 the start and the end of a CTA (one to an SM). Tiles of 64 rows with two CTAs to an SM measured
// the same (257 -> 263 us before the steps above; 2048 tokens 91 -> 94), an issuer for each key tile 243 for 244, old sums asked for by the producer 240 for 240.
#include <cuda_bf16.h>

#include <algorithm>

#include "../common/launch.h"
#include "../common/launch_count.h"
#include "../common/ptx.cuh"
#include "../common/tma_host.h"
#include "../common/weights_args.h"

namespace eredu {

constexpr int kPwThreads = 320;
constexpr int kPwTile = 128;                 // keys, and rows, of a tile
constexpr int kPwKeys = 2 * kPwTile;         // keys of a CTA
constexpr int kPwHalf = kPwTile * 64 * 2;    // one [128][64] half tile
constexpr int kPwStages = 4;
constexpr int kPwPage = 16;
constexpr int kPwCluster = 8;

struct PwParams {
  const float* lse;
  const int *block_table, *seq_lens, *cu_q;
  float* weights;
  int* status;
  int wide, num_pages, n_q, n_kv, group, gshift, window, observed;
  float scale_log2, unscale;   // and 1 / scale_log2
};

// shared memory: key tiles a, b (NK halves each) | query ring | ones | lse ring | sums of the keys | barriers
constexpr int kPwExtra = kPwTile * 16 * 2;   // a tile [128][16] of the step that brings the rows' lse
// (more than half of an SM's in any case: a CTA has all of its tensor memory, and one that waited for a neighbour's while its own cluster waits for it would never get it)
constexpr int pw_smem(int nk) { return std::max(120 * 1024, 1024 + (2 * nk + kPwStages * nk) * kPwHalf + (1 + kPwStages) * kPwExtra + kPwKeys * 4 + 256); }

// Operand [rows][16] without swizzle: blocks of eight rows of 16 bytes (128 bytes each), the two of a row side by side along K.
__device__ __forceinline__ uint64_t pw_desc_plain(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 16;            // along K: 128 bytes
  d |= static_cast<uint64_t>(256 >> 4) << 32;            // eight rows on: 256 bytes
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}
__device__ __forceinline__ int pw_plain(int row, int col) { return (row >> 3) * 256 + (col >> 3) * 128 + (row & 7) * 16 + (col & 7) * 2; }
// Uses of the registers stay behind the wait in front of this.
__device__ __forceinline__ void pw_settled(uint32_t (&r)[4][16]) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    asm volatile("" : "+r"(r[c][0]), "+r"(r[c][1]), "+r"(r[c][2]), "+r"(r[c][3]), "+r"(r[c][4]), "+r"(r[c][5]), "+r"(r[c][6]), "+r"(r[c][7]), "+r"(r[c][8]),
                 "+r"(r[c][9]), "+r"(r[c][10]), "+r"(r[c][11]), "+r"(r[c][12]), "+r"(r[c][13]), "+r"(r[c][14]), "+r"(r[c][15]));
}

__device__ __forceinline__ void pw_load_page(void* dst, const CUtensorMap* map, int x, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(0), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

template <int NK>
__global__ void __launch_bounds__(kPwThreads, 1) prompt_weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const PwParams p) {
  extern __shared__ __align__(1024) uint8_t pw_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pw_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* k_s = smem;
  uint8_t* q_s = k_s + 2 * NK * kPwHalf;
  uint8_t* one_s = q_s + kPwStages * NK * kPwHalf;
  uint8_t* lse_s = one_s + kPwExtra;
  float* sum_s = reinterpret_cast<float*>(lse_s + kPwStages * kPwExtra);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sum_s + kPwKeys);
  uint64_t* k_full = bars;                               // 1
  uint64_t* q_full = bars + 1;                           // [stages]: bytes, and the 32 lanes that wrote lse
  uint64_t* q_empty = q_full + kPwStages;                // [stages]: the MMA's commit
  uint64_t* s_full = q_empty + kPwStages;                // [tile][2]
  uint64_t* s_empty = s_full + 4;                        // [tile][2], 128 arrivals
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_empty + 4);

  pdl_launch_early();
  const int warp = static_cast<int>(warp_uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  int ranks, rank;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  ranks = static_cast<int>(warp_uniform(ranks));
  rank = static_cast<int>(warp_uniform(rank));
  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    for (int s = 0; s < kPwStages; ++s) {
      mbar_init(&q_full[s], 1 + 32);
      mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 128);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
  }
  // the step's A operand is three ones a key, its B operand what is left in three pieces; columns behind them are zero on both sides
  for (int i = threadIdx.x; i < (1 + kPwStages) * kPwExtra / 16; i += kPwThreads) reinterpret_cast<uint4*>(one_s)[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  for (int i = threadIdx.x; i < kPwTile; i += kPwThreads) *reinterpret_cast<uint2*>(one_s + pw_plain(i, 0)) = make_uint2(0x3F803F80u, 0x3F80u);
  fence_proxy_async_smem();
  pdl_wait();

  // (blocks of keys vary slowest: the first ones are seen by the most rows)
  const int h = static_cast<int>(blockIdx.x) / ranks, b = blockIdx.y, key0 = blockIdx.z * kPwKeys;
  const int q0 = static_cast<int>(warp_uniform(p.cu_q[b])), q_len = static_cast<int>(warp_uniform(p.cu_q[b + 1])) - q0;
  const int n = static_cast<int>(warp_uniform(p.seq_lens[b])), kv_len = min(n, p.wide * kPwPage);
  if ((n > kv_len || kv_len > static_cast<int>(gridDim.z) * kPwKeys) && threadIdx.x == 0) report_status(p.status, kStatusBadArgument);
  const int before = kv_len - q_len;                                    // tokens in front of the call's own
  // query tokens [t0, t1) that count and see some of this CTA's keys
  int t0 = p.observed > 0 ? max(0, q_len - p.observed) : 0, t1 = q_len;
  t0 = max(t0, key0 - before);
  if (p.window > 0) t1 = min(t1, key0 + kPwKeys - 1 - before + p.window);
  const int tile_tokens = kPwTile >> p.gshift, per_head = max(0, t1 - t0 + tile_tokens - 1) / tile_tokens;
  const int tiles = key0 < kv_len ? per_head * (p.group >> p.gshift) : 0;
  const int begin = static_cast<int>(static_cast<long long>(tiles) * rank / ranks), end = static_cast<int>(static_cast<long long>(tiles) * (rank + 1) / ranks);
  // nothing to do (the same for all CTAs of a cluster): behind the sequence's last token, or older tokens that no row sees
  if (key0 >= kv_len || q_len <= 0 || (tiles == 0 && key0 + kPwKeys <= before)) return;
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = warp_uniform(*tmem_slot);
  pdl_launch_dependents();                               // (behind the allocation: what comes next may want tensor memory too)
  // (tile i of the CTA: tokens from t0 + i / heads on, heads varying fastest, so that CTAs of one head read the same rows at about the same time)
  const int head_tiles = p.group >> p.gshift;

  bool ok = true;
  float total = 0.f;
  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    const bool one = elect_one();
    if (begin < end) {
      const int entry = key0 / kPwPage + (lane & 15);
      int page = entry < p.wide && entry * kPwPage < kv_len ? p.block_table[static_cast<size_t>(b) * p.wide + entry] : 0;
      if (page < 0 || page >= p.num_pages) {
        report_status(p.status, kStatusBadArgument);
        page = 0;
      }
      if (one) mbar_arrive_expect_tx(k_full, 2 * NK * kPwHalf);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int pg = __shfl_sync(0xffffffffu, page, i);
        if (one)
          for (int x = 0; x < NK; ++x) pw_load_page(k_s + ((i >> 3) * NK + x) * kPwHalf + (i & 7) * 2048, &tmK, x * 64, h, pg, k_full);
      }
      for (int i = begin; i < end; ++i) {
        const int it = i - begin, s = it % kPwStages;
        const int token = t0 + i / head_tiles * tile_tokens, head = h * p.group + (i % head_tiles << p.gshift);
        // rows of this tile: lane l has columns l, l + 32, ..
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = lane + 32 * j, t = token + (c >> p.gshift);
          v[j] = t < q_len ? -p.lse[static_cast<size_t>(q0 + t) * p.n_q + head + (c & ((1 << p.gshift) - 1))] * p.unscale : -INFINITY;
          if (v[j] == INFINITY) v[j] = -INFINITY;                       // a row that saw nothing gives nothing
        }
        if (it >= kPwStages) ok = mbar_wait_warp(&q_empty[s], (it / kPwStages - 1) & 1, p.status, kStatusSmemEmptyTimeout);
        if (!ok) break;
        if (one) {
          mbar_arrive_expect_tx(&q_full[s], NK * kPwHalf);
          for (int x = 0; x < NK; ++x) tma_load_3d(q_s + (s * NK + x) * kPwHalf, &tmQ, x * 64, head, q0 + token, &q_full[s]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // 24 bits in three pieces of eight
          const float high = __bfloat162float(__float2bfloat16(v[j])), rest = high == -INFINITY ? 0.f : v[j] - high;
          const float mid = __bfloat162float(__float2bfloat16(rest));
          *reinterpret_cast<uint2*>(lse_s + s * kPwExtra + pw_plain(lane + 32 * j, 0)) = make_uint2(pack_bf16x2(high, mid), pack_bf16x2(rest - mid, 0.f));
        }
        fence_proxy_async_smem();
        mbar_arrive(&q_full[s]);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const bool one = elect_one();
    constexpr uint32_t idesc = umma_idesc_bf16(kPwTile, kPwTile);
    if (begin < end) ok = mbar_wait_warp(k_full, 0, p.status, kStatusTmaFullTimeout);
    for (int i = begin; i < end && ok; ++i) {
      const int it = i - begin, s = it % kPwStages, buf = it & 1;
      ok = mbar_wait_warp(&q_full[s], (it / kPwStages) & 1, p.status, kStatusTmaFullTimeout);
      for (int w = 0; w < 2 && ok; ++w) {
        if (it >= 2) ok = mbar_wait_warp(&s_empty[w * 2 + buf], ((it >> 1) - 1) & 1, p.status, kStatusAccumTimeout);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t ka = smem_u32(k_s + w * NK * kPwHalf), qa = smem_u32(q_s + s * NK * kPwHalf), d = tmem + (w * 2 + buf) * kPwTile;
        if (one) {
#pragma unroll
          for (int kk = 0; kk < NK * 4; ++kk) {
            const uint32_t off = (kk >> 2) * kPwHalf + (kk & 3) * 32;
            umma_f16(d, umma_desc_k_sw128(ka + off), umma_desc_k_sw128(qa + off), idesc, kk > 0 ? 1u : 0u);
          }
          umma_f16(d, pw_desc_plain(smem_u32(one_s)), pw_desc_plain(smem_u32(lse_s + s * kPwExtra)), idesc, 1u);
          umma_commit(&s_full[w * 2 + buf]);
          if (w == 1) umma_commit(&q_empty[s]);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ sums, one key per thread
    const int w = (warp - 2) >> 2, quarter = warp & 3;
    const int key = key0 + w * kPwTile + quarter * 32 + lane;
    const int tile_first = key0 + w * kPwTile, tile_last = min(kv_len, tile_first + kPwTile) - 1;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    uint64_t acc[4] = {0ull, 0ull, 0ull, 0ull};
    // the first column and the one behind the last of a tile that see this thread's key; all of them where no row or key of the tile is at an edge
    auto seen = [&](int i, int& low, int& high) {
      const int token = t0 + i / head_tiles * tile_tokens, pos = before + token;     // positions of the tile's rows: [pos, pos + tile_tokens)
      low = 0;
      high = kPwTile;
      const bool edge = pos < tile_last || token + tile_tokens > q_len || (p.window > 0 && pos + tile_tokens - 1 >= tile_first + p.window);
      if (edge) {
        const int high_t = p.window > 0 ? min(q_len, key - before + p.window) : q_len;
        low = (key - pos) * (1 << p.gshift);
        high = (high_t - token) * (1 << p.gshift);
      }
      return edge;
    };
    auto add = [&](const uint32_t (&sc)[4][16], int first, bool edge, int low, int high) {
      if (edge) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int col = first + c * 16 + e;
            const float v = ex2_approx(__uint_as_float(sc[c][e]) * p.scale_log2);
            total += col >= low && col < high ? v : 0.f;
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float x0 = __uint_as_float(sc[c][e]) * p.scale_log2, x1 = __uint_as_float(sc[c][e + 1]) * p.scale_log2;
            acc[(e >> 1) & 3] = add_f32x2(acc[(e >> 1) & 3], pack_f32x2(ex2_approx(x0), ex2_approx(x1)));
          }
        }
      }
    };
    // A score row comes in two halves; while one is added up the next is on its way, the next tile's first half as well.
    uint32_t left[4][16], right[4][16];
    auto ask = [&](uint32_t (&sc)[4][16], int i, int first) {
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld16(tmem + lanes + (w * 2 + ((i - begin) & 1)) * kPwTile + first + c * 16, sc[c]);
    };
    auto ready = [&](int i) {
      ok = mbar_wait_warp(&s_full[w * 2 + ((i - begin) & 1)], ((i - begin) >> 1) & 1, p.status, kStatusAccumTimeout);
      if (ok) {
        tc_fence_after_sync();
        ask(left, i, 0);
      }
    };
    if (begin < end) ready(begin);
    for (int i = begin; i < end && ok; ++i) {
      int low, high;
      const bool edge = seen(i, low, high);
      tmem_wait_ld();
      pw_settled(left);
      ask(right, i, 64);
      add(left, 0, edge, low, high);
      tmem_wait_ld();
      pw_settled(right);
      tc_fence_before_sync();
      mbar_arrive(&s_empty[w * 2 + ((i - begin) & 1)]);
      if (i + 1 < end) ready(i + 1);
      add(right, 64, edge, low, high);
    }
    float s0, s1;
    unpack_f32x2(add_f32x2(add_f32x2(acc[0], acc[1]), add_f32x2(acc[2], acc[3])), s0, s1);
    total += s0 + s1;
    if (ranks > 1) sum_s[w * kPwTile + quarter * 32 + lane] = total;
  }
  if (ranks > 1) {
    __syncwarp();
    cluster_arrive_release();
    cluster_wait_acquire();
  }
  if (warp >= 2 && rank == 0) {
    const int w = (warp - 2) >> 2, at = w * kPwTile + (warp & 3) * 32 + lane, key = key0 + at;
    for (int r = 1; r < ranks; ++r) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(sum_s + at), r)) : "memory");
      total += v;
    }
    if (key < kv_len && (tiles > 0 || key >= before)) {
      const int page = p.block_table[static_cast<size_t>(b) * p.wide + key / kPwPage];
      if (page >= 0 && page < p.num_pages) {
        float* at_w = p.weights + (static_cast<size_t>(page) * p.n_kv + h) * kPwPage + key % kPwPage;
        *at_w = key >= before ? total : *at_w + total;
      }
    }
  }
  if (ranks > 1) {
    __syncwarp();
    cluster_arrive_release();                                           // nobody leaves while its sums are read
    cluster_wait_acquire();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <int NK>
static int pw_launch(const CUtensorMap& tmQ, const CUtensorMap& tmK, const PwParams& p, int blocks, int ranks, int batch, cudaStream_t stream) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    if (cudaFuncSetAttribute(prompt_weights_kernel<NK>, cudaFuncAttributeMaxDynamicSharedMemorySize, pw_smem(NK)) != cudaSuccess) return -1;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_kv * ranks, batch, blocks);
  cfg.blockDim = dim3(kPwThreads);
  cfg.dynamicSmemBytes = pw_smem(NK);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, prompt_weights_kernel<NK>, tmQ, tmK, p);
  eredu_count_launches(1);
  return static_cast<int>(e);
}

}  // namespace eredu

using namespace eredu;

extern "C" int eredu_attn_prefill_tc_lse(const void* q, const void* k_cache, const void* v_cache, void* out, float* lse, const int* block_table,
                                         const int* seq_lens, const int* cu_q, const float* sinks, int batch, int total_q, int max_q_len,
                                         int max_pages, int num_pages, int n_q_heads, int n_kv_heads, int dim, int window, int max_kv_len, int sm_count,
                                         float scale, int* status, cudaStream_t stream);

// Attention of prompts or portions of them (attention_tc.cu), and the weights behind it.
extern "C" int eredu_weighed_prefill(const void* args, int bytes) {
  WeighedPrefillArgs a;
  if (!weights_args(a, args, bytes)) return -2;
  if (a.batch <= 0 || a.total_q <= 0 || a.max_kv_len <= 0) return 0;
  const int blocks = (std::min(a.max_kv_len, a.wide * kPwPage) + kPwKeys - 1) / kPwKeys;
  if ((a.D != 64 && a.D != 128) || a.n_kv <= 0 || a.n_q % a.n_kv != 0 || a.num_pages <= 0 || a.batch > 65535 || blocks > 65535 || a.window < 0 || a.observed < 0 ||
      (a.ranks != 1 && a.ranks != 2 && a.ranks != 4 && a.ranks != kPwCluster))
    return -2;
  const int e = eredu_attn_prefill_tc_lse(a.q, a.k, a.v, a.out, a.lse, a.block_table, a.seq_lens, a.cu_q, a.sinks, a.batch, a.total_q, a.max_q_len, a.wide, a.num_pages,
                                          a.n_q, a.n_kv, a.D, a.window, a.max_kv_len, a.sm_count, a.scale, a.status, a.stream);
  if (e != 0) return e;
  PwParams p = {};
  p.lse = a.lse;
  p.block_table = a.block_table;
  p.seq_lens = a.seq_lens;
  p.cu_q = a.cu_q;
  p.weights = a.weights;
  p.status = a.status;
  p.wide = a.wide;
  p.num_pages = a.num_pages;
  p.n_q = a.n_q;
  p.n_kv = a.n_kv;
  p.group = a.n_q / a.n_kv;
  while (p.gshift < 5 && p.group % (2 << p.gshift) == 0) ++p.gshift;    // query heads of a tile: a power of two that divides the group, 32 at most
  p.window = a.window;
  p.observed = a.observed;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.unscale = 1.f / p.scale_log2;
  const uint64_t D = static_cast<uint64_t>(a.D), H = static_cast<uint64_t>(a.n_kv), Q = static_cast<uint64_t>(a.n_q);
  CUtensorMap tmQ, tmK;
  int r = make_tma_3d(&tmQ, a.q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, D, Q, static_cast<uint64_t>(a.total_q), D * 2, Q * D * 2, 64, 1 << p.gshift, kPwTile >> p.gshift);
  if (r != 0) return -100 + r;
  r = make_tma_4d(&tmK, a.k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, D, 16, H, static_cast<uint64_t>(a.num_pages), D * 2, 16 * D * 2, H * 16 * D * 2, 64, 16, 1, 1);
  if (r != 0) return -200 + r;
  return a.D == 128 ? pw_launch<2>(tmQ, tmK, p, blocks, a.ranks, a.batch, a.stream) : pw_launch<1>(tmQ, tmK, p, blocks, a.ranks, a.batch, a.stream);
}
