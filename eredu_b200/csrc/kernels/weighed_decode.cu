// Decode attention that adds up the weight it gives: out = softmax(scale q k^T) v over the pages of a sequence, as attention.cu has it, and
// for every cached token and key / value head the sum of the softmax weights over the query rows and the query heads that share the head,
// added to what earlier calls gave the token (the tokens that the call brings begin with it).
//
// A weight is known when the sum of its row is, behind the last key, so the scores have to be kept until then: 4 bytes for every
// row and token beside the 512 (head size 128) of its key and value, in memory that stays in L2, where reading the keys a second time would be half as much again.
//
// grid (splits, n_kv, batch), four warps. A warp walks every fourth page of the split's share through a ring of its own, filled by TMA (page blocks
// [16][64] with the 128-byte swizzle that ldmatrix reads without conflicts). Scores come as S^T = K Q^T (mma.sync m16n8k16: the sixteen keys of a page by eight rows, so
// that the four to eight rows of a group fill the narrow side), and so does O^T = V^T P^T: a lane has two rows in both, whose maxima rescale its own accumulators. The
// row maximum is a bound that is moved when a score is above it by more than 2^8: most pages need no exchange between lanes.
// The splits of a sequence and head (up to sixteen, or to the largest cluster that the device has room for) are a cluster: maxima, sums and outputs meet in shared memory, and
// every CTA weighs its own tokens. More splits leave their part in memory, and a second kernel does the same. Up to sixteen rows that share a head are a warp's; with more, two
// or four warps walk the same pages with sixteen rows each.
//
// Probabilities are rounded to bf16 in front of the product with the values, the type of its other operand: outputs are 0.0018 to 0.0023 off 64 bits, where bf16 outputs alone
// make it 0.0017; the weights are made of unrounded ones, and all sums are held in 32 bits.
//
// Measured (floor: K, V and weights at 6.54 TB/s; launches of a graph on inputs that together exceed the second-level cache): 64 sequences of 2048 to 4096 tokens, 32 heads of
// 128 over 8, 135 us (floor 124, 6.0 TB/s); 32 of 1088 to 2175 45 us (33: what is left is the start and the end of the CTAs, about 8 us); one of 32768, 64 heads over 8, 32 us (21:
// 24 splits to a head and the second kernel); one of 512, 32 heads of 64 over 8, 6.0 us, a chain of latencies. Storing the scores and adding up the weights took 18 us of 144 in the
// first of these before keys and values were kept from pushing the scores out of the second-level cache. A page costs a warp some 300 instructions at five cycles each while
// it is alone on its scheduler, so that twelve warps to an SM (two stages to a ring) move more than eight with three stages: 64 x 4096 156 -> 148 us.
#include <cuda_bf16.h>

#include <algorithm>

#include "../common/launch.h"
#include "../common/launch_count.h"
#include "../common/ptx.cuh"
#include "../common/tma_host.h"
#include "../common/weights_args.h"

namespace eredu {

constexpr int kWdPage = 16;
constexpr int kWdWarps = 4;
constexpr int kWdPages = 8;              // of the rings of a CTA: 64 KB with heads of 128, three CTAs to an SM
constexpr int kWdMaxRows = 64;
constexpr int kWdHeld = 16 * 1024;       // bytes of scores that a CTA may hold in shared memory
constexpr int kWdCluster = 16;           // splits of a cluster (more than eight: where the device has room for it)
constexpr int kWdMaxSplits = 64;
constexpr float kWdGrow = 8.f;           // log2 units a score may lie above the bound in use

struct WdParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const int *block_table, *seq_lens;
  const float* sinks;
  float *weights, *scores, *part_o, *part_ml;
  int* status;
  int q_per_seq, pitch, max_tokens, room, num_pages, n_q, n_kv, group, rows, pad, splits, window;
  float scale_log2;
};

__device__ __forceinline__ void wd_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void wd_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t wd_transposed(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ void wd_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void wd_load_page(void* dst, const CUtensorMap* map, int x, int head, int page, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(0), "r"(head), "r"(page), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}
__device__ __forceinline__ float wd_remote(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// What a (sequence, split) walks.
struct WdShare {
  int kv_len, first_pos;     // tokens, position of the first query row
  int low;                   // first token that some row sees
  int page0, page1;
};
__device__ __forceinline__ WdShare wd_share(const WdParams& p, int b, int split) {
  WdShare s;
  const int n = p.seq_lens[b];
  s.kv_len = min(n, min(p.max_tokens, p.room));
  if (n > s.kv_len) report_status(p.status, kStatusBadArgument);
  s.first_pos = s.kv_len - p.q_per_seq;
  s.low = p.window > 0 ? max(0, s.first_pos - p.window + 1) : 0;
  const int base = s.low / kWdPage, pages = (s.kv_len + kWdPage - 1) / kWdPage;
  const int per = max(0, (pages - base + p.splits - 1) / p.splits);
  s.page0 = min(pages, base + split * per);
  s.page1 = min(pages, s.page0 + per);
  return s;
}

// Tokens of pages [page0, page1): thread i has i, i + threads, .. of them, kWdDeep at a time. Where their weights lie, and what they are, does not hang on the
// attention and is asked for ahead; one token after the other, a thread waited for two reads for each (32768 tokens in one CTA: 400 us of 494).
constexpr int kWdDeep = 4;
struct WdCells {
  float* at[kWdDeep];                      // null: none
  float held[kWdDeep];
  float4 score[kWdDeep][2];                // of the first eight rows
};
// Where a CTA finds its scores: memory, or shared memory behind everything else where they are few.
struct WdScores {
  float* at;
  int first;                               // token that lies there
  __device__ __forceinline__ float* row(int t, int pad) const { return at + static_cast<size_t>(t - first) * pad; }
};
__device__ __forceinline__ void wd_scores(const WdParams& p, const WdScores& scores, int t0, int r, int threads, const WdCells& c, float4 (&score)[kWdDeep][2]) {
#pragma unroll
  for (int u = 0; u < kWdDeep; ++u)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      score[u][i] = c.at[u] != nullptr && r + 4 * i < p.pad ? *reinterpret_cast<const float4*>(scores.row(t0 + u * threads, p.pad) + r + 4 * i)
                                                              : make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ void wd_cells(const WdParams& p, const WdShare& s, const WdScores& scores, int b, int h, int t0, int threads, WdCells& c) {
  int page[kWdDeep];
#pragma unroll
  for (int u = 0; u < kWdDeep; ++u) {
    const int t = t0 + u * threads;
    page[u] = t < s.page1 * kWdPage && t < s.kv_len && t >= s.low ? p.block_table[static_cast<size_t>(b) * p.pitch + t / kWdPage] : -1;
  }
#pragma unroll
  for (int u = 0; u < kWdDeep; ++u) {
    const int t = t0 + u * threads;
    c.at[u] = page[u] >= 0 && page[u] < p.num_pages ? p.weights + (static_cast<size_t>(page[u]) * p.n_kv + h) * kWdPage + t % kWdPage : nullptr;
    c.held[u] = c.at[u] != nullptr && t < s.first_pos ? *c.at[u] : 0.f;
  }
  wd_scores(p, scores, t0, 0, threads, c, c.score);
}
// Their weights, summed over rows: 2^(score - top) / sum. `c`: the first cells.
__device__ __forceinline__ void wd_weigh(const WdParams& p, const WdShare& s, const WdScores& scores, int b, int h, const float* top, const float* inv, int threads,
                                         WdCells& c) {
  for (int t0 = s.page0 * kWdPage + static_cast<int>(threadIdx.x); t0 < s.page1 * kWdPage; t0 += kWdDeep * threads) {
    if (t0 >= s.page0 * kWdPage + threads) wd_cells(p, s, scores, b, h, t0, threads, c);
    float sum[kWdDeep];
#pragma unroll
    for (int u = 0; u < kWdDeep; ++u) sum[u] = 0.f;
    for (int r = 0; r < p.pad; r += 8) {
      float4 next[kWdDeep][2];                       // of the next eight rows, on their way while these are added up
      if (r + 8 < p.pad) wd_scores(p, scores, t0, r + 8, threads, c, next);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (r + 4 * i >= p.pad) break;
        const float4 m = *reinterpret_cast<const float4*>(top + r + 4 * i), f = *reinterpret_cast<const float4*>(inv + r + 4 * i);   // (rows behind the last have f = 0)
#pragma unroll
        for (int u = 0; u < kWdDeep; ++u) {
          const float4 v = c.score[u][i];
          sum[u] += ex2_approx(v.x - m.x) * f.x + ex2_approx(v.y - m.y) * f.y + (ex2_approx(v.z - m.z) * f.z + ex2_approx(v.w - m.w) * f.w);
        }
      }
      if (r + 8 < p.pad) {
#pragma unroll
        for (int u = 0; u < kWdDeep; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) c.score[u][i] = next[u][i];
      }
    }
#pragma unroll
    for (int u = 0; u < kWdDeep; ++u)
      if (c.at[u] != nullptr) *c.at[u] = c.held[u] + sum[u];
  }
}

// Shared memory: the rings [page groups][stages][K, V]; behind the last page the warps' parts [warps][ROWS][D + 4], maxima and sums, then
// the CTA's part [RG * ROWS][D], maxima and sums.
template <int D, int NT, int RG>
constexpr int wd_smem() {
  constexpr int ring = kWdPages * 2 * kWdPage * D * 2;
  constexpr int rows = 8 * NT;
  constexpr int merge = (kWdWarps * rows * (D + 4) + 2 * kWdWarps * rows + RG * rows * D + 2 * RG * rows) * 4;
  return 1024 + (ring > merge ? ring : merge);
}

// RG: warps that share the pages of a ring, with 8 NT query rows each.
template <int D, int NT, int RG>
__global__ void __launch_bounds__(32 * kWdWarps, 3) weighed_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const WdParams p) {
  constexpr int KS = D / 16, HALVES = D / 64, ROWS = 8 * NT, ALL = RG * ROWS, NTH = 32 * kWdWarps;
  constexpr int PG = kWdWarps / RG, STAGES = kWdPages / PG;            // page groups, pages of a ring
  constexpr int BLOCK = kWdPage * D * 2, STAGE = 2 * BLOCK;
  extern __shared__ __align__(1024) uint8_t wd_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(wd_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full[PG][STAGES], empty[PG][STAGES];
  __shared__ __align__(16) float s_top[ALL], s_inv[ALL];
  __shared__ float s_part[ALL][kWdCluster];
  const int warp = static_cast<int>(warp_uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z, pgroup = warp / RG, rgroup = warp % RG, row0 = rgroup * ROWS;
  pdl_launch_early();
  if (threadIdx.x == 0) {
    for (int i = 0; i < PG * STAGES; ++i) {
      mbar_init(&full[0][0] + i, 1);
      mbar_init(&empty[0][0] + i, RG);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const WdShare s = wd_share(p, b, split);
  const int* table = p.block_table + static_cast<size_t>(b) * p.pitch;
  const bool one = elect_one();
  // keys and values are read once, and leave the second-level cache to the scores, which are read again (64 x 4096 144 -> 135 us, 32 x 2175 48 -> 44, 1 x 32768 39 -> 33)
  const uint64_t policy = l2_policy_evict_first();
  uint8_t* ring = smem + pgroup * STAGES * STAGE;
  const int first = s.page0 + pgroup;
  bool ok = true;
  int ids = 0;                                                        // lane l: the page of this ring's iteration 32 i + l
  auto next_ids = [&](int it) {
    const int pg = first + (it + lane) * PG;
    ids = pg < s.page1 ? table[pg] : 0;
    if (ids < 0 || ids >= p.num_pages) {
      report_status(p.status, kStatusBadArgument);
      ids = 0;
    }
  };
  // called with it = 0, 1, 2, ..; one warp of those that share a ring fills it, when all of them have read the page
  auto fetch = [&](int it) {
    if (RG > 1 && rgroup != 0) return;
    if ((it & 31) == 0) next_ids(it);
    const int page = __shfl_sync(0xffffffffu, ids, it & 31);
    if (first + it * PG >= s.page1) return;
    const int st = it % STAGES;
    if (RG > 1 && it >= STAGES && ok) ok = mbar_wait_warp(&empty[pgroup][st], (it / STAGES - 1) & 1, p.status, kStatusSmemEmptyTimeout);
    if (one && ok) {
      mbar_arrive_expect_tx(&full[pgroup][st], STAGE);
#pragma unroll
      for (int i = 0; i < HALVES; ++i) {
        wd_load_page(ring + st * STAGE + i * 2048, &tmK, i * 64, h, page, &full[pgroup][st], policy);
        wd_load_page(ring + st * STAGE + BLOCK + i * 2048, &tmV, i * 64, h, page, &full[pgroup][st], policy);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES; ++i) fetch(i);
  // queries as B fragments: lane (g, t) has row g of every eight, dims 16 ks + 2 t and + 8
  uint32_t qf[NT][KS][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = row0 + nt * 8 + g;
    const int token = r / p.group, head = h * p.group + r % p.group;
    const uint32_t* row = reinterpret_cast<const uint32_t*>(p.q + (static_cast<size_t>(b * p.q_per_seq + token) * p.n_q + head) * D);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[nt][ks][0] = r < p.rows ? row[ks * 8 + tig] : 0u;
      qf[nt][ks][1] = r < p.rows ? row[ks * 8 + tig + 4] : 0u;
    }
  }
  float o[NT][KS][4], top[NT][2], sum[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    top[nt][0] = top[nt][1] = -INFINITY;
    sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
  }
  const bool held = p.scores == nullptr;
  const WdScores scores{held ? reinterpret_cast<float*>(smem + wd_smem<D, NT, RG>() - 1024) : p.scores + (static_cast<size_t>(b) * p.n_kv + h) * p.room * p.pad,
                        held ? s.page0 * kWdPage : 0};
  // A row of 128 bytes has its 16-byte pieces permuted by the row's number: piece 2 i + half of a lane's row is the half's place with bits 5 and 6 flipped by i
  const uint32_t ring_addr = smem_u32(ring);
  const uint32_t a_off = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_off = ((lane >> 4) * 8 + (lane & 7)) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
  float* score_at = scores.row(first * kWdPage + g, p.pad) + row0 + 2 * tig;
  int it = 0;
  for (int pg = first; pg < s.page1 && ok; pg += PG, ++it, score_at += PG * kWdPage * p.pad) {
    const int st = it % STAGES;
    ok = mbar_wait_warp(&full[pgroup][st], (it / STAGES) & 1, p.status, kStatusTmaFullTimeout);
    if (!ok) break;
    const uint32_t k_addr = ring_addr + st * STAGE, v_addr = k_addr + BLOCK;
    // all fragments of the keys are on their way ahead of the first product, which run in two chains; those of the values during the softmax
    uint32_t a[KS][4];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      wd_ldsm(((k_addr + a_off) ^ ((ks & 3) << 5)) + (ks >> 2) * 2048, a[ks]);
    }
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float odd[4] = {0.f, 0.f, 0.f, 0.f};
      sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks += 2) {
        wd_mma(sc[nt], a[ks], qf[nt][ks][0], qf[nt][ks][1]);
        wd_mma(odd, a[ks + 1], qf[nt][ks + 1][0], qf[nt][ks + 1][1]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nt][e] = (sc[nt][e] + odd[e]) * p.scale_log2;
    }
    const int key0 = pg * kWdPage;
    const bool edge = key0 + kWdPage - 1 > s.first_pos || (p.window > 0 && key0 < s.kv_len - p.window);
    // values of tokens that no row sees, in front of the window or behind the last one: a weight of zero does not make a number of what is none
    if (key0 < s.low || key0 + kWdPage > s.kv_len) {
      for (int i = lane; i < kWdPage * (D / 8); i += 32) {
        const int r = i / (D / 8), c = i % (D / 8);
        if (key0 + r < s.low || key0 + r >= s.kv_len)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_addr + (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4)), "r"(0) : "memory");
      }
      fence_proxy_async_smem();                                       // the stage is filled again by TMA
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      wd_ldsm_t(((v_addr + v_off) ^ ((i & 3) << 5)) + (i >> 2) * 2048, a[i]);
    }
    __syncwarp();
    if (RG > 1 && lane == 0) mbar_arrive(&empty[pgroup][st]);
    fetch(it + STAGES);
    uint32_t pf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (edge) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + g + (e >> 1) * 8, r = row0 + nt * 8 + 2 * tig + (e & 1), pos = s.first_pos + r / p.group;
          if (key > pos || (p.window > 0 && key <= pos - p.window)) sc[nt][e] = -INFINITY;
        }
      }
      if (row0 + nt * 8 + 2 * tig < p.pad) {
        // (rows behind the last are nothing, whatever zeros make of a key that is no number)
        const int r = row0 + nt * 8 + 2 * tig;
        const bool r0 = r < p.rows, r1 = r + 1 < p.rows;
        float* at = score_at + nt * 8;
        *reinterpret_cast<float2*>(at) = make_float2(r0 ? sc[nt][0] : -INFINITY, r1 ? sc[nt][1] : -INFINITY);
        *reinterpret_cast<float2*>(at + 8 * p.pad) = make_float2(r0 ? sc[nt][2] : -INFINITY, r1 ? sc[nt][3] : -INFINITY);
      }
      float mx0 = fmaxf(sc[nt][0], sc[nt][2]), mx1 = fmaxf(sc[nt][1], sc[nt][3]);
      const bool grow = (mx0 > top[nt][0] + kWdGrow) || (mx1 > top[nt][1] + kWdGrow);
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int m = 4; m < 32; m <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, m));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, m));
        }
        mx0 = fmaxf(mx0, top[nt][0]);
        mx1 = fmaxf(mx1, top[nt][1]);
        // (a row that has seen nothing has nothing to rescale)
        const float c0 = top[nt][0] == -INFINITY ? 0.f : ex2_approx(top[nt][0] - mx0), c1 = top[nt][1] == -INFINITY ? 0.f : ex2_approx(top[nt][1] - mx1);
        top[nt][0] = mx0;
        top[nt][1] = mx1;
        sum[nt][0] *= c0;
        sum[nt][1] *= c1;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          o[nt][i][0] *= c0;
          o[nt][i][1] *= c1;
          o[nt][i][2] *= c0;
          o[nt][i][3] *= c1;
        }
      }
      const float m0 = top[nt][0] == -INFINITY ? 0.f : top[nt][0], m1 = top[nt][1] == -INFINITY ? 0.f : top[nt][1];
      const float p0 = ex2_approx(sc[nt][0] - m0), p1 = ex2_approx(sc[nt][1] - m1), p2 = ex2_approx(sc[nt][2] - m0), p3 = ex2_approx(sc[nt][3] - m1);
      sum[nt][0] += p0 + p2;
      sum[nt][1] += p1 + p3;
      pf[nt][0] = wd_transposed(pack_bf16x2(p0, p1));
      pf[nt][1] = wd_transposed(pack_bf16x2(p2, p3));
    }
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) wd_mma(o[nt][i], a[i], pf[nt][0], pf[nt][1]);
  }
  // (a wait that ran out: what is on its way must have landed before the rings are used for anything else)
  if (!ok)
    for (int i = 0; i < STAGES; ++i)
      if (first + (it + i) * PG < s.page1) mbar_wait(&full[pgroup][(it + i) % STAGES], ((it + i) / STAGES) & 1, p.status, kStatusTmaFullTimeout);
  __syncthreads();
  // ---- the warps' parts
  float* mo = reinterpret_cast<float*>(smem);                         // [warps][ROWS][D + 4]
  float* mm = mo + kWdWarps * ROWS * (D + 4);                         // [warps][ROWS]
  float* ml = mm + kWdWarps * ROWS;
  float* po = ml + kWdWarps * ROWS;                                   // [ALL][D]
  float* pm = po + ALL * D;
  float* pl = pm + ALL;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float l = sum[nt][j];
#pragma unroll
      for (int m = 4; m < 32; m <<= 1) l += __shfl_xor_sync(0xffffffffu, l, m);
      const int r = nt * 8 + 2 * tig + j;
      if (g == 0) {
        mm[warp * ROWS + r] = top[nt][j];
        ml[warp * ROWS + r] = l;
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        mo[(warp * ROWS + r) * (D + 4) + i * 16 + g] = o[nt][i][j];
        mo[(warp * ROWS + r) * (D + 4) + i * 16 + g + 8] = o[nt][i][2 + j];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.rows * D; i += NTH) {
    const int r = i / D, d = i % D;
    float M = -INFINITY;
    const int w0 = r / ROWS, own = r % ROWS;                          // the first of the warps that have this row (every RG-th), and its place there
#pragma unroll
    for (int w = 0; w < PG; ++w) M = fmaxf(M, mm[(w0 + w * RG) * ROWS + own]);
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < PG; ++w) {
      const int at = (w0 + w * RG) * ROWS + own;
      const float m = mm[at], c = m == -INFINITY ? (ml[at] != 0.f ? 1.f : 0.f) : ex2_approx(m - M);   // (a sum without a maximum is no number, and stays)
      L += ml[at] * c;
      acc += mo[at * (D + 4) + d] * c;
    }
    po[r * D + d] = acc;
    if (d == 0) {
      pm[r] = M;
      pl[r] = L;
    }
  }
  if (p.part_o != nullptr) {
    // a second kernel joins the splits
    __syncthreads();
    const size_t at = (static_cast<size_t>(b) * p.n_kv + h) * p.splits + split;
    for (int i = threadIdx.x; i < p.rows * D; i += NTH) p.part_o[at * p.rows * D + i] = po[i];
    for (int i = threadIdx.x; i < p.rows; i += NTH) {
      p.part_ml[(at * p.rows + i) * 2] = pm[i];
      p.part_ml[(at * p.rows + i) * 2 + 1] = pl[i];
    }
    return;
  }
  const bool many = p.splits > 1;
  WdCells cells;
  if (many) {
    __syncwarp();
    cluster_arrive_release();
    wd_cells(p, s, scores, b, h, s.page0 * kWdPage + static_cast<int>(threadIdx.x), NTH, cells);
    __syncwarp();
    cluster_wait_acquire();
  } else {
    wd_cells(p, s, scores, b, h, s.page0 * kWdPage + static_cast<int>(threadIdx.x), NTH, cells);
    __syncthreads();
  }
  const uint32_t a_o = smem_u32(po), a_m = smem_u32(pm), a_l = smem_u32(pl);
  for (int r = threadIdx.x; r < ALL; r += NTH) {
    if (r >= p.rows) {
      s_top[r] = s_inv[r] = 0.f;
      continue;
    }
    float ms[kWdCluster], ls[kWdCluster], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < kWdCluster; ++i) {
      ms[i] = -INFINITY;
      ls[i] = 0.f;
      if (i < p.splits) {
        ms[i] = many ? wd_remote(mapa_shared(a_m + r * 4, i)) : pm[r];
        ls[i] = many ? wd_remote(mapa_shared(a_l + r * 4, i)) : pl[r];
      }
      M = fmaxf(M, ms[i]);
    }
    const float sink = p.sinks != nullptr ? p.sinks[h * p.group + r % p.group] * 1.4426950408889634f : -INFINITY;
    if (M > -INFINITY && sink > M + 64.f) M = sink;                    // (a sink far above all scores: its own term stays finite)
#pragma unroll
    for (int i = 0; i < kWdCluster; ++i) {
      const float c = ms[i] == -INFINITY ? (ls[i] != 0.f ? 1.f : 0.f) : ex2_approx(ms[i] - M);
      s_part[r][i] = c;
      L += ls[i] * c;
    }
    if (M > -INFINITY && p.sinks != nullptr) L += ex2_approx(sink - M);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    s_top[r] = M == -INFINITY ? 0.f : M;
    s_inv[r] = inv;
  }
  __syncthreads();
  for (int i = threadIdx.x + split * NTH; i < p.rows * D; i += NTH * p.splits) {
    const int r = i / D, d = i % D;
    float acc = 0.f;
    if (many) {
#pragma unroll
      for (int sp = 0; sp < kWdCluster; ++sp)
        if (sp < p.splits) acc += wd_remote(mapa_shared(a_o + i * 4, sp)) * s_part[r][sp];
    } else {
      acc = po[i] * s_part[r][0];
    }
    p.out[(static_cast<size_t>(b * p.q_per_seq + r / p.group) * p.n_q + h * p.group + r % p.group) * D + d] = __float2bfloat16(acc * s_inv[r]);
  }
  if (many) {
    __syncwarp();
    cluster_arrive_release();                                         // done with the peers' shared memory
  }
  wd_weigh(p, s, scores, b, h, s_top, s_inv, NTH, cells);
  if (many) {
    __syncwarp();
    cluster_wait_acquire();                                           // nobody leaves while a peer reads its part
  }
}

// grid (splits, n_kv, batch): joins what the splits have left, a share of the output and of the tokens each.
constexpr int kWdJoinThreads = 256;
__global__ void __launch_bounds__(kWdJoinThreads) weighed_join_kernel(const WdParams p, const int D) {
  __shared__ __align__(16) float s_top[kWdMaxRows], s_inv[kWdMaxRows];
  __shared__ float s_part[kWdMaxRows][kWdMaxSplits];
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const WdShare s = wd_share(p, b, split);
  const size_t at = (static_cast<size_t>(b) * p.n_kv + h) * p.splits;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kWdMaxRows && static_cast<int>(threadIdx.x) >= p.rows) s_top[threadIdx.x] = s_inv[threadIdx.x] = 0.f;
  for (int r = warp; r < p.rows; r += kWdJoinThreads / 32) {
    float M = -INFINITY, L = 0.f;
    float2 v[kWdMaxSplits / 32];
#pragma unroll
    for (int i = 0; i < kWdMaxSplits / 32; ++i) {
      const int sp = i * 32 + lane;
      v[i] = sp < p.splits ? *reinterpret_cast<const float2*>(p.part_ml + ((at + sp) * p.rows + r) * 2) : make_float2(-INFINITY, 0.f);
      M = fmaxf(M, v[i].x);
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, m));
    const float sink = p.sinks != nullptr ? p.sinks[h * p.group + r % p.group] * 1.4426950408889634f : -INFINITY;
    if (M > -INFINITY && sink > M + 64.f) M = sink;
#pragma unroll
    for (int i = 0; i < kWdMaxSplits / 32; ++i) {
      const float c = v[i].x == -INFINITY ? (v[i].y != 0.f ? 1.f : 0.f) : ex2_approx(v[i].x - M);
      s_part[r][i * 32 + lane] = c;
      L += v[i].y * c;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) L += __shfl_xor_sync(0xffffffffu, L, m);
    if (M > -INFINITY && p.sinks != nullptr) L += ex2_approx(sink - M);
    if (lane == 0) {
      s_top[r] = M == -INFINITY ? 0.f : M;
      s_inv[r] = L == 0.f ? 0.f : 1.f / L;
    }
  }
  const WdScores scores{p.scores + (static_cast<size_t>(b) * p.n_kv + h) * p.room * p.pad, 0};
  WdCells cells;
  wd_cells(p, s, scores, b, h, s.page0 * kWdPage + static_cast<int>(threadIdx.x), kWdJoinThreads, cells);
  __syncthreads();
  for (int i = threadIdx.x + split * kWdJoinThreads; i < p.rows * D; i += kWdJoinThreads * p.splits) {
    const int r = i / D, d = i % D;
    float acc = 0.f;
#pragma unroll 8
    for (int sp = 0; sp < p.splits; ++sp) acc += p.part_o[(at + sp) * p.rows * D + i] * s_part[r][sp];
    p.out[(static_cast<size_t>(b * p.q_per_seq + r / p.group) * p.n_q + h * p.group + r % p.group) * D + d] = __float2bfloat16(acc * s_inv[r]);
  }
  wd_weigh(p, s, scores, b, h, s_top, s_inv, kWdJoinThreads, cells);
}

// What every launch of a kernel may want, whoever asks first.
template <int D, int NT, int RG>
static bool wd_configure() {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && configured[dev]) return true;
  if (cudaFuncSetAttribute(weighed_decode_kernel<D, NT, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, wd_smem<D, NT, RG>() + kWdHeld) != cudaSuccess ||
      cudaFuncSetAttribute(weighed_decode_kernel<D, NT, RG>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return false;
  if (dev >= 0 && dev < 64) configured[dev] = true;
  return true;
}

template <int D, int NT, int RG>
static int wd_launch(const CUtensorMap& tmK, const CUtensorMap& tmV, const WdParams& p, int batch, int held, cudaStream_t stream) {
  if (!wd_configure<D, NT, RG>()) return -1;
  const bool cluster = p.part_o == nullptr && p.splits > 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.splits, p.n_kv, batch);
  cfg.blockDim = dim3(32 * kWdWarps);
  cfg.dynamicSmemBytes = wd_smem<D, NT, RG>() + held;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = p.splits;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cudaError_t e = cudaLaunchKernelEx(&cfg, weighed_decode_kernel<D, NT, RG>, tmK, tmV, p);
  eredu_count_launches(1);
  if (e == cudaSuccess && p.part_o != nullptr) {
    e = launch_pdl(weighed_join_kernel, dim3(p.splits, p.n_kv, batch), dim3(kWdJoinThreads), 0, stream, p, D);
    eredu_count_launches(1);
  }
  return static_cast<int>(e);
}

}  // namespace eredu

using namespace eredu;

extern "C" int eredu_weighed_decode(const void* args, int bytes) {
  WeighedDecodeArgs a;
  if (!weights_args(a, args, bytes)) return -2;
  if (a.batch <= 0 || a.q_per_seq <= 0) return 0;
  if ((a.D != 64 && a.D != 128) || a.n_kv <= 0 || a.n_q % a.n_kv != 0 || a.num_pages <= 0 || a.batch > 65535 || a.n_kv > 65535 || a.splits < 1 ||
      a.splits > kWdMaxSplits || a.window < 0 || a.room <= 0 || a.room % kWdPage != 0 || (a.part_o != nullptr ? a.splits < 2 || a.part_ml == nullptr : a.splits > kWdCluster))
    return -2;
  WdParams p = {};
  p.group = a.n_q / a.n_kv;
  if (static_cast<long long>(a.q_per_seq) * p.group > kWdMaxRows) return -2;
  p.rows = a.q_per_seq * p.group;
  p.pad = (p.rows + 3) / 4 * 4;
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.block_table = a.block_table;
  p.seq_lens = a.seq_lens;
  p.sinks = a.sinks;
  p.weights = a.weights;
  p.scores = a.scores;
  p.part_o = a.part_o;
  p.part_ml = a.part_ml;
  p.status = a.status;
  p.q_per_seq = a.q_per_seq;
  p.pitch = a.pitch;
  p.max_tokens = a.max_tokens;
  p.room = a.room;
  p.num_pages = a.num_pages;
  p.n_q = a.n_q;
  p.n_kv = a.n_kv;
  p.splits = a.splits;
  p.window = a.window;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  // (the pages of a split, however short the others are)
  const long long few = static_cast<long long>((a.room / kWdPage + a.splits - 1) / a.splits) * kWdPage * p.pad * 4;
  if (a.scores == nullptr && (few > kWdHeld || a.part_o != nullptr)) return -2;
  const int held = a.scores == nullptr ? static_cast<int>(few) : 0;
  const uint64_t D = static_cast<uint64_t>(a.D), H = static_cast<uint64_t>(a.n_kv);
  CUtensorMap tmK, tmV;
  int r = make_tma_4d(&tmK, a.k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, D, 16, H, static_cast<uint64_t>(a.num_pages), D * 2, 16 * D * 2, H * 16 * D * 2, 64, 16, 1, 1);
  if (r != 0) return -100 + r;
  r = make_tma_4d(&tmV, a.v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, D, 16, H, static_cast<uint64_t>(a.num_pages), D * 2, 16 * D * 2, H * 16 * D * 2, 64, 16, 1, 1);
  if (r != 0) return -200 + r;
#define ER_WD(D_)                                                                                                          \
  return p.rows <= 8    ? wd_launch<D_, 1, 1>(tmK, tmV, p, a.batch, held, a.stream)                                                  \
         : p.rows <= 16 ? wd_launch<D_, 2, 1>(tmK, tmV, p, a.batch, held, a.stream)                                                  \
         : p.rows <= 32 ? wd_launch<D_, 2, 2>(tmK, tmV, p, a.batch, held, a.stream)                                                  \
                        : wd_launch<D_, 2, 4>(tmK, tmV, p, a.batch, held, a.stream)
  if (a.D == 128) ER_WD(128);
  ER_WD(64);
#undef ER_WD
}

// Whether clusters of sixteen find room on the current device (1, or 0).
extern "C" int eredu_weighed_clusters() {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kWdCluster);
  cfg.blockDim = dim3(32 * kWdWarps);
  cfg.dynamicSmemBytes = wd_smem<128, 2, 1>() + kWdHeld;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kWdCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (!wd_configure<128, 2, 1>() || cudaOccupancyMaxActiveClusters(&n, weighed_decode_kernel<128, 2, 1>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return n > 0 ? 1 : 0;
}
