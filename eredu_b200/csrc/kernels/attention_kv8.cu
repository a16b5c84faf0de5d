// Decode attention over a cache held in 8 bits (common/kv8.cuh): a few queries per sequence, 1 to k + 1 new tokens.
//
//   s_j = (q . c_j) scale ks,   o = sum_j 2^(s_j log2 e - m) vs c'_j / sum_j 2^(s_j log2 e - m)     (ks, vs: scales of token j's blocks)
//
// Bound by memory: every cached token is read once per key / value head, 2 D bytes. A warp walks pages of its own; codes go from
// memory straight into the registers that mma.sync m16n8k16 takes, without shared memory:
//   scores  S^T[16 tokens, 8 query rows] = K[16, D] Q^T: the page is the A operand. The sum over D may run in any order, so a lane takes 16
//           neighbouring bytes of two token rows and the query fragment is laid out to match.
//   output  O^T[D, 8 rows] = V^T[D, 16] P^T: a lane takes 16 neighbouring bytes (8 where D = 64) of four token rows and pairs tokens by byte
//           permutation; which accumulator row is which value channel is settled when they are written out. P^T comes from S^T by movmatrix.
// The 8 query rows of a tile are the query heads that share the key / value head, times the new tokens; two tiles side by side above 8.
// Codes are exact as f16, and so are queries scaled by a power of two per row (to a largest magnitude of 2^14: what f16 drops is below 2^-38 of that).
// Probabilities are rounded to f16 (11 bits). The page's value scale goes into their exponent, with a running maximum of its own (m2, of s_j + log2 vs): the largest
// contribution to the output is near 1 whatever the scales are. The maxima are raised only where a score passes one by more than 2^8.
#include <cuda_bf16.h>

#include "../common/kv8.cuh"
#include "../common/launch.h"
#include "../common/launch_count.h"
#include "../common/ptx.cuh"
#include "../common/trace.cuh"

namespace eredu {

struct AttnKv8Params {
  const __nv_bfloat16* q;          // [B * q_per_seq, n_q, D]
  const int8_t *k_codes, *v_codes; // [pages, n_kv, 16, D]
  const float *k_scales, *v_scales;
  __nv_bfloat16* out;              // [B * q_per_seq, n_q, D]
  const int* block_table;          // [B, max_pages]
  const int* seq_lens;             // [B], new tokens included
  const float* sinks;              // optional [n_q]
  float* part_o;                   // more splits than a cluster holds: [B, n_kv, tiles, splits, rows of a tile, D]
  float* part_ml;                  //                                   [B, n_kv, tiles, splits, rows of a tile, 4]
  int max_pages, num_pages, n_q, n_kv, q_per_seq, tiles, splits, window, chunk;
  float scale_log2;
  int* status;
};
constexpr int kKv8Warps = 8;
constexpr int kKv8Cluster = 8;      // splits that meet in a cluster
constexpr float kKv8Slack = 8.f;    // log2 units by which a score may pass the maximum in use
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(v));
  return v;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Codes of the cache; a step reads each of them once.
__device__ __forceinline__ uint4 ld_codes16(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld_codes8(const int8_t* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int kv8_lowest_key(const AttnKv8Params& p, int pos) {
  if (p.window > 0) return max(0, pos - p.window + 1);
  return p.chunk > 0 && pos > 0 ? pos - pos % p.chunk : 0;
}

// What a row has gathered: maximum and sum of the scores, maximum the output is relative to.
struct Kv8Row {
  float m, l, m2;
};
// Output of a row: `o` relative to 2^m2, the sum to 2^m; a sink is a key of zero value. A row that sees nothing is zero.
__device__ __forceinline__ float kv8_finish(float o, const Kv8Row& r, const float* sink) {
  float m = r.m, l = r.l;
  if (sink != nullptr) {
    const float s = *sink * 1.4426950408889634f;
    const float top = fmaxf(m, s);
    l = l * ex2_approx(m - top) + ex2_approx(s - top);
    m = top;
  }
  return l == 0.f || r.l == 0.f ? 0.f : o / l * ex2_approx(r.m2 - m);
}

// grid (splits, n_kv * tiles, B)
template <int D, int NT>
__global__ void __launch_bounds__(32 * kKv8Warps, NT == 1 ? 2 : 1) attn_kv8_kernel(AttnKv8Params p) {
  constexpr int ROWS = 8 * NT, KC = D / 64, STEPS = D / 16, VW = D / 32;   // KC: 16-byte pieces of a token row per lane; VW: value words per token and lane
  extern __shared__ float smem[];
  float* o_warp = smem;                                  // [warps][ROWS][D]
  float* o_s = o_warp + kKv8Warps * ROWS * D;            // [ROWS][D]
  Kv8Row* row_warp = reinterpret_cast<Kv8Row*>(o_s + ROWS * D);   // [warps][ROWS]
  Kv8Row* row_s = row_warp + kKv8Warps * ROWS;           // [ROWS]
  pdl_launch_early();
  trace_mark(kTraceAttnDecode, kTraceStart);
  pdl_wait();
  trace_mark(kTraceAttnDecode, kTraceAfterWait);
  pdl_launch_dependents();
  const int b = blockIdx.z, kvh = blockIdx.y / p.tiles, tile = blockIdx.y % p.tiles, split = blockIdx.x;
  const int warp = static_cast<int>(warp_uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = p.n_q / p.n_kv, rows_all = p.q_per_seq * group, r0 = tile * ROWS, rows = min(ROWS, rows_all - r0);
  const int kv_len = p.seq_lens[b], pos_new = kv_len - p.q_per_seq;
  const int pos_first = pos_new + r0 / group, pos_last = pos_new + (r0 + rows - 1) / group;   // positions of the tile's first and last row
  const int page_lo = kv8_lowest_key(p, pos_first) / kKv8Page, page_hi = min(pos_last / kKv8Page + (pos_last >= 0), p.max_pages);
  const int per = max(0, page_hi - page_lo + p.splits - 1) / p.splits;
  const int page0 = page_lo + split * per, page1 = min(page_hi, page0 + per);
  const int mask_hi = pos_first, mask_lo = kv8_lowest_key(p, pos_last);   // pages inside need no mask

  // ---- the query rows: f16 fragments, and what takes a score back to log2 units
  uint32_t qf[NT][STEPS][2];
  float back[NT][2];                                    // of the lane's columns 2t, 2t + 1
  int pos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + nt * 8 + g;
    const bool in = nt * 8 + g < rows;
    const __nv_bfloat16* src = p.q + (static_cast<size_t>(b * p.q_per_seq + (in ? r / group : 0)) * p.n_q + kvh * group + (in ? r % group : 0)) * D;
    uint4 raw[KC][2];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < KC; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        raw[j][h] = in ? *reinterpret_cast<const uint4*>(src + 64 * j + 16 * t + 8 * h) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {raw[j][h].x, raw[j][h].y, raw[j][h].z, raw[j][h].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
      }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = top >= 0x7f80u || top < 0x0080u ? 0 : max(-110, min(110, 141 - static_cast<int>(top >> 7)));   // 2^e brings the largest to 2^14
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23), down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
    for (int j = 0; j < KC; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w[4] = {raw[j][h].x, raw[j][h].y, raw[j][h].z, raw[j][h].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[nt][4 * j + 2 * h + (i >> 1)][i & 1] = pack_f16x2(bf16_lo(w[i]) * up, bf16_hi(w[i]) * up);
      }
    const float mine = p.scale_log2 * down;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      back[nt][c] = __shfl_sync(0xffffffffu, mine, (2 * t + c) * 4);
      pos[nt][c] = pos_new + (r0 + min(nt * 8 + 2 * t + c, rows - 1)) / group;
    }
  }

  float o[NT][STEPS][4], m[NT][2], m2[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    m[nt][0] = m[nt][1] = m2[nt][0] = m2[nt][1] = kLowest;
    l[nt][0] = l[nt][1] = 0.f;
  }

  // ---- pages warp, warp + 8, ... of the split. Lane i holds page id and scales of the i-th of 32 turns.
  const int* table = p.block_table + static_cast<size_t>(b) * p.max_pages;
  const int turns = page1 > page0 + warp ? (page1 - page0 - warp + kKv8Warps - 1) / kKv8Warps : 0;
  int ids = 0;
  float ks = 0.f, ev = 0.f;
  auto look_up = [&](int turn) {
    const int pg = page0 + warp + kKv8Warps * (turn + lane);
    ids = pg < page1 ? table[pg] : 0;
    if (ids < 0 || ids >= p.num_pages) {
      report_status(p.status, kStatusBadArgument);
      ids = 0;
    }
    const size_t cell = static_cast<size_t>(ids) * p.n_kv + kvh;
    ks = p.k_scales[cell];
    ev = log2f(p.v_scales[cell]);
  };
  uint4 kr[2][KC];
  uint32_t vr[4][VW];
  float ks_next = 0.f, ev_next = 0.f;
  auto fetch_k = [&](int turn) {
    const int id = __shfl_sync(0xffffffffu, ids, turn & 31);
    const int8_t* at = p.k_codes + (static_cast<size_t>(id) * p.n_kv + kvh) * (kKv8Page * D) + g * D + 16 * t;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < KC; ++j) kr[h][j] = ld_codes16(at + h * 8 * D + 64 * j);
  };
  auto fetch_v = [&](int turn) {
    const int id = __shfl_sync(0xffffffffu, ids, turn & 31);
    const int8_t* at = p.v_codes + (static_cast<size_t>(id) * p.n_kv + kvh) * (kKv8Page * D) + 2 * t * D + g * (D / 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // tokens 2t, 2t + 1, 2t + 8, 2t + 9
      const int8_t* row = at + ((i >> 1) * 8 + (i & 1)) * D;
      if (VW == 4) {
        const uint4 u = ld_codes16(row);
        vr[i][0] = u.x; vr[i][1] = u.y; vr[i][VW - 2] = u.z; vr[i][VW - 1] = u.w;
      } else {
        const uint2 u = ld_codes8(row);
        vr[i][0] = u.x; vr[i][1] = u.y;
      }
    }
    ks_next = __shfl_sync(0xffffffffu, ks, turn & 31);
    ev_next = __shfl_sync(0xffffffffu, ev, turn & 31);
  };
  if (turns > 0) {
    look_up(0);
    fetch_k(0);
    fetch_v(0);
  }
  for (int turn = 0; turn < turns; ++turn) {
    const int tok = (page0 + warp + kKv8Warps * turn) * kKv8Page;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const uint32_t lo[4] = {kr[0][j].x, kr[0][j].y, kr[0][j].z, kr[0][j].w}, hi[4] = {kr[1][j].x, kr[1][j].y, kr[1][j].z, kr[1][j].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t x = lo[w] ^ 0x80808080u, y = hi[w] ^ 0x80808080u;
        const uint32_t a0 = kv8_halves<0x4140>(x), a1 = kv8_halves<0x4140>(y), a2 = kv8_halves<0x4342>(x), a3 = kv8_halves<0x4342>(y);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], a0, a1, a2, a3, qf[nt][4 * j + w][0], qf[nt][4 * j + w][1]);
      }
    }
    const float ks_now = ks_next, ev_now = ev_next;
    const bool more = turn + 1 < turns;
    if (more) {
      if (((turn + 1) & 31) == 0) look_up(turn + 1);
      fetch_k(turn + 1);
    }
    // ---- scores in log2 units, masks, maxima
    bool passes = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 4; ++c) s[nt][c] *= back[nt][c & 1] * ks_now;
    }
    if (tok + kKv8Page - 1 > mask_hi || tok < mask_lo) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = tok + g + (c >> 1) * 8, at = pos[nt][c & 1];
          if (key > at || key < kv8_lowest_key(p, at)) s[nt][c] = -INFINITY;
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float top = fmaxf(s[nt][c], s[nt][c + 2]);
        passes |= top > m[nt][c] + kKv8Slack || top + ev_now > m2[nt][c] + kKv8Slack;
      }
    if (__any_sync(0xffffffffu, passes)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float down[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = fmaxf(s[nt][c], s[nt][c + 2]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          const float up = fmaxf(m[nt][c], top), up2 = fmaxf(m2[nt][c], top + ev_now);
          l[nt][c] *= ex2_approx(m[nt][c] - up);
          down[c] = ex2_approx(m2[nt][c] - up2);
          m[nt][c] = up;
          m2[nt][c] = up2;
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          o[nt][i][0] *= down[0];
          o[nt][i][1] *= down[1];
          o[nt][i][2] *= down[0];
          o[nt][i][3] *= down[1];
        }
      }
    }
    uint32_t pf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        l[nt][c & 1] += ex2_approx(s[nt][c] - m[nt][c & 1]);
        // a masked place is zero whatever the scale of its block is
        w[c] = s[nt][c] == -INFINITY ? 0.f : ex2_approx(s[nt][c] + ev_now - m2[nt][c & 1]);
      }
      pf[nt][0] = transposed(pack_f16x2(w[0], w[1]));
      pf[nt][1] = transposed(pack_f16x2(w[2], w[3]));
    }
    // ---- output
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const uint32_t a = vr[0][w] ^ 0x80808080u, bb = vr[1][w] ^ 0x80808080u, c = vr[2][w] ^ 0x80808080u, d = vr[3][w] ^ 0x80808080u;
      const uint32_t x0 = __byte_perm(a, bb, 0x5140), x1 = __byte_perm(a, bb, 0x7362), y0 = __byte_perm(c, d, 0x5140), y1 = __byte_perm(c, d, 0x7362);
      const uint32_t e0 = kv8_halves<0x4140>(x0), e1 = kv8_halves<0x4342>(x0), e2 = kv8_halves<0x4140>(y0), e3 = kv8_halves<0x4342>(y0);
      const uint32_t f0 = kv8_halves<0x4140>(x1), f1 = kv8_halves<0x4342>(x1), f2 = kv8_halves<0x4140>(y1), f3 = kv8_halves<0x4342>(y1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_f16(o[nt][2 * w], e0, e1, e2, e3, pf[nt][0], pf[nt][1]);
        mma_f16(o[nt][2 * w + 1], f0, f1, f2, f3, pf[nt][0], pf[nt][1]);
      }
    }
    if (more) fetch_v(turn + 1);
  }

  // ---- the warps of the CTA together
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float sum = l[nt][c];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      const int row = nt * 8 + 2 * t + c;
      if (g == 0) row_warp[warp * ROWS + row] = Kv8Row{m[nt][c], sum, m2[nt][c]};
      float2* dst = reinterpret_cast<float2*>(o_warp + (warp * ROWS + row) * D + g * (D / 8));
#pragma unroll
      for (int i = 0; i < STEPS; ++i) dst[i] = make_float2(o[nt][i][c], o[nt][i][c + 2]);
    }
  __syncthreads();
  if (threadIdx.x < ROWS) {
    Kv8Row r = {kLowest, 0.f, kLowest};
    for (int w = 0; w < kKv8Warps; ++w) {
      r.m = fmaxf(r.m, row_warp[w * ROWS + threadIdx.x].m);
      r.m2 = fmaxf(r.m2, row_warp[w * ROWS + threadIdx.x].m2);
    }
    for (int w = 0; w < kKv8Warps; ++w) r.l += row_warp[w * ROWS + threadIdx.x].l * ex2_approx(row_warp[w * ROWS + threadIdx.x].m - r.m);
    row_s[threadIdx.x] = r;
  }
  __syncthreads();
  const bool alone = p.splits == 1, cluster = p.splits > 1 && p.splits <= kKv8Cluster;
  const size_t part = ((static_cast<size_t>(b) * p.n_kv * p.tiles + blockIdx.y) * p.splits + split) * ROWS;
  for (int i = threadIdx.x; i < rows * D; i += 32 * kKv8Warps) {
    const int row = i / D, d = i % D;
    const Kv8Row r = row_s[row];
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kKv8Warps; ++w) sum += o_warp[(w * ROWS + row) * D + d] * ex2_approx(row_warp[w * ROWS + row].m2 - r.m2);
    if (alone) {
      const int at = r0 + row, head = kvh * group + at % group;
      p.out[(static_cast<size_t>(b * p.q_per_seq + at / group) * p.n_q + head) * D + d] =
          __float2bfloat16(kv8_finish(sum, r, p.sinks == nullptr ? nullptr : p.sinks + head));
    } else if (cluster) {
      o_s[i] = sum;
    } else {
      p.part_o[part * D + i] = sum;
      if (d == 0) *reinterpret_cast<float4*>(p.part_ml + (part + row) * 4) = make_float4(r.m, r.l, r.m2, 0.f);
    }
  }
  if (!cluster) return;
  // ---- the splits: every CTA of the cluster finishes some of the values
  cluster_arrive_release();
  cluster_wait_acquire();
  for (int i = split * 32 * kKv8Warps + threadIdx.x; i < rows * D; i += p.splits * 32 * kKv8Warps) {
    const int row = i / D;
    Kv8Row part_row[kKv8Cluster], r = {kLowest, 0.f, kLowest};
#pragma unroll
    for (int s = 0; s < kKv8Cluster; ++s) {
      if (s >= p.splits) break;
      const uint32_t at = mapa_shared(smem_u32(row_s + row), s);
      part_row[s] = Kv8Row{ld_cluster_f32(at), ld_cluster_f32(at + 4), ld_cluster_f32(at + 8)};
      r.m = fmaxf(r.m, part_row[s].m);
      r.m2 = fmaxf(r.m2, part_row[s].m2);
    }
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < kKv8Cluster; ++s) {
      if (s >= p.splits) break;
      r.l += part_row[s].l * ex2_approx(part_row[s].m - r.m);
      sum += ld_cluster_f32(mapa_shared(smem_u32(o_s + i), s)) * ex2_approx(part_row[s].m2 - r.m2);
    }
    const int at = r0 + row, head = kvh * group + at % group;
    p.out[(static_cast<size_t>(b * p.q_per_seq + at / group) * p.n_q + head) * D + i % D] =
        __float2bfloat16(kv8_finish(sum, r, p.sinks == nullptr ? nullptr : p.sinks + head));
  }
  cluster_arrive_release();   // nobody leaves while its shared memory is read
  cluster_wait_acquire();
}

// More splits than a cluster holds: a warp per query row. grid (rows, n_kv, B), 32 threads
template <int D>
__global__ void __launch_bounds__(32) attn_kv8_combine_kernel(AttnKv8Params p, int tile_rows) {
  constexpr int PER = D / 32;
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, kvh = blockIdx.y, at = blockIdx.x, lane = threadIdx.x, group = p.n_q / p.n_kv;
  const int tile = at / tile_rows, row = at % tile_rows;
  const size_t first = ((static_cast<size_t>(b) * p.n_kv + kvh) * p.tiles + tile) * p.splits * tile_rows + row;
  Kv8Row r = {kLowest, 0.f, kLowest};
  for (int s = lane; s < p.splits; s += 32) {
    const float* ml = p.part_ml + (first + static_cast<size_t>(s) * tile_rows) * 4;
    r.m = fmaxf(r.m, ml[0]);
    r.m2 = fmaxf(r.m2, ml[2]);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    r.m = fmaxf(r.m, __shfl_xor_sync(0xffffffffu, r.m, x));
    r.m2 = fmaxf(r.m2, __shfl_xor_sync(0xffffffffu, r.m2, x));
  }
  float sum[PER] = {};
  for (int s = 0; s < p.splits; ++s) {
    const size_t i = first + static_cast<size_t>(s) * tile_rows;
    const float4 ml = *reinterpret_cast<const float4*>(p.part_ml + i * 4);
    r.l += ml.y * ex2_approx(ml.x - r.m);
    const float w = ex2_approx(ml.z - r.m2);
#pragma unroll
    for (int j = 0; j < PER; ++j) sum[j] += p.part_o[i * D + lane + 32 * j] * w;
  }
  const int head = kvh * group + at % group;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    p.out[(static_cast<size_t>(b * p.q_per_seq + at / group) * p.n_q + head) * D + lane + 32 * j] =
        __float2bfloat16(kv8_finish(sum[j], r, p.sinks == nullptr ? nullptr : p.sinks + head));
}

template <int D, int NT>
static cudaError_t launch_attn_kv8(const AttnKv8Params& p, int batch, cudaStream_t stream) {
  constexpr int ROWS = 8 * NT;
  const size_t smem = static_cast<size_t>(kKv8Warps + 1) * ROWS * (D * sizeof(float) + sizeof(Kv8Row));
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_kv8_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.splits, p.n_kv * p.tiles, batch);
  cfg.blockDim = dim3(32 * kKv8Warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.splits > 1 && p.splits <= kKv8Cluster) {
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
  cudaError_t e = cudaLaunchKernelEx(&cfg, attn_kv8_kernel<D, NT>, p);
  eredu_count_launches(1);
  if (e == cudaSuccess && p.splits > kKv8Cluster) {
    e = launch_pdl(attn_kv8_combine_kernel<D>, dim3(p.q_per_seq * (p.n_q / p.n_kv), p.n_kv, batch), dim3(32), 0, stream, p, ROWS);
    eredu_count_launches(1);
  }
  return e;
}

}  // namespace eredu

using namespace eredu;

EREDU_TRACE_INSTALLER(attention_kv8)

// Query rows of one key / value head that a CTA takes at once; beyond 16, a tile more of them reads the pages again.
static int kv8_tile_rows(int rows) { return rows <= 8 ? 8 : 16; }

extern "C" int eredu_attn_kv8_decode(const void* q, const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales, void* out,
                                     const int* block_table, const int* seq_lens, const float* sinks, float* part_o, float* part_ml, int batch,
                                     int q_per_seq, int max_pages, int num_pages, int n_q, int n_kv, int D, int splits, int window, int chunk, float scale,
                                     int* status, cudaStream_t stream) {
  if (batch <= 0) return 0;
  if ((D != 64 && D != 128) || n_kv <= 0 || n_q % n_kv != 0 || n_q <= 0 || q_per_seq <= 0 || splits <= 0 || max_pages <= 0 || num_pages <= 0 ||
      window < 0 || chunk < 0 || batch > 65535 || (splits > kKv8Cluster && (part_o == nullptr || part_ml == nullptr)))
    return -2;
  AttnKv8Params p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k_codes = static_cast<const int8_t*>(k_codes);
  p.v_codes = static_cast<const int8_t*>(v_codes);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.sinks = sinks;
  p.part_o = part_o;
  p.part_ml = part_ml;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.n_q = n_q;
  p.n_kv = n_kv;
  p.q_per_seq = q_per_seq;
  const int rows = q_per_seq * (n_q / n_kv), tile = kv8_tile_rows(rows);
  p.tiles = (rows + tile - 1) / tile;
  p.splits = splits;
  p.window = window;
  p.chunk = chunk;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = status;
  if (static_cast<long long>(n_kv) * p.tiles > 65535) return -2;
  cudaError_t e;
  if (D == 128) e = tile == 8 ? launch_attn_kv8<128, 1>(p, batch, stream) : launch_attn_kv8<128, 2>(p, batch, stream);
  else e = tile == 8 ? launch_attn_kv8<64, 1>(p, batch, stream) : launch_attn_kv8<64, 2>(p, batch, stream);
  return static_cast<int>(e);
}
