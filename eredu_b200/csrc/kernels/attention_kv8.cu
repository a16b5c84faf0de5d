// Decode attention over a cache held in 8 bits (common/kv8.cuh): a few queries per sequence, 1 to k + 1 new tokens.
//
//   s_j = (q . c_j) scale ks,   o = sum_j 2^(s_j log2 e - m) vs c'_j / sum_j 2^(s_j log2 e - m)     (ks, vs: scales of token j's blocks)
//
// Bound by memory where contexts are long: every cached token is read once per key / value head, 2 D bytes. A warp walks pairs of pages of its own, which
// come into its ring in shared memory by cp.async, one pair on its way while another is worked on, and go from there into the registers of mma.sync by ldmatrix:
//   scores  S^T[16 tokens, 8 query rows] = K[16, D] Q^T as integers (m16n8k32): the codes are the A operand as they are. A query row is rounded to 16 bits,
//           with a power of two that brings its largest magnitude to 2^14 (a bf16 query keeps all its bits down to 2^-7 of that), and taken as a signed upper and
//           an unsigned lower byte.
//   output  O^T[D, 8 rows] = V^T[D, 16] P^T in f16 (m16n8k16): ldmatrix transposes pairs of channels; the two bytes of a pair are parted into an upper
//           and a lower accumulator row. P^T comes from S^T by movmatrix.
// The 8 query rows of a tile are the query heads that share the key / value head, times the new tokens; two tiles side by side above 8.
// Probabilities are rounded to f16 (11 bits; codes are exact in it). The page's value scale goes into what a probability weighs, relative to a running maximum of its
// own (m2, of s_j + log2 vs): the largest weight of a row is near 1 whatever the scales are, and one
// below 2^-14 of it is off by 2^-25 of it at most. The maxima are raised only where a score passes one by far.
//
// What it measured. Pages have to be read as they lie: with each lane fetching the bytes of its own fragments (pieces of 64 bytes) memory gives 4.85 TB/s at best,
// in order 6.5. Scores in f16 take 280 instructions a page and head, most of them conversions of codes; as integers 200, issued in 40 % of the cycles of 12 warps
// an SM, where most waiting is for memory. 64 sequences of 8192 tokens, 32 heads over 8: 142 us (6.0 TB/s; bf16 pages 305), split three ways 136; 32 of 2048
// 28 (46); one of 65536 31.6 (58), of which some 10 are the way in, to the CTA's place and the first pages, and the second kernel; of 512, head size 64, 5.2 (4.9).
#include <cuda_bf16.h>

#include <algorithm>

#include "../common/kv8_args.h"
#include "../common/kv8_store.cuh"
#include "../common/launch.h"
#include "../common/launch_count.h"
#include "../common/mma.cuh"
#include "../common/ptx.cuh"
#include "../common/trace.cuh"

namespace eredu {

struct AttnKv8Params {
  const __nv_bfloat16* q;          // [B * q_per_seq] rows of ld_q elements, n_q heads of D; or
  const float* q32;                // the same in 32 bits
  const int8_t *k_codes, *v_codes; // [pages, n_kv, 16, D]
  const float *k_scales, *v_scales;
  __nv_bfloat16* out;              // [B * q_per_seq, n_q, D]
  const int* block_table;          // [B rows of `pitch`], max_pages of them
  const int* seq_lens;             // [B], new tokens included
  const float* sinks;              // optional [n_q]
  float* part_o;                   // even shares: [CTAs, 2, rows of a tile, D]
  float* part_ml;                  //              [CTAs, 2, rows of a tile, 4]
  int4* joins;                     //              [CTAs]: what of the CTA's first part is to be added up, see attn_kv8_combine_kernel
  int batch, max_pages, pitch, num_pages, n_q, n_kv, q_per_seq, tiles, splits, window, chunk;
  int ctas, stretch;               // of even shares; joins that a CTA of the second kernel looks through, 32 at most
  int ld_q;
  uint32_t per_group;              // 2^32 / (n_q / n_kv), rounded up; 0 for a group of one
  float scale_log2;
  int* status;
  // A step from the projection's output (q, st.k and st.v in the same rows): queries are normalised and rotated as they are read, and the CTA that has the
  // page of a new token writes its rows there.
  Kv8StoreParams st;
  int settled;      // the kernel just before this one writes the projection's output only: no pages, tables, lengths, positions, slots or frequencies
};
// Token of query row r among those that share a key / value head (r < 2^16: exact), in place of a division of some thirty instructions.
__device__ __forceinline__ int kv8_token(const AttnKv8Params& p, int r) { return p.per_group == 0 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), p.per_group)); }

constexpr int kKv8Warps = 4;         // three CTAs of four warps to an SM: four pages a warp fill shared memory
constexpr int kKv8Threads = 32 * kKv8Warps;
constexpr int kKv8Cluster = 8;      // splits that meet in a cluster
// log2 units by which a score may pass the maximum in use, and a probability's weight the probability: what they give together, 2^14, f16 holds.
constexpr float kKv8Slack = 6.f, kKv8Weight = 8.f;
constexpr float kLowest = -3.402823466e38f;
constexpr uint32_t kNone = 0xffffffffu;   // bits of no scale
// Integer sums start at the bits of 1.5 * 2^23: as floats they are that plus the sum, which stays below 2^22 (128 * 127 * 255).
constexpr int kMagicBits = 0x4b400000;
constexpr float kMagic = 12582912.f;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes times the upper (signed) and the lower (unsigned) byte of queries. d = a b + c.
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ void mma_u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The smaller one, or no number where one of them is none (fminf gives the other).
__device__ __forceinline__ float min_or_none(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(v));
  return v;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void copy16(uint32_t smem, const int8_t* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(from) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int kv8_lowest_key(const AttnKv8Params& p, int pos) {
  if (p.window > 0) return max(0, pos - p.window + 1);
  return p.chunk > 0 && pos > 0 ? pos - pos % p.chunk : 0;
}

// Pages of a sequence that one of its queries sees: [first, end).
struct Kv8Pages {
  int first, end;
};
__device__ __forceinline__ Kv8Pages kv8_pages(const AttnKv8Params& p, int kv_len) {
  const int last = min((kv_len + kKv8Page - 1) >> 4, p.max_pages);
  return Kv8Pages{min(kv8_lowest_key(p, kv_len - p.q_per_seq) >> 4, last), last};
}
// Even shares: the pairs of pages of all sequences, heads and tiles of rows in one line, of which every CTA takes as many. A sequence has one pair at
// least, so that somebody writes its rows.
__device__ __forceinline__ int kv8_pairs(const AttnKv8Params& p, int b) {
  const Kv8Pages r = kv8_pages(p, p.seq_lens[b]);
  return max(1, (r.end - r.first + 1) / 2);
}
constexpr int kKv8LeastPairs = 4;   // of a CTA: one per warp
struct Kv8Place {
  int total, share;      // pairs in all, pairs of a CTA
  int b, begin, pairs;   // sequence in which pair `at` lies, where its pairs begin, and how many a head and tile of it has
};
// Place of pair share * i, by one warp; b = -1 behind the last.
__device__ __forceinline__ Kv8Place kv8_place(const AttnKv8Params& p, int i, int ctas, int lane) {
  const int heads = p.n_kv * p.tiles;
  Kv8Place r = {0, 0, -1, 0, 0};
  int pairs = lane < p.batch ? kv8_pairs(p, lane) : 0;
  r.total = __reduce_add_sync(0xffffffffu, pairs);
  for (int base = 32; base < p.batch; base += 32) r.total += __reduce_add_sync(0xffffffffu, base + lane < p.batch ? kv8_pairs(p, base + lane) : 0);
  r.total *= heads;
  r.share = max(kKv8LeastPairs, (r.total + ctas - 1) / ctas);
  const int at = r.share * i;
  if (at >= r.total) return r;
  for (int base = 0;; base += 32) {
    if (base > 0) pairs = base + lane < p.batch ? kv8_pairs(p, base + lane) : 0;
    int end = pairs;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, end, x);
      if (lane >= x) end += o;
    }
    const uint32_t behind = __ballot_sync(0xffffffffu, r.begin + end * heads > at);
    if (behind != 0) {   // at < total: it comes
      const int l = __ffs(behind) - 1;
      r.b = base + l;
      r.pairs = __shfl_sync(0xffffffffu, pairs, l);
      r.begin += __shfl_sync(0xffffffffu, end - pairs, l) * heads;
      return r;
    }
    r.begin += __shfl_sync(0xffffffffu, end, 31) * heads;
  }
}

// What a row has gathered: maximum and sum of the scores, maximum the output is relative to.
struct Kv8Row {
  float m, l, m2;
};
// What takes a row's output, relative to 2^m2, to the sum of its probabilities: o * over * up. A sink is a key of zero value. A row that sees nothing is zero.
struct Kv8Finish {
  float over, up;
};
__device__ __forceinline__ Kv8Finish kv8_finish(const Kv8Row& r, const float* sink) {
  float m = r.m, l = r.l;
  if (sink != nullptr) {
    const float s = *sink * 1.4426950408889634f;
    const float top = fmaxf(m, s);
    l = l * ex2_approx(m - top) + ex2_approx(s - top);
    m = top;
  }
  if (l == 0.f || r.l == 0.f) return Kv8Finish{0.f, 0.f};
  return Kv8Finish{1.f / l, ex2_approx(r.m2 - m)};
}
__device__ __forceinline__ float4 fma4(float4 a, float w, float4 c) { return make_float4(fmaf(a.x, w, c.x), fmaf(a.y, w, c.y), fmaf(a.z, w, c.z), fmaf(a.w, w, c.w)); }
__device__ __forceinline__ void store_out(__nv_bfloat16* to, float4 v, float up) {
  *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(v.x * up, v.y * up), pack_bf16x2(v.z * up, v.w * up));
}

__device__ __forceinline__ float exp2_of(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }   // -126 <= e <= 127
// Four values of a query row times two powers of two, rounded to 16 bits: their upper bytes and their lower bytes.
__device__ __forceinline__ uint2 query_bytes(float4 x, float up, float more) {
  auto whole = [&](float v) { return static_cast<uint32_t>(min(__float2int_rn(v * up * more), 32767)); };
  const uint32_t a = whole(x.x), b = whole(x.y), c = whole(x.z), d = whole(x.w);
  return make_uint2(__byte_perm(__byte_perm(a, b, 0x0051), __byte_perm(c, d, 0x0051), 0x5410), __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410));
}

// grid (splits, n_kv * tiles, B): the splits of a sequence and head form a cluster and meet in its shared memory.
// EVEN: grid (CTAs): even shares of all pairs, so that long and short sequences, and few and many, fill the SMs alike. What a CTA has of a sequence and head
// that others have a part of as well goes to memory, and attn_kv8_combine_kernel adds it up.
template <int D, int NT, bool EVEN, bool STEP>
__global__ void __launch_bounds__(kKv8Threads, 3) attn_kv8_kernel(AttnKv8Params p) {
  constexpr int ROWS = 8 * NT, KC = D / 64, STEPS = D / 16, WIDE = D + 4;   // WIDE: lanes of four rows meet all banks
  constexpr int PAGE_BYTES = 2 * kKv8Page * D;
  // on lines of 128 bytes: rings 16 bytes off them cost 17 % (32 sequences of 2048 29.8 -> 34.9 us)
  extern __shared__ __align__(128) uint8_t smem[];
  // queries as bytes [NT][2 KC][32 lanes], then the rings [warps][2 pairs][2 pages]; behind the last page, what the warps have gathered takes their place
  uint4* q_s = reinterpret_cast<uint4*>(smem);
  uint8_t* rings = smem + NT * 2 * KC * 512;
  float* o_warp = reinterpret_cast<float*>(rings);       // [warps][ROWS][WIDE]
  float* o_s = o_warp + kKv8Warps * ROWS * WIDE;         // [ROWS][D]
  Kv8Row* row_warp = reinterpret_cast<Kv8Row*>(o_s + ROWS * D);   // [warps][ROWS]
  Kv8Row* row_s = row_warp + kKv8Warps * ROWS;           // [ROWS]
  float* weight = reinterpret_cast<float*>(row_s + ROWS);         // [warps, or splits][ROWS]
  __shared__ float back_s[ROWS], up_s[ROWS];
  __shared__ size_t out_s[ROWS];          // where a row's output goes
  __shared__ float scale_s[kKv8Warps];    // scales of blocks with new rows
  __shared__ __align__(16) float turns_s[STEP ? kKv8StepTokens * D : 1];   // cosines and sines of the tile's tokens
  pdl_launch_early();
  trace_mark(kTraceAttnDecode, kTraceStart);
  // settled: what lies in front of the projection's output in time - places, pages, angles - is read ahead of the wait; nothing is written
  bool waited = !(STEP && p.settled);
  auto wait_for_input = [&]() {
    pdl_wait();
    trace_mark(kTraceAttnDecode, kTraceAfterWait);
    pdl_launch_dependents();
    waited = true;
  };
  if (waited) wait_for_input();
  const int warp = static_cast<int>(warp_uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = p.n_q / p.n_kv, rows_all = p.q_per_seq * group;
  // the CTA's share: pairs [at, end) of the line; or one split
  Kv8Place place = {};
  int at = 0, end = 0, slot = 0;
  int4 join = make_int4(0, 0, 0, 0);
  if (EVEN) {
    place = kv8_place(p, blockIdx.x, gridDim.x, lane);
    at = place.share * blockIdx.x;
    if (place.b < 0) {
      if (!waited) wait_for_input();
      if (threadIdx.x == 0) p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
    end = min(place.total, at + place.share);
    // of the CTAs that have a part of the first rows, the second one stands for all: it begins behind their first pair, and the CTA in front does not
    const int head_tile = (at - place.begin) / place.pairs, begin = place.begin + head_tile * place.pairs;
    if (at > begin && at - place.share <= begin)
      join = make_int4((begin + place.pairs - 1) / place.share - blockIdx.x + 2, place.b, head_tile, at - place.share == begin);
  }
  do {
  const int b = EVEN ? place.b : blockIdx.z, head_tile = EVEN ? (at - place.begin) / place.pairs : blockIdx.y, split = EVEN ? 0 : blockIdx.x;
  const int kvh = p.tiles == 1 ? head_tile : head_tile / p.tiles, r0 = (head_tile - kvh * p.tiles) * ROWS, rows = min(ROWS, rows_all - r0);
  const int kv_len = p.seq_lens[b], pos_new = kv_len - p.q_per_seq;
  const int token0 = kv8_token(p, r0), pos_first = pos_new + token0, pos_last = pos_new + kv8_token(p, r0 + rows - 1);   // positions of the tile's first and last row
  const Kv8Pages pages = kv8_pages(p, kv_len);
  int page0, page1;
  bool whole = p.splits == 1;                                                                 // nobody else has a part of these rows
  if (EVEN) {
    const int first = (at - place.begin) % place.pairs, n = min(end - at, place.pairs - first);
    whole = n == place.pairs;
    at += n;
    page0 = pages.first + 2 * first;
    page1 = min(pages.end, page0 + 2 * n);
  } else {
    const int per = whole ? pages.end - pages.first : (pages.end - pages.first + p.splits - 1) / p.splits;
    page0 = pages.first + split * per;
    page1 = min(pages.end, page0 + per);
  }
  const int last_key = page1 * kKv8Page - 1;                                                  // of this part
  const int mask_hi = min(pos_first, last_key), mask_lo = kv8_lowest_key(p, pos_last);        // pages inside need no mask

  // ---- pairs warp, warp + 4, ... of the part. Lanes 2 i and 2 i + 1 hold page ids and scales of the i-th of 16 turns; those of the 16 before stay at hand.
  const int* table = p.block_table + static_cast<size_t>(b) * p.pitch;
  const int turns = page1 > page0 + 2 * warp ? (page1 - page0 - 2 * warp + 2 * kKv8Warps - 1) / (2 * kKv8Warps) : 0;
  int ids = 0;
  float ks = 0.f, ev = 0.f, ks_before = 0.f, ev_before = 0.f;
  auto look_up = [&](int turn) {
    const int pg = page0 + 2 * (warp + kKv8Warps * (turn + (lane >> 1))) + (lane & 1);
    ids = pg < page1 ? table[pg] : 0;
    if (ids < 0 || ids >= p.num_pages) {
      report_status(p.status, kStatusBadArgument);
      ids = 0;
    }
    const size_t cell = static_cast<size_t>(ids) * p.n_kv + kvh;
    ks_before = ks;
    ev_before = ev;
    ks = p.k_scales[cell];
    ev = p.v_scales[cell];
  };
  // A page comes in as it lies in memory, 512 bytes at a time. ldmatrix: lane i names row i & 7 of matrix i >> 3; the four are tokens 0 to 7 and 8 to 15 of one
  // piece, then of the next.
  const uint8_t* mine = rings + warp * (4 * PAGE_BYTES);
  const int in_at = kv8_piece<D>(lane / (D / 16), lane % (D / 16));
  const int out_at = kv8_piece<D>(lane & 15, lane >> 4);
  const uint32_t ring = smem_u32(mine);
  auto fetch = [&](int turn) {
    if ((turn & 15) == 0) look_up(turn);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int id = __shfl_sync(0xffffffffu, ids, 2 * (turn & 15) + u);
      const size_t cell = (static_cast<size_t>(id) * p.n_kv + kvh) * (kKv8Page * D) + lane * 16;
      const uint32_t to = ring + ((turn & 1) * 2 + u) * PAGE_BYTES;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int at = i * 512 + (D == 128 && (i & 1) ? in_at ^ 64 : in_at);   // rows 4 i and on, of which every second four have bit 2
        copy16(to + at, p.k_codes + cell + i * 512);
        copy16(to + PAGE_BYTES / 2 + at, p.v_codes + cell + i * 512);
      }
    }
  };
  if (turns > 0) fetch(0);
  cp_async_commit();
  if (turns > 1) fetch(1);
  cp_async_commit();

  constexpr int RPI = 128 / D;                          // query rows a warp holds at once, four channels a lane
  const int half = STEP ? p.st.rot / 2 : 0;
  if (STEP) {
    const int tokens = pos_last - pos_first + 1;
    const int* positions = p.st.positions + static_cast<size_t>(b) * p.q_per_seq + token0;
    for (int n = threadIdx.x / (D / 2), i = threadIdx.x % (D / 2); n < tokens; n += kKv8Threads / (D / 2))
      if (i < half) turn_of(positions[n], p.st.inv_freq[i], p.st.attn_factor, turns_s[n * p.st.rot + i], turns_s[n * p.st.rot + half + i]);
    __syncthreads();
  }
  // The new rows lie in two pages of this part at most, from new_page on. Warps 0 and 2 write their keys, 1 and 3 their values - to memory, and to the ring where
  // the page is on its way to it already.
  const int new_page = STEP ? max(page0, pos_new < 0 ? 0 : pos_new / kKv8Page) : page1;
  const bool news = new_page < page1;
  const int my_page = new_page + (warp >> 1);
  const int my_row = STEP ? max(0, my_page * kKv8Page - pos_new) : 0, my_end = STEP && my_page < page1 ? min(p.q_per_seq, (my_page + 1) * kKv8Page - pos_new) : 0;
  long long my_slot = -1;
  float my_scale = 0.f;
  int my_id = -1;                  // the page's number in the table
  uint8_t* my_held = nullptr;
  if (STEP && my_row < my_end) {
    my_slot = p.st.slots[b * p.q_per_seq + my_row];
    if (my_slot >= 0 && (my_slot >> 4) < p.num_pages) my_scale = ((warp & 1) == 0 ? p.k_scales : p.v_scales)[(my_slot >> 4) * p.n_kv + kvh];
    my_id = table[my_page];
    const int i = my_page - page0;
    if (i < 4 * kKv8Warps)
      my_held = rings + (i >> 1) % kKv8Warps * (4 * PAGE_BYTES) + (i / (2 * kKv8Warps) * 2 + (i & 1)) * PAGE_BYTES + (warp & 1) * (PAGE_BYTES / 2);
  }
  if (STEP && !waited) wait_for_input();
  if (EVEN && slot == 0 && threadIdx.x == 0) p.joins[blockIdx.x] = join;
  constexpr int QUERIES = ROWS / (kKv8Warps * RPI);     // of a warp, all on their way before the first is looked at
  float4 query[QUERIES];
#pragma unroll
  for (int i = 0; i < QUERIES; ++i) {
    const int r = r0 + min((i * kKv8Warps + warp) * RPI + lane / (D / 4), rows - 1), token = kv8_token(p, r);
    const size_t at = static_cast<size_t>(b * p.q_per_seq + token) * p.ld_q + (kvh * group + r - token * group) * D;
    query[i] = !STEP && p.q32 != nullptr ? *reinterpret_cast<const float4*>(p.q32 + at + lane % (D / 4) * 4) : load_row4<D>(p.q + at, lane);
  }
  Kv8Few<D> few;
  if (STEP && my_row < my_end)
    few.load(((warp & 1) == 0 ? p.st.k : p.st.v) + static_cast<size_t>(b * p.q_per_seq + my_row) * ((warp & 1) == 0 ? p.st.ld_k : p.st.ld_v) + kvh * D,
             (warp & 1) == 0 ? p.st.ld_k : p.st.ld_v, my_end - my_row, lane);
  // ---- the query rows: bytes into shared memory, and what takes a score back to log2 units
#pragma unroll(STEP ? 1 : QUERIES)
  for (int i = 0; i < QUERIES; ++i) {      // (a step's rows one after the other: what rotates them is long, and read once)
    const int row = (i * kKv8Warps + warp) * RPI + lane / (D / 4), c = lane % (D / 4);       // this lane has channels 4 c and three more
    const bool in = row < rows;
    float4 x = query[0];
#pragma unroll
    for (int j = 1; j < QUERIES; ++j)
      if (i == j) x = query[j];
    if (STEP) x = prepared<D>(p.st, x, p.st.q_norm_w, turns_s + (kv8_token(p, r0 + min(row, rows - 1)) - token0) * p.st.rot, lane);
    if (!in) x = make_float4(0.f, 0.f, 0.f, 0.f);
    uint32_t top = max(max(__float_as_uint(fabsf(x.x)), __float_as_uint(fabsf(x.y))), max(__float_as_uint(fabsf(x.z)), __float_as_uint(fabsf(x.w))));
#pragma unroll
    for (int o = D / 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool fine = top < 0x7f800000u;
    const int e = static_cast<int>(top >> 23), up = !fine || e == 0 ? 0 : 141 - e, up0 = up / 2;   // 2^(e - 127) <= top; 2^up brings it to 2^14
    const uint2 bytes = query_bytes(x, exp2_of(up0), exp2_of(up - up0));
    // the B fragments of lane 4 g + t: channels 32 j + 4 t and 32 j + 16 + 4 t of row g, upper bytes of either, then lower bytes
    uint32_t* to = reinterpret_cast<uint32_t*>(q_s + ((row >> 3) * 2 * KC + (c >> 3)) * 32 + (row & 7) * 4 + (c & 3)) + (c >> 2 & 1);
    to[0] = bytes.x;
    to[2] = bytes.y;
    if (c == 0) back_s[row] = fine ? p.scale_log2 * exp2_of(-up0) * exp2_of(up0 - up) : __uint_as_float(0x7fc00000u);
  }
  // ---- the new rows
  if (STEP && news) {
    float scale = __uint_as_float(kNone);
    const int row0 = b * p.q_per_seq;
    cp_async_wait<0>();
    __syncthreads();      // what the rings hold of all warps has landed
#pragma unroll 1
    for (int r = my_row; r < my_end;) {
      const long long to = r == my_row ? my_slot : p.st.slots[row0 + r];
      int n = 1;
      if (to >= 0 && (to >> 4) < p.num_pages) {
        while (r + n < my_end && (to + n) % kKv8Page != 0 && p.st.slots[row0 + r + n] == to + n) ++n;
        const long long cell = (to >> 4) * p.n_kv + kvh;
        const float before = r == my_row ? my_scale : ((warp & 1) == 0 ? p.k_scales : p.v_scales)[cell];
        const bool seen = to >> 4 == my_id;
        uint8_t* held = seen ? my_held : nullptr;
        float now;
        if ((warp & 1) == 0) now = store_few<D, true>(p.st, few, r - my_row, n, static_cast<int>(to & 15), cell, turns_s + my_row * p.st.rot, lane, before, held);
        else now = store_few<D, false>(p.st, few, r - my_row, n, static_cast<int>(to & 15), cell, turns_s, lane, before, held);
        __syncwarp();
        if (seen) scale = now;
      } else if (to >= 0) {
        report_status(p.status, kStatusBadArgument);
      }
      r += n;
    }
    if (lane == 0) scale_s[warp] = scale;
  }
  __syncthreads();
  if (STEP && news) {      // looked up in front of the write
    const int i = page0 + 2 * (warp + kKv8Warps * (lane >> 1)) + (lane & 1) - new_page;
    if (i >= 0 && i < page1 - new_page) {
      const float k = scale_s[2 * min(i, 1)], v = scale_s[2 * min(i, 1) + 1];
      if (__float_as_uint(k) != kNone) ks = k;
      if (__float_as_uint(v) != kNone) ev = v;
    }
  }
  float back[NT][2];                                    // of the lane's columns 2t, 2t + 1
  int pos[NT][2];
  float o[NT][STEPS][4], m[NT][2], m2[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      back[nt][c] = back_s[nt * 8 + 2 * t + c];
      pos[nt][c] = pos_new + kv8_token(p, r0 + min(nt * 8 + 2 * t + c, rows - 1));
      m[nt][c] = m2[nt][c] = kLowest;
      l[nt][c] = 0.f;
    }
  }

  for (int turn = 0; turn < turns; ++turn) {
    const int tok = (page0 + 2 * (warp + kKv8Warps * turn)) * kKv8Page;
    cp_async_wait<1>();
    __syncwarp();
    const uint32_t from = ring + (turn & 1) * 2 * PAGE_BYTES;
    // scales of this turn: its 16 may have been followed by the next ones already
    const bool before = (turn >> 4) != (min(turn + 1, turns - 1) >> 4);
    float s[2][NT][4], ev_now[2];
    {
      int hi[2][NT][4], lo[2][NT][4];
      const int magic[4] = {kMagicBits, kMagicBits, kMagicBits, kMagicBits};
#pragma unroll
      for (int j = 0; j < 2 * KC; ++j) {          // 32 channels at a time
        uint32_t a[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) ldsm_x4(from + u * PAGE_BYTES + (out_at ^ (32 * j)), a[u][0], a[u][1], a[u][2], a[u][3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 q = q_s[(nt * 2 * KC + j) * 32 + lane];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (j == 0) {
              mma_s8(hi[u][nt], a[u], q.x, q.y, magic);
              mma_u8(lo[u][nt], a[u], q.z, q.w, magic);
            } else {
              mma_s8(hi[u][nt], a[u], q.x, q.y, hi[u][nt]);
              mma_u8(lo[u][nt], a[u], q.z, q.w, lo[u][nt]);
            }
          }
        }
      }
      // ---- scores in log2 units
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = 2 * (turn & 15) + u;
        const float ks_now = __shfl_sync(0xffffffffu, before ? ks_before : ks, at);
        ev_now[u] = lg2_approx(__shfl_sync(0xffffffffu, before ? ev_before : ev, at));   // (exact for powers of two)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float f0 = back[nt][0] * ks_now, f1 = back[nt][1] * ks_now;
#pragma unroll
          for (int c = 0; c < 4; ++c) s[u][nt][c] = (fmaf(__int_as_float(hi[u][nt][c]), 256.f, -257.f * kMagic) + __int_as_float(lo[u][nt][c])) * (c & 1 ? f1 : f0);
        }
      }
    }
    const bool edge = tok + 2 * kKv8Page - 1 > mask_hi || tok < mask_lo;
    if (edge) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int high = min(pos[nt][c], last_key) - tok - g, low = kv8_lowest_key(p, pos[nt][c]) - tok - g;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (u * kKv8Page + h * 8 > high || u * kKv8Page + h * 8 < low) s[u][nt][c + 2 * h] = -INFINITY;
        }
    }
    // ---- d: score against the maximum in use. f: what a probability weighs in the output, against m2
    float d[2][NT][4], f[2][NT][2];
    auto relate = [&]() {
      bool passes = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            d[u][nt][c] = s[u][nt][c] - m[nt][c];
            d[u][nt][c + 2] = s[u][nt][c + 2] - m[nt][c];
            f[u][nt][c] = ev_now[u] + (m[nt][c] - m2[nt][c]);
          }
          passes |= fmaxf(fmaxf(d[0][nt][c], d[0][nt][c + 2]), fmaxf(d[1][nt][c], d[1][nt][c + 2])) > kKv8Slack ||
                    fmaxf(f[0][nt][c], f[1][nt][c]) > kKv8Weight;
        }
      return passes;
    };
    if (__any_sync(0xffffffffu, relate())) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float down[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float t0 = fmaxf(s[0][nt][c], s[0][nt][c + 2]), t1 = fmaxf(s[1][nt][c], s[1][nt][c + 2]);
          float up = fmaxf(m[nt][c], fmaxf(t0, t1)), up2 = fmaxf(m2[nt][c], fmaxf(t0 + ev_now[0], t1 + ev_now[1]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, x));
            up2 = fmaxf(up2, __shfl_xor_sync(0xffffffffu, up2, x));
          }
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
      relate();
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
        // (value scales that are further apart than this has room for, over 2^126, lose the smaller ones; the scale of a block that is no number stays none)
        const float f0 = ex2_approx(min_or_none(f[u][nt][0], 126.f)), f1 = ex2_approx(min_or_none(f[u][nt][1], 126.f));
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float e = ex2_approx(d[u][nt][c]);
          l[nt][c & 1] += e;
          w[c] = e * (c & 1 ? f1 : f0);
        }
        if (edge) {   // a masked place is zero whatever the scale of its block is
#pragma unroll
          for (int c = 0; c < 4; ++c) w[c] = s[u][nt][c] == -INFINITY ? 0.f : w[c];
        }
        pf[nt][0] = transposed(pack_f16x2(w[0], w[1]));
        pf[nt][1] = transposed(pack_f16x2(w[2], w[3]));
      }
      // ---- output
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        // channels 2g and 2g + 1 of a piece, tokens 2t, 2t + 1 and 8 more: bytes {2t: a, b; 2t + 1: a, b}
        uint32_t v[4];
        ldsm_x4_t(from + u * PAGE_BYTES + PAGE_BYTES / 2 + (out_at ^ (32 * j)), v[0], v[1], v[2], v[3]);
        uint32_t a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = kv8_parted<false>(v[i]);
          b[i] = kv8_parted<true>(v[i]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(o[nt][2 * j], a[0], b[0], a[1], b[1], pf[nt][0], pf[nt][1]);
          mma_f16(o[nt][2 * j + 1], a[2], b[2], a[3], b[3], pf[nt][0], pf[nt][1]);
        }
      }
    }
    __syncwarp();
    if (turn + 2 < turns) fetch(turn + 2);
    cp_async_commit();
  }

  // ---- the warps of the CTA together
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float sum = l[nt][c];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      const int row = nt * 8 + 2 * t + c;
      if (g == 0) row_warp[warp * ROWS + row] = Kv8Row{m[nt][c], sum, m2[nt][c]};
      float2* dst = reinterpret_cast<float2*>(o_warp + (warp * ROWS + row) * WIDE + 2 * g);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) dst[8 * i] = make_float2(o[nt][i][c], o[nt][i][c + 2]);
    }
  __syncthreads();
  if (threadIdx.x < ROWS) {
    const int row = threadIdx.x;
    Kv8Row r = {kLowest, 0.f, kLowest};
    for (int w = 0; w < kKv8Warps; ++w) {
      r.m = fmaxf(r.m, row_warp[w * ROWS + row].m);
      r.m2 = fmaxf(r.m2, row_warp[w * ROWS + row].m2);
    }
    for (int w = 0; w < kKv8Warps; ++w) r.l += row_warp[w * ROWS + row].l * ex2_approx(row_warp[w * ROWS + row].m - r.m);
    const int n = r0 + min(row, rows - 1), token = kv8_token(p, n), head = kvh * group + n - token * group;
    out_s[row] = (static_cast<size_t>(b * p.q_per_seq + token) * p.n_q + head) * D;
    const Kv8Finish f = whole ? kv8_finish(r, p.sinks == nullptr ? nullptr : p.sinks + head) : Kv8Finish{1.f, 1.f};
    for (int w = 0; w < kKv8Warps; ++w) weight[w * ROWS + row] = ex2_approx(row_warp[w * ROWS + row].m2 - r.m2) * f.over;
    up_s[row] = f.up;
    row_s[row] = r;
  }
  __syncthreads();
  const size_t part = (static_cast<size_t>(blockIdx.x) * 2 + slot) * ROWS;
  for (int i = threadIdx.x; i < rows * (D / 4); i += kKv8Threads) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kKv8Warps; ++w) sum = fma4(*reinterpret_cast<const float4*>(o_warp + (w * ROWS + row) * WIDE + d), weight[w * ROWS + row], sum);
    if (whole) {
      store_out(p.out + out_s[row] + d, sum, up_s[row]);
    } else if (!EVEN) {
      *reinterpret_cast<float4*>(o_s + row * D + d) = sum;
    } else {
      *reinterpret_cast<float4*>(p.part_o + (part + row) * D + d) = sum;
      if (d == 0) *reinterpret_cast<float4*>(p.part_ml + (part + row) * 4) = make_float4(row_s[row].m, row_s[row].l, row_s[row].m2, 0.f);
    }
  }
  if (EVEN) {
    slot = 1;
    if (at < end && at == place.begin + place.pairs * p.n_kv * p.tiles) {
      place.begin = at;
      place.pairs = kv8_pairs(p, ++place.b);
    }
    __syncthreads();   // shared memory is free again
    continue;
  }
  if (whole) return;
  // ---- the splits: every CTA of the cluster finishes some of the values
  cluster_arrive_release();
  cluster_wait_acquire();
  if (threadIdx.x < ROWS) {
    const int row = threadIdx.x;
    Kv8Row part_row[kKv8Cluster], r = {kLowest, 0.f, kLowest};
#pragma unroll
    for (int s = 0; s < kKv8Cluster; ++s) {
      if (s >= p.splits) break;
      const uint32_t at = mapa_shared(smem_u32(row_s + row), s);
      part_row[s] = Kv8Row{ld_cluster_f32(at), ld_cluster_f32(at + 4), ld_cluster_f32(at + 8)};
    }
#pragma unroll
    for (int s = 0; s < kKv8Cluster; ++s) {
      if (s >= p.splits) break;
      r.m = fmaxf(r.m, part_row[s].m);
      r.m2 = fmaxf(r.m2, part_row[s].m2);
    }
#pragma unroll
    for (int s = 0; s < kKv8Cluster; ++s) {
      if (s >= p.splits) break;
      r.l += part_row[s].l * ex2_approx(part_row[s].m - r.m);
    }
    const int n = r0 + min(row, rows - 1);
    const Kv8Finish f = kv8_finish(r, p.sinks == nullptr ? nullptr : p.sinks + kvh * group + n - kv8_token(p, n) * group);
#pragma unroll
    for (int s = 0; s < kKv8Cluster; ++s) {
      if (s >= p.splits) break;
      weight[s * ROWS + row] = ex2_approx(part_row[s].m2 - r.m2) * f.over;
    }
    up_s[row] = f.up;
  }
  __syncthreads();
  for (int i = split * kKv8Threads + threadIdx.x; i < rows * (D / 4); i += p.splits * kKv8Threads) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float4 o4[kKv8Cluster], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < kKv8Cluster; ++s) {
      if (s >= p.splits) break;
      o4[s] = ld_cluster_f32x4(mapa_shared(smem_u32(o_s + row * D + d), s));
    }
#pragma unroll
    for (int s = 0; s < kKv8Cluster; ++s) {
      if (s >= p.splits) break;
      sum = fma4(o4[s], weight[s * ROWS + row], sum);
    }
    store_out(p.out + out_s[row] + d, sum, up_s[row]);
  }
  cluster_arrive_relaxed();   // nobody leaves while its shared memory is read; nothing is handed over (with release: 0.1 to 0.3 us for stores on their way)
  cluster_wait_acquire();
  } while (EVEN && at < end);
}

// Rows of a sequence and head of which several CTAs have a part: joins[i] = {parts, sequence, head and tile, whether the first part, that of CTA i - 1, is also
// the first of that CTA}, no parts where there is nothing to add up. grid (stretches of joins, rows of a tile): two stretches for each sequence and head, a CTA
// for each of all joins, mostly without work, only where there are no fewer of those. Four warps take some parts each.
// One sequence of 65536 tokens, attention in all: a CTA for every join 33.1 (64 query heads 35.0) us, stretches 31.6 (31.9), with eight warps 30.8 (31.5); 64 of
// 8192, where parts are two or three: 141.7, 142.8, with eight warps 148.7.
constexpr int kCombineWarps = 4;
template <int D, int NT>
__global__ void __launch_bounds__(32 * kCombineWarps) attn_kv8_combine_kernel(AttnKv8Params p) {
  constexpr int PER = D / 32, ROWS = 8 * NT;
  __shared__ Kv8Row row_s[kCombineWarps];
  __shared__ float sum_s[kCombineWarps][D];
  pdl_launch_early();
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.n_q / p.n_kv;
  const int i0 = blockIdx.x * p.stretch;
  const int4 held = lane < p.stretch && i0 + lane < p.ctas ? p.joins[i0 + lane] : make_int4(0, 0, 0, 0);
  for (uint32_t there = __ballot_sync(0xffffffffu, held.x != 0); there != 0; there &= there - 1) {
    const int from = __ffs(there) - 1, c0 = i0 + from - 1;
    const int parts = __shfl_sync(0xffffffffu, held.x, from), b = __shfl_sync(0xffffffffu, held.y, from), head_tile = __shfl_sync(0xffffffffu, held.z, from);
    const int first = __shfl_sync(0xffffffffu, held.w, from);
    const int kvh = p.tiles == 1 ? head_tile : head_tile / p.tiles, n = (head_tile - kvh * p.tiles) * ROWS + row;
    if (n >= p.q_per_seq * group) continue;
    // the first of the CTAs has it as its last part, the others as their first
    auto place_of = [&](int s) { return (static_cast<size_t>(c0 + s) * 2 + (s == 0 && first == 0 ? 1 : 0)) * ROWS + row; };
    Kv8Row r = {kLowest, 0.f, kLowest};
    float sum[PER] = {};
    // up to eight parts a warp at once, so that their loads are on the way together
    for (int s0 = warp; s0 < parts; s0 += 8 * kCombineWarps) {
      float4 ml[8];
      float part[8][PER];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int s = s0 + i * kCombineWarps;
        const size_t at = place_of(min(s, parts - 1));
        ml[i] = s < parts ? *reinterpret_cast<const float4*>(p.part_ml + at * 4) : make_float4(kLowest, 0.f, kLowest, 0.f);
#pragma unroll
        for (int j = 0; j < PER; ++j) part[i][j] = s < parts ? p.part_o[at * D + lane + 32 * j] : 0.f;
      }
      float m = r.m, m2 = r.m2;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m = fmaxf(m, ml[i].x);
        m2 = fmaxf(m2, ml[i].z);
      }
      r.l *= ex2_approx(r.m - m);
      const float down = ex2_approx(r.m2 - m2);
#pragma unroll
      for (int j = 0; j < PER; ++j) sum[j] *= down;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r.l += ml[i].y * ex2_approx(ml[i].x - m);
        const float w = ex2_approx(ml[i].z - m2);
#pragma unroll
        for (int j = 0; j < PER; ++j) sum[j] += part[i][j] * w;
      }
      r.m = m;
      r.m2 = m2;
    }
    if (lane == 0) row_s[warp] = r;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum_s[warp][lane + 32 * j] = sum[j];
    __syncthreads();
    if (threadIdx.x < D) {   // (D is at most the number of threads)
      r = Kv8Row{kLowest, 0.f, kLowest};
#pragma unroll
      for (int w = 0; w < kCombineWarps; ++w) {
        r.m = fmaxf(r.m, row_s[w].m);
        r.m2 = fmaxf(r.m2, row_s[w].m2);
      }
      float all = 0.f;
#pragma unroll
      for (int w = 0; w < kCombineWarps; ++w) {
        r.l += row_s[w].l * ex2_approx(row_s[w].m - r.m);
        all += sum_s[w][threadIdx.x] * ex2_approx(row_s[w].m2 - r.m2);
      }
      const int token = kv8_token(p, n), head = kvh * group + n - token * group;
      const Kv8Finish f = kv8_finish(r, p.sinks == nullptr ? nullptr : p.sinks + head);
      p.out[(static_cast<size_t>(b * p.q_per_seq + token) * p.n_q + head) * D + threadIdx.x] = __float2bfloat16(all * f.over * f.up);
    }
    if ((there & (there - 1)) != 0) __syncthreads();   // the next rows go to the same places
  }
}

template <int D, int NT, bool EVEN, bool STEP>
static cudaError_t launch_attn_kv8(const AttnKv8Params& p, int ctas, cudaStream_t stream) {
  constexpr int ROWS = 8 * NT;
  constexpr size_t rings = static_cast<size_t>(kKv8Warps) * 4 * 2 * kKv8Page * D;
  constexpr size_t gathered = static_cast<size_t>(ROWS) * ((kKv8Warps * (D + 4) + D) * sizeof(float) + (kKv8Warps + 1) * sizeof(Kv8Row) + kKv8Cluster * sizeof(float));
  constexpr size_t smem = NT * (D / 32) * 512 + (rings > gathered ? rings : gathered);
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_kv8_kernel<D, NT, EVEN, STEP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = EVEN ? dim3(ctas) : dim3(p.splits, p.n_kv * p.tiles, p.batch);
  cfg.blockDim = dim3(kKv8Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (!EVEN && p.splits > 1) {
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
  cudaError_t e = cudaLaunchKernelEx(&cfg, attn_kv8_kernel<D, NT, EVEN, STEP>, p);
  eredu_count_launches(1);
  if (EVEN && e == cudaSuccess) {
    e = launch_pdl(attn_kv8_combine_kernel<D, NT>, dim3((ctas + p.stretch - 1) / p.stretch, p.tiles == 1 ? p.q_per_seq * (p.n_q / p.n_kv) : ROWS), dim3(32 * kCombineWarps), 0, stream, p);
    eredu_count_launches(1);
  }
  return e;
}

}  // namespace eredu

using namespace eredu;

EREDU_TRACE_INSTALLER(attention_kv8)

// Query rows of one key / value head that a CTA takes at once; beyond 16, a tile more of them reads the pages again.
static int kv8_tile_rows(int rows) { return rows <= 8 ? 8 : 16; }

static int attn_kv8(AttnKv8Params& p, int D, int ctas, bool step, cudaStream_t stream) {
  if (p.batch <= 0) return 0;
  if ((D != 64 && D != 128) || p.n_kv <= 0 || p.n_q % p.n_kv != 0 || p.n_q <= 0 || p.q_per_seq <= 0 || p.splits < 0 || p.splits > kKv8Cluster ||
      p.max_pages <= 0 || p.num_pages <= 0 || p.window < 0 || p.chunk < 0 || p.ld_q % 4 != 0)
    return -2;
  const int rows = p.q_per_seq * (p.n_q / p.n_kv), tile = kv8_tile_rows(rows);
  if (rows >= 1 << 16) return -2;
  p.tiles = (rows + tile - 1) / tile;
  p.ctas = ctas;
  p.stretch = static_cast<int>(std::clamp(ctas / (2LL * p.batch * p.n_kv * p.tiles), 1LL, 32LL));
  const uint32_t group = p.n_q / p.n_kv;
  p.per_group = group == 1 ? 0 : static_cast<uint32_t>(((1ULL << 32) + group - 1) / group);
  const long long line = static_cast<long long>(p.batch) * p.n_kv * p.tiles * (p.max_pages / 2 + 1);
  if (p.splits == 0 ? ctas <= 0 || p.part_o == nullptr || p.part_ml == nullptr || p.joins == nullptr || line > (1LL << 30)
                    : p.batch > 65535 || static_cast<long long>(p.n_kv) * p.tiles > 65535)
    return -2;
  cudaError_t e;
#define ER_KV8(D_, NT_)                                                                                                                            \
  e = step ? (p.splits == 0 ? launch_attn_kv8<D_, NT_, true, true>(p, ctas, stream) : launch_attn_kv8<D_, NT_, false, true>(p, ctas, stream))      \
           : (p.splits == 0 ? launch_attn_kv8<D_, NT_, true, false>(p, ctas, stream) : launch_attn_kv8<D_, NT_, false, false>(p, ctas, stream))
  if (D == 128 && tile == 8) ER_KV8(128, 1);
  else if (D == 128) ER_KV8(128, 2);
  else if (tile == 8) ER_KV8(64, 1);
  else ER_KV8(64, 2);
#undef ER_KV8
  return static_cast<int>(e);
}

static AttnKv8Params attn_kv8_params(const Kv8AttentionArgs& a, int ld_q) {
  AttnKv8Params p = {};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.ld_q = ld_q;
  p.k_codes = static_cast<const int8_t*>(a.k_codes);
  p.v_codes = static_cast<const int8_t*>(a.v_codes);
  p.k_scales = a.k_scales;
  p.v_scales = a.v_scales;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.block_table = a.block_table;
  p.seq_lens = a.seq_lens;
  p.sinks = a.sinks;
  p.part_o = a.part_o;
  p.part_ml = a.part_ml;
  p.joins = static_cast<int4*>(a.joins);
  p.batch = a.batch;
  p.max_pages = a.max_pages;
  p.pitch = a.pitch;
  p.num_pages = a.num_pages;
  p.n_q = a.n_q;
  p.n_kv = a.n_kv;
  p.q_per_seq = a.q_per_seq;
  p.splits = a.splits;
  p.window = a.window;
  p.chunk = a.chunk;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = a.status;
  return p;
}

// splits 1 to 8: CTAs of a sequence and head. 0: even shares for `ctas` CTAs, with scratch for 2 * ctas tiles of 8 rows (16 where a head has more than 8).
extern "C" int eredu_attn_kv8_decode(const void* args, int bytes) {
  Kv8AttentionArgs a;
  if (!kv8_args(a, args, bytes)) return -2;
  AttnKv8Params p = attn_kv8_params(a, a.n_q * a.D);
  return attn_kv8(p, a.D, a.ctas, false, a.stream);
}

// The same from the projection's output, rows [q heads | k heads | v heads] x D of ld elements. The attention kernel rotates queries and writes the new
// rows itself where one tile holds all query rows of a head, so that one CTA has a page; else kv8_store goes in front and leaves the queries in
// q32 [batch * q_per_seq, n_q, D] (four sequences of 3000 tokens, five new ones, 32 heads over 4: 17 us; rotated in each of three tiles 20).
extern "C" int eredu_attn_kv8_step(const void* args, int bytes) {
  Kv8AttentionArgs a;
  if (!kv8_args(a, args, bytes)) return -2;
  if (a.batch <= 0) return 0;
  if (a.n_kv <= 0 || a.n_q <= 0 || a.n_q % a.n_kv != 0 || a.q_per_seq <= 0 || a.rot < 0 || a.rot > a.D || a.rot % 8 != 0) return -2;
  const bool own = a.q_per_seq * (a.n_q / a.n_kv) <= 16 && a.q_per_seq <= kKv8StepTokens;
  const __nv_bfloat16 *row = static_cast<const __nv_bfloat16*>(a.q), *k = row + a.n_q * a.D, *v = k + a.n_kv * a.D;
  AttnKv8Params p = attn_kv8_params(a, a.ld);
  if (!own) {
    if (a.q32 == nullptr) return -2;
    const int e = kv8_store(Kv8StoreArgs{a.q, k, v, a.q32, a.k_codes, a.v_codes, a.k_scales, a.v_scales, a.positions, a.slots, a.inv_freq, a.q_norm_w, a.k_norm_w, a.status,
                                         a.stream, a.batch * a.q_per_seq, a.ld, a.ld, a.ld, a.n_q, a.n_kv, a.D, a.rot, a.interleaved, a.num_pages, 1, a.attn_factor,
                                         a.norm_eps, a.norm_w_off});
    if (e != 0) return e;
    p.q32 = a.q32;
    p.ld_q = a.n_q * a.D;
    return attn_kv8(p, a.D, a.ctas, false, a.stream);
  }
  p.settled = !EREDU_PDL_EARLY && pdl_enabled() && a.settled != 0;
  p.st.k = k;
  p.st.v = v;
  p.st.ld_k = p.st.ld_v = a.ld;
  p.st.k_codes = static_cast<int8_t*>(a.k_codes);
  p.st.v_codes = static_cast<int8_t*>(a.v_codes);
  p.st.k_scales = a.k_scales;
  p.st.v_scales = a.v_scales;
  p.st.positions = a.positions;
  p.st.slots = a.slots;
  p.st.inv_freq = a.inv_freq;
  p.st.q_norm_w = a.q_norm_w;
  p.st.k_norm_w = a.k_norm_w;
  p.st.rot = a.rot;
  p.st.interleaved = a.interleaved;
  p.st.attn_factor = a.attn_factor;
  p.st.norm_eps = a.norm_eps;
  p.st.norm_w_off = a.norm_w_off;
  return attn_kv8(p, a.D, a.ctas, true, a.stream);
}
