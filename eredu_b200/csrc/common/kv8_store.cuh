// Rows of keys and values into blocks of 8 bits (kv8.cuh), rotated and normalised on the way.
#pragma once
#include "kv8.cuh"
#include "ptx.cuh"

namespace eredu {

struct Kv8StoreParams {
  const __nv_bfloat16 *q, *k, *v;   // [M, heads, D], rows of ld_q, ld_k, ld_v elements
  void* q_out;                      // [M, n_q, D] bf16, or fp32
  int q_out_fp32;
  int8_t *k_codes, *v_codes;        // [pages, n_kv, 16, D]
  float *k_scales, *v_scales;       // [pages, n_kv]
  const int* positions;             // [M]
  const long long* slots;           // [M] page * 16 + offset, < 0: not stored
  const float* inv_freq;            // [rot / 2]
  const float *q_norm_w, *k_norm_w; // optional [D]
  int M, ld_q, ld_k, ld_v, n_q, n_kv, rot, interleaved, tile, num_pages;
  float attn_factor, norm_eps, norm_w_off;
  int* status;
};

// Cosine and sine of pos * freq, times `factor`, off by 2^-23 or so. The product in two parts, so that far positions keep their digits; quarter turns are taken
// off with pi / 2 in two parts (the reduction of Cody and Waite; fma makes the first difference exact), and what is left, pi / 4 at most, goes into the Taylor
// series up to x^9 and x^10 (the next terms are below 2^-28). For angles below 2^22; sincosf costs more than twice as much, and its fast forms are off by 2^-21.
__device__ __forceinline__ void turn_of(int pos, float freq, float factor, float& c, float& s) {
  constexpr float kWhole = 12582912.f;                       // 1.5 * 2^23
  const float p = static_cast<float>(pos);
  const float a = p * freq, rest = fmaf(p, freq, -a);
  const float t = fmaf(a, 0.636619772f, kWhole), k = t - kWhole;
  const float r = fmaf(-k, -4.37113883e-8f, fmaf(-k, 1.57079637f, a)) + rest, z = r * r;
  const float sine = fmaf(r * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), r);
  const float cosine = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const int quarter = __float_as_int(t);
  s = ((quarter & 1) ? cosine : sine) * ((quarter & 2) ? -factor : factor);
  c = ((quarter & 1) ? sine : cosine) * (((quarter + 1) & 2) ? -factor : factor);
}

template <int D>
__device__ __forceinline__ float4 load_row4(const __nv_bfloat16* row, int lane) {
  const uint2 u = *reinterpret_cast<const uint2*>(row + 4 * (lane & (D / 4 - 1)));
  return make_float4(bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y));
}
// The D / 4 lanes of a row together: norm, then rotation. `turns`: rot / 2 cosines of the row's angles, then as many sines.
template <int D>
__device__ __forceinline__ float4 prepared(const Kv8StoreParams& p, float4 x, const float* w, const float* turns, int lane) {
  const int d = 4 * (lane & (D / 4 - 1));
  if (w != nullptr) {
    float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
#pragma unroll
    for (int o = D / 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss / static_cast<float>(D) + p.norm_eps);
    x.x *= inv * (w[d] + p.norm_w_off);
    x.y *= inv * (w[d + 1] + p.norm_w_off);
    x.z *= inv * (w[d + 2] + p.norm_w_off);
    x.w *= inv * (w[d + 3] + p.norm_w_off);
  }
  if (p.rot == 0) return x;
  const int half = p.rot / 2;
  if (p.interleaved) {
    if (d < p.rot) {
      const float2 c = *reinterpret_cast<const float2*>(turns + d / 2), n = *reinterpret_cast<const float2*>(turns + half + d / 2);
      x = make_float4(x.x * c.x - x.y * n.x, x.y * c.x + x.x * n.x, x.z * c.y - x.w * n.y, x.w * c.y + x.z * n.y);
    }
    return x;
  }
  const int from = d < half ? lane + half / 4 : d < p.rot ? lane - half / 4 : lane;
  const float4 o = make_float4(__shfl_sync(0xffffffffu, x.x, from), __shfl_sync(0xffffffffu, x.y, from), __shfl_sync(0xffffffffu, x.z, from),
                               __shfl_sync(0xffffffffu, x.w, from));
  if (d < p.rot) {
    const float sign = d < half ? -1.f : 1.f;
    const int i = d < half ? d : d - half;
    const float4 c = *reinterpret_cast<const float4*>(turns + i), n = *reinterpret_cast<const float4*>(turns + half + i);
    x = make_float4(x.x * c.x + sign * o.x * n.x, x.y * c.y + sign * o.y * n.y, x.z * c.z + sign * o.z * n.z, x.w * c.w + sign * o.w * n.w);
  }
  return x;
}
// How a warp holds rows. WHOLE, all of a row is rotated, in halves: a lane has four channels of the lower half and their partners of the upper, so that a rotation
// stays in the lane and a warp holds two rows of 128 (or four of 64). Else a lane has four neighbouring channels, and `prepared` above finds the partners.
template <int D, bool WHOLE>
struct Kv8Rows {
  static constexpr int PER = WHOLE ? 2 : 1, LANES = D / (4 * PER), ROWS = 32 / LANES;
  float4 x[PER];
  static __device__ __forceinline__ int row(int lane) { return LANES == 32 ? 0 : lane / LANES; }
  static __device__ __forceinline__ int channel(int lane, int j) { return 4 * (lane & (LANES - 1)) + j * (D / 2); }
  __device__ __forceinline__ void take(const uint2 (&u)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = make_float4(bf16_lo(u[j].x), bf16_hi(u[j].x), bf16_lo(u[j].y), bf16_hi(u[j].y));
  }
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int lane) {
    uint2 u[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) u[j] = *reinterpret_cast<const uint2*>(row + channel(lane, j));
    take(u);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // Norm, then rotation, by the LANES lanes of a row together.
  __device__ __forceinline__ void prepare(const Kv8StoreParams& p, const float* w, const float* turns, int lane) {
    if constexpr (!WHOLE) {
      x[0] = prepared<D>(p, x[0], w, turns, lane);
    } else {
      float4 &a = x[0], &b = x[1];
      const int d = channel(lane, 0);
      if (w != nullptr) {
        float ss = a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w + b.x * b.x + b.y * b.y + b.z * b.z + b.w * b.w;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(ss / static_cast<float>(D) + p.norm_eps);
        const float* u = w + D / 2;
        a = make_float4(a.x * (inv * (w[d] + p.norm_w_off)), a.y * (inv * (w[d + 1] + p.norm_w_off)), a.z * (inv * (w[d + 2] + p.norm_w_off)),
                        a.w * (inv * (w[d + 3] + p.norm_w_off)));
        b = make_float4(b.x * (inv * (u[d] + p.norm_w_off)), b.y * (inv * (u[d + 1] + p.norm_w_off)), b.z * (inv * (u[d + 2] + p.norm_w_off)),
                        b.w * (inv * (u[d + 3] + p.norm_w_off)));
      }
      const float4 c = *reinterpret_cast<const float4*>(turns + d), n = *reinterpret_cast<const float4*>(turns + D / 2 + d);
      const float4 lo = make_float4(a.x * c.x - b.x * n.x, a.y * c.y - b.y * n.y, a.z * c.z - b.z * n.z, a.w * c.w - b.w * n.w);
      b = make_float4(b.x * c.x + a.x * n.x, b.y * c.y + a.y * n.y, b.z * c.z + a.z * n.z, b.w * c.w + a.w * n.w);
      a = lo;
    }
  }
};

// The scale of a block whose new rows have the largest magnitude `top` (as bits); `before`: that of the rows in front, if any. The larger of the two, and what is
// no number stays none.
__device__ __forceinline__ float kv8_raised(uint32_t top, int first, float before) {
  const float scale = kv8_needed(__uint_as_float(top));
  return first > 0 && !(before <= scale) ? (scale != scale ? scale : before) : scale;
}
__device__ __forceinline__ uint32_t kv8_top(uint32_t top, float4 x) {
  top = max(max(top, __float_as_uint(fabsf(x.x))), __float_as_uint(fabsf(x.y)));
  return max(max(top, __float_as_uint(fabsf(x.z))), __float_as_uint(fabsf(x.w)));
}

constexpr int kKv8StepTokens = 8;   // new tokens of a sequence in a step that writes its own rows
// The keys or values of a step's new rows, as they are, on their way to one warp: two registers for every 128 values.
template <int D>
struct Kv8Few {
  static constexpr int RPI = 128 / D, N = kKv8StepTokens / RPI;
  uint2 raw[N];
  // rows [0, n) of head h from `from` on
  __device__ __forceinline__ void load(const __nv_bfloat16* from, int ld, int n, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * RPI < n) raw[i] = *reinterpret_cast<const uint2*>(from + static_cast<size_t>(min(i * RPI + lane / (D / 4), n - 1)) * ld + 4 * (lane & (D / 4 - 1)));
  }
  // row `at`, one of this lane's
  __device__ __forceinline__ float4 row(int at) const {
    uint2 u = raw[0];
#pragma unroll
    for (int i = 1; i < N; ++i)
      if (at / RPI == i) u = raw[i];
    return make_float4(bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y));
  }
};

// Rows [row, row + n) of a step, of `few`, into the block at `cell` = (page, head), from offset `first` on, by one warp that has other things in its registers: they are
// looked at twice, one after the other. A lane has rows lane / (D / 4) + RPI i of them (those in front of `row`, and behind, do not count). `before`: the block's
// scale. `held`: where the page's codes of the head lie in shared memory as well, if they do (kv8_piece). Gives the scale.
template <int D, bool KEYS>
__device__ __forceinline__ float store_few(const Kv8StoreParams& p, const Kv8Few<D>& few, int row, int n, int first, long long cell, const float* turns, int lane, float before,
                                           uint8_t* held) {
  constexpr int RPI = 128 / D;
  int8_t* codes = (KEYS ? p.k_codes : p.v_codes) + cell * (kKv8Page * D);
  const int sub = RPI == 1 ? 0 : lane >> 4, c = 4 * (lane & (D / 4 - 1)), row0 = row / RPI * RPI;
  auto row_of = [&](int r) {      // (all lanes of the warp)
    const float4 y = few.row(r);
    return KEYS ? prepared<D>(p, y, p.k_norm_w, turns + min(r, row + n - 1) * p.rot, lane) : y;
  };
  auto beside = [&](int r) { return reinterpret_cast<uint32_t*>(held + kv8_piece<D>(r, c >> 4) + (c & 15)); };
  uint32_t top = 0;
  float4 x;
#pragma unroll 1
  for (int r = row0 + sub; r - sub < row + n; r += RPI) {
    x = row_of(r);
    if (r >= row && r < row + n) top = kv8_top(top, x);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  const float scale = kv8_raised(top, first, before), inv = kv8_inverse(scale);
  if (first > 0 && scale != before) {
#pragma unroll 1
    for (int r = sub; r < first; r += RPI) {
      uint32_t* w = reinterpret_cast<uint32_t*>(codes + r * D + c);
      const uint32_t u = held != nullptr ? *beside(r) : *w;
      const uint32_t now = kv8_pack(kv8_code(u, 0), kv8_code(u, 1), kv8_code(u, 2), kv8_code(u, 3), before * inv);
      *w = now;
      if (held != nullptr) *beside(r) = now;
    }
  }
#pragma unroll 1
  for (int r = row0 + sub; r - sub < row + n; r += RPI) {
    if (row + n - row0 > RPI) x = row_of(r);
    const uint32_t now = kv8_pack(x.x, x.y, x.z, x.w, inv);
    if (r >= row && r < row + n) {
      *reinterpret_cast<uint32_t*>(codes + (first + r - row) * D + c) = now;
      if (held != nullptr) *beside(first + r - row) = now;
    }
  }
  if (lane == 0) (KEYS ? p.k_scales : p.v_scales)[cell] = scale;
  return scale;
}

}  // namespace eredu
