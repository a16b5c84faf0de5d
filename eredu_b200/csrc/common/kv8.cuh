// Blocks of a cache held in 8 bits: the 16 rows of one key / value head in a page, int8 codes [16, D] and one scale, a power of two.
// value = code * scale; code = round(x / scale), ties to even; the scale is the smallest that keeps |code| <= 127, at least 2^-100.
// A power of two: products and quotients by it are exact, and a block whose scale was raised several times (each time at least twofold) is off
// by less than one step of the last scale in all, where scales of any value would add up half a step for every time.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace eredu {

constexpr int kKv8Page = 16;
constexpr float kKv8Floor = 7.888609052210118e-31f;   // 2^-100

// Scale that the largest magnitude `amax` needs; not a number where amax is none (or infinite).
__device__ __forceinline__ float kv8_needed(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  // amax = f 2^e, 1 <= f < 2, and 127 = 1.984375 * 2^6
  const int e = static_cast<int>(u >> 23) - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return e < 27 ? kKv8Floor : __uint_as_float(static_cast<uint32_t>(e) << 23);
}
// 1 / scale of a power of two (not a number stays none).
__device__ __forceinline__ float kv8_inverse(float scale) {
  const uint32_t u = __float_as_uint(scale);
  return u >= 0x7f800000u ? scale : __uint_as_float(0x7f000000u - u);
}
// Codes of four values times `inv`, a power of two: the sum with 1.5 * 2^23 rounds to a whole number, ties to even, and ends in its byte.
__device__ __forceinline__ uint32_t kv8_pack(float a, float b, float c, float d, float inv) {
  constexpr float kWhole = 12582912.f;
  const uint32_t i = __float_as_uint(fmaf(a, inv, kWhole)), j = __float_as_uint(fmaf(b, inv, kWhole)), k = __float_as_uint(fmaf(c, inv, kWhole)),
                 l = __float_as_uint(fmaf(d, inv, kWhole));
  return __byte_perm(__byte_perm(i, j, 0x0040), __byte_perm(k, l, 0x0040), 0x5410);
}
__device__ __forceinline__ float kv8_code(uint32_t word, int i) { return static_cast<float>(static_cast<int8_t>(word >> (8 * i))); }

// The lower (UPPER: the upper) bytes of both halves of a word as exact f16: 0x6400 | c + 128 is 1152 + c.
template <bool UPPER>
__device__ __forceinline__ uint32_t kv8_parted(uint32_t word) {
  uint32_t h = ((UPPER ? word >> 8 : word) & 0x00ff00ffu) ^ 0x64806480u;
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(h) : "r"(0x64806480u));
  return h;
}


// Where 16-byte piece c of token row r lies in a page's half of a ring slot: pieces change places within 128 bytes, so that the eight rows of an 8 x 8 matrix
// that ldmatrix reads meet all banks.
template <int D>
__device__ __forceinline__ int kv8_piece(int r, int c) {
  return D == 128 ? r * 128 + (c ^ (r & 7)) * 16 : (r >> 1) * 128 + (((r & 1) << 2 | c) ^ (r >> 1 & 3)) * 16;
}

}  // namespace eredu
