// The format of a key/value cache in 4 bits, and how its kernels take it apart.
//
// A token's key (value) of one kv head: `padded` = head_dim rounded up to whole 64s numbers (zeros behind head_dim) in groups of 32. Of a
// group with lo = min(0, least) and hi = max(0, largest):
//     s = (hi - lo) / 15 in float, at least 2^-100, rounded up to three significant bits
//     z = rint(-lo / s),  code = clamp(rint(x / s) + z, 0, 15),  value = s (code - z)
// |code - z| <= 15 has four bits and s three, so every value is a bfloat16 number (seven bits), and so are s (16 + z) (eight) and every
// step on the way: the products run on the tensor cores without another rounding. The quotients by s are correctly rounded floats; for a
// divisor of three bits no quotient rounds to a tie that it is not (a quotient's distance from k + 1/2, if any, is more than half its ulp), so
// rint() gives what exact arithmetic gives.
// Codes: padded / 2 bytes, dimension d in byte d / 2, the even one in the low bits; eight dimensions are one 32-bit word. A group's 16-bit
// word: s as bfloat16 (its low five bits are zero) with z in the low four bits.
// A token and head with a number that is not finite, or from 2^120 up, in its key or value has the key words 0x7fc0 (s is NaN) and zero
// value words and codes: who sees the key gets NaN, and nothing else does, since the values stay finite where weights are zero.
// Planes: codes [pages, kv_heads, page_size, padded / 2] bytes, words [pages, kv_heads, page_size, padded / 32] of 16 bits.
#pragma once

#include "common.cuh"

namespace tie {

constexpr uint32_t kKv4NaN = 0x7fc0;
constexpr float kKv4Limit = 1.329227995784916e36f;        // 2^120
constexpr float kKv4LeastScale = 7.888609052210118e-31f;  // 2^-100
constexpr int kStatusBadPage = 15;                        // a block table that names a page outside the cache, or is too short for its context
constexpr int kStatusBadSlot = 16;                        // a slot outside the cache

// Bits 4 i .. 4 i + 3 of both halves of w as two bfloat16 numbers 16 + code: the code becomes the upper four bits of the mantissa of 16.
template <int i> __device__ __forceinline__ uint32_t kv4_pair(uint32_t w) {
  return ((i == 0 ? w << 3 : w >> (i == 0 ? 0 : 4 * i - 3)) & 0x00780078u) | 0x41804180u;
}
__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t bf16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Of two groups' words (one in each half; the same one twice where both numbers of a pair belong to one group): their s, and -(16 + z) s,
// so that a pair's values are fma(16 + code, s, -(16 + z) s).
struct Kv4Scale {
  uint32_t s, off;
};
__device__ __forceinline__ Kv4Scale kv4_scale(uint32_t words) {
  Kv4Scale k;
  k.s = words & 0xffe0ffe0u;
  k.off = bf16x2_mul(((words & 0x000f000fu) << 3) | 0xc180c180u, k.s);
  return k;
}

// The smallest number of three significant bits that is not below (hi - lo) / 15; the float division rounds first.
__device__ __forceinline__ float kv4_step(float lo, float hi) {
  const float least = fmaxf(__fdiv_rn(hi - lo, 15.0f), kKv4LeastScale);
  return __uint_as_float((__float_as_uint(least) + 0x1fffffu) & ~0x1fffffu);
}

}  // namespace tie
