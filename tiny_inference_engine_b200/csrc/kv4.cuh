// The format of a key/value cache in 4 bits, and how its kernels take it apart.
//
// A token's key (value) of one kv head: `padded` = head_dim rounded up to whole 64s numbers (zeros behind head_dim) in groups of 32. Of a
// group with lo = min(0, least) and hi = max(0, largest):
//     s = (hi - lo) / 15 in float, at least 2^-100, rounded up to three significant bits
//     z = rint(-lo / s),  code = clamp(rint(x / s) + z, 0, 15),  value = s (code - z)
// |code - z| <= 15 has four bits and s three, so every value is a bfloat16 number (seven bits), and so is s z: the products run on the tensor
// cores without another rounding. The quotients by s are correctly rounded floats; for a
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
// Taking codes apart without shifts. A bfloat16 pattern whose exponent field is 0 or 1 is its lower eight bits as a whole number times 2^-133:
// subnormal numbers and the first normal ones lie on one line. So a code in bits 0..3 or 4..7 of a half word is a number as it stands, once
// the other bits are masked away, code 2^-133 or code 2^-129, and one fma with s 2^102 or s 2^98 and -z s 2^-31 makes the value times 2^-31
// of it, exactly (the products take 2^31 back in float): the least step, 2^-100, leaves whole multiples of 2^-133. Against the code put into the
// mantissa of 16, which takes a shift and two constants: eight contexts of 32,768 keys 81 us against 94 (then); logical operations and shifts
// share the pipe that bounds these kernels.
// s 2^102 is finite for steps below 2^26. Where there are larger ones (BIG), one product more brings the codes to code 2^-6, and s 2^-25 takes them
// to the same numbers. Whoever takes words apart looks for them first (kv4_big): no model's keys come near, so that costs a few instructions
// a tile, and attention sees every step of the format.
constexpr float kKv4Unscale = 2147483648.0f;               // 2^31
// Weights are 2^8 times what they are (their sums too, so quotients stay): products with the smallest values of the format, 2^-131, then are
// no subnormal floats, and sums of 2^20 of the largest, 2^120 with weights of up to 2^8, stay below 2^128.
constexpr float kKv4WeightShift = 8.0f;
// Two words side by side: whether either's step is 2^26 or above, or NaN: 0x4c80 in bfloat16. (Bits 15 and 31 of the sum, no carry.)
__device__ __forceinline__ uint32_t kv4_big(uint32_t words) { return words + 0x33803380u; }
constexpr uint32_t kKv4BigBits = 0x80008000u;
// `words`: two groups' words, one in each half (the same one twice where both numbers of a pair belong to one group).
struct Kv4Scale {
  uint32_t low, high, off;      // for codes in bits 0..3 and 4..7; -z s 2^-31
};
// (signs: two sign bits, in a register: with a constant the compiler makes two operations of the and-or)
__device__ __forceinline__ uint32_t kv4_signs() {
  uint32_t signs;
  asm volatile("mov.b32 %0, 0x80008000;" : "=r"(signs));
  return signs;
}
template <bool BIG> __device__ __forceinline__ Kv4Scale kv4_scale(uint32_t words, uint32_t signs) {
  Kv4Scale k;
  uint32_t z;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(z) : "r"(words), "r"(signs));                  // -z 2^-133
  k.low = bf16x2_mul(words & 0xffe0ffe0u, BIG ? 0x33003300u : 0x72807280u);                         // 2^-25, 2^102
  k.high = BIG ? k.low : bf16x2_mul(k.low, 0x3d803d80u);                                            // 2^-4
  k.off = bf16x2_mul(BIG ? bf16x2_mul(z, 0x7f007f00u) : z, k.low);                                  // 2^127
  return k;
}
// The values 2^-31 of the codes in bits 0..3 (4..7) of both halves of w.
template <bool BIG> __device__ __forceinline__ uint32_t kv4_low(uint32_t w, const Kv4Scale& k) {
  const uint32_t codes = w & 0x000f000fu;
  return bf16x2_fma(BIG ? bf16x2_mul(codes, 0x7f007f00u) : codes, k.low, k.off);                    // 2^127
}
template <bool BIG> __device__ __forceinline__ uint32_t kv4_high(uint32_t w, const Kv4Scale& k) {
  const uint32_t codes = w & 0x00f000f0u;
  return bf16x2_fma(BIG ? bf16x2_mul(codes, 0x7d007d00u) : codes, k.high, k.off);                   // 2^123
}

// Eight dimensions of a row, `dims` of them there (the others are zero); vec: rows are 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int dims, bool vec, float (&x)[8]) {
  if (vec && dims >= 8) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      Vec16<T> t;
      t.load(p + i);
#pragma unroll
      for (int e = 0; e < N; ++e) x[i + e] = t.v[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < dims ? ld(p + i) : 0.0f;
  }
}

// Two floats that sm_100a works on as one.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float low_of(Pair p) { return __uint_as_float(static_cast<uint32_t>(p)); }
__device__ __forceinline__ float high_of(Pair p) { return __uint_as_float(static_cast<uint32_t>(p >> 32)); }
__device__ __forceinline__ Pair fma_pair(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Pair mul_pair(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair add_pair(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The smallest number of three significant bits that is not below (hi - lo) / 15; the float division rounds first.
__device__ __forceinline__ float kv4_step(float lo, float hi) {
  const float least = fmaxf(__fdiv_rn(hi - lo, 15.0f), kKv4LeastScale);
  return __uint_as_float((__float_as_uint(least) + 0x1fffffu) & ~0x1fffffu);
}

}  // namespace tie
