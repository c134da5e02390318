// Keys and values into a cache in 4 bits (the format: kv4.cuh), and out of it again.
//
// Both move memory: a token and head has 4 head_dim bytes of bfloat16 keys and values on one side and 9/8 head_dim bytes of codes and words on
// the other. 8,192 tokens of 8 heads of 128 in bfloat16: in 10.3 us, out 10.0 us (38 MB each; 33 MB filled with zeros take 9.5 us, copied from
// L2 6.8 us). What is stored is bound by instructions: with 8 dimensions a thread, whose group's step, its reciprocal and the places of what is stored
// were worked out four times instead of twice, 14.8 us; with one float at a time instead of two 16.3 us.
#include "kv4.cuh"
#include "launchers.h"

namespace tie {

int* status_word();

constexpr int kKv4Blocks = 65535;        // of a head, before blockIdx.z counts on

struct Kv4Planes {
  uint32_t *k_codes, *v_codes;
  uint16_t *k_words, *v_words;
  int kv_heads, page_size, page_shift, head_dim;     // page_shift -1: no power of two
  unsigned int slots;       // pages * page_size
};

// Row of the planes (token slots of one head) of a slot; a plane has less than 2^31.
__device__ __forceinline__ int kv4_row(int slot, int head, const Kv4Planes& c) {
  const int page = c.page_shift >= 0 ? slot >> c.page_shift : slot / c.page_size;
  return (page * c.kv_heads + head - page) * c.page_size + slot;
}

// Where a thread of kv4_append works: 16 dimensions (half a group) of a token's key or value of one head. The lanes of a token and head, its key's first, lie side by
// side in a warp; blockIdx.x is the head, the block's tokens come in turn.
template <int NG> struct Kv4Lanes {
  static constexpr int PLANE = 4 * NG;                                 // lanes of a key, or of a value
  static constexpr int LANES = NG == 1 ? 8 : NG == 2 ? 16 : 32;        // (heads of three 64s leave eight idle)
  static constexpr int STEP = 256 / LANES;                             // tokens that a block has at a time
};

// Adding it rounds a float below 2^22 to a whole number, ties to even, and leaves that number in the low bits.
constexpr float kRoundMagic = 12582912.0f;      // 1.5 * 2^23
// rint(x / s) for |x / s| < 16, x / s as the correctly rounded quotient: Markstein's method (1990), which takes the correctly rounded reciprocal, a
// quotient by it, the remainder by one fma (exact) and a second fma that corrects the quotient. (Ties of bfloat16 numbers are common: a
// quotient that is only near would send most warps through a division.)
// The whole number comes plus `add` (which is whole, too).
__device__ __forceinline__ float kv4_quotient(float x, float s, float reciprocal, float add) {
  const float q = x * reciprocal;
  return __fadd_rn(__fadd_rn(fmaf(fmaf(-q, s, x), reciprocal, q), kRoundMagic), add - kRoundMagic);
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Eight values as codes. Four codes are the digits of one number, whose bits 2^23 shows; dimensions 0-3 and 4-7 side by side.
// rint(x / s) >= rint(lo / s) = -z, and rint(x / s) + z is above 15 only where both x / s and -lo / s are halves that round up, and then
// 16: `top` says so for the group.
__device__ __forceinline__ uint32_t kv4_codes(const float* x, float s, float reciprocal, float z, bool top) {
  if (!top) {
    const Pair s2 = pair(-s, -s), r2 = pair(reciprocal, reciprocal), magic = pair(kRoundMagic, kRoundMagic), back = pair(z - kRoundMagic, z - kRoundMagic);
    Pair four = pair(128.0f, 128.0f);       // 2^23 when four digits have come in
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      const Pair v2 = pair(x[e], x[4 + e]), q = mul_pair(v2, r2);
      four = fma_pair(four, pair(16.0f, 16.0f), add_pair(add_pair(fma_pair(fma_pair(q, s2, v2), r2, q), magic), back));
    }
    return __byte_perm(static_cast<uint32_t>(four), static_cast<uint32_t>(four >> 32), 0x5410);
  }
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) codes |= (__float_as_uint(fminf(kv4_quotient(x[e], s, reciprocal, z), 15.0f) + 8388608.0f) & 15u) << (4 * e);
  return codes;
}

// ROUNDS: tokens that a thread takes one after the other, and works out its place in a head for once.
template <typename T, int NG, int ROUNDS>
__global__ void __launch_bounds__(256) kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, long long k_stride, long long v_stride,
                                                         const int* __restrict__ slots, Kv4Planes c, int tokens, int vec, int* status) {
  pdl_sync();
  using L = Kv4Lanes<NG>;
  const int lane = threadIdx.x & (L::LANES - 1), head = blockIdx.x, is_v = lane >= L::PLANE, part = lane - (is_v ? L::PLANE : 0);
  const uint32_t mine = L::LANES == 32 ? 0xffffffffu : ((1u << (L::LANES & 31)) - 1u) << (threadIdx.x & (32 - L::LANES));
  const int dims = part < L::PLANE ? c.head_dim - part * 16 : 0;
  const long long stride = is_v ? v_stride : k_stride;
  const int first = (blockIdx.z * kKv4Blocks + blockIdx.y) * (ROUNDS * L::STEP) + threadIdx.x / L::LANES;
  const T* src = (is_v ? v : k) + static_cast<long long>(head) * c.head_dim + part * 16 + first * stride;
  uint32_t* const codes = is_v ? c.v_codes : c.k_codes;
  uint16_t* const words = is_v ? c.v_words : c.k_words;
#pragma unroll 1          // (2: 32,768 tokens 49 us instead of 43)
  for (int round = 0; round < ROUNDS; ++round) {
    const int token = first + round * L::STEP;
    const int slot = token < tokens ? slots[token] : -1;
    const bool writes = slot >= 0 && static_cast<unsigned int>(slot) < c.slots;
    if (slot >= 0 && !writes && lane == 0) *reinterpret_cast<volatile int*>(status) = kStatusBadSlot;
    float x[16];
    load8(src + round * L::STEP * stride, writes ? dims : 0, vec != 0, reinterpret_cast<float(&)[8]>(x[0]));
    load8(src + round * L::STEP * stride + 8, writes ? dims - 8 : 0, vec != 0, reinterpret_cast<float(&)[8]>(x[8]));
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; e += 2) lo = min_nan(lo, x[e], x[e + 1]), hi = max_nan(hi, x[e], x[e + 1]);
    const bool fine = (__ballot_sync(0xffffffffu, hi < kKv4Limit && lo > -kKv4Limit) & mine) == mine;      // (false for NaN)
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
    uint2 out = make_uint2(0u, 0u);
    uint32_t w = is_v ? 0u : kKv4NaN;
    if (fine) {
      const float s = kv4_step(lo, hi), reciprocal = __frcp_rn(s);
      const float z = kv4_quotient(-lo, s, reciprocal, 0.0f);
      const bool top = kv4_quotient(hi, s, reciprocal, z) > 15.0f;
      out = make_uint2(kv4_codes(x, s, reciprocal, z, top), kv4_codes(x + 8, s, reciprocal, z, top));
      w = (__float_as_uint(s) >> 16) | (__float_as_uint(z + 8388608.0f) & 15u);
    }
    if (writes && part < L::PLANE) {
      const long long at = static_cast<long long>(kv4_row(slot, head, c)) * L::PLANE + part;
      reinterpret_cast<uint2*>(codes)[at] = out;
      if ((part & 1) == 0) words[at >> 1] = static_cast<uint16_t>(w);
    }
  }
}

// Where a thread of kv4_read works: 8 dimensions, so that neighbours write 16 bytes side by side (with 16 dimensions 2,049 tokens of 5 heads of 96 in
// float 4.8 us instead of 3.5). A head's token: up to two 64s its key and value are the lanes of a warp (one 64: of half a warp), else every lane has
// a word of both. blockIdx.x is the head, the block's warps (halves) take tokens in turn.
template <int NG> struct Kv4ReadLanes {
  static constexpr int W = 8 * NG;                        // words of codes of a head
  static constexpr int ITEMS = NG <= 2 ? 1 : 2;           // words of a lane
  static constexpr int LANES = NG == 1 ? 16 : 32;
  static constexpr int STEP = 256 / LANES;                // tokens that a block has at a time
  static __device__ __forceinline__ bool is_value(int lane, int item) { return ITEMS == 2 ? item == 1 : lane >= W; }
  static __device__ __forceinline__ int word(int lane) { return ITEMS == 2 ? lane : lane % W; }
};

template <typename T, int NG, int ROUNDS>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4Planes c, const int* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, long long k_stride,
                                                       long long v_stride, int tokens, int vec, int* status) {
  pdl_sync();
  using L = Kv4ReadLanes<NG>;
  const int lane = threadIdx.x & (L::LANES - 1), head = blockIdx.x, word = L::word(lane), left = c.head_dim - word * 8;
  if (word >= L::W || left <= 0) return;
#pragma unroll 4
  for (int round = 0; round < ROUNDS; ++round) {
    const int token = (blockIdx.z * kKv4Blocks + blockIdx.y) * (ROUNDS * L::STEP) + round * L::STEP + threadIdx.x / L::LANES;
    const int slot = token < tokens ? slots[token] : -1;
    if (slot < 0) continue;
    if (static_cast<unsigned int>(slot) >= c.slots) {
      if (lane == 0) *reinterpret_cast<volatile int*>(status) = kStatusBadSlot;
      continue;
    }
    const int at = kv4_row(slot, head, c);
#pragma unroll
    for (int i = 0; i < L::ITEMS; ++i) {
      const bool is_v = L::is_value(lane, i);
      const uint32_t codes = (is_v ? c.v_codes : c.k_codes)[static_cast<long long>(at) * L::W + word];
      const uint32_t w = (is_v ? c.v_words : c.k_words)[static_cast<long long>(at) * (L::W / 4) + word / 4];
      const float s = __uint_as_float((w & 0xffe0u) << 16);
      const float z = __uint_as_float((w & 15u) | 0x4b000000u);          // 2^23 + z, and 2^23 + code: their difference is exact
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s * (__uint_as_float(((codes >> (4 * e)) & 15u) | 0x4b000000u) - z);
      T* dst = (is_v ? v + token * v_stride : k + token * k_stride) + static_cast<long long>(head) * c.head_dim + word * 8;
      if (vec && left >= 8) {
        constexpr int N = Vec16<T>::N;
#pragma unroll
        for (int j = 0; j < 8; j += N) {
          Vec16<T> t;
#pragma unroll
          for (int e = 0; e < N; ++e) t.v[e] = x[j + e];
          t.store(dst + j);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) st(dst + e, x[e]);
      }
    }
  }
}

static bool kv4_rows_aligned(const void* k, const void* v, long long k_stride, long long v_stride, int head_dim, int size) {
  return reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 && k_stride * size % 16 == 0 && v_stride * size % 16 == 0 &&
         head_dim * size % 16 == 0;
}

template <typename T, int NG, int ROUNDS>
static void launch_kv4(bool append, T* k, T* v, long long k_stride, long long v_stride, const int* slots, const Kv4Planes& c, int tokens, cudaStream_t s) {
  const int vec = kv4_rows_aligned(k, v, k_stride, v_stride, c.head_dim, sizeof(T)) ? 1 : 0;
  const int blocks = ceil_div(tokens, ROUNDS * (append ? Kv4Lanes<NG>::STEP : Kv4ReadLanes<NG>::STEP));
  const dim3 grid(c.kv_heads, min(blocks, kKv4Blocks), ceil_div(blocks, kKv4Blocks));
  if (append) TIE_LAUNCH((kv4_append_kernel<T, NG, ROUNDS>), grid, 256, 0, s, k, v, k_stride, v_stride, slots, c, tokens, vec, status_word());
  else TIE_LAUNCH((kv4_read_kernel<T, NG, ROUNDS>), grid, 256, 0, s, c, slots, k, v, k_stride, v_stride, tokens, vec, status_word());
}

// Four tokens a thread where that still leaves every SM eight blocks. (One token: 8,192 of 8 heads of 128 in and out 2 us more; four everywhere: 2,049
// of 5 heads of 96 11.1 us instead of 8.8, eight tokens 4.8 instead of 3.3.)
template <typename T, int NG>
static void launch_kv4(bool append, T* k, T* v, long long k_stride, long long v_stride, const int* slots, const Kv4Planes& c, int tokens, cudaStream_t s) {
  const int blocks = tokens / (4 * (append ? Kv4Lanes<NG>::STEP : Kv4ReadLanes<NG>::STEP));
  if (static_cast<long long>(blocks) * c.kv_heads >= 148 * 8) launch_kv4<T, NG, 4>(append, k, v, k_stride, v_stride, slots, c, tokens, s);
  else launch_kv4<T, NG, 1>(append, k, v, k_stride, v_stride, slots, c, tokens, s);
}

template <typename T>
static void launch_kv4(bool append, void* k, void* v, long long k_stride, long long v_stride, const int* slots, const Kv4Planes& c, int tokens, cudaStream_t s) {
  T *kt = static_cast<T*>(k), *vt = static_cast<T*>(v);
  switch ((c.head_dim + 63) / 64) {
    case 1: launch_kv4<T, 1>(append, kt, vt, k_stride, v_stride, slots, c, tokens, s); break;
    case 2: launch_kv4<T, 2>(append, kt, vt, k_stride, v_stride, slots, c, tokens, s); break;
    case 3: launch_kv4<T, 3>(append, kt, vt, k_stride, v_stride, slots, c, tokens, s); break;
    default: launch_kv4<T, 4>(append, kt, vt, k_stride, v_stride, slots, c, tokens, s); break;
  }
}

static Kv4Planes kv4_planes(const void* k_codes, const void* k_words, const void* v_codes, const void* v_words, int kv_heads, int head_dim, int page_size, long long pages) {
  int shift = 0;
  while (shift < 30 && (1 << shift) < page_size) ++shift;
  return {static_cast<uint32_t*>(const_cast<void*>(k_codes)), static_cast<uint32_t*>(const_cast<void*>(v_codes)), static_cast<uint16_t*>(const_cast<void*>(k_words)),
          static_cast<uint16_t*>(const_cast<void*>(v_words)), kv_heads, page_size, (1 << shift) == page_size ? shift : -1, head_dim,
          static_cast<unsigned int>(pages * page_size)};
}

static int launch_kv4(const char* name, bool append, int dtype, const Kv4Planes& c, void* k, void* v, long long k_stride, long long v_stride, const int* slots, int tokens,
                      long long pages, cudaStream_t s) {
  TIE_REQUIRE(tokens >= 0 && tokens <= (1 << 30) && c.kv_heads > 0 && c.kv_heads <= 65535 && c.page_size > 0 && c.head_dim > 0 && c.head_dim <= 256,
              "%s: bad sizes (tokens %d, kv heads %d, page size %d, head size %d)", name, tokens, c.kv_heads, c.page_size, c.head_dim);
  TIE_REQUIRE(pages > 0 && pages * c.page_size < (1LL << 31), "%s: %lld pages of %d tokens: slots are 32-bit numbers", name, pages, c.page_size);
  TIE_REQUIRE(pages * c.page_size * c.kv_heads < (1LL << 31), "%s: planes of %lld x %d x %d rows: rows are 32-bit numbers", name, pages, c.kv_heads, c.page_size);
  TIE_REQUIRE(status_word() != nullptr, "%s: cannot allocate the status word", name);
  if (tokens == 0) return kOk;
  if (dtype == TIE_F32) launch_kv4<float>(append, k, v, k_stride, v_stride, slots, c, tokens, s);
  else launch_kv4<__nv_bfloat16>(append, k, v, k_stride, v_stride, slots, c, tokens, s);
  TIE_RETURN_LAUNCH(name);
}

}  // namespace tie

using namespace tie;

// k, v [tokens, kv_heads * head_dim] (rows strides apart) into the planes at slots[t]; a slot below zero writes nothing.
TIE_API int tie_kv4_append(int dtype, const void* k, const void* v, long long k_stride, long long v_stride, const int* slots, void* k_codes, void* k_words,
                           void* v_codes, void* v_words, int tokens, int kv_heads, int head_dim, int page_size, long long pages, cudaStream_t s) {
  return launch_kv4("kv4_append", true, dtype, kv4_planes(k_codes, k_words, v_codes, v_words, kv_heads, head_dim, page_size, pages), const_cast<void*>(k),
                    const_cast<void*>(v), k_stride, v_stride, slots, tokens, pages, s);
}

// The values at slots[t] into k, v [tokens, kv_heads * head_dim]; rows whose slot is below zero are left as they are.
TIE_API int tie_kv4_read(int dtype, const void* k_codes, const void* k_words, const void* v_codes, const void* v_words, const int* slots, void* k, void* v,
                         long long k_stride, long long v_stride, int tokens, int kv_heads, int head_dim, int page_size, long long pages, cudaStream_t s) {
  return launch_kv4("kv4_read", false, dtype, kv4_planes(k_codes, k_words, v_codes, v_words, kv_heads, head_dim, page_size, pages), k, v, k_stride, v_stride, slots,
                    tokens, pages, s);
}
