// Keys and values into a cache in 4 bits (the format: kv4.cuh), and out of it again.
//
// Both move memory: a token and head has 4 head_dim bytes of bfloat16 keys and values on one side and 9/8 head_dim bytes of codes and words on
// the other. Eight dimensions (one 32-bit word of codes, 16 bytes of bfloat16) are one thread's; four threads share a group and meet in two
// shuffles; a token and head is one warp (half of one up to 64 dimensions), which also settles by one vote whether all its numbers are finite.
#include "kv4.cuh"

namespace tie {

int* status_word();

struct Kv4Planes {
  uint32_t *k_codes, *v_codes;
  uint16_t *k_words, *v_words;
  int kv_heads, page_size, head_dim;
  unsigned int slots;       // pages * page_size
};

// Row of the planes (token slots of one head) of a slot.
__device__ __forceinline__ long long kv4_row(int slot, int head, int kv_heads, int page_size) {
  return (static_cast<long long>(slot / page_size) * kv_heads + head) * page_size + slot % page_size;
}

// NG: head_dim in 64s. Up to two a key and value fit a warp's lanes side by side (one: half a warp), else the lanes hold a word of both.
template <typename T, int NG>
__global__ void __launch_bounds__(256) kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, long long k_stride, long long v_stride,
                                                         const int* __restrict__ slots, Kv4Planes c, long long units, int vec, int* status) {
  pdl_sync();
  constexpr int W = 8 * NG;                        // words of codes of a head
  constexpr int ITEMS = NG <= 2 ? 1 : 2;           // of a lane
  constexpr int LANES = NG == 1 ? 16 : 32;
  const int lane = threadIdx.x & (LANES - 1);
  const long long unit = static_cast<long long>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  const bool there = unit < units;
  const long long token = there ? unit / c.kv_heads : 0;
  const int head = there ? static_cast<int>(unit % c.kv_heads) : 0;
  const int slot = there ? slots[token] : -1;
  const bool writes = slot >= 0 && static_cast<unsigned int>(slot) < c.slots;
  if (slot >= 0 && !writes && lane == 0) *reinterpret_cast<volatile int*>(status) = kStatusBadSlot;
  float x[ITEMS][8];
  bool fine = true;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const bool is_v = ITEMS == 2 ? i == 1 : lane >= W;
    const int word = ITEMS == 2 ? lane : lane % W;
    const T* row = is_v ? v + token * v_stride : k + token * k_stride;
    const int dims = writes && word < W ? c.head_dim - word * 8 : 0;
    load8(row + static_cast<long long>(head) * c.head_dim + word * 8, dims, vec != 0, x[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) fine = fine && fabsf(x[i][e]) < kKv4Limit;
  }
  const uint32_t all = __ballot_sync(0xffffffffu, fine);
  const uint32_t mine = NG == 1 ? 0xffffu << (threadIdx.x & 16) : 0xffffffffu;
  fine = (all & mine) == mine;
  const long long at = kv4_row(writes ? slot : 0, head, c.kv_heads, c.page_size);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const bool is_v = ITEMS == 2 ? i == 1 : lane >= W;
    const int word = ITEMS == 2 ? lane : lane % W;
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) lo = fminf(lo, x[i][e]), hi = fmaxf(hi, x[i][e]);
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    uint32_t codes = 0, w = is_v ? 0u : kKv4NaN;
    if (fine) {
      const float s = kv4_step(lo, hi);
      const float z = rintf(__fdiv_rn(-lo, s));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q = fminf(fmaxf(rintf(__fdiv_rn(x[i][e], s)) + z, 0.0f), 15.0f);
        codes |= static_cast<uint32_t>(q) << (4 * e);
      }
      w = (__float_as_uint(s) >> 16) | static_cast<uint32_t>(z);
    }
    if (writes && word < W) {
      (is_v ? c.v_codes : c.k_codes)[at * W + word] = codes;
      if ((word & 3) == 0) (is_v ? c.v_words : c.k_words)[at * (W / 4) + word / 4] = static_cast<uint16_t>(w);
    }
  }
}

// A thread: eight dimensions of a row of keys or of values.
template <typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4Planes c, const int* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, long long k_stride,
                                                       long long v_stride, int words, long long items, int vec, int* status) {
  pdl_sync();
  const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (id >= items) return;
  const int word = static_cast<int>(id % words);
  const long long rest = id / words;
  const bool is_v = rest & 1;
  const long long unit = rest >> 1, token = unit / c.kv_heads;
  const int head = static_cast<int>(unit % c.kv_heads);
  const int slot = slots[token];
  if (slot < 0) return;
  if (static_cast<unsigned int>(slot) >= c.slots) {
    *reinterpret_cast<volatile int*>(status) = kStatusBadSlot;
    return;
  }
  const int left = c.head_dim - word * 8;
  if (left <= 0) return;
  const long long at = kv4_row(slot, head, c.kv_heads, c.page_size);
  const uint32_t codes = (is_v ? c.v_codes : c.k_codes)[at * words + word];
  const uint32_t w = (is_v ? c.v_words : c.k_words)[at * (words / 4) + word / 4];
  const float s = __uint_as_float((w & 0xffe0u) << 16);
  const int z = w & 15;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = s * static_cast<float>(static_cast<int>((codes >> (4 * e)) & 15) - z);
  T* dst = (is_v ? v + token * v_stride : k + token * k_stride) + static_cast<long long>(head) * c.head_dim + word * 8;
  if (vec && left >= 8) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      Vec16<T> t;
#pragma unroll
      for (int e = 0; e < N; ++e) t.v[e] = x[i + e];
      t.store(dst + i);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) st(dst + e, x[e]);
  }
}

static bool kv4_rows_aligned(const void* k, const void* v, long long k_stride, long long v_stride, int head_dim, int size) {
  return reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 && k_stride * size % 16 == 0 && v_stride * size % 16 == 0 &&
         head_dim * size % 16 == 0;
}

template <typename T>
static void launch_kv4_append(const T* k, const T* v, long long k_stride, long long v_stride, const int* slots, const Kv4Planes& c, int tokens, cudaStream_t s) {
  const long long units = static_cast<long long>(tokens) * c.kv_heads;
  const int vec = kv4_rows_aligned(k, v, k_stride, v_stride, c.head_dim, sizeof(T)) ? 1 : 0;
  const int ng = (c.head_dim + 63) / 64;
  const int blocks = ceil_div(units, ng == 1 ? 16 : 8);
  switch (ng) {
    case 1: TIE_LAUNCH((kv4_append_kernel<T, 1>), blocks, 256, 0, s, k, v, k_stride, v_stride, slots, c, units, vec, status_word()); break;
    case 2: TIE_LAUNCH((kv4_append_kernel<T, 2>), blocks, 256, 0, s, k, v, k_stride, v_stride, slots, c, units, vec, status_word()); break;
    case 3: TIE_LAUNCH((kv4_append_kernel<T, 3>), blocks, 256, 0, s, k, v, k_stride, v_stride, slots, c, units, vec, status_word()); break;
    default: TIE_LAUNCH((kv4_append_kernel<T, 4>), blocks, 256, 0, s, k, v, k_stride, v_stride, slots, c, units, vec, status_word()); break;
  }
}

template <typename T>
static void launch_kv4_read(T* k, T* v, long long k_stride, long long v_stride, const int* slots, const Kv4Planes& c, int tokens, cudaStream_t s) {
  const int words = (c.head_dim + 63) / 64 * 8;
  const long long items = static_cast<long long>(tokens) * c.kv_heads * 2 * words;
  const int vec = kv4_rows_aligned(k, v, k_stride, v_stride, c.head_dim, sizeof(T)) ? 1 : 0;
  TIE_LAUNCH(kv4_read_kernel<T>, ceil_div(items, 256), 256, 0, s, c, slots, k, v, k_stride, v_stride, words, items, vec, status_word());
}

static int kv4_check(const char* name, const Kv4Planes& c, int tokens, long long pages) {
  TIE_REQUIRE(tokens >= 0 && c.kv_heads > 0 && c.page_size > 0 && c.head_dim > 0 && c.head_dim <= 256, "%s: bad sizes (tokens %d, kv heads %d, page size %d, head size %d)",
              name, tokens, c.kv_heads, c.page_size, c.head_dim);
  TIE_REQUIRE(pages > 0 && pages * c.page_size < (1LL << 31), "%s: %lld pages of %d tokens: slots are 32-bit numbers", name, pages, c.page_size);
  TIE_REQUIRE(static_cast<long long>(tokens) * c.kv_heads * 64 < (1LL << 31) * 256, "%s: too many rows", name);
  TIE_REQUIRE(status_word() != nullptr, "%s: cannot allocate the status word", name);
  return kOk;
}

}  // namespace tie

using namespace tie;

// k, v [tokens, kv_heads * head_dim] (rows strides apart) into the planes at slots[t]; a slot below zero writes nothing.
TIE_API int tie_kv4_append(int dtype, const void* k, const void* v, long long k_stride, long long v_stride, const int* slots, void* k_codes, void* k_words,
                           void* v_codes, void* v_words, int tokens, int kv_heads, int head_dim, int page_size, long long pages, cudaStream_t s) {
  const Kv4Planes c{static_cast<uint32_t*>(k_codes), static_cast<uint32_t*>(v_codes), static_cast<uint16_t*>(k_words), static_cast<uint16_t*>(v_words),
                    kv_heads, page_size, head_dim, static_cast<unsigned int>(pages * page_size)};
  if (const int bad = kv4_check("kv4_append", c, tokens, pages)) return bad;
  if (tokens == 0) return kOk;
  if (dtype == TIE_F32) launch_kv4_append(static_cast<const float*>(k), static_cast<const float*>(v), k_stride, v_stride, slots, c, tokens, s);
  else launch_kv4_append(static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), k_stride, v_stride, slots, c, tokens, s);
  TIE_RETURN_LAUNCH("kv4_append");
}

// The values at slots[t] into k, v [tokens, kv_heads * head_dim]; rows whose slot is below zero are left as they are.
TIE_API int tie_kv4_read(int dtype, const void* k_codes, const void* k_words, const void* v_codes, const void* v_words, const int* slots, void* k, void* v,
                         long long k_stride, long long v_stride, int tokens, int kv_heads, int head_dim, int page_size, long long pages, cudaStream_t s) {
  const Kv4Planes c{static_cast<uint32_t*>(const_cast<void*>(k_codes)), static_cast<uint32_t*>(const_cast<void*>(v_codes)),
                    static_cast<uint16_t*>(const_cast<void*>(k_words)), static_cast<uint16_t*>(const_cast<void*>(v_words)),
                    kv_heads, page_size, head_dim, static_cast<unsigned int>(pages * page_size)};
  if (const int bad = kv4_check("kv4_read", c, tokens, pages)) return bad;
  if (tokens == 0) return kOk;
  if (dtype == TIE_F32) launch_kv4_read(static_cast<float*>(k), static_cast<float*>(v), k_stride, v_stride, slots, c, tokens, s);
  else launch_kv4_read(static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), k_stride, v_stride, slots, c, tokens, s);
  TIE_RETURN_LAUNCH("kv4_read");
}
