// Attention over a cache in 4 bits (the format: kv4.cuh) for few rows at a time: sequences that bring one token, short portions, the 32-bit
// path, and every head size up to 256. Long bfloat16 portions of heads up to 128 run in attention_prompt_kv4.cu.
//
// What it computes, for row (query j of sequence s, head h): pos = context - queries + j, keys lo..pos (lo > 0 only with a window),
//     out = sum_k softmax_k(scale q . K_k) V_k,   K_k, V_k the bfloat16 values that the codes stand for;  no key: zeros.
//
// The cache has to be read once: 9/8 head_dim bytes a token and kv head, a quarter of a bfloat16 cache's, so at the same memory rate a value has a
// quarter of the time. What an SM can spend on one is then about two instructions of a warp for 32 values, and the kernel is laid out around
// that:
//   - The products run transposed, S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16: keys (then dimensions) are the 16 rows and the
//     query heads of a kv head the 8 columns, so eight heads fill a tile that would be half empty the other way round, and what is taken
//     apart is the A operand, whose registers a thread makes itself out of words it loads as they lie in memory. A sum does not care about
//     the order of its terms, so which dimension (or key) stands at which place of a tile is chosen such that every thread reads whole
//     words: a thread of a quad a quarter of a key's row, a thread of eight an eighth of a value's.
//   - Two codes become two bfloat16 values in three instructions: shift, (and | or) that puts the codes into the mantissa of 16, one
//     fma with the group's s and -(16 + z) s. Every one of them is exact.
//   - The scores' accumulators have keys as rows; movmatrix turns the weights into the B operand of the second product.
//   - The maximum moves only when a score exceeds it by 2^8 (any reference gives the same quotient), which costs one vote a tile.
// A CTA is four warps that share (sequence, kv head, 8 or 16 rows, a split of the keys); each warp has its own 32-key tiles (every fourth of the
// split) and its own ring of stages, filled by bulk copies of whole pages (or, for pages that are no power of two from 4 up, by cp.async row by
// row), so that warps wait for memory only, never for one another. At the end the warps put their sums together in shared memory, and the
// splits theirs in the workspace: the last CTA to arrive adds them in split order, so the result does not depend on who came last.
//
// The weights enter the second product as two bfloat16 terms (16 bits), the queries of float rows and their weights as three (24 bits):
// the operands then have the bits that the result's type can show.
#include "attention_mma.cuh"
#include "kv4.cuh"
#include "tma.cuh"

namespace tie {

constexpr int kKv4Threads = 128;
constexpr int kKv4Tile = 32;              // keys of a warp's tile
constexpr int kKv4Stages = 3;
constexpr int kKv4MinTiles = 8;           // tiles of a split at least (two a warp), where there is a choice
constexpr int kKv4MaxCtas = 2368;         // CTAs that leave partial sums (the workspace's size): 16 an SM

struct Kv4Args {
  const void* q;
  void* out;
  const uint8_t *k_codes, *v_codes, *k_words, *v_words;
  const int *query_start, *context_lens, *block_tables, *seq_list;
  float* scratch;           // [grid z][grid x][max_splits][rows of a CTA][head_dim + 2]
  int* counters;            // [grid z][grid x], zero between launches
  int* status;
  long long q_stride, tokens;
  int max_blocks, pages, q_heads, kv_heads, head_dim, page_size, page_shift, window, max_splits, seqs, row_blocks;
  float scale_log2;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// a and b as TERMS pairs of bfloat16 numbers whose sums they are (to 8 TERMS bits).
template <int TERMS> __device__ __forceinline__ void split_terms(float a, float b, uint32_t (&t)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    t[i] = pack_bf16(a, b);
    if (i + 1 < TERMS) a -= bf16_lo(t[i]), b -= bf16_hi(t[i]);
  }
}

template <int N> __device__ __forceinline__ void lds_words(uint32_t (&r)[N], const uint8_t* p) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      r[i] = v.x, r[i + 1] = v.y, r[i + 2] = v.z, r[i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p + 4 * i);
      r[i] = v.x, r[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
  }
}

// NG: padded head size in 64s; HN: tiles of 8 rows a CTA; F32: float queries and outputs (three terms), else bfloat16 (queries as they are, two
// terms of the weights); BULK: pages are copied whole.
template <int NG, int HN, bool F32, bool BULK>
__global__ void __launch_bounds__(kKv4Threads, NG <= 2 && HN == 1 && !F32 ? 4 : 2) attn_kv4_kernel(Kv4Args a) {
  pdl_sync();
  constexpr int DP = 64 * NG, ROWS = 8 * HN;
  constexpr int CODE_ROW = 32 * NG, WORD_ROW = 4 * NG;                     // bytes of a token
  constexpr int CODES = kKv4Tile * CODE_ROW, WORDS = kKv4Tile * WORD_ROW;
  constexpr int STAGE = 2 * (CODES + WORDS);
  constexpr int QT = F32 ? 3 : 1, PT = F32 ? 3 : 2;
  constexpr int QK = 4 * NG;                                               // steps of 16 dimensions
  constexpr bool Q_REGS = !F32;
  constexpr int Q_BYTES = Q_REGS ? 0 : QT * HN * QK * 32 * 8;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (kKv4Stages * STAGE);
  uint2* q_frag = reinterpret_cast<uint2*>(smem + 4 * kKv4Stages * STAGE);          // [term][tile][step][lane], float rows only
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + 4 * kKv4Stages * STAGE + Q_BYTES) + warp * kKv4Stages;
  int* flags = reinterpret_cast<int*>(smem + 4 * kKv4Stages * STAGE + Q_BYTES + 4 * kKv4Stages * 8);    // [0] a wait gave up, [1] last to arrive

  const int split = blockIdx.y, kvh = blockIdx.x % a.kv_heads, rb = blockIdx.x / a.kv_heads;
  const int seq = a.seq_list ? a.seq_list[blockIdx.z] : static_cast<int>(blockIdx.z);
  if (seq < 0 || seq >= a.seqs) return;
  const int G = a.q_heads / a.kv_heads;
  const int t0 = a.query_start[seq], nq = a.query_start[seq + 1] - t0, context = a.context_lens[seq];
  const int rows = min(nq * G - rb * ROWS, ROWS);
  if (rows <= 0) return;
  const int pos0 = context - nq;                                           // position of the sequence's first row
  const int q_first = rb * ROWS / G, q_last = (rb * ROWS + rows - 1) / G;
  const int hi = pos0 + q_last;
  const int lo = a.window > 0 ? max(0, pos0 + q_first - a.window + 1) : 0;
  const int tile0 = lo / kKv4Tile;
  const int tiles = hi < lo ? 0 : hi / kKv4Tile - tile0 + 1;
  const int n_splits = max(1, min(a.max_splits, (tiles + kKv4MinTiles - 1) / kKv4MinTiles));
  if (split >= n_splits) return;
  const int per = (tiles + n_splits - 1) / n_splits;
  const int first = tile0 + split * per, last = min(tile0 + tiles, first + per);       // this CTA's tiles [first, last)
  const int mine = last - first - warp > 0 ? (last - first - warp + 3) / 4 : 0;         // this warp's: first + warp, + 4, ...

  if (threadIdx.x == 0) {
    flags[0] = 0;
    flags[1] = 0;
  }
  if constexpr (BULK) {
    if (lane == 0) {
      for (int s = 0; s < kKv4Stages; ++s) mbar_init(full + s, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
  }
  const int* table = a.block_tables + static_cast<long long>(seq) * a.max_blocks;
  const int box = BULK ? min(a.page_size, kKv4Tile) : 1;                   // keys of one copy
  // the page of this lane's key (its copy's first key) in tile i of this warp, or -1
  const auto page_of = [&](int i) {
    const int key = (first + warp + 4 * i) * kKv4Tile + (BULK ? (lane >> 2) * box : lane);
    if (i >= mine || key > hi || (BULK && (lane >> 2) * box >= kKv4Tile)) return -1;
    const int idx = BULK ? key >> a.page_shift : key / a.page_size;
    const int page = idx < a.max_blocks ? table[idx] : -1;
    if (page < 0 || page >= a.pages) {
      if (key + box > lo) *reinterpret_cast<volatile int*>(a.status) = kStatusBadPage;     // (pages below a window are gone)
      return -1;
    }
    return page;
  };
  // copies of tile i into its stage; `page` as page_of gave it
  const auto fetch = [&](int i, int page) {
    uint8_t* stage = ring + (i % kKv4Stages) * STAGE;
    const int key0 = (first + warp + 4 * i) * kKv4Tile;
    if constexpr (BULK) {
      const int key = key0 + (lane >> 2) * box;
      const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, page >= 0)) >> 2;      // (four lanes a box)
      uint64_t* bar = full + i % kKv4Stages;
      if (lane == 0) mbar_expect_tx(bar, boxes * box * 2 * (CODE_ROW + WORD_ROW));
      __syncwarp();
      if (page >= 0) {
        const long long row = (static_cast<long long>(page) * a.kv_heads + kvh) * a.page_size + (key & (a.page_size - 1));
        const int at = (lane >> 2) * box;
        if (t < 2) bulk_load(stage + t * CODES + at * CODE_ROW, (t == 0 ? a.k_codes : a.v_codes) + row * CODE_ROW, box * CODE_ROW, bar);
        else bulk_load(stage + 2 * CODES + (t - 2) * WORDS + at * WORD_ROW, (t == 2 ? a.k_words : a.v_words) + row * WORD_ROW, box * WORD_ROW, bar);
      }
    } else {
      const long long row = page >= 0 ? (static_cast<long long>(page) * a.kv_heads + kvh) * a.page_size + (key0 + lane) % a.page_size : 0;
      constexpr int CHUNKS = CODE_ROW / 16;
      const uint32_t dst = smem_u32(stage);
#pragma unroll 2
      for (int j = 0; j < CHUNKS; ++j) {
        const int id = j * 32 + lane, key = id / CHUNKS, c = id % CHUNKS;
        const long long r = __shfl_sync(0xffffffffu, row, key);
        const int bytes = __shfl_sync(0xffffffffu, page, key) >= 0 ? 16 : 0;
        cp_async16(dst + id * 16, a.k_codes + r * CODE_ROW + c * 16, bytes);
        cp_async16(dst + CODES + id * 16, a.v_codes + r * CODE_ROW + c * 16, bytes);
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        cp_async4(dst + 2 * CODES + (lane * NG + j) * 4, a.k_words + row * WORD_ROW + j * 4, page >= 0 ? 4 : 0);
        cp_async4(dst + 2 * CODES + WORDS + (lane * NG + j) * 4, a.v_words + row * WORD_ROW + j * 4, page >= 0 ? 4 : 0);
      }
      cp_async_commit();
    }
  };
  int next_page = page_of(0);
#pragma unroll 1
  for (int i = 0; i < kKv4Stages - 1; ++i) {
    const int page = next_page;
    next_page = page_of(i + 1);
    if (i < mine) fetch(i, page);
    else if constexpr (!BULK) cp_async_commit();
  }

  // Queries: the B operand's registers of row g of a tile, dimensions (2 NG t + w) 8 + {i, i + 4} of word w of this thread's part of a row
  uint32_t qf[Q_REGS ? HN : 1][Q_REGS ? QK : 1][2];
#pragma unroll
  for (int n = 0; n < HN; ++n) {
    const int r = rb * ROWS + n * 8 + g;
    const bool there = n * 8 + g < rows && t0 + r / G < a.tokens;
    const T* src = static_cast<const T*>(a.q) + (there ? static_cast<long long>(t0 + r / G) * a.q_stride + static_cast<long long>(kvh * G + r % G) * a.head_dim : 0);
    if (!F32 || warp == 0) {
#pragma unroll
      for (int k = 0; k < QK; ++k) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int d = (2 * NG * t + k / 2) * 8 + 2 * (k & 1) + half;
          const float x = there && d < a.head_dim ? ld(src + d) : 0.0f, y = there && d + 4 < a.head_dim ? ld(src + d + 4) : 0.0f;
          uint32_t terms[QT];
          split_terms<QT>(x, y, terms);
          if constexpr (Q_REGS) {
            qf[n][k][half] = terms[0];
          } else {
#pragma unroll
            for (int e = 0; e < QT; ++e) reinterpret_cast<uint32_t*>(q_frag + ((e * HN + n) * QK + k) * 32 + lane)[half] = terms[e];
          }
        }
      }
    }
  }
  __syncthreads();

  float acc[HN][4 * NG][4];
  float m[HN][2], l[HN][2];
  int pos[HN][2];               // of rows 2 t and 2 t + 1 of a tile; -1: no such row
#pragma unroll
  for (int n = 0; n < HN; ++n) {
#pragma unroll
    for (int i = 0; i < 4 * NG; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[n][e] = -INFINITY, l[n][e] = 0.0f;
      const int r = n * 8 + 2 * t + e;
      pos[n][e] = r < rows ? pos0 + (rb * ROWS + r) / G : -1;
    }
  }
  const int kappa = g ^ ((g >> 1) & 1);                    // the key at row g of an 8-key half (neighbouring rows lie in different bank halves)
  const int ka = 2 * t ^ (t & 1), kb = (2 * t + 1) ^ (t & 1);      // the keys at rows 2 t and 2 t + 1
  const int all_from = a.window > 0 ? pos0 + q_last - a.window + 1 : 0;       // keys that every row sees: all_from..all_to
  const int all_to = pos0 + q_first;

#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    const uint8_t* stage = ring + (i % kKv4Stages) * STAGE;
    const int key0 = (first + warp + 4 * i) * kKv4Tile;
    {
      // the stage that the tile before this one left
      const int page = next_page;
      next_page = page_of(i + kKv4Stages);
      if (i + kKv4Stages - 1 < mine) fetch(i + kKv4Stages - 1, page);
      else if constexpr (!BULK) cp_async_commit();
    }
    if constexpr (BULK) {
      if (!__all_sync(0xffffffffu, mbar_wait(full + i % kKv4Stages, (i / kKv4Stages) & 1, flags, a.status, 12) ? 1 : 0)) break;
    } else {
      cp_async_wait<kKv4Stages - 1>();
      __syncwarp();
    }
    const bool edge = key0 < all_from || key0 + kKv4Tile - 1 > all_to;
    // ---- scores
    float sc[2][HN][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int n = 0; n < HN; ++n) sc[b][n][0] = sc[b][n][1] = sc[b][n][2] = sc[b][n][3] = 0.0f;
      uint32_t w[2][2 * NG];
      Kv4Scale s0[2], s1[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = 16 * b + 8 * h + kappa;
        lds_words(w[h], stage + key * CODE_ROW + t * 8 * NG);
        const uint16_t* words = reinterpret_cast<const uint16_t*>(stage + 2 * CODES + key * WORD_ROW);
        s0[h] = kv4_scale(words[(2 * NG * t) >> 2] * 0x10001u);
        if constexpr (NG > 2) s1[h] = kv4_scale(words[((2 * NG * t) >> 2) + 1] * 0x10001u);
        else s1[h] = s0[h];
      }
#pragma unroll
      for (int x = 0; x < 2 * NG; ++x) {
        // words of a second group: the upper half of four words; of three 64s, those behind the first whole group's end
        uint32_t v[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool second = NG == 4 ? x >= 4 : (NG == 3 ? x >= ((t & 1) ? 2 : 4) : false);
          const Kv4Scale& s = second ? s1[h] : s0[h];
          v[h][0] = bf16x2_fma(kv4_pair<0>(w[h][x]), s.s, s.off);
          v[h][1] = bf16x2_fma(kv4_pair<1>(w[h][x]), s.s, s.off);
          v[h][2] = bf16x2_fma(kv4_pair<2>(w[h][x]), s.s, s.off);
          v[h][3] = bf16x2_fma(kv4_pair<3>(w[h][x]), s.s, s.off);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t af[4] = {v[0][2 * y], v[1][2 * y], v[0][2 * y + 1], v[1][2 * y + 1]};
#pragma unroll
          for (int n = 0; n < HN; ++n) {
            if constexpr (Q_REGS) {
              mma_bf16(sc[b][n], af, qf[n][2 * x + y][0], qf[n][2 * x + y][1]);
            } else {
#pragma unroll
              for (int e = QT - 1; e >= 0; --e) {
                const uint2 f = q_frag[((e * HN + n) * QK + 2 * x + y) * 32 + lane];
                mma_bf16(sc[b][n], af, f.x, f.y);
              }
            }
          }
        }
      }
    }
    // ---- softmax: rows of the accumulators are keys kappa, 8 + kappa of a half tile, columns the rows 2 t, 2 t + 1
    bool grow = false;
#pragma unroll
    for (int n = 0; n < HN; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& v = sc[b][n][2 * h + e];
            v *= a.scale_log2;
            if (edge) {
              const int key = key0 + 16 * b + 8 * h + kappa;
              const bool seen = key <= pos[n][e] && (a.window <= 0 || key > pos[n][e] - a.window);
              v = seen ? v : -INFINITY;
            }
            top = fmaxf(top, v);
          }
        }
        grow = grow || top > m[n][e] + 8.0f;
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < HN; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(fmaxf(sc[0][n][e], sc[0][n][2 + e]), fmaxf(sc[1][n][e], sc[1][n][2 + e]));
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (top > m[n][e]) {
            const float f = m[n][e] == -INFINITY ? 0.0f : exp2f(m[n][e] - top);
            m[n][e] = top;
            l[n][e] *= f;
#pragma unroll
            for (int j = 0; j < 4 * NG; ++j) acc[n][j][e] *= f, acc[n][j][2 + e] *= f;
          }
        }
      }
    }
    uint32_t pf[2][HN][PT][2];
#pragma unroll
    for (int n = 0; n < HN; ++n) {
      const float base0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], base1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = exp2f(sc[b][n][2 * h] - base0), p1 = exp2f(sc[b][n][2 * h + 1] - base1);
          l[n][0] += p0, l[n][1] += p1;
          uint32_t terms[PT];
          split_terms<PT>(p0, p1, terms);
#pragma unroll
          for (int e = 0; e < PT; ++e) pf[b][n][e][h] = transpose8x8(terms[e]);
        }
      }
    }
    // ---- values
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t w[4][NG];
      uint32_t words[2][2];       // group words of keys (ka, kb) of either half, of the first and second group of this thread's dimensions
      constexpr int SECOND = NG == 3 ? 1 : 0;
      const int group = (g * NG) >> 2;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k0 = 16 * b + 8 * h + ka, k1 = 16 * b + 8 * h + kb;
        lds_words(w[2 * h], stage + CODES + k0 * CODE_ROW + g * 4 * NG);
        lds_words(w[2 * h + 1], stage + CODES + k1 * CODE_ROW + g * 4 * NG);
        const uint16_t* wa = reinterpret_cast<const uint16_t*>(stage + 2 * CODES + WORDS + k0 * WORD_ROW) + group;
        const uint16_t* wb = reinterpret_cast<const uint16_t*>(stage + 2 * CODES + WORDS + k1 * WORD_ROW) + group;
        words[h][0] = wa[0] | (static_cast<uint32_t>(wb[0]) << 16);
        words[h][1] = words[h][0];
        // (of three 64s, a thread's words may reach into the next group; the last one's does not)
        if constexpr (SECOND != 0) words[h][1] = ((g * NG) & 3) != 0 && group < 2 * NG - 1 ? wa[1] | (static_cast<uint32_t>(wb[1]) << 16) : words[h][0];
        if (edge) {                // what lies outside of the keys may be anything (a page below a window was not even copied): its values are zero
          const int x0 = key0 + k0, x1 = key0 + k1;
          const uint32_t keep = (x0 >= lo && x0 <= hi ? 0xffffu : 0u) | (x1 >= lo && x1 <= hi ? 0xffff0000u : 0u);
          words[h][0] &= keep, words[h][1] &= keep;
        }
      }
      const Kv4Scale s0[2] = {kv4_scale(words[0][0]), kv4_scale(words[1][0])};
      const Kv4Scale s1[2] = {SECOND ? kv4_scale(words[0][1]) : s0[0], SECOND ? kv4_scale(words[1][1]) : s0[1]};
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const bool second = NG == 3 && ((g * NG) & 3) + x >= 4;
        uint32_t v[2][8];          // [half][dimension of the word]: the value of key ka in the low, of kb in the high bits
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Kv4Scale& s = second ? s1[h] : s0[h];
          const uint32_t low = __byte_perm(w[2 * h][x], w[2 * h + 1][x], 0x5410), high = __byte_perm(w[2 * h][x], w[2 * h + 1][x], 0x7632);
          v[h][0] = bf16x2_fma(kv4_pair<0>(low), s.s, s.off);
          v[h][1] = bf16x2_fma(kv4_pair<1>(low), s.s, s.off);
          v[h][2] = bf16x2_fma(kv4_pair<2>(low), s.s, s.off);
          v[h][3] = bf16x2_fma(kv4_pair<3>(low), s.s, s.off);
          v[h][4] = bf16x2_fma(kv4_pair<0>(high), s.s, s.off);
          v[h][5] = bf16x2_fma(kv4_pair<1>(high), s.s, s.off);
          v[h][6] = bf16x2_fma(kv4_pair<2>(high), s.s, s.off);
          v[h][7] = bf16x2_fma(kv4_pair<3>(high), s.s, s.off);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t af[4] = {v[0][y], v[0][y + 4], v[1][y], v[1][y + 4]};
#pragma unroll
          for (int n = 0; n < HN; ++n) {
#pragma unroll
            for (int e = PT - 1; e >= 0; --e) mma_bf16(acc[n][4 * x + y], af, pf[b][n][e][0], pf[b][n][e][1]);
          }
        }
      }
    }
    __syncwarp();        // (the next fetch writes the stage that was just read)
  }
  if constexpr (!BULK) cp_async_wait<0>();
  __syncthreads();
  if (flags[0] != 0) {   // a wait ran out: let copies that are still in flight land before the ring is reused
    const unsigned long long start = clock64();
    while (clock64() - start < 4000000ull) {
    }
    __syncthreads();
  }

  // The warps' sums: [warp][row][DP + 2] floats, over the ring
  constexpr int RS = DP + 2;
  float* part = reinterpret_cast<float*>(smem);
  static_assert(4 * ROWS * RS * 4 + 6 * ROWS * 4 <= 4 * kKv4Stages * STAGE, "the warps' sums fit the ring");
#pragma unroll
  for (int n = 0; n < HN; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* dst = part + (warp * ROWS + n * 8 + 2 * t + e) * RS;
#pragma unroll
      for (int x = 0; x < NG; ++x) {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int d = (g * NG + x) * 8 + y;
          dst[d] = acc[n][4 * x + y][e];
          dst[d + 4] = acc[n][4 * x + y][2 + e];
        }
      }
      float sum = l[n][e];
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (g == 0) dst[DP] = m[n][e], dst[DP + 1] = sum;
    }
  }
  __syncthreads();
  float* fac = part + 4 * ROWS * RS;         // [row][4] factors, [row] maximum, [row] sum
  if (threadIdx.x < ROWS) {
    const int r = threadIdx.x;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, part[(w * ROWS + r) * RS + DP]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = part[(w * ROWS + r) * RS + DP], lw = part[(w * ROWS + r) * RS + DP + 1];
      // a warp without keys has the sum zero; one whose scores were all NaN has no maximum, but a NaN sum that has to count
      const float f = mw == -INFINITY ? (lw == 0.0f ? 0.0f : lw) : exp2f(mw - top);
      fac[r * 4 + w] = f;
      sum += lw * f;
    }
    fac[4 * ROWS + r] = top;
    fac[5 * ROWS + r] = sum;
  }
  __syncthreads();
  T* out = static_cast<T*>(a.out);
  if (n_splits == 1) {
    for (int id = threadIdx.x; id < rows * a.head_dim; id += kKv4Threads) {
      const int n = id / a.head_dim, d = id % a.head_dim, r = rb * ROWS + n;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) v = fmaf(part[(w * ROWS + n) * RS + d], fac[n * 4 + w], v);
      const float sum = fac[5 * ROWS + n];
      if (t0 + r / G < a.tokens) st(out + (static_cast<long long>(t0 + r / G) * a.q_heads + kvh * G + r % G) * a.head_dim + d, sum == 0.0f ? 0.0f : v / sum);
    }
    return;
  }
  const int sw = a.head_dim + 2;
  const long long cta = static_cast<long long>(blockIdx.z) * gridDim.x + blockIdx.x;
  float* sums = a.scratch + cta * a.max_splits * ROWS * sw;
  for (int id = threadIdx.x; id < rows * sw; id += kKv4Threads) {
    const int n = id / sw, d = id % sw;
    float v = 0.0f;
    if (d < a.head_dim) {
#pragma unroll
      for (int w = 0; w < 4; ++w) v = fmaf(part[(w * ROWS + n) * RS + d], fac[n * 4 + w], v);
    } else {
      v = fac[(d == a.head_dim ? 4 : 5) * ROWS + n];
    }
    sums[(static_cast<long long>(split) * ROWS + n) * sw + d] = v;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) flags[1] = atomicAdd(a.counters + cta, 1) == n_splits - 1;
  __syncthreads();
  if (flags[1] == 0) return;
  __threadfence();
  if (threadIdx.x == 0) a.counters[cta] = 0;
  float* weight = part;                      // [row][split] weights, maxima and sums of the splits, then [row] sums
  for (int id = threadIdx.x; id < rows * n_splits; id += kKv4Threads) {
    const int n = id / n_splits, i = id % n_splits;
    weight[ROWS * n_splits + id] = __ldcg(sums + (static_cast<long long>(i) * ROWS + n) * sw + a.head_dim);
    weight[ROWS * n_splits * 2 + id] = __ldcg(sums + (static_cast<long long>(i) * ROWS + n) * sw + a.head_dim + 1);
  }
  __syncthreads();
  for (int n = warp; n < rows; n += 4) {
    float top = -INFINITY, sum = 0.0f;
    for (int i = lane; i < n_splits; i += 32) top = fmaxf(top, weight[ROWS * n_splits + n * n_splits + i]);
    top = warp_max(top);
    for (int i = lane; i < n_splits; i += 32) {
      const float mi = weight[ROWS * n_splits + n * n_splits + i], li = weight[ROWS * n_splits * 2 + n * n_splits + i];
      const float f = mi == -INFINITY ? (li == 0.0f ? 0.0f : li) : exp2f(mi - top);
      weight[n * n_splits + i] = f;
      sum += li * f;
    }
    sum = warp_sum(sum);
    if (lane == 0) weight[ROWS * n_splits * 3 + n] = sum;
  }
  __syncthreads();
  for (int id = threadIdx.x; id < rows * a.head_dim; id += kKv4Threads) {
    const int n = id / a.head_dim, d = id % a.head_dim, r = rb * ROWS + n;
    float v = 0.0f;
#pragma unroll 4
    for (int i = 0; i < n_splits; ++i) v = fmaf(__ldcg(sums + (static_cast<long long>(i) * ROWS + n) * sw + d), weight[n * n_splits + i], v);
    const float sum = weight[ROWS * n_splits * 3 + n];
    if (t0 + r / G < a.tokens) st(out + (static_cast<long long>(t0 + r / G) * a.q_heads + kvh * G + r % G) * a.head_dim + d, sum == 0.0f ? 0.0f : v / sum);
  }
}

template <int NG, int HN, bool F32, bool BULK>
static int launch_attn_kv4(const Kv4Args& a, int n_list, cudaStream_t s) {
  constexpr int STAGE = 2 * kKv4Tile * 36 * NG;
  constexpr size_t smem = 4 * kKv4Stages * STAGE + (F32 ? 3 * HN * 4 * NG * 32 * 8 : 0) + 4 * kKv4Stages * 8 + 16;
  static_assert(smem <= 227 * 1024, "shared memory of one CTA");
  if (cudaFuncSetAttribute(attn_kv4_kernel<NG, HN, F32, BULK>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) {
    set_error("attention_kv4: cannot reserve %zu bytes of shared memory", smem);
    return kCudaError;
  }
  TIE_LAUNCH((attn_kv4_kernel<NG, HN, F32, BULK>), dim3(a.kv_heads * a.row_blocks, a.max_splits, n_list), kKv4Threads, smem, s, a);
  return kOk;
}

template <int NG, int HN, bool F32>
static int launch_attn_kv4(const Kv4Args& a, bool bulk, int n_list, cudaStream_t s) {
  return bulk ? launch_attn_kv4<NG, HN, F32, true>(a, n_list, s) : launch_attn_kv4<NG, HN, F32, false>(a, n_list, s);
}

template <int NG>
static int launch_attn_kv4(const Kv4Args& a, int hn, bool f32, bool bulk, int n_list, cudaStream_t s) {
  if (f32) return launch_attn_kv4<NG, 1, true>(a, bulk, n_list, s);
  return hn == 1 ? launch_attn_kv4<NG, 1, false>(a, bulk, n_list, s) : launch_attn_kv4<NG, 2, false>(a, bulk, n_list, s);
}

}  // namespace tie

using namespace tie;

TIE_API int tie_attention_kv4_ctas() { return kKv4MaxCtas; }

// Sequences seq_list[0..n_list) (null: 0..n_list-1) of the step, each bringing up to max_queries tokens; max_context: about the longest context
// among them (how the launch is cut, not what it computes). scratch and counters: the workspace, kKv4MaxCtas x 16 x (head_dim + 2)
// floats and kKv4MaxCtas zeros.
TIE_API int tie_attention_kv4(int dtype, const void* q, long long q_stride, long long tokens, const void* k_codes, const void* k_words, const void* v_codes,
                              const void* v_words, void* out, const int* query_start, const int* context_lens, const int* block_tables, int max_blocks, int seqs,
                              int max_queries, int q_heads, int kv_heads, int head_dim, int page_size, long long pages, int window, float scale, const int* seq_list,
                              int n_list, int max_context, float* scratch, int* counters, cudaStream_t s) {
  TIE_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && head_dim > 0 && head_dim <= 256, "attention_kv4: %d query heads over %d kv heads of size %d (at most 256)",
              q_heads, kv_heads, head_dim);
  TIE_REQUIRE(page_size > 0 && pages > 0 && pages * page_size < (1LL << 31) && max_blocks >= 0 && n_list >= 0 && n_list <= 65535 && max_queries >= 0,
              "attention_kv4: bad sizes (%lld pages of %d, %d sequences, %d queries)", pages, page_size, n_list, max_queries);
  TIE_REQUIRE(scale > 0.0f, "attention_kv4: the scale must be positive");
  if (n_list == 0 || max_queries == 0) return kOk;
  TIE_REQUIRE(status_word() != nullptr, "attention_kv4: cannot allocate the status word");
  const bool f32 = dtype == TIE_F32;
  const long long rows = static_cast<long long>(max_queries) * (q_heads / kv_heads);
  const int hn = !f32 && rows > 8 ? 2 : 1;
  const long long row_blocks = (rows + 8 * hn - 1) / (8 * hn), x = row_blocks * kv_heads;
  TIE_REQUIRE(x < (1LL << 30), "attention_kv4: %d queries in one portion are too many", max_queries);
  const int ng = (head_dim + 63) / 64;
  // Splits: as many as fill the SMs once (CTAs that one SM holds at a time: by registers four, or two of the larger forms), no more than the
  // longest context has work for.
  const int places = 148 * (ng <= 2 && hn == 1 && !f32 ? 4 : 2);
  const long long ctas = x * n_list;
  const int keys = window > 0 ? (max_context < window + max_queries ? max_context : window + max_queries) : max_context;
  long long splits = places / ctas;
  const long long most = (keys / kKv4Tile + kKv4MinTiles) / kKv4MinTiles;
  if (splits > most) splits = most;
  if (splits * ctas > kKv4MaxCtas) splits = kKv4MaxCtas / ctas;
  if (splits < 1) splits = 1;
  if (splits > 128) splits = 128;             // (the merge keeps three numbers a row and split in shared memory)
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  const bool bulk = (1 << shift) == page_size && page_size >= 4;
  const Kv4Args a{q, out, static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(v_codes), static_cast<const uint8_t*>(k_words),
                  static_cast<const uint8_t*>(v_words), query_start, context_lens, block_tables, seq_list, scratch, counters, status_word(), q_stride, tokens,
                  max_blocks, static_cast<int>(pages), q_heads, kv_heads, head_dim, page_size, shift, window, static_cast<int>(splits), seqs,
                  static_cast<int>(row_blocks), scale * 1.4426950408889634f};
  int st;
  switch (ng) {
    case 1: st = launch_attn_kv4<1>(a, hn, f32, bulk, n_list, s); break;
    case 2: st = launch_attn_kv4<2>(a, hn, f32, bulk, n_list, s); break;
    case 3: st = launch_attn_kv4<3>(a, hn, f32, bulk, n_list, s); break;
    default: st = launch_attn_kv4<4>(a, hn, f32, bulk, n_list, s); break;
  }
  if (st != kOk) return st;
  TIE_RETURN_LAUNCH("attention_kv4");
}
