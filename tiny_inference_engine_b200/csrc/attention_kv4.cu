// Attention over a cache in 4 bits (the format: kv4.cuh) for few rows at a time: sequences that bring one token, short portions, rows and heads of
// any alignment and size up to 256. Long portions run in attention_prompt_umma.cu (bfloat16 heads up to 256, float up to 128).
//
// What it computes, for row (query j of sequence s, head h): pos = context - queries + j, keys lo..pos (lo > 0 only with a window),
//     out = sum_k softmax_k(scale q . K_k) V_k,   K_k, V_k the bfloat16 values that the codes stand for;  no key: zeros.
//
// The cache has to be read once: 9/8 head_dim bytes a token and kv head, a quarter of a bfloat16 cache's, so at the same memory rate a value has a
// quarter of the time. What bounds the kernel is therefore not the memory but how many instructions a value takes, and the layout follows from
// that:
//   - The products run transposed, S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16: keys (then dimensions) are the 16 rows and the
//     query heads of a kv head the 8 columns, so eight heads fill a tile that would be half empty the other way round, and what is taken
//     apart is the A operand, whose registers a thread makes itself out of words it loads as they lie in memory. A sum does not care about
//     the order of its terms, so which dimension (or key) stands at which place of a tile is chosen such that every thread reads whole
//     words: a thread of a quad a quarter of a key's row, a thread of eight an eighth of a value's.
//   - Two codes become two bfloat16 values by a mask and an fma (kv4.cuh); a shift for every other pair, or, where two keys' words are put side by
//     side anyway, none.
//   - The scores' accumulators have keys as rows; movmatrix turns the weights into the B operand of the second product.
//   - Up to four rows stand in the eight columns twice, and the weights' second terms take the columns that would be empty.
//   - The maximum moves only when a score exceeds it by 2^8 (any reference gives the same quotient), which costs one vote a tile.
// A CTA is four warps that share (sequence, kv head, 4, 8 or 16 rows, a split of the keys); each warp has its own 32-key tiles (every fourth of the
// split) and its own ring of stages, filled by cp.async, so that warps wait for memory only, never for one another. (Bulk copies
// of pages, one an instruction, come out slower: a warp issues them one after the other, and with pages of 16 tokens eight a tile cost more
// instructions than a tile's cp.asyncs and their addresses.) At the end the warps put their sums together in shared memory, and the
// splits theirs in the workspace: the last CTA to arrive adds them in split order, so the result does not depend on who came last.
// Measured (one B200, in a graph): 32 heads over 8 of 128, eight contexts of 32,768 keys 74 us: 302 MB at 4.1 TB/s, 0.63 of the copy rate; 64 contexts of 512
// to 4,096 keys 52 us; one of 4,096 keys 9.6 us. Counters of the first with half the keys: 178 instructions a warp for 8 keys, 2.3 a cycle and
// SM of 4, logical pipe 49 %, fma pipe 33 %, tensor pipe 20 %, 16 warps an SM: no unit is full. What bounds it is the work of a key, and warps too few
// (for their registers) to hide what waits for other work or for a pipe that is taken.
//
// The weights enter the second product as two bfloat16 terms (16 bits), the queries of float rows and their weights as three (24 bits):
// the operands then have the bits that the result's type can show.
#include <type_traits>

#include "attention_mma.cuh"
#include "kv4.cuh"
#include "launchers.h"
#include "umma.cuh"

namespace tie {

constexpr int kKv4Threads = 128;
constexpr int kKv4Tile = 32;              // keys of a warp's tile
constexpr int kKv4Stages = 2;
constexpr int kKv4MaxCtas = 2368;         // CTAs that leave partial sums (the workspace's size): 16 an SM

struct Kv4Args {
  const void* q;
  void* out;
  const uint8_t *k_codes, *v_codes, *k_words, *v_words;
  const int *query_start, *context_lens, *block_tables, *seq_list;
  float* scratch;           // [grid z][grid x][max_splits][rows of a CTA][DP + 2]
  int* counters;            // [grid z][grid x], zero between launches
  int* status;
  long long q_stride, tokens;
  int max_blocks, pages, q_heads, kv_heads, head_dim, page_size, page_shift, window, max_splits, seqs, row_blocks, min_tiles, q_aligned, max_queries;
  float scale_log2;
};

template <int BYTES> __device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// (Not volatile: the compiler may put other work between products that wait for one another.)
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
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

// NG: padded head size in 64s; ROWS: rows of a CTA: 16, 8, or 4, which stand in a tile of 8 twice: the first four columns of the weights are then
// their first terms, the others their second, and one product takes both. F32: float queries and outputs (three terms), else bfloat16
// (queries as they are, two terms of the weights).
template <int NG, int ROWS, bool F32>
__global__ void __launch_bounds__(kKv4Threads, NG <= 2 && ROWS <= 8 && !F32 ? 4 : 2) attn_kv4_kernel(Kv4Args a) {
  pdl_sync();
  constexpr int DP = 64 * NG, HN = (ROWS + 7) / 8;                         // HN tiles of eight columns
  constexpr bool TWICE = ROWS == 4;
  static_assert(!(TWICE && F32), "two terms of the weights");
  constexpr int CODE_ROW = 32 * NG, WORD_ROW = 4 * NG;                     // bytes of a token
  constexpr int CODES = kKv4Tile * CODE_ROW, WORDS = kKv4Tile * WORD_ROW;
  constexpr int STAGE = 2 * (CODES + WORDS);
  constexpr int QT = F32 ? 3 : 1, PT = F32 ? 3 : TWICE ? 1 : 2;
  constexpr int QK = 4 * NG;                                               // steps of 16 dimensions
  constexpr bool Q_REGS = !F32;
  constexpr int Q_BYTES = Q_REGS ? 0 : QT * HN * QK * 32 * 8;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (kKv4Stages * STAGE);
  uint2* q_frag = reinterpret_cast<uint2*>(smem + 4 * kKv4Stages * STAGE);          // [term][tile][step][lane], float rows only
  int* last_one = reinterpret_cast<int*>(smem + 4 * kKv4Stages * STAGE + Q_BYTES);       // whether this CTA is the last of its splits

  const int split = blockIdx.y, kvh = blockIdx.x % a.kv_heads, rb = blockIdx.x / a.kv_heads;
  const int seq = a.seq_list ? a.seq_list[blockIdx.z] : static_cast<int>(blockIdx.z);
  if (seq < 0 || seq >= a.seqs) return;
  const int G = a.q_heads / a.kv_heads;
  const int t0 = a.query_start[seq], nq = a.query_start[seq + 1] - t0, context = a.context_lens[seq];
  const int rows = min(min(nq, a.max_queries) * G - rb * ROWS, ROWS);      // (the first max_queries tokens only; the others' rows stay)
  if (rows <= 0 || t0 < 0) return;
  const int pos0 = context - nq;                                           // position of the sequence's first row
  const int q_first = rb * ROWS / G, q_last = (rb * ROWS + rows - 1) / G;
  int hi = pos0 + q_last;
  if (hi >= static_cast<long long>(a.max_blocks) * a.page_size) {          // a table too short for the context: what it names is read, and the host is told
    if (threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.status) = kStatusBadPage;
    hi = a.max_blocks * a.page_size - 1;
  }
  const int lo = a.window > 0 ? max(0, pos0 + q_first - a.window + 1) : 0;
  const int tile0 = lo / kKv4Tile;
  const int tiles = hi < lo ? 0 : hi / kKv4Tile - tile0 + 1;
  const int n_splits = max(1, min(a.max_splits, (tiles + a.min_tiles - 1) / a.min_tiles));
  if (split >= n_splits) return;
  const int per = (tiles + n_splits - 1) / n_splits;
  const int first = tile0 + split * per, last = min(tile0 + tiles, first + per);       // this CTA's tiles [first, last)
  const int mine = last - first - warp > 0 ? (last - first - warp + 3) / 4 : 0;         // this warp's: first + warp, + 4, ...

  const int* table = a.block_tables + static_cast<long long>(seq) * a.max_blocks;
  // The row of the planes (a token slot of this head) that holds this lane's key of this warp's next tile. Keys beyond the context, below a
  // window or on a page that cannot be have row 0: what is read there is masked. (hi may be below lo: a context of 0, rows ahead of the first
  // key, a table that is too short; then no key is looked up.)
  const unsigned int n_keys = static_cast<unsigned int>(max(hi - lo + 1, 0));
  int next_key = (first + warp) * kKv4Tile + lane;
  const auto row_of_next = [&] {
    const int key = next_key;
    next_key += 4 * kKv4Tile;
    if (static_cast<unsigned int>(key - lo) >= n_keys) return 0;
    const int idx = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
    const int page = table[idx];
    if (static_cast<unsigned int>(page) >= static_cast<unsigned int>(a.pages)) {
      *reinterpret_cast<volatile int*>(a.status) = kStatusBadPage;
      return 0;
    }
    return (page * a.kv_heads + kvh - idx) * a.page_size + key;
  };
  // Copies of a tile into stage s; `row` as row_of_next gave it. Four lanes (of one 64, two) copy a key's codes, 16 bytes each at a time.
  const uint32_t my_dst = smem_u32(ring) + lane * 16;
  const auto fetch = [&](int s, int row) {
    constexpr int CHUNKS = CODE_ROW / 16;
    const uint32_t dst = my_dst + s * STAGE;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
      const int id = j * 32 + lane;
      const long long at = static_cast<long long>(__shfl_sync(0xffffffffu, row, id / CHUNKS)) * CODE_ROW + id % CHUNKS * 16;
      cp_async<16>(dst + j * 512, a.k_codes + at);
      cp_async<16>(dst + CODES + j * 512, a.v_codes + at);
    }
    constexpr int BYTES = NG % 4 == 0 ? 16 : NG % 2 == 0 ? 8 : 4;
    const long long at = static_cast<long long>(row) * WORD_ROW;
    const uint32_t words = smem_u32(ring) + s * STAGE + 2 * CODES + lane * WORD_ROW;
#pragma unroll
    for (int j = 0; j < WORD_ROW; j += BYTES) {
      cp_async<BYTES>(words + j, a.k_words + at + j);
      cp_async<BYTES>(words + WORDS + j, a.v_words + at + j);
    }
  };
  int next_row = row_of_next();
#pragma unroll 1
  for (int i = 0; i < kKv4Stages - 1; ++i) {
    const int row = next_row;
    next_row = row_of_next();
    if (i < mine) fetch(i, row);
    cp_async_commit();
  }

  // Queries: the B operand's registers of row g of a tile, dimensions (2 NG t + w) 8 + {i, i + 4} of word w of this thread's part of a row
  uint32_t qf[Q_REGS ? HN : 1][Q_REGS ? QK : 1][2];
#pragma unroll
  for (int n = 0; n < HN; ++n) {
    const int column = TWICE ? g & 3 : n * 8 + g, r = rb * ROWS + column;
    const bool there = column < rows && t0 + r / G < a.tokens;
    const T* src = static_cast<const T*>(a.q) + (there ? static_cast<long long>(t0 + r / G) * a.q_stride + static_cast<long long>(kvh * G + r % G) * a.head_dim : 0);
    if (!F32 || warp == 0) {
#pragma unroll
      for (int w = 0; w < 2 * NG; ++w) {
        const int d = (2 * NG * t + w) * 8;
        float x[8];
        load8(src + d, there ? a.head_dim - d : 0, a.q_aligned != 0, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 2 * w + i / 2, half = i % 2;
          uint32_t terms[QT];
          split_terms<QT>(x[i], x[i + 4], terms);
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
      const int r = TWICE ? (2 * t + e) & 3 : n * 8 + 2 * t + e;
      pos[n][e] = r < rows ? pos0 + (rb * ROWS + r) / G : -1;
    }
  }
  const int kappa = g ^ ((g >> 1) & 1);                    // the key at row g of an 8-key half (neighbouring rows lie in different bank halves)
  const int ka = 2 * t ^ (t & 1), kb = (2 * t + 1) ^ (t & 1);      // the keys at rows 2 t and 2 t + 1
  const int all_from = a.window > 0 ? pos0 + q_last - a.window + 1 : 0;       // keys that every row sees: all_from..all_to
  const int all_to = pos0 + q_first;

  const uint32_t signs = kv4_signs();
  // One tile. EDGE: not every row sees every key of it (its own form, so that the others do without the comparisons); BIG: with steps that need
  // a product more (kv4.cuh), in the edges' form whatever the rows see
  const auto work = [&](auto edge, auto big, const uint8_t* stage, int key0) {
    constexpr bool EDGE = decltype(edge)::value, BIG = decltype(big)::value;
    // ---- scores, of both halves of the tile side by side
    float sc[2][HN][4];
    uint32_t w[2][2][2 * NG];
    Kv4Scale s0[2][2], s1[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int n = 0; n < HN; ++n) sc[b][n][0] = sc[b][n][1] = sc[b][n][2] = sc[b][n][3] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = 16 * b + 8 * h + kappa;
        lds_words(w[b][h], stage + key * CODE_ROW + t * 8 * NG);
        const uint16_t* words = reinterpret_cast<const uint16_t*>(stage + 2 * CODES + key * WORD_ROW);
        s0[b][h] = kv4_scale<BIG>(words[(2 * NG * t) >> 2] * 0x10001u, signs);
        if constexpr (NG > 2) s1[b][h] = kv4_scale<BIG>(words[((2 * NG * t) >> 2) + 1] * 0x10001u, signs);
        else s1[b][h] = s0[b][h];
      }
    }
#pragma unroll
    for (int x = 0; x < 2 * NG; ++x) {
      uint32_t v[2][2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // words of a second group: the upper half of four words; of three 64s, those behind the first whole group's end
          const bool second = NG == 4 ? x >= 4 : (NG == 3 ? x >= ((t & 1) ? 2 : 4) : false);
          const Kv4Scale& s = second ? s1[b][h] : s0[b][h];
          const uint32_t word = w[b][h][x], next = word >> 8;
          v[b][h][0] = kv4_low<BIG>(word, s);
          v[b][h][1] = kv4_high<BIG>(word, s);
          v[b][h][2] = kv4_low<BIG>(next, s);
          v[b][h][3] = kv4_high<BIG>(next, s);
        }
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int e = QT - 1; e >= 0; --e) {
#pragma unroll
          for (int n = 0; n < HN; ++n) {
            uint2 f;
            if constexpr (Q_REGS) f = make_uint2(qf[n][2 * x + y][0], qf[n][2 * x + y][1]);
            else f = q_frag[((e * HN + n) * QK + 2 * x + y) * 32 + lane];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const uint32_t af[4] = {v[b][0][2 * y], v[b][1][2 * y], v[b][0][2 * y + 1], v[b][1][2 * y + 1]};
              mma(sc[b][n], af, f.x, f.y);
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
            if constexpr (EDGE) {
              const int key = key0 + 16 * b + 8 * h + kappa;
              const bool seen = key <= pos[n][e] && (a.window <= 0 || key > pos[n][e] - a.window);
              v = seen ? v : -INFINITY;
            }
            top = fmaxf(top, v);
          }
        }
        grow = grow || top * a.scale_log2 > m[n][e] + 8.0f;
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
          top *= a.scale_log2;
          if (top > m[n][e]) {
            const float f = m[n][e] == -INFINITY ? 0.0f : ex2(m[n][e] - top);
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
      const float base0 = m[n][0] == -INFINITY ? 0.0f : kKv4WeightShift - m[n][0], base1 = m[n][1] == -INFINITY ? 0.0f : kKv4WeightShift - m[n][1];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = ex2(fmaf(sc[b][n][2 * h], a.scale_log2, base0)), p1 = ex2(fmaf(sc[b][n][2 * h + 1], a.scale_log2, base1));
          l[n][0] += p0, l[n][1] += p1;
          uint32_t terms[TWICE ? 2 : PT];
          split_terms<TWICE ? 2 : PT>(p0, p1, terms);
          if constexpr (TWICE) terms[0] = t < 2 ? terms[0] : terms[1];
#pragma unroll
          for (int e = 0; e < PT; ++e) pf[b][n][e][h] = transpose8x8(terms[e]);
        }
      }
    }
    // ---- values
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t vw[4][NG];
      uint32_t words[2][2];       // group words of keys (ka, kb) of either half, of the first and second group of this thread's dimensions
      constexpr int SECOND = NG == 3 ? 1 : 0;
      const int group = (g * NG) >> 2;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k0 = 16 * b + 8 * h + ka, k1 = 16 * b + 8 * h + kb;
        lds_words(vw[2 * h], stage + CODES + k0 * CODE_ROW + g * 4 * NG);
        lds_words(vw[2 * h + 1], stage + CODES + k1 * CODE_ROW + g * 4 * NG);
        const uint16_t* wa = reinterpret_cast<const uint16_t*>(stage + 2 * CODES + WORDS + k0 * WORD_ROW) + group;
        const uint16_t* wb = reinterpret_cast<const uint16_t*>(stage + 2 * CODES + WORDS + k1 * WORD_ROW) + group;
        words[h][0] = wa[0] | (static_cast<uint32_t>(wb[0]) << 16);
        words[h][1] = words[h][0];
        // (of three 64s, a thread's words may reach into the next group; the last one's does not)
        if constexpr (SECOND != 0) words[h][1] = ((g * NG) & 3) != 0 && group < 2 * NG - 1 ? wa[1] | (static_cast<uint32_t>(wb[1]) << 16) : words[h][0];
        if constexpr (EDGE) {      // what lies outside of the keys may be anything: its values are zero
          const int x0 = key0 + k0, x1 = key0 + k1;
          const uint32_t keep = (x0 >= lo && x0 <= hi ? 0xffffu : 0u) | (x1 >= lo && x1 <= hi ? 0xffff0000u : 0u);
          words[h][0] &= keep, words[h][1] &= keep;
        }
      }
      const Kv4Scale g0[2] = {kv4_scale<BIG>(words[0][0], signs), kv4_scale<BIG>(words[1][0], signs)};
      const Kv4Scale g1[2] = {SECOND ? kv4_scale<BIG>(words[0][1], signs) : g0[0], SECOND ? kv4_scale<BIG>(words[1][1], signs) : g0[1]};
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const bool second = NG == 3 && ((g * NG) & 3) + x >= 4;
        uint32_t v[2][8];          // [half][dimension of the word]: the value of key ka in the low, of kb in the high bits
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Kv4Scale& s = second ? g1[h] : g0[h];
#pragma unroll
          for (int j = 0; j < 4; ++j) {        // byte j of both keys' words
            const uint32_t both = __byte_perm(vw[2 * h][x], vw[2 * h + 1][x], 0x4400 + 0x1111 * j);
            v[h][2 * j] = kv4_low<BIG>(both, s);
            v[h][2 * j + 1] = kv4_high<BIG>(both, s);
          }
        }
        // (a row's terms one round after the other, so that no product waits for the one ahead of it)
#pragma unroll
        for (int e = PT - 1; e >= 0; --e) {
#pragma unroll
          for (int n = 0; n < HN; ++n) {
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t af[4] = {v[0][y], v[0][y + 4], v[1][y], v[1][y + 4]};
              mma(acc[n][4 * x + y], af, pf[b][n][e][0], pf[b][n][e][1]);
            }
          }
        }
      }
    }
  };
  int at = 0;                             // the tile's stage
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    const uint8_t* stage = ring + at * STAGE;
    const int key0 = (first + warp + 4 * i) * kKv4Tile;
    {
      // into the stage that the tile before this one left
      const int row = next_row;
      next_row = row_of_next();
      if (i + kKv4Stages - 1 < mine) fetch(at == 0 ? kKv4Stages - 1 : at - 1, row);
      cp_async_commit();
    }
    cp_async_wait<kKv4Stages - 1>();
    __syncwarp();
    uint32_t big = 0;                     // of this lane's key and value (a key that no row sees: of row 0)
    {
      uint32_t words[2][NG];
      lds_words(words[0], stage + 2 * CODES + lane * WORD_ROW);
      lds_words(words[1], stage + 2 * CODES + WORDS + lane * WORD_ROW);
#pragma unroll
      for (int j = 0; j < NG; ++j) big |= kv4_big(words[0][j]) | kv4_big(words[1][j]);
    }
    if (__any_sync(0xffffffffu, (big & kKv4BigBits) != 0)) work(std::true_type{}, std::true_type{}, stage, key0);
    else if (key0 < all_from || key0 + kKv4Tile - 1 > all_to) work(std::true_type{}, std::false_type{}, stage, key0);
    else work(std::false_type{}, std::false_type{}, stage, key0);
    __syncwarp();        // (the next fetch writes the stage that was just read)
    if (++at == kKv4Stages) at = 0;
  }
  cp_async_wait<0>();
  __syncthreads();

  // The warps' sums over the ring: [warp][row][RS] floats, in a row DP sums, the maximum and the row sum
  constexpr int RS = DP + 4;
  float* part = reinterpret_cast<float*>(smem);
  static_assert(4 * ROWS * RS * 4 + 6 * ROWS * 4 <= 4 * kKv4Stages * STAGE, "the warps' sums fit the ring");
#pragma unroll
  for (int n = 0; n < HN; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if constexpr (TWICE) {       // the sums of a row's second terms are in the lane two on
#pragma unroll
        for (int j = 0; j < 4 * NG; ++j) {
          acc[n][j][e] += __shfl_xor_sync(0xffffffffu, acc[n][j][e], 2);
          acc[n][j][2 + e] += __shfl_xor_sync(0xffffffffu, acc[n][j][2 + e], 2);
        }
      }
      float* dst = part + (warp * ROWS + (TWICE ? (2 * t + e) & 3 : n * 8 + 2 * t + e)) * RS;
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const int d = (g * NG + x) * 8;
        const float4 low = make_float4(acc[n][4 * x][e], acc[n][4 * x + 1][e], acc[n][4 * x + 2][e], acc[n][4 * x + 3][e]);
        const float4 high = make_float4(acc[n][4 * x][2 + e], acc[n][4 * x + 1][2 + e], acc[n][4 * x + 2][2 + e], acc[n][4 * x + 3][2 + e]);
        if (!TWICE || t < 2) *reinterpret_cast<float4*>(dst + d) = low;
        if (!TWICE || t >= 2) *reinterpret_cast<float4*>(dst + d + 4) = high;
      }
      float sum = l[n][e];
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (g == 0 && (!TWICE || t < 2)) dst[DP] = m[n][e], dst[DP + 1] = sum;
    }
  }
  __syncthreads();
  float* fac = part + 4 * ROWS * RS;         // [row][4] factors, [row] maximum, [row] sum
  if (threadIdx.x < ROWS) {
    const int r = threadIdx.x;
    float top = -INFINITY, sum = 0.0f, mw[4], lw[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mw[w] = part[(w * ROWS + r) * RS + DP], lw[w] = part[(w * ROWS + r) * RS + DP + 1], top = fmaxf(top, mw[w]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // a warp without keys has the sum zero; one whose scores were all NaN has no maximum, but a NaN sum that has to count
      const float f = mw[w] == -INFINITY ? lw[w] : exp2f(mw[w] - top);
      fac[r * 4 + w] = f;
      sum += lw[w] * f;
    }
    fac[4 * ROWS + r] = top;
    fac[5 * ROWS + r] = sum;
  }
  __syncthreads();
  // Four columns of a row at a time: from the four warps, and then from the splits
  constexpr int COLS = DP / 4;
  const auto of_warps = [&](int n, int d) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(part + (w * ROWS + n) * RS + d);
      const float f = fac[n * 4 + w];
      v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
    }
    return v;
  };
  const auto store = [&](int n, int d, const float4& v, float sum) {
    const int r = rb * ROWS + n, row = t0 + r / G;
    if (d >= a.head_dim || row >= a.tokens) return;
    T* out = static_cast<T*>(a.out) + (static_cast<long long>(row) * a.q_heads + kvh * G + r % G) * a.head_dim + d;
    const float f = sum == 0.0f ? 0.0f : kKv4Unscale / sum;
    const float x[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
    if ((a.head_dim & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0) {
      store4(out, x);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < a.head_dim) st(out + e, x[e]);
    }
  };
  if (n_splits == 1) {
    for (int id = threadIdx.x; id < rows * COLS; id += kKv4Threads) store(id / COLS, id % COLS * 4, of_warps(id / COLS, id % COLS * 4), fac[5 * ROWS + id / COLS]);
    return;
  }
  const long long cta = static_cast<long long>(blockIdx.z) * gridDim.x + blockIdx.x;
  float* sums = a.scratch + cta * a.max_splits * ROWS * (DP + 2);            // [split][row][DP], then [split][row] maximum and sum
  float2* stats = reinterpret_cast<float2*>(sums + static_cast<long long>(a.max_splits) * ROWS * DP);
  for (int id = threadIdx.x; id < rows * COLS; id += kKv4Threads)
    *reinterpret_cast<float4*>(sums + (static_cast<long long>(split) * ROWS + id / COLS) * DP + id % COLS * 4) = of_warps(id / COLS, id % COLS * 4);
  if (threadIdx.x < rows) stats[split * ROWS + threadIdx.x] = make_float2(fac[4 * ROWS + threadIdx.x], fac[5 * ROWS + threadIdx.x]);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *last_one = atomicAdd(a.counters + cta, 1) == n_splits - 1;
  __syncthreads();
  if (*last_one == 0) return;
  __threadfence();
  if (threadIdx.x == 0) a.counters[cta] = 0;
  float* weight = part;                      // [row][split] weights of the splits, then [row] sums
  for (int n = warp; n < rows; n += 4) {
    float2 of[4];                            // (at most 128 splits)
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = lane + 32 * j;
      of[j] = i < n_splits ? __ldcg(stats + i * ROWS + n) : make_float2(-INFINITY, 0.0f);
      top = fmaxf(top, of[j].x);
    }
    top = warp_max(top);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = lane + 32 * j;
      const float f = of[j].x == -INFINITY ? of[j].y : exp2f(of[j].x - top);
      if (i < n_splits) weight[n * n_splits + i] = f;
      sum += of[j].y * f;
    }
    sum = warp_sum(sum);
    if (lane == 0) weight[ROWS * n_splits + n] = sum;
  }
  __syncthreads();
  for (int id = threadIdx.x; id < rows * COLS; id += kKv4Threads) {
    const int n = id / COLS, d = id % COLS * 4;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int i = 0; i < n_splits; ++i) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(sums + (static_cast<long long>(i) * ROWS + n) * DP + d));
      const float f = weight[n * n_splits + i];
      v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
    }
    store(n, d, v, weight[ROWS * n_splits + n]);
  }
}

template <int NG, int ROWS, bool F32>
static int launch_attn_kv4(const Kv4Args& a, int n_list, cudaStream_t s) {
  constexpr int STAGE = 2 * kKv4Tile * 36 * NG;
  constexpr size_t smem = 4 * kKv4Stages * STAGE + (F32 ? 3 * 4 * NG * 32 * 8 : 0) + 16;
  static_assert(smem <= 227 * 1024 && !(F32 && ROWS != 8), "shared memory of one CTA");
  if (smem > 48 * 1024 && cudaFuncSetAttribute(attn_kv4_kernel<NG, ROWS, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) {
    set_error("attention_kv4: cannot reserve %zu bytes of shared memory", smem);
    return kCudaError;
  }
  TIE_LAUNCH((attn_kv4_kernel<NG, ROWS, F32>), dim3(a.kv_heads * a.row_blocks, a.max_splits, n_list), kKv4Threads, smem, s, a);
  return kOk;
}

template <int NG>
static int launch_attn_kv4(const Kv4Args& a, int cta_rows, bool f32, int n_list, cudaStream_t s) {
  if (f32) return launch_attn_kv4<NG, 8, true>(a, n_list, s);
  if (cta_rows == 4) return launch_attn_kv4<NG, 4, false>(a, n_list, s);
  return cta_rows == 8 ? launch_attn_kv4<NG, 8, false>(a, n_list, s) : launch_attn_kv4<NG, 16, false>(a, n_list, s);
}

}  // namespace tie

using namespace tie;

TIE_API int tie_attention_kv4_ctas() { return kKv4MaxCtas; }

// Sequences seq_list[0..n_list) (null: 0..n_list-1) of the step, each bringing up to max_queries tokens; max_context: about the longest context
// among them (how the launch is cut, not what it computes). scratch and counters: the workspace, kKv4MaxCtas x 16 x (padded head_dim + 2)
// floats and kKv4MaxCtas zeros.
TIE_API int tie_attention_kv4(int dtype, const void* q, long long q_stride, long long tokens, const void* k_codes, const void* k_words, const void* v_codes,
                              const void* v_words, void* out, const int* query_start, const int* context_lens, const int* block_tables, int max_blocks, int seqs,
                              int max_queries, int q_heads, int kv_heads, int head_dim, int page_size, long long pages, int window, float scale, const int* seq_list,
                              int n_list, int max_context, float* scratch, int* counters, cudaStream_t s) {
  TIE_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && head_dim > 0 && head_dim <= 256, "attention_kv4: %d query heads over %d kv heads of size %d (at most 256)",
              q_heads, kv_heads, head_dim);
  TIE_REQUIRE(page_size > 0 && pages > 0 && pages * page_size < (1LL << 31) && max_blocks >= 0 && n_list >= 0 && n_list <= 65535 && max_queries >= 0,
              "attention_kv4: bad sizes (%lld pages of %d, %d sequences, %d queries)", pages, page_size, n_list, max_queries);
  TIE_REQUIRE(pages * page_size * kv_heads < (1LL << 31), "attention_kv4: planes of %lld x %d x %d rows: rows are 32-bit numbers", pages, kv_heads, page_size);
  TIE_REQUIRE(scale > 0.0f, "attention_kv4: the scale must be positive");
  if (n_list == 0 || max_queries == 0) return kOk;
  TIE_REQUIRE(status_word() != nullptr, "attention_kv4: cannot allocate the status word");
  const bool f32 = dtype == TIE_F32;
  const long long rows = static_cast<long long>(max_queries) * (q_heads / kv_heads);
  const int cta_rows = f32 ? 8 : rows > 8 ? 16 : rows > 4 ? 8 : 4;
  const long long row_blocks = (rows + cta_rows - 1) / cta_rows, x = row_blocks * kv_heads;
  TIE_REQUIRE(x < (1LL << 30), "attention_kv4: %d queries in one portion are too many", max_queries);
  const int ng = (head_dim + 63) / 64;
  // Splits. Few (sequence, kv head, row block)s: as many as fill the SMs once (what one SM holds at a time: four CTAs, two of the larger forms), of
  // 256 keys at least (one request at 4,096 keys, 8 kv heads: 17 splits 10.0 us, 9 splits 11.2, 34 10.7). Where not even four fit, contexts are
  // cut into pieces of 1,024 keys at least, enough for two rounds, so that the longest does not set the pace alone (64 contexts of 512 to
  // 4,096 keys: three splits 53 us, one 69; pieces of 256 keys 58).
  const int places = 148 * (ng <= 2 && cta_rows <= 8 && !f32 ? 4 : 2);
  const long long ctas = x * n_list;
  const int keys = window > 0 ? (max_context < window + max_queries ? max_context : window + max_queries) : max_context;
  long long splits = places / ctas;
  int min_tiles = 8;
  if (splits < 4) splits = (2 * places + ctas - 1) / ctas, min_tiles = 32;
  const long long most = (keys / kKv4Tile + min_tiles) / min_tiles;
  if (splits > most) splits = most;
  if (splits * ctas > kKv4MaxCtas) splits = kKv4MaxCtas / ctas;
  if (splits > 128) splits = 128;             // (four a lane in the merge)
  if (splits < 1) splits = 1;
  int shift = 0;
  while (shift < 30 && (1 << shift) < page_size) ++shift;
  if ((1 << shift) != page_size) shift = -1;
  const int size = f32 ? 4 : 2;
  const int q_aligned = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride * size % 16 == 0 && head_dim * size % 16 == 0;
  const Kv4Args a{q, out, static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(v_codes), static_cast<const uint8_t*>(k_words),
                  static_cast<const uint8_t*>(v_words), query_start, context_lens, block_tables, seq_list, scratch, counters, status_word(), q_stride, tokens,
                  max_blocks, static_cast<int>(pages), q_heads, kv_heads, head_dim, page_size, shift, window, static_cast<int>(splits), seqs,
                  static_cast<int>(row_blocks), min_tiles, q_aligned, max_queries, scale * 1.4426950408889634f * kKv4Unscale};
  int st;
  switch (ng) {
    case 1: st = launch_attn_kv4<1>(a, cta_rows, f32, n_list, s); break;
    case 2: st = launch_attn_kv4<2>(a, cta_rows, f32, n_list, s); break;
    case 3: st = launch_attn_kv4<3>(a, cta_rows, f32, n_list, s); break;
    default: st = launch_attn_kv4<4>(a, cta_rows, f32, n_list, s); break;
  }
  if (st != kOk) return st;
  TIE_RETURN_LAUNCH("attention_kv4");
}
