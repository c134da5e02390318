// Causal attention of prompt portions on the 5th-generation tensor cores: S = Q K^T and O += P V are
// tcgen05.mma with the scores and the output accumulator in tensor memory; keys and values come page by
// page through TMA. Head sizes 64 and 128, up to 16 query heads per kv head, pages that are powers
// of two from 8 up; other sizes stay with the mma.sync kernels.
//
// Contract as in attention_prompt.cu (the reference's paged_attention,
// src/backend/cpu/cpu_backend.cpp:261-319): row t of sequence s sits at
// pos = context_len[s] - n_queries(s) + (t - query_start[s]) and sees keys 0..pos (window w > 0:
// pos-w+1..pos), all read from the pages.
//
// One CTA owns 256 rows (rows = queries x the query heads of one kv head) as two tiles of 128, so
// that the tensor cores work on one tile while the other tile's softmax runs, and both share every
// key/value tile of 64 keys. The MMAs' operand reads are what shared memory has to feed, so Q, which
// every key tile needs again, sits in tensor memory (the A operand of Q K^T comes from there; of heads of 128 one half), P too
// where it has room, and only K, V and what has none are read from shared memory. Ten warps:
//   0-3, 4-7  softmax of tile 0 and 1: thread = one row. Puts its Q row into tensor memory once. Per key
//             tile it reads its 64 scores out of tensor memory, masks, exponentiates in float, writes P as
//             bfloat16 into one of its buffers (in shared memory in the layout the MMA reads) and keeps the row
//             sum. The accumulator O stays in tensor memory; it is rescaled only when a row's maximum has
//             grown by more than 2^8 since the value it was last scaled for (any reference point gives
//             the same O / sum, as long as nothing overflows).
//   8         TMA producer: lane b fetches box b (a page, or 64 keys of a larger page) of every tile.
//   9         one thread issues the MMAs: for one row tile and then the other, P V of a key tile and Q K^T of the one after the next.
// Barriers: kv_full/kv_empty per stage, and for each row tile s_full (scores written), s_empty
// (scores read), p_full[2] (P written, O rescaled), p_empty[2] (P V retired). Every wait on an mbarrier is bounded.
// Where the rows are few and the keys many, 2 or 4 CTAs of a thread-block cluster share out the keys of 256 rows and put their sums
// together through distributed shared memory. (The cluster's two barriers have no limit; every path of a CTA reaches them, one that
// gave up a wait too, and the CTAs of a cluster leave ahead of them together or not at all.)
// grid = (kv heads, row tiles, sequences x splits): CTAs start in that order with the last row tiles first, so the
// tiles with the most keys of every kv head run first.
//
// KV4: the same over a cache in 4 bits (kv4.cuh), heads of up to 256 (a multiple of 8; what is missing is zeros) and pages of any size.
// Warps take the place of the TMA producer: they read codes and words some tiles ahead, take them apart and write the
// tile as TMA would have. Heads above 128 leave tensor memory for one row tile a CTA; so do float queries, which
// stand there as three bfloat16 terms (24 bits), as the weights do in shared memory. 4 portions of 512 queries at 2,048 keys, 32 heads over 8,
// us against the kernel whose warps take 16 rows each: heads of 128 90 and 405 (float 194 and 655), of 64 79 and 280 (148 and 422), of 192
// 148 and 604, of 256 193 and 803. Eight dimensions lie in a tile in the order 0 4 1 5 2 6 3 7, in which a word of codes comes apart; Q is put into tensor
// memory in the same order and the outputs are taken out of it again. Keys and values are exact in bfloat16, times 2^-31 (kv4.cuh).
#include <type_traits>

#include "attention_mma.cuh"
#include "kv4.cuh"
#include "umma.cuh"
#include "launchers.h"

namespace tie {

constexpr int kUmmaMaxSplits = 4;
constexpr int kUmmaSplitKeys = 2049;

// Where dimension d of eight lies in a tile of a cache in 4 bits (KV4 below).
__host__ __device__ constexpr int ordered(int d) { return (d & ~7) | ((d & 3) << 1) | ((d >> 2) & 1); }

struct UmmaPromptArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const int* query_start;
  const int* context_lens;
  const int* block_tables;
  int* status;
  long long q_stride;
  int max_blocks, q_heads, kv_heads, page_size, page_shift, window;
  float scale_log2;
  int splits;     // CTAs of a cluster that share out the keys of 256 rows (1: no cluster)
  int cta_rows;   // 256: a CTA works on two row tiles side by side; 128: on one (more CTAs when there are few rows)
  // KV4 only
  const uint8_t *k_codes, *v_codes;
  const uint16_t *k_words, *v_words;
  int head_dim, pages, max_queries;
  long long tokens;       // rows of q and out
};

// Eight outputs of a row from element `at` on; a row's start is 16-byte aligned.
template <bool F32>
__device__ __forceinline__ void store8(__nv_bfloat16* out, long long at, const float (&v)[8]) {
  if constexpr (F32) {
    float* dst = reinterpret_cast<float*>(out) + at;
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(out + at) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
}

// The form of a kernel: heads of up to DH; RT row tiles of 128 a CTA; F32: float queries and outputs, in three bfloat16 terms.
template <int DH_, bool KV4_, int RT_, bool F32_>
struct UmmaForm {
  static constexpr int DH = DH_, RT = RT_, TERMS = F32_ ? 3 : 1;
  static constexpr bool KV4 = KV4_, F32 = F32_;
  // (KV4: with one warp more the softmax's 64 scores a thread would have too few registers)
  static constexpr int THREADS = !KV4 ? 320 : RT == 2 ? 384 : 352;
  static constexpr int PRODUCERS = RT == 2 ? 96 : 192;            // threads that take a KV4 tile apart
  static constexpr int STAGES = DH <= 64 ? (F32 ? 4 : 6) : DH == 128 ? (KV4 ? 3 : 4) : DH == 192 ? 3 : 2;
  static constexpr int AHEAD = 2;                                   // tiles that a producer copies ahead (3: heads of 64 88.6 us instead of 87.3, the others alike)
  static constexpr int ROUNDS = (kKeysPerTile * DH / 32 + PRODUCERS - 1) / PRODUCERS;     // keys (and values) of a producer thread in a tile
  static constexpr int RAW = ROUNDS * PRODUCERS * 40;             // bytes of a tile on its way: a thread's two times 16 bytes of codes and two words
  // Pairs of barriers a stage: 1 for keys and values together; 2 with one for the keys, which are filled again while the values are still read. That
  // pays where the producers are what the others wait for (4 portions of 512 queries at 2,048 keys, 32 heads over 8 of 256: 210 us instead of
  // 235, of 64: 87 instead of 91, with P in shared memory) and else costs waits (of 128: 109 instead of 98; of 192: 174 instead of 159).
  static constexpr int RINGS = KV4_ && !F32_ && (DH <= 64 || DH == 256) ? 2 : 1;
  static constexpr int P_BYTES = 128 * 128;                       // 128 rows x 64 keys
  static constexpr int STAGE_BYTES = 2 * (DH / 64) * 64 * 128;    // keys and values of a tile
  // Where its 512 columns hold scores, Q, accumulators and two tiles' weights P (32 columns a term), P stands in tensor memory too: nothing to store
  // in shared memory and to read there again (KV4, 4 portions of 512 at 2,048 keys: heads of 64 79 us instead of 87, of 192 148 instead of 159,
  // of 256 192 instead of 211, float of 64 149 instead of 163; bfloat16 pages, 16 heads of 64 over 4 at 8,192 keys 138 instead of 170). Two row tiles with heads of
  // 128 make room for one tile's weights each by leaving the second half of Q in shared memory, which is written once (88 us instead of 97; bfloat16
  // pages, 512 queries of 32 heads over 8 at 8,192 keys 85 instead of 98).
  static constexpr bool Q_HALF = DH == 128 && RT == 2;
  static constexpr int Q_COLS = TERMS * DH / 2 / (Q_HALF ? 2 : 1), P_BUFS = Q_HALF ? 1 : 2;
  static constexpr bool P_TMEM = RT * (64 + Q_COLS + DH + 32 * P_BUFS * TERMS) <= 512;
  static constexpr int P_ALL = Q_HALF ? RT * P_BYTES : P_TMEM ? 0 : RT * 2 * TERMS * P_BYTES;         // [row tile][buffer][term]
  static constexpr int SMEM = P_ALL + STAGES * STAGE_BYTES + (KV4 ? AHEAD * RAW : 0) + (2 * RINGS * STAGES + 12) * 8 + 16 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
  static_assert(SMEM >= RT * 128 * (DH + 4) * 4 + (2 * RINGS * STAGES + 12) * 8 + 16 + 1024, "the sums of a CTA's rows");
};

// What the producer warps of a CTA do (KV4); `id` numbers their threads. A thread takes 32 dimensions (16 bytes of codes, one group) of
// some keys and values of every tile. It copies them with cp.async into places of shared memory that are its own, AHEAD tiles ahead, so
// nobody has to be told when they have landed; their pages it looks up another tile ahead.
template <typename Form>
__device__ __forceinline__ void kv4_produce(const UmmaPromptArgs& a, uint8_t* ring, uint8_t* raw, uint64_t* kv_full, uint64_t* kv_empty, volatile int* abort_flag,
                                            int id, int seq, int kvh, int kt_first, int n_tiles, int lo, int hi) {
  constexpr int GROUPS = Form::DH / 32, PER = Form::ROUNDS, RAW = Form::RAW, STAGES = Form::STAGES, PLANE_BYTES = Form::STAGE_BYTES / 2;
  static_assert(Form::PRODUCERS % (4 * GROUPS) == 0, "a thread's keys have one group");
  // Eight threads have four keys' 64 dimensions: what they store at a time lies in eight different places of a row of 128 bytes. (With a key's groups
  // side by side it lies in two to four: with P in shared memory heads of 256 330 us instead of 235, of 192 203 instead of 159, of 128 105 instead of 98.)
  const int group = (id >> 3) % (GROUPS / 2) * 2 + (id & 1), first = (id >> 3) / (GROUPS / 2) * 4 + ((id >> 1) & 3);
  constexpr int STEP = Form::PRODUCERS / GROUPS;                  // its keys: first + j * STEP of a tile, below its 64
  const int* table = a.block_tables + static_cast<long long>(seq) * a.max_blocks;
  const uint32_t signs = kv4_signs();
  int rows[PER];                  // of the tile that is copied next; what no row sees is row 0, and masked below
  const auto find = [&](int i) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int key = (kt_first + i) * kKeysPerTile + first + j * STEP;
      rows[j] = 0;
      if (i >= n_tiles || first + j * STEP >= kKeysPerTile || key < lo || key > hi) continue;
      const int idx = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
      const int page = idx < a.max_blocks ? table[idx] : -1;
      if (page < 0 || page >= a.pages) *reinterpret_cast<volatile int*>(a.status) = kStatusBadPage;
      else rows[j] = (page * a.kv_heads + kvh - idx) * a.page_size + key;
    }
  };
  const auto copy = [&](int i) {
    if (i < n_tiles) {
      const uint32_t dst = smem_u32(raw + (i % Form::AHEAD) * RAW);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (first + j * STEP >= kKeysPerTile) break;
        const long long at = static_cast<long long>(rows[j]) * GROUPS + group;
        const uint32_t codes = dst + (j * Form::PRODUCERS + id) * 16, words = dst + PER * Form::PRODUCERS * 32 + (j * Form::PRODUCERS + id) * 8;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(codes), "l"(a.k_codes + at * 16) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(codes + PER * Form::PRODUCERS * 16), "l"(a.v_codes + at * 16) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(words), "l"(a.k_words + (at & ~1LL)) : "memory");          // two groups' words
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(words + 4), "l"(a.v_words + (at & ~1LL)) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const auto put = [&](auto big, uint8_t* plane, int row, const uint4& codes, uint32_t words) {
    constexpr bool BIG = decltype(big)::value;
    const Kv4Scale s = kv4_scale<BIG>(__byte_perm(words, 0, (group & 1) ? 0x3232 : 0x1010), signs);
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    uint8_t* dst = plane + (group >> 1) * (64 * 128) + row * 128;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t next = w[c] >> 8;
      *reinterpret_cast<uint4*>(dst + ((((group & 1) * 4 + c) ^ (row & 7)) << 4)) =
          make_uint4(kv4_low<BIG>(w[c], s), kv4_high<BIG>(w[c], s), kv4_low<BIG>(next, s), kv4_high<BIG>(next, s));
    }
  };
  const auto filled = [&](uint64_t* bar) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if ((id & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
  };
  find(0);
#pragma unroll 1
  for (int i = 0; i < Form::AHEAD; ++i) {
    copy(i);
    find(i + 1);
  }
  // Tiles from i on; true where the usual form met steps that need a product more (kv4.cuh), and from there on all tiles are taken apart that way. (So
  // the usual form stays one run of instructions: 4 portions of 512 queries at 2,048 keys, 32 heads over 8 of 128, 90.7 us; with a branch a tile 94, a branch a
  // word 102, without looking 89.)
  int i = 0;
  const auto walk = [&](auto form) {
    constexpr bool BIG = decltype(form)::value;
#pragma unroll 1
    for (; i < n_tiles; ++i) {
      const int st = i % STAGES;
      asm volatile("cp.async.wait_group %0;" ::"n"(Form::AHEAD - 1) : "memory");
      const uint8_t* src = raw + (i % Form::AHEAD) * RAW;
      uint4 kc[PER], vc[PER];
      uint2 words[PER];
      uint32_t found = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int key = (kt_first + i) * kKeysPerTile + first + j * STEP;
        if (first + j * STEP >= kKeysPerTile) break;
        kc[j] = *reinterpret_cast<const uint4*>(src + (j * Form::PRODUCERS + id) * 16);
        vc[j] = *reinterpret_cast<const uint4*>(src + ((PER + j) * Form::PRODUCERS + id) * 16);
        words[j] = *reinterpret_cast<const uint2*>(src + PER * Form::PRODUCERS * 32 + (j * Form::PRODUCERS + id) * 8);
        if (key < lo || key > hi) words[j] = make_uint2(0u, 0u);       // what no row sees: zeros
        found |= kv4_big(words[j].x) | kv4_big(words[j].y);
      }
      if (!BIG && __any_sync(0xffffffffu, (found & kKv4BigBits) != 0)) return true;
      copy(i + Form::AHEAD);          // (this thread's own place, whose words it holds)
      find(i + Form::AHEAD + 1);
      uint8_t* k_plane = ring + st * 2 * PLANE_BYTES;
      if (!__all_sync(0xffffffffu, mbar_wait(kv_empty + st, ((i / STAGES) & 1) ^ 1, abort_flag, a.status, 11) ? 1 : 0)) return false;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (first + j * STEP >= kKeysPerTile) break;
        put(form, k_plane, first + j * STEP, kc[j], words[j].x);
        if (Form::RINGS == 1) put(form, k_plane + PLANE_BYTES, first + j * STEP, vc[j], words[j].y);
      }
      if constexpr (Form::RINGS == 2) {
        filled(kv_full + st);
        if (!__all_sync(0xffffffffu, mbar_wait(kv_empty + STAGES + st, ((i / STAGES) & 1) ^ 1, abort_flag, a.status, 11) ? 1 : 0)) return false;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (first + j * STEP >= kKeysPerTile) break;
          put(form, k_plane + PLANE_BYTES, first + j * STEP, vc[j], words[j].y);
        }
      }
      filled(kv_full + (Form::RINGS - 1) * STAGES + st);
    }
    return false;
  };
  if (walk(std::false_type{})) walk(std::true_type{});
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename Form>
__global__ void __launch_bounds__(Form::THREADS, 1)
attn_prompt_umma_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, UmmaPromptArgs a) {
  pdl_sync();
  constexpr int DH = Form::DH, STAGES = Form::STAGES, RINGS = Form::RINGS, RT = Form::RT, TERMS = Form::TERMS;
  constexpr bool KV4 = Form::KV4, F32 = Form::F32, P_TMEM = Form::P_TMEM;
  constexpr int HALVES = DH / 64, P_BYTES = Form::P_BYTES, STAGE_BYTES = Form::STAGE_BYTES;
  constexpr int PLANE_BYTES = STAGE_BYTES / 2;    // 64 keys
  // columns: the row tiles' scores, their Q (two elements a column, a term behind the other), their accumulators; of one row tile the
  // accumulator first
  constexpr int S_COL = RT == 1 ? DH : 0, Q_COL = S_COL + 64 * RT, O_COL = RT == 1 ? 0 : Q_COL + RT * Form::Q_COLS;
  constexpr int P_COL = RT * (64 + Form::Q_COLS + DH), P_BUFS = Form::P_BUFS, Q_COLS = Form::Q_COLS;      // P_TMEM: [row tile][buffer][term]
  constexpr bool Q_HALF = Form::Q_HALF;
  constexpr uint32_t TMEM_COLS = 512;
  static_assert(64 * RT + RT * Form::Q_COLS + RT * DH <= 512, "tensor memory");
  constexpr float kRescaleStep = 8.0f;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);      // (an offset, so that the compiler still sees shared memory)
  uint8_t* p_smem = smem;                 // [row tile][buffer][term]; Q_HALF: dimensions 64.. of Q, [row tile]
  uint8_t* ring = p_smem + Form::P_ALL;
  uint8_t* raw = ring + STAGES * STAGE_BYTES;      // KV4: codes and words on their way
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(raw + (KV4 ? Form::AHEAD * Form::RAW : 0));
  uint64_t* kv_empty = kv_full + RINGS * STAGES;
  uint64_t* s_full = kv_empty + RINGS * STAGES;   // [2]
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_empty + 2;         // [row tile][buffer]
  uint64_t* p_empty = p_full + 4;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(p_empty + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.z / a.splits, rank = blockIdx.z % a.splits, kvh = blockIdx.x;
  const int G = a.q_heads / a.kv_heads;
  const int t0 = a.query_start[seq];
  const int nq = a.query_start[seq + 1] - t0;
  const int rows = (KV4 ? min(nq, a.max_queries) : nq) * G;
  const int row0 = (static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y)) * a.cta_rows;   // last rows (most keys) first
  if (row0 >= rows || (KV4 && t0 < 0)) return;
  const int pos0 = a.context_lens[seq] - nq;

  // key tiles each row tile needs: first[q]..last[q]; the CTA walks first[0]..last[1] (or last[0])
  bool has[2];
  int first[2], last[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r0 = row0 + 128 * q;
    has[q] = r0 < rows && 128 * q < a.cta_rows;
    const int lo_pos = pos0 + r0 / G, hi_pos = pos0 + min(rows - 1, r0 + 127) / G;
    first[q] = a.window > 0 ? max(0, lo_pos - a.window + 1) / kKeysPerTile : 0;
    last[q] = (KV4 ? max(hi_pos, 0) : hi_pos) / kKeysPerTile;
  }
  int kt_first = first[0], kt_last = has[1] ? last[1] : last[0];
  if (a.splits > 1) {             // this CTA's share of the key tiles
    const int per = (kt_last - kt_first + a.splits) / a.splits;
    kt_first += rank * per;
    kt_last = min(kt_last, kt_first + per - 1);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      first[q] = max(first[q], kt_first);
      last[q] = min(last[q], kt_last);
      has[q] = has[q] && first[q] <= last[q];
    }
  }
  const int n_tiles = kt_last - kt_first + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < RINGS * STAGES; ++s) {
      mbar_init(kv_full + s, KV4 ? Form::PRODUCERS / 32 : 1);
      mbar_init(kv_empty + s, 1);
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(s_full + q, 1);
      mbar_init(s_empty + q, 4);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(p_full + b, 4);
      mbar_init(p_empty + b, 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_holder;
  if (warp < 4 * RT) {
    // Q: every softmax thread puts its own row into tensor memory (rows beyond the sequence: zeros)
    const int q = warp >> 2, rr = (warp & 3) * 32 + lane;
    const int row = row0 + 128 * q + rr;
    const int head_dim = KV4 ? a.head_dim : DH;
    const bool there = row < rows && (!KV4 || t0 + row / G < a.tokens);
    const long long at = there ? static_cast<long long>(t0 + row / G) * a.q_stride + static_cast<long long>(kvh * G + row % G) * head_dim : 0;
    const uint32_t q_tmem = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + Q_COL + q * Q_COLS;
#pragma unroll
    for (int c0 = 0; c0 < DH / 2; c0 += 16) {
      uint32_t w[TERMS][16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool some = there && (!KV4 || 2 * c0 + 8 * e < head_dim);
        if constexpr (F32) {
          float x[8] = {};
          if (some) load4(reinterpret_cast<const float*>(a.q) + at + 2 * c0 + 8 * e, reinterpret_cast<float(&)[4]>(x[0])),
                    load4(reinterpret_cast<const float*>(a.q) + at + 2 * c0 + 8 * e + 4, reinterpret_cast<float(&)[4]>(x[4]));
#pragma unroll
          for (int y = 0; y < 4; ++y) {             // dimensions 0 4 1 5 2 6 3 7
            uint32_t terms[TERMS];
            split_terms<TERMS>(x[y], x[y + 4], terms);
#pragma unroll
            for (int term = 0; term < TERMS; ++term) w[term][4 * e + y] = terms[term];
          }
        } else {
          const uint4 v = some ? reinterpret_cast<const uint4*>(a.q + at)[c0 / 4 + e] : make_uint4(0u, 0u, 0u, 0u);
          if constexpr (KV4) {        // dimensions 0 4 1 5 2 6 3 7
            w[0][4 * e] = __byte_perm(v.x, v.z, 0x5410), w[0][4 * e + 1] = __byte_perm(v.x, v.z, 0x7632);
            w[0][4 * e + 2] = __byte_perm(v.y, v.w, 0x5410), w[0][4 * e + 3] = __byte_perm(v.y, v.w, 0x7632);
          } else {
            w[0][4 * e] = v.x, w[0][4 * e + 1] = v.y, w[0][4 * e + 2] = v.z, w[0][4 * e + 3] = v.w;
          }
        }
      }
#pragma unroll
      for (int term = 0; term < TERMS; ++term) {
        if (Q_HALF && c0 >= DH / 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(p_smem + q * P_BYTES + rr * 128 + (((c0 - DH / 4) / 4 + e) ^ (rr & 7)) * 16) = make_uint4(w[0][4 * e], w[0][4 * e + 1], w[0][4 * e + 2], w[0][4 * e + 3]);
        } else {
          tmem_st16(q_tmem + term * (DH / 2) + c0, w[term]);
        }
      }
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    if (Q_HALF) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");

  if (KV4 && warp != 9 && warp >= 4 * RT) {
    const int hi = pos0 + min(rows - 1, row0 + a.cta_rows - 1) / G, lo = a.window > 0 ? max(0, pos0 + row0 / G - a.window + 1) : 0;
    kv4_produce<Form>(a, ring, raw, kv_full, kv_empty, abort_flag, (warp - 4 * RT - (warp > 9 ? 1 : 0)) * 32 + lane, seq, kvh, kt_first, n_tiles, lo, hi);
  } else if (!KV4 && warp == 8) {
    // ---- producer
    const int box_rows = min(a.page_size, kKeysPerTile);
    const int boxes_per_tile = kKeysPerTile / box_rows;
    const int* table = a.block_tables + static_cast<long long>(seq) * a.max_blocks;
    for (int i = 0; i < n_tiles; ++i) {
      const int s = i % STAGES;
      int ok = 1;
      if (lane == 0) {
        ok = mbar_wait(kv_empty + s, ((i / STAGES) & 1) ^ 1, abort_flag, a.status, 11) ? 1 : 0;
        if (ok) mbar_expect_tx(kv_full + s, STAGE_BYTES);
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      if (lane < boxes_per_tile) {
        const int key = (kt_first + i) * kKeysPerTile + lane * box_rows;
        const int idx = key >> a.page_shift;
        const int page = idx < a.max_blocks ? table[idx] : 0;   // beyond the table: any real page; those keys are masked
        const int row = (page * a.kv_heads + kvh) * a.page_size + (key & (a.page_size - 1));
        uint8_t* kdst = ring + s * STAGE_BYTES + lane * box_rows * 128;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          tma_load_2d(kdst + h * (64 * 128), &k_map, h * 64, row, kv_full + s);
          tma_load_2d(kdst + PLANE_BYTES + h * (64 * 128), &v_map, h * 64, row, kv_full + s);
        }
      }
    }
  } else if (warp == 9) {
    // ---- MMA issuer: the whole warp walks the loop (uniform), one elected lane issues
    {
      constexpr uint32_t idesc_qk = instr_desc(kKeysPerTile);          // 128 x 64, both operands k-major
      constexpr uint32_t idesc_pv = instr_desc(DH) | (1u << 16);       // 128 x DH, B (= V) with its N extent contiguous
      // Descriptors as (low word, constant high word): one thread issues every MMA, so what it computes
      // per MMA is on the critical path of the tensor cores.
      const uint32_t k_lo0 = desc_lo_sw128(smem_u32(ring));
      const uint32_t v_lo0 = desc_lo_sw128(smem_u32(ring + PLANE_BYTES), 64 * 128);   // blocks of 64 head-dim columns lie 64 rows apart
      const uint32_t p_lo0 = desc_lo_sw128(smem_u32(p_smem));
      int n_qk[2] = {0, 0}, n_pv[2] = {0, 0};
      bool ok = true;
      const auto on = [&](int q, int i) { return has[q] && i >= 0 && i < n_tiles && kt_first + i >= first[q] && kt_first + i <= last[q]; };
      const auto qk = [&](int q, int i) {
        const uint32_t k_lo = k_lo0 + (i % STAGES) * (STAGE_BYTES >> 4);
        if (elect_one()) {
#pragma unroll
          for (int term = TERMS - 1; term >= 0; --term) {
#pragma unroll
            for (int ks = 0; ks < DH / 16; ++ks) {
              const uint64_t k_desc = desc_from_words(k_lo + (((ks >> 2) * (64 * 128) + (ks & 3) * 32) >> 4), kDescHiSw128);
              const uint32_t add = ks > 0 || term < TERMS - 1 ? 1u : 0u;
              if (Q_HALF && ks >= 4) umma_bf16(tmem_base + S_COL + q * kKeysPerTile, desc_from_words(p_lo0 + ((q * P_BYTES + (ks & 3) * 32) >> 4), kDescHiSw128), k_desc, idesc_qk, add);
              else umma_bf16_a_tmem(tmem_base + S_COL + q * kKeysPerTile, tmem_base + Q_COL + q * Q_COLS + term * (DH / 2) + ks * 8, k_desc, idesc_qk, add);
            }
          }
          umma_commit(s_full + q);
        }
        __syncwarp();
        ++n_qk[q];
      };
      const auto pv = [&](int q, int i) {
        const uint32_t v_lo = v_lo0 + (i % STAGES) * (STAGE_BYTES >> 4);
        const int pb = 2 * q + n_pv[q] % P_BUFS;
        const uint32_t p_lo = p_lo0 + pb * (TERMS * P_BYTES >> 4);
        const uint32_t keep = n_pv[q] > 0 ? 1u : 0u;
        if (elect_one()) {
#pragma unroll
          for (int term = TERMS - 1; term >= 0; --term) {
#pragma unroll
            for (int kk = 0; kk < kKeysPerTile / 16; ++kk) {
              const uint64_t v_desc = desc_from_words(v_lo + ((kk * 16 * 128) >> 4), kDescHiSw128);
              const uint32_t add = kk > 0 || term < TERMS - 1 ? 1u : keep;
              if constexpr (P_TMEM) umma_bf16_a_tmem(tmem_base + O_COL + q * DH, tmem_base + P_COL + ((q * P_BUFS + n_pv[q] % P_BUFS) * TERMS + term) * 32 + kk * 8, v_desc, idesc_pv, add);
              else umma_bf16(tmem_base + O_COL + q * DH, desc_from_words(p_lo + ((term * P_BYTES + kk * 32) >> 4), kDescHiSw128), v_desc, idesc_pv, add);
            }
          }
          umma_commit(p_empty + pb);
        }
        __syncwarp();
        ++n_pv[q];
      };
      // Step i, for row tile 0 and then for row tile 1: P V of key tile i - 1, once the softmax has written its weights, and Q K^T of key tile
      // i + 1, once it has taken the scores of tile i, which happens right behind that. The row tiles have waits of their own, so one's products
      // run while the other's softmax does: 8,192 tokens of 32 heads over 8 of 128 545 us (517 now), 649 with one wait for both row tiles' scores and one for
      // their weights. A wait costs this one thread a couple of hundred cycles even when the barrier has long flipped, so a row tile's are
      // one (two: 606 us); but where a few stages are filled by warps, P V and the stage's release come first (KV4, 4 portions of 512 at 2,048
      // keys: heads of 128 88 us against 96, of 256 210 against 271; not of 192, 163 against 159).
      constexpr bool TOGETHER = !KV4 || (DH == 64 && RT == 2) || DH == 192;
      const BarrierPhase none{nullptr, 0u, false};
      const auto wait = [&](const BarrierPhase& w0, const BarrierPhase& w1, const BarrierPhase& w2) {
        if (!w0.on && !w1.on && !w2.on) return;
        ok = __all_sync(0xffffffffu, mbar_wait_all(w0, w1, w2, abort_flag, a.status, 12) ? 1 : 0) != 0;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      };
      for (int i = -1; i <= n_tiles && ok; ++i) {
#pragma unroll
        for (int q = 0; q < RT; ++q) {
          const bool next = on(q, i + 1), last_one = on(q, i - 1);
          const BarrierPhase keys{kv_full + (i + 1) % STAGES, static_cast<uint32_t>(((i + 1) / STAGES) & 1), q == 0 && i + 1 < n_tiles};
          const BarrierPhase taken{s_empty + q, static_cast<uint32_t>((n_qk[q] & 1) ^ 1), next};
          const BarrierPhase weights{p_full + 2 * q + n_pv[q] % P_BUFS, static_cast<uint32_t>(n_pv[q] / P_BUFS & 1), last_one};
          const BarrierPhase values{kv_full + STAGES + (i + STAGES - 1) % STAGES, static_cast<uint32_t>(((i - 1) / STAGES) & 1), RINGS == 2 && q == 0 && i >= 1};
          if (TOGETHER) wait(keys, taken, weights);
          else wait(weights, values, none);
          if (!ok) break;
          if (RINGS == 2 && TOGETHER) wait(values, none, none);
          if (!ok) break;
          if (last_one) pv(q, i - 1);
          if (q == RT - 1 && i >= 1) {        // all row tiles are done with the values of key tile i - 1 (and with its keys)
            if (elect_one()) umma_commit(kv_empty + (RINGS - 1) * STAGES + (i - 1) % STAGES);
            __syncwarp();
          }
          if (!TOGETHER) wait(keys, taken, none);
          if (!ok) break;
          if (next) qk(q, i + 1);
          if (RINGS == 2 && q == RT - 1 && i + 1 < n_tiles) {      // with the keys of i + 1
            if (elect_one()) umma_commit(kv_empty + (i + 1) % STAGES);
            __syncwarp();
          }
        }
      }
    }
  } else {
    // ---- softmax: warps 0-3 own tile 0, warps 4-7 tile 1; thread = row
    const int q = warp >> 2, wq = warp & 3;
    const int rr = wq * 32 + lane;                           // row inside the tile = lane of tensor memory
    const int row = row0 + 128 * q + rr;
    // Rows beyond the sequence (their queries are zeros, nothing of them is written) see what its last one sees: with no key at all they would
    // take the whole warp through the masks in every tile (portions of 512, 512, 512 and 2 tokens at 8,192 keys 344 us instead of 173).
    const int pos = pos0 + min(row, rows - 1) / G;
    const uint32_t lane_base = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t s_tmem = tmem_base + lane_base + S_COL + q * kKeysPerTile;
    const uint32_t o_tmem = tmem_base + lane_base + O_COL + q * DH;
    uint8_t* p_rows = p_smem + 2 * q * TERMS * P_BYTES + rr * 128;
    float m_run = -INFINITY, m_used = -INFINITY, l = 0.0f;
    bool ok = has[q];
    const int my_tiles = has[q] ? last[q] - first[q] + 1 : 0;
    for (int n = 0; n < my_tiles && ok; ++n) {
      const int key0 = (first[q] + n) * kKeysPerTile;
      ok = __all_sync(0xffffffffu, mbar_wait(s_full + q, n & 1, abort_flag, a.status, 13) ? 1 : 0) != 0;
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      uint32_t sr[64];
      {
        uint32_t c0[16], c1[16], c2[16], c3[16];
        tmem_ld16(s_tmem, c0);
        tmem_ld16(s_tmem + 16, c1);
        tmem_ld16(s_tmem + 32, c2);
        tmem_ld16(s_tmem + 48, c3);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          sr[e] = c0[e];
          sr[16 + e] = c1[e];
          sr[32 + e] = c2[e];
          sr[48 + e] = c3[e];
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(s_empty + q)) : "memory");

      const bool full_tile = key0 + 63 <= pos && (a.window <= 0 || key0 > pos - a.window);
      if (!full_tile) {
#pragma unroll
        for (int c = 0; c < 64; ++c) {
          const int key = key0 + c;
          const bool seen = key <= pos && (a.window <= 0 || key > pos - a.window);
          sr[c] = seen ? sr[c] : 0xff800000u;   // -inf
        }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) mx4[e] = fmaxf(mx4[e], __uint_as_float(sr[c + e]));
      }
      m_run = fmaxf(m_run, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2);
      const bool need = m_run > m_used + kRescaleStep;       // also: the first finite maximum of the row
      if (__any_sync(0xffffffffu, need)) {
        float f = 1.0f;
        if (need) {
          f = m_used == -INFINITY ? 1.0f : ex2(m_used - m_run);
          m_used = m_run;
          l *= f;
        }
        if (n > 0) {
          // O may be touched once P V of the tile before has retired
          ok = __all_sync(0xffffffffu, mbar_wait(p_empty + 2 * q + (n - 1) % P_BUFS, (n - 1) / P_BUFS & 1, abort_flag, a.status, 13) ? 1 : 0) != 0;
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
          for (int c0 = 0; c0 < DH; c0 += 16) {
            uint32_t o[16];
            tmem_ld16(o_tmem + c0, o);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(o_tmem + c0, o);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
      }
      const float base = m_used == -INFINITY ? 0.0f : KV4 ? m_used - kKv4WeightShift : m_used;
      float sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      // this buffer held P of the tile before the last one (of the last one where there is one buffer): its P V has to have retired
      const int pb = 2 * q + n % P_BUFS;
      uint8_t* p_row = p_rows + (n & 1) * TERMS * P_BYTES;
      const uint32_t p_tmem = tmem_base + lane_base + P_COL + (q * P_BUFS + n % P_BUFS) * TERMS * 32;
      if constexpr (F32) {
        ok = __all_sync(0xffffffffu, mbar_wait(p_empty + pb, (n / P_BUFS & 1) ^ 1, abort_flag, a.status, 13) ? 1 : 0) != 0;
        if (!ok) break;
        if constexpr (P_TMEM) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t w[TERMS][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = ex2(fmaf(__uint_as_float(sr[8 * c + 2 * e]), a.scale_log2, -base));
            const float p1 = ex2(fmaf(__uint_as_float(sr[8 * c + 2 * e + 1]), a.scale_log2, -base));
            sum4[e] += p0 + p1;
            uint32_t terms[TERMS];
            split_terms<TERMS>(p0, p1, terms);
#pragma unroll
            for (int term = 0; term < TERMS; ++term) w[term][e] = terms[term];
          }
#pragma unroll
          for (int term = 0; term < TERMS; ++term) {
            if constexpr (P_TMEM) tmem_st4(p_tmem + term * 32 + 4 * c, w[term]);
            else *reinterpret_cast<uint4*>(p_row + term * P_BYTES + ((c ^ (rr & 7)) << 4)) = make_uint4(w[term][0], w[term][1], w[term][2], w[term][3]);
          }
        }
      } else {
        // two scores an instruction (1,024 queries at 4,096 keys, 32 heads over 8 of 128: 81 us instead of 87, in 4 bits 93 instead of 95)
        const Pair scale2 = pair(a.scale_log2, a.scale_log2), base2 = pair(-base, -base);
        Pair sums[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const Pair x = fma_pair(pair(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), scale2, base2);
          const float p0 = ex2(low_of(x)), p1 = ex2(high_of(x));
          sums[(c >> 1) & 1] = add_pair(sums[(c >> 1) & 1], pair(p0, p1));
          sr[c >> 1] = pack_bf16(p0, p1);
        }
        sums[0] = add_pair(sums[0], sums[1]);
        sum4[0] = low_of(sums[0]), sum4[1] = high_of(sums[0]);
        ok = __all_sync(0xffffffffu, mbar_wait(p_empty + pb, (n / P_BUFS & 1) ^ 1, abort_flag, a.status, 13) ? 1 : 0) != 0;
        if (!ok) break;
        if constexpr (P_TMEM) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          uint32_t w0[16], w1[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w0[e] = sr[e], w1[e] = sr[16 + e];
          tmem_st16(p_tmem, w0);
          tmem_st16(p_tmem + 16, w1);
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(p_row + ((c ^ (rr & 7)) << 4)) = make_uint4(sr[4 * c], sr[4 * c + 1], sr[4 * c + 2], sr[4 * c + 3]);
        }
      }
      l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
      if constexpr (P_TMEM) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      else asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(p_full + pb)) : "memory");
    }
    if (ok && my_tiles > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(p_empty + 2 * q + (my_tiles - 1) % P_BUFS, (my_tiles - 1) / P_BUFS & 1, abort_flag, a.status, 13) ? 1 : 0) != 0;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    const bool mine = ok && my_tiles > 0;
    if (a.splits > 1) {
      // The CTAs of the cluster leave their sums, references and row sums in shared memory (once neither row tile's products read there any
      // more); every CTA puts together a slice of the columns of all rows.
      float* const sums = reinterpret_cast<float*>(smem) + (128 * q + rr) * (DH + 4);
      asm volatile("bar.sync 1, %0;" ::"n"(128 * RT) : "memory");
      if (mine) {
#pragma unroll 1
        for (int c0 = 0; c0 < DH; c0 += 16) {
          uint32_t o[16];
          tmem_ld16(o_tmem + c0, o);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int e = 0; e < 16; e += 4) *reinterpret_cast<uint4*>(sums + c0 + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      sums[DH] = mine ? m_used : -INFINITY;
      sums[DH + 1] = mine ? l : 0.0f;
    } else if (mine) {
      const float inv = KV4 ? (l == 0.0f ? 0.0f : kKv4Unscale / l) : l > 0.0f ? 1.0f / l : 0.0f;
      const int head_dim = KV4 ? a.head_dim : DH;
      const bool there = row < rows && (!KV4 || t0 + row / G < a.tokens);
      const long long at = there ? (static_cast<long long>(t0 + row / G) * a.q_heads + kvh * G + row % G) * head_dim : 0;
#pragma unroll 1
      for (int c0 = 0; c0 < DH; c0 += 16) {
        uint32_t o[16];
        tmem_ld16(o_tmem + c0, o);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int h = 0; h < 16; h += 8) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[h + (KV4 ? ordered(e) : e)]) * inv;
          if (there && (!KV4 || c0 + h < head_dim)) store8<F32>(a.out, at + c0 + h, v);
        }
      }
    }
  }
  if (a.splits > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp < 4 * RT) {
      const int row = row0 + threadIdx.x;
      const uint32_t here = smem_u32(reinterpret_cast<float*>(smem) + threadIdx.x * (DH + 4));
      auto peer = [&](int r, int column) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(here + column * 4), "r"(r));
        return at;
      };
      // A share that met no key of the row (reference -inf, row sum 0) is left out; every other one counts, whatever its factor: a share
      // whose scores were NaN has the reference -inf too, but a NaN row sum, and one with a NaN among its values may have a factor
      // that came to zero. Both leave NaN, as without shares.
      float top = -INFINITY, f[kUmmaMaxSplits], l[kUmmaMaxSplits], total = 0.0f;
#pragma unroll
      for (int r = 0; r < kUmmaMaxSplits; ++r) {
        f[r] = -INFINITY, l[r] = 0.0f;
        if (r < a.splits) {
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[r]) : "r"(peer(r, DH)));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(l[r]) : "r"(peer(r, DH + 1)));
        }
        top = fmaxf(top, f[r]);
      }
      bool left_out[kUmmaMaxSplits];
#pragma unroll
      for (int r = 0; r < kUmmaMaxSplits; ++r) {
        left_out[r] = f[r] == -INFINITY && l[r] == 0.0f;
        f[r] = f[r] == -INFINITY ? l[r] : ex2(f[r] - top);      // (-inf with a row sum: that is NaN)
        if (!left_out[r]) total = fmaf(l[r], f[r], total);
      }
      const float inv = KV4 ? (total == 0.0f ? 0.0f : kKv4Unscale / total) : total > 0.0f ? 1.0f / total : 0.0f;
      const int cols = DH / a.splits;
      const int head_dim = KV4 ? a.head_dim : DH;
      if (row < rows && (!KV4 || t0 + row / G < a.tokens)) {
        const long long at = (static_cast<long long>(t0 + row / G) * a.q_heads + kvh * G + row % G) * head_dim;
        for (int c = rank * cols; c < (rank + 1) * cols; c += 8) {
          float v[8] = {};
#pragma unroll
          for (int r = 0; r < kUmmaMaxSplits; ++r) {
            if (left_out[r]) continue;      // (its sums were not written)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
              float x[4];
              asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(peer(r, c + e)));
#pragma unroll
              for (int y = 0; y < 4; ++y) v[e + y] = fmaf(x[y], f[r] * inv, v[e + y]);
            }
          }
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = v[KV4 ? ordered(e) : e];
          if (!KV4 || c < head_dim) store8<F32>(a.out, at + c, o);
        }
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");      // nobody leaves while its sums are read
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag != 0) {   // a wait ran out: let copies and MMAs that are still in flight finish before the CTA goes away
    const unsigned long long t_start = clock64();
    while (clock64() - t_start < 4000000ull) {
    }
    __syncthreads();
  }
  if (warp == 8) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

template <typename Form>
static int launch_prompt_umma(const CUtensorMap& km, const CUtensorMap& vm, const UmmaPromptArgs& a, int n_seqs, int max_rows,
                              cudaStream_t s) {
  constexpr size_t smem = Form::SMEM;
  static bool configured = false;
  if (Form::KV4 || !configured) {      // (the attribute belongs to a device: KV4 asks for it on whichever is the current one)
    if (cudaFuncSetAttribute(attn_prompt_umma_kernel<Form>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) {
      set_error("attention_prompt_umma: cannot reserve %zu bytes of shared memory", smem);
      return kCudaError;
    }
    configured = true;
  }
  const dim3 grid(a.kv_heads, ceil_div(max_rows, a.cta_rows), n_seqs * a.splits);
  if (a.splits == 1) {
    TIE_LAUNCH((attn_prompt_umma_kernel<Form>), grid, Form::THREADS, smem, s, km, vm, a);
    return kOk;
  }
  // clusters of CTAs that hold tensor memory are not started beside the kernel ahead
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(Form::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = a.splits;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, attn_prompt_umma_kernel<Form>, km, vm, a);
  return kOk;
}

// How the rows and keys of a launch are shared out over its CTAs.
static void cut_prompt_umma(UmmaPromptArgs& a, int max_queries, int n_seqs, int max_keys) {
  const int max_rows = max_queries * (a.q_heads / a.kv_heads);
  // Few rows: with two row tiles a CTA, half of the SMs or more would have none
  int sms = 148;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, 0);
  // ...; with many keys they share out the keys instead: what bounds either is the keys and values that L2 feeds the SMs, and tiles of
  // 256 rows read them half as often. 128 rows a CTA against shares, us: two shares, 512 tokens of 32 heads over 8, heads of 128: 2,100 keys
  // 35.9 / 33.8, 3,000 47.8 / 41.0, 8,192 115 / 81, 16,384 224 / 147 (at 1,024 21.7 / 24.8: the merge costs about 8 us); heads of 64 28.9 / 26.9, 38.1 / 33.3,
  // 93 / 73, 179 / 135 (17.1 / 18.8). Four shares, 128 tokens: heads of 128 2,100 keys 35.5 / 30.1, 3,000 47.0 / 33.1, 8,192 114 / 53; 16 heads of 64 over
  // 4 28.3 / 22.0, 37.3 / 25.0, 91 / 45; 8 over 8 of 128 34.4 / 22.1, 46.0 / 24.6, 113 / 42.
  const long long ctas = static_cast<long long>(a.kv_heads) * ceil_div(max_rows, 256) * n_seqs;
  const int keys = a.window > 0 && a.window + max_queries < max_keys ? a.window + max_queries : max_keys;
  if (ctas * 2 <= sms) {
    if (keys >= kUmmaSplitKeys) a.splits = ctas * 4 <= sms ? 4 : 2;
    else a.cta_rows = 128;
  }
}

// The same with KV4, by what the ways cost in tiles of 64 keys by 256 rows: the CTAs' rounds on the SMs times a CTA's tiles. Two shares of the
// keys add the time of 8 tiles to a round, four 12 (and four CTAs of a cluster find room on about 132 of the SMs); CTAs of 128 rows take 0.86 of a
// tile's time. How many CTAs have rows is estimated from all rows of the step, since portions differ. (The terms were fitted when a tile took a
// tenth to a third longer; a merge is about 11 tiles now.) What it picks, against all ways, us: portions of 512, 342, 172 and 2 tokens of 16 heads of
// 64 over 4 at 8,192 keys: one share 146, of 128 rows 137, two shares 83, four 142 (the rule: two); 512 tokens of 32 heads of 128 over 8 at 8,192 keys 158, 144,
// 93, 123 (two); 128 tokens at 4,096 keys 84, 76, 55, 41 (four); 1,024 tokens at 4,096 keys 86, 134, 102, 163 (one); eight portions of 300 to 2 tokens at
// 4,096 keys 168, 225, 164, 239 (two); 300 tokens at 300 keys 14.7, 13.0, 19.6, 39 (128 rows); 2,048 tokens at 2,048 keys 55, 94, 105, 218 (one). Forms of one
// row tile, 512 tokens at 8,192 keys, one, two and four shares: heads of 192 139, 155, 200, of 256 193, 210, 262, float of 128 184, 198, 236 (one).
static void cut_prompt_kv4(UmmaPromptArgs& a, int row_tiles, int max_queries, int n_seqs, int max_keys) {
  const long long group = a.q_heads / a.kv_heads, max_rows = max_queries * group;
  const int keys = a.window > 0 && a.window + max_queries < max_keys ? a.window + max_queries : max_keys;
  const double tiles = (keys + kKeysPerTile - 1) / kKeysPerTile;
  double best = 0.0;
  const int whole = 128 * row_tiles;      // (forms of one row tile a CTA: only shares)
  const int ways[4][3] = {{1, whole, 0}, {1, 128, 0}, {2, whole, 8}, {4, whole, 12}};
  for (int i = 0; i < 4; ++i) {
    const int splits = ways[i][0], rows = ways[i][1];
    const long long most = n_seqs * ((max_rows + rows - 1) / rows), about = (2 * a.tokens * group + (n_seqs + 1) * rows) / (2 * rows);
    const long long ctas = a.kv_heads * (most < about ? most : about) * splits, places = splits == 4 ? 132 : 148;
    const double cost = static_cast<double>((ctas + places - 1) / places) * (rows < whole ? 0.86 : 1.0) * (tiles / splits + ways[i][2]);
    if (i == 0 || cost < best) best = cost, a.splits = splits, a.cta_rows = rows;
  }
}

}  // namespace tie

using namespace tie;

// Rows [0, rows) of the step belong to sequences 0..n_seqs-1, each bringing several tokens;
// max_queries is the largest number of tokens one of them brings, max_keys the longest context of one; pages is the
// number of pages of the cache planes.
TIE_API int tie_attention_prompt_umma(const void* q, long long q_stride, const void* k_cache, const void* v_cache, void* out,
                                      const int* query_start, const int* context_lens, const int* block_tables,
                                      int max_blocks, int n_seqs, int max_queries, int q_heads, int kv_heads, int head_dim,
                                      int page_size, int pages, int window, float scale, int max_keys, cudaStream_t s) {
  TIE_REQUIRE(head_dim == 64 || head_dim == 128, "attention_prompt_umma: head_dim %d is not 64 or 128", head_dim);
  TIE_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && q_heads / kv_heads <= 16,
              "attention_prompt_umma: %d query heads over %d kv heads (at most 16 per group)", q_heads, kv_heads);
  TIE_REQUIRE(page_size >= 8 && (page_size & (page_size - 1)) == 0, "attention_prompt_umma: page size %d is not a power of two from 8 up", page_size);
  TIE_REQUIRE(q_stride % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
              "attention_prompt_umma: q and out rows must be 16-byte aligned");
  TIE_REQUIRE(scale > 0.0f, "attention_prompt_umma: the scale must be positive");
  if (n_seqs == 0 || max_queries == 0) return kOk;
  TIE_REQUIRE(static_cast<long long>(max_queries) * (q_heads / kv_heads) <= 65535LL * 256, "attention_prompt_umma: %d queries in one portion are too many", max_queries);
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  const int box_rows = page_size < kKeysPerTile ? page_size : kKeysPerTile;
  CUtensorMap km, vm;
  const long long rows = static_cast<long long>(pages) * kv_heads * page_size;
  TIE_REQUIRE(make_map_bf16(&km, k_cache, rows, head_dim, head_dim, 64, box_rows) &&
                  make_map_bf16(&vm, v_cache, rows, head_dim, head_dim, 64, box_rows),
              "attention_prompt_umma: cuTensorMapEncodeTiled failed");
  TIE_REQUIRE(status_word() != nullptr, "attention_prompt_umma: cannot allocate the status word");
  UmmaPromptArgs a{static_cast<const __nv_bfloat16*>(q), static_cast<__nv_bfloat16*>(out), query_start, context_lens, block_tables,
                   status_word(), q_stride, max_blocks, q_heads, kv_heads, page_size, shift, window, scale * 1.4426950408889634f, 1, 256};
  const int max_rows = max_queries * (q_heads / kv_heads);
  cut_prompt_umma(a, max_queries, n_seqs, max_keys);
  const int st = head_dim == 64 ? launch_prompt_umma<UmmaForm<64, false, 2, false>>(km, vm, a, n_seqs, max_rows, s)
                                : launch_prompt_umma<UmmaForm<128, false, 2, false>>(km, vm, a, n_seqs, max_rows, s);
  if (st != kOk) return st;
  TIE_RETURN_LAUNCH("attention_prompt_umma");
}

// The same over a cache in 4 bits: heads of a multiple of 8 up to 256 (float rows: 128); pages of any size; rows of q 16-byte aligned.
TIE_API int tie_attention_prompt_kv4(int dtype, const void* q, long long q_stride, long long tokens, const void* k_codes, const void* k_words,
                                     const void* v_codes, const void* v_words, void* out, const int* query_start, const int* context_lens,
                                     const int* block_tables, int max_blocks, int n_seqs, int max_queries, int q_heads, int kv_heads, int head_dim, int page_size,
                                     long long pages, int window, float scale, int max_keys, cudaStream_t s) {
  const bool f32 = dtype == TIE_F32;
  TIE_REQUIRE(head_dim > 0 && head_dim <= (f32 ? 128 : 256) && head_dim % 8 == 0, "attention_prompt_kv4: head_dim %d is not a multiple of 8 up to %d", head_dim,
              f32 ? 128 : 256);
  TIE_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0, "attention_prompt_kv4: %d query heads over %d kv heads", q_heads, kv_heads);
  TIE_REQUIRE(q_stride * (f32 ? 4 : 2) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
              "attention_prompt_kv4: q and out rows must be 16-byte aligned");
  TIE_REQUIRE(page_size > 0 && pages > 0 && pages * page_size * kv_heads < (1LL << 31) && max_blocks >= 0 && n_seqs >= 0 && n_seqs <= 16383 && max_queries >= 0,
              "attention_prompt_kv4: bad sizes (%lld pages of %d, %d sequences, %d queries)", pages, page_size, n_seqs, max_queries);
  TIE_REQUIRE(scale > 0.0f, "attention_prompt_kv4: the scale must be positive");
  if (n_seqs == 0 || max_queries == 0) return kOk;
  const long long all_rows = static_cast<long long>(max_queries) * (q_heads / kv_heads);
  TIE_REQUIRE(all_rows <= 65535LL * 128, "attention_prompt_kv4: %d queries in one portion are too many", max_queries);
  TIE_REQUIRE(status_word() != nullptr, "attention_prompt_kv4: cannot allocate the status word");
  int shift = 0;
  while (shift < 30 && (1 << shift) < page_size) ++shift;
  if ((1 << shift) != page_size) shift = -1;
  UmmaPromptArgs a{static_cast<const __nv_bfloat16*>(q), static_cast<__nv_bfloat16*>(out), query_start, context_lens, block_tables, status_word(), q_stride, max_blocks,
                   q_heads, kv_heads, page_size, shift, window, scale * 1.4426950408889634f * kKv4Unscale, 1, 256, static_cast<const uint8_t*>(k_codes),
                   static_cast<const uint8_t*>(v_codes), static_cast<const uint16_t*>(k_words), static_cast<const uint16_t*>(v_words), head_dim,
                   static_cast<int>(pages), max_queries, tokens};
  cut_prompt_kv4(a, f32 || head_dim > 128 ? 1 : 2, max_queries, n_seqs, max_keys);
  const CUtensorMap none = {};
  const int rows = static_cast<int>(all_rows);
  int st;
  if (f32) st = head_dim <= 64 ? launch_prompt_umma<UmmaForm<64, true, 1, true>>(none, none, a, n_seqs, rows, s)
                               : launch_prompt_umma<UmmaForm<128, true, 1, true>>(none, none, a, n_seqs, rows, s);
  else if (head_dim <= 64) st = launch_prompt_umma<UmmaForm<64, true, 2, false>>(none, none, a, n_seqs, rows, s);
  else if (head_dim <= 128) st = launch_prompt_umma<UmmaForm<128, true, 2, false>>(none, none, a, n_seqs, rows, s);
  else if (head_dim <= 192) st = launch_prompt_umma<UmmaForm<192, true, 1, false>>(none, none, a, n_seqs, rows, s);
  else st = launch_prompt_umma<UmmaForm<256, true, 1, false>>(none, none, a, n_seqs, rows, s);
  if (st != kOk) return st;
  TIE_RETURN_LAUNCH("attention_prompt_kv4");
}
