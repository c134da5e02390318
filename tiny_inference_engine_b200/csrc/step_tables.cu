// The index arrays of a step, built on the GPU from the requests' lengths.
//
// A request's row of `tables` names its pages, lens[request] the tokens they hold; the free pages are a stack (free_pages, free_count). A
// sequence i of the step brings counts[i] tokens of request requests[i]:
//     query_start  = prefix sums of counts;  context_lens = lens + counts
//     pages        : a request that crosses into new pages takes them from the end of the stack, in the order of the sequences and of their pages
//     positions, seq_of_row, slots of every row: lens + (row - query_start), page * page_size + position % page_size
//     block_tables : the sequences' pages side by side, zeros behind them
// What is written is 4 (3 rows + sequences * columns) bytes; the time goes to latency: the chain lengths -> prefix sums -> rows. So there is one
// kernel whose blocks each work out all prefix sums themselves (a few thousand integers from L2, one scan a block) and then fill their share of
// rows and tables: a grid-wide barrier or a second launch would cost more than the repeated scan (512 sequences: 2 us a block).
// A step that cannot be is refused whole (status != 0): nothing is taken, every slot is -1, every context 0.
// `commit`: a second small kernel writes the new lengths and the new free count, behind the first one, whose blocks all read the old ones.
#include "common.cuh"

namespace tie {

constexpr int kTableThreads = 512;
constexpr int kMaxTableSeqs = 8192;
constexpr int kMaxTableRequests = 1 << 17;
// status bits
constexpr int kNoPages = 1, kTableShort = 2, kRowsShort = 4, kBadRequest = 8;

struct TableArgs {
  const int *requests, *counts, *lens;
  int* tables;
  const int *free_pages, *free_count;
  int *query_start, *context_lens, *positions, *seq_of_row, *slots, *block_tables, *free_left, *status;
  int seqs, rows, columns, table_columns, n_requests, free_capacity, page_size;
};

// Sums before and up to this thread's value of a pair of numbers, over the block; `total` the block's. scratch: 2 * 17 long longs.
__device__ __forceinline__ void block_scan2(long long a, long long b, long long& a_before, long long& b_before, long long& a_total, long long& b_total,
                                            long long* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long x = a, y = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, x, o), w = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) x += u, y += w;
  }
  __syncthreads();      // scratch may still be read from the call before
  if (lane == 31) scratch[warp] = x, scratch[17 + warp] = y;
  __syncthreads();
  a_total = 0, b_total = 0;
  long long pa = 0, pb = 0;
  for (int i = 0; i < warps; ++i) {
    if (i == warp) pa = a_total, pb = b_total;
    a_total += scratch[i], b_total += scratch[17 + i];
  }
  a_before = pa + x - a, b_before = pb + y - b;
}

__global__ void __launch_bounds__(kTableThreads) step_tables_kernel(TableArgs t) {
  // (the kernel behind is not started early: attention kernels read tables and lengths ahead of their wait)
  pdl_wait();
  extern __shared__ int smem[];
  int* start = smem;                       // [seqs + 1] first row of a sequence
  int* held = start + t.seqs + 1;          // [seqs] tokens in the cache
  int* fresh = held + t.seqs;              // [seqs] pages that the sequences ahead take
  unsigned int* listed = reinterpret_cast<unsigned int*>(fresh + t.seqs);      // a bit a request
  __shared__ long long scratch[34];
  __shared__ int flags;
  if (threadIdx.x == 0) flags = 0;
  for (int i = threadIdx.x; i < (t.n_requests + 31) / 32; i += kTableThreads) listed[i] = 0;
  __syncthreads();
  const int free_count = *t.free_count;
  long long row = 0, taken = 0;
  int bad = free_count < 0 || free_count > t.free_capacity ? kBadRequest : 0;
  for (int i0 = 0; i0 < t.seqs; i0 += kTableThreads) {
    const int i = i0 + threadIdx.x;
    long long count = 0, pages = 0;
    int have = 0;
    if (i < t.seqs) {
      const int request = t.requests[i];
      count = t.counts[i];
      if (count < 0 || count > t.rows) bad |= count < 0 ? kBadRequest : kRowsShort, count = 0;
      if (request >= 0 && request < t.n_requests) {
        have = t.lens[request];
        const long long end = static_cast<long long>(have) + count;
        if (atomicOr(listed + request / 32, 1u << (request & 31)) >> (request & 31) & 1u) bad |= kBadRequest;
        else if (have < 0) bad |= kBadRequest, have = 0;
        else if (end > static_cast<long long>(t.columns) * t.page_size || end > 0x7fffffffLL) bad |= kTableShort;
        else pages = (end + t.page_size - 1) / t.page_size - (have + static_cast<long long>(t.page_size) - 1) / t.page_size;
      } else if (request != -1) {
        bad |= kBadRequest;
      }
    }
    long long before_rows, before_pages, all_rows, all_pages;
    block_scan2(count, pages, before_rows, before_pages, all_rows, all_pages, scratch);
    if (i < t.seqs) {
      start[i] = static_cast<int>(min(row + before_rows, 0x7fffffffLL));
      held[i] = have;
      fresh[i] = static_cast<int>(min(taken + before_pages, 0x7fffffffLL));
    }
    row += all_rows, taken += all_pages;
  }
  if (threadIdx.x == 0) start[t.seqs] = static_cast<int>(min(row, 0x7fffffffLL));
  if (row > t.rows) bad |= kRowsShort;
  if (taken > free_count) bad |= kNoPages;
  if (bad != 0) atomicOr(&flags, bad);
  __syncthreads();
  const int status = flags;
  const bool ok = status == 0;
  const int live = ok ? start[t.seqs] : 0;
  const long long threads = static_cast<long long>(gridDim.x) * kTableThreads, id = static_cast<long long>(blockIdx.x) * kTableThreads + threadIdx.x;
  if (id == 0) {
    *t.status = status;
    *t.free_left = ok ? free_count - static_cast<int>(taken) : free_count;
  }
  // page number `place` of sequence i: from the request's table, or the page that it takes now
  const auto page_of = [&](int i, int request, int place) {
    const int old = static_cast<int>((held[i] + static_cast<long long>(t.page_size) - 1) / t.page_size);
    return place < old ? t.tables[static_cast<long long>(request) * t.table_columns + place] : t.free_pages[free_count - 1 - (fresh[i] + place - old)];
  };
  for (long long i = id; i <= t.seqs; i += threads) {
    t.query_start[i] = ok ? start[i] : 0;
    if (i < t.seqs) t.context_lens[i] = ok && t.requests[i] >= 0 ? held[i] + start[i + 1] - start[i] : 0;
  }
  for (long long r = id; r < t.rows; r += threads) {
    int seq = -1, position = 0, slot = -1;
    if (r < live) {
      int lo = 0, hi = t.seqs;             // start[lo] <= r < start[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= r) lo = mid;
        else hi = mid;
      }
      seq = lo;
      const int request = t.requests[seq];
      if (request >= 0) {
        position = held[seq] + static_cast<int>(r) - start[seq];
        slot = page_of(seq, request, position / t.page_size) * t.page_size + position % t.page_size;
      }
    }
    t.positions[r] = position;
    t.seq_of_row[r] = seq;
    t.slots[r] = slot;
  }
  // A warp a table row at a time: the columns are read and written in order, and what belongs to the sequence is worked out once. The
  // request's new pages go into its own table here too; nobody else reads those entries in this launch.
  const int warps = static_cast<int>(threads >> 5), lane = threadIdx.x & 31;
  const int parts = max(1, min((t.columns + 127) / 128, warps / max(1, t.seqs)));      // warps that share a row, where there are more warps than rows
  const int per = ((t.columns + parts - 1) / parts + 3) / 4 * 4;
  for (long long job = id >> 5; job < static_cast<long long>(t.seqs) * parts; job += warps) {
    const int i = static_cast<int>(job / parts), c0 = static_cast<int>(job % parts) * per, c1 = min(t.columns, c0 + per);
    const int request = t.requests[i];
    int old = 0, now = 0;
    if (ok && request >= 0) {
      old = static_cast<int>((held[i] + static_cast<long long>(t.page_size) - 1) / t.page_size);
      now = static_cast<int>((held[i] + static_cast<long long>(start[i + 1] - start[i]) + t.page_size - 1) / t.page_size);
    }
    int* out = t.block_tables + static_cast<long long>(i) * t.columns;
    int* own = t.tables + static_cast<long long>(max(request, 0)) * t.table_columns;
    for (int c = c0 + lane; c < c1; c += 32) {
      int page = 0;
      if (c < old) {
        page = own[c];
      } else if (c < now) {
        page = t.free_pages[free_count - 1 - (fresh[i] + c - old)];
        own[c] = page;
      }
      out[c] = page;
    }
  }
}

__global__ void __launch_bounds__(256) commit_tables_kernel(const int* __restrict__ requests, const int* __restrict__ context_lens, const int* __restrict__ free_left,
                                                            const int* __restrict__ status, int* lens, int* free_count, int seqs) {
  pdl_wait();
  if (*status != 0) return;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i == 0) *free_count = *free_left;
  if (i < seqs && requests[i] >= 0) lens[requests[i]] = context_lens[i];
}

// The pages of `requests` go back: onto the end of the stack, the requests in their order, each one's pages in theirs. One block.
__global__ void __launch_bounds__(kTableThreads) release_tables_kernel(const int* __restrict__ requests, int* lens, const int* __restrict__ tables, int* free_pages,
                                                                       int* free_count, int* status, int seqs, int n_requests, int table_columns,
                                                                       int free_capacity, int page_size) {
  pdl_wait();
  extern __shared__ int smem[];
  int* fresh = smem;                       // [seqs + 1] pages of the requests ahead
  unsigned int* listed = reinterpret_cast<unsigned int*>(fresh + seqs + 1);
  __shared__ long long scratch[34];
  __shared__ int flags;
  if (threadIdx.x == 0) flags = 0;
  for (int i = threadIdx.x; i < (n_requests + 31) / 32; i += kTableThreads) listed[i] = 0;
  __syncthreads();
  const int count = *free_count;
  int bad = count < 0 || count > free_capacity ? kBadRequest : 0;
  long long pages_before = 0;
  for (int i0 = 0; i0 < seqs; i0 += kTableThreads) {
    const int i = i0 + threadIdx.x;
    long long pages = 0;
    if (i < seqs) {
      const int request = requests[i];
      if (request >= 0 && request < n_requests) {
        const int have = lens[request];
        if (atomicOr(listed + request / 32, 1u << (request & 31)) >> (request & 31) & 1u) bad |= kBadRequest;
        else if (have < 0 || have > static_cast<long long>(table_columns) * page_size) bad |= kBadRequest;
        else pages = (have + static_cast<long long>(page_size) - 1) / page_size;
      } else if (request != -1) {
        bad |= kBadRequest;
      }
    }
    long long a, b, unused, all;
    block_scan2(0, pages, a, b, unused, all, scratch);
    if (i < seqs) fresh[i] = static_cast<int>(min(pages_before + b, 0x7fffffffLL));
    pages_before += all;
  }
  if (threadIdx.x == 0) fresh[seqs] = static_cast<int>(min(pages_before, 0x7fffffffLL));
  if (count + pages_before > free_capacity) bad |= kNoPages;
  if (bad != 0) atomicOr(&flags, bad);
  __syncthreads();
  if (threadIdx.x == 0) *status = flags;
  if (flags != 0) return;
  for (int i = threadIdx.x >> 5; i < seqs; i += kTableThreads / 32) {
    const int pages = fresh[i + 1] - fresh[i];
    for (int c = threadIdx.x & 31; c < pages; c += 32)
      free_pages[count + fresh[i] + c] = tables[static_cast<long long>(requests[i]) * table_columns + c];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < seqs; i += kTableThreads)
    if (requests[i] >= 0) lens[requests[i]] = 0;
  if (threadIdx.x == 0) *free_count = count + fresh[seqs];
}

static int tables_check(const char* name, int seqs, int n_requests, int table_columns, int free_capacity, int page_size) {
  TIE_REQUIRE(seqs >= 0 && seqs <= kMaxTableSeqs, "%s: %d sequences (at most %d)", name, seqs, kMaxTableSeqs);
  TIE_REQUIRE(n_requests > 0 && n_requests <= kMaxTableRequests, "%s: %d requests (1 to %d)", name, n_requests, kMaxTableRequests);
  TIE_REQUIRE(table_columns > 0 && free_capacity > 0 && page_size > 0 && static_cast<long long>(free_capacity) * page_size < (1LL << 31),
              "%s: bad sizes (columns %d, pages %d of %d tokens)", name, table_columns, free_capacity, page_size);
  return kOk;
}

template <typename Kernel> static bool allow_smem(Kernel kernel, size_t smem) {
  return smem <= 48 * 1024 || cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) == cudaSuccess;
}

}  // namespace tie

using namespace tie;

TIE_API int tie_step_tables(const int* requests, const int* counts, int* lens, int* tables, const int* free_pages, int* free_count, int* query_start,
                            int* context_lens, int* positions, int* seq_of_row, int* slots, int* block_tables, int* free_left, int* status, int seqs, int rows,
                            int columns, int table_columns, int n_requests, int free_capacity, int page_size, int commit, cudaStream_t s) {
  if (const int bad = tables_check("step_tables", seqs, n_requests, table_columns, free_capacity, page_size)) return bad;
  TIE_REQUIRE(rows >= 0 && rows < (1 << 30) && columns > 0 && columns <= table_columns, "step_tables: bad sizes (%d rows, %d columns of %d)", rows, columns, table_columns);
  const TableArgs t{requests, counts, lens, tables, free_pages, free_count, query_start, context_lens, positions, seq_of_row, slots, block_tables, free_left, status,
                    seqs, rows, columns, table_columns, n_requests, free_capacity, page_size};
  const size_t smem = (3 * static_cast<size_t>(seqs) + 1 + (n_requests + 31) / 32) * 4;
  TIE_REQUIRE(allow_smem(step_tables_kernel, smem), "step_tables: cannot reserve %zu bytes of shared memory", smem);
  // a block for every 4,096 numbers that are written, up to one an SM
  const int blocks = static_cast<int>(min(148LL, max(1LL, (3LL * rows + static_cast<long long>(seqs) * columns + 4095) / 4096)));
  TIE_LAUNCH(step_tables_kernel, blocks, kTableThreads, smem, s, t);
  if (commit) TIE_LAUNCH(commit_tables_kernel, ceil_div(max(seqs, 1), 256), 256, 0, s, requests, context_lens, free_left, status, lens, free_count, seqs);
  TIE_RETURN_LAUNCH("step_tables");
}

TIE_API int tie_release_tables(const int* requests, int* lens, const int* tables, int* free_pages, int* free_count, int* status, int seqs, int n_requests,
                               int table_columns, int free_capacity, int page_size, cudaStream_t s) {
  if (const int bad = tables_check("release_tables", seqs, n_requests, table_columns, free_capacity, page_size)) return bad;
  const size_t smem = (static_cast<size_t>(seqs) + 1 + (n_requests + 31) / 32) * 4;
  TIE_REQUIRE(allow_smem(release_tables_kernel, smem), "release_tables: cannot reserve %zu bytes of shared memory", smem);
  TIE_LAUNCH(release_tables_kernel, 1, kTableThreads, smem, s, requests, lens, tables, free_pages, free_count, status, seqs, n_requests, table_columns,
             free_capacity, page_size);
  TIE_RETURN_LAUNCH("release_tables");
}
