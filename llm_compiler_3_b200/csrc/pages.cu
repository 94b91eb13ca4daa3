// Bookkeeping of a paged cache: page tables of the next step, compaction of a
// pool, and the copies of pages that both ask for.
//
// page_update and page_compact work on whole numbers only: tables and reference
// counts of a few thousand to a few hundred thousand words, in phases that each
// need the previous one finished everywhere.  They are bound by latency (256 rows of 96
// entries and 12000 pages: 14 us; 8192 rows of 64 and 600000 pages, 227 us, are bound by what 8
// SMs read), so one launch does it all: a single cluster of 8 CTAs, whose hardware barrier orders
// the phases (and their global writes) without flags or further launches, and
// whose distributed shared memory carries the counts of the prefix sums.  Every
// result is a count, a rank or a lowest index, so no order of atomics shows.
#include <limits.h>

#include "paged.cuh"

namespace npu_b200 {
namespace {

constexpr int kCtas = 8;
constexpr int kThreads = 1024;
constexpr int kWarpsPerCta = kThreads / 32;
constexpr int kMaxRows = 8192;
constexpr int kRowPiece = 256;  // table entries of one warp's turn
constexpr int kAtOnce = 4;      // groups of 32 pages whose counts a warp loads together
// What a copying row adds to the count of a page that others hold too, so that it is not
// free in this step, whoever gives it up: 8192 of them and a count stay below 2^31.
constexpr int kHold = 1 << 17;

// Exclusive prefix of `v` over the CTA's threads and the CTA's total.
__device__ __forceinline__ long long block_scan(long long v, long long* s_warp, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto inclusive = [&](long long x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  const long long x = inclusive(v);
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  const long long upto = inclusive(s_warp[lane]);  // every warp scans the 32 warps' sums
  *total = __shfl_sync(0xffffffffu, upto, 31);
  return x - v + (warp > 0 ? __shfl_sync(0xffffffffu, upto, warp - 1) : 0);
}

// Sum over the CTA's warps of `v`, one value per warp; in every thread.  s_warp keeps
// the warps' values.
__device__ __forceinline__ int block_sum(int v, int* s_warp) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) s_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, s_warp[lane]);
}

// Sum of the values of the warps before this one.
__device__ __forceinline__ int warps_before(const int* s_warp) {
  const int lane = threadIdx.x & 31;
  return __reduce_add_sync(0xffffffffu, lane < static_cast<int>(threadIdx.x >> 5) ? s_warp[lane] : 0);
}

// Every CTA's `mine` into s_all[kCtas] of every CTA (needs a cluster barrier
// before it is read, and one before the kernel's first call: all CTAs have started).
__device__ __forceinline__ void cluster_share(int mine, int* s_all) {
  if (threadIdx.x < kCtas) {
    const uint32_t to = cluster_map(smem_u32(s_all + cluster_ctarank()), threadIdx.x);
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(mine) : "memory");
  }
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

__device__ __forceinline__ int ld_fresh(const int32_t* p) { return __ldcg(p); }

// The pages of warp w of the cluster: a contiguous stretch, so that ranks follow
// from one count per warp.
struct Stretch {
  int begin, end;
  __device__ __forceinline__ Stretch(int count) {
    const int warps = kCtas * kWarpsPerCta;
    const int each = ((count + warps - 1) / warps + 31) & ~31;
    const int w = cluster_ctarank() * kWarpsPerCta + (threadIdx.x >> 5);
    begin = static_cast<int>(min(static_cast<long long>(w) * each, static_cast<long long>(count)));
    end = static_cast<int>(min(static_cast<long long>(begin) + each, static_cast<long long>(count)));
  }
};

struct UpdateParams {
  const int32_t *table, *lens, *parents, *capacity, *refs;
  int32_t *new_table, *new_lens, *new_refs, *copies, *info;
  int rows, new_rows, entries, page_size, num_pages;
  Divisor by_page;
};

// One new row, in shared memory: what it keeps of its parent.
struct Row {
  int parent;  // or -1
  int len;     // tokens
  int last;    // the partly filled page, or -1
  int need;    // fresh pages of the rows before
  int copy;    // 2 x the copying rows before, + 1 if this one copies its last page
};

// Grid: one cluster.  Phases, a cluster barrier after each of the first three:
//   1. new_refs = refs; every CTA lays out the rows' needs in its shared memory
//   2. the old rows' holds leave new_refs, the shared pages' enter; entries kept
//      are written, the others cleared
//   3. free pages are counted per warp
//   4. the k-th free page goes to the k-th need
// and, if a page that others hold too is copied, a fifth that lets go of it.
__global__ void __launch_bounds__(kThreads) page_update_kernel(const UpdateParams p) {
  extern __shared__ int32_t smem_i[];
  int32_t* first = smem_i;                             // [rows] lowest new row of each old one
  Row* row = reinterpret_cast<Row*>(first + p.rows);   // [new_rows]
  __shared__ long long s_scan[kWarpsPerCta];
  __shared__ int s_sum[kWarpsPerCta], s_free[kCtas];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster_ctarank());
  const int all_threads = kCtas * kThreads, me = rank * kThreads + tid;
  const int reach = p.entries * p.page_size;
  pdl_launch_dependents();
  pdl_wait();

#pragma unroll 4
  for (int i = me; i < p.num_pages; i += all_threads) p.new_refs[i] = p.refs[i];
  cluster_arrive();  // the counts are waited for once the rows are laid out
  for (int r = tid; r < p.rows; r += kThreads) first[r] = INT_MAX;
  __syncthreads();
  const int each = (p.new_rows + kThreads - 1) / kThreads;
  const int b0 = min(tid * each, p.new_rows), b1 = min(b0 + each, p.new_rows);
  int held = 0;  // a page to copy is held elsewhere
  for (int b = b0; b < b1; ++b) {
    Row r;
    r.parent = p.parents[b];
    const int cap = min(max(p.capacity[b], 0), reach);
    r.len = 0;
    r.last = -1;
    r.copy = 0;
    if (r.parent >= 0 && r.parent < p.rows) {
      atomicMin(&first[r.parent], b);
      r.len = min(max(p.lens[r.parent], 0), reach);
    } else {
      r.parent = -1;
    }
    const int full = p.by_page.quotient(r.len), part = r.len - full * p.page_size;
    if (part > 0) {
      r.last = p.table[static_cast<size_t>(r.parent) * p.entries + full];
      if (r.last >= 0 && r.last < p.num_pages)
        held |= r.copy = p.refs[r.last] != 1;
      else
        r.last = -1;
    }
    r.need = p.by_page.quotient(max(cap, r.len) + p.page_size - 1) - full - (part > 0);
    row[b] = r;
  }
  const bool holds = __syncthreads_or(held);  // the same in every CTA
  long long mine = 0;  // needs, and copying rows in the upper half
  for (int b = b0; b < b1; ++b) {
    Row& r = row[b];
    if (r.last >= 0 && first[r.parent] != b) r.copy = 1;
    r.need += r.copy;
    mine += static_cast<long long>(r.copy) << 32 | r.need;
  }
  long long total, at_row = block_scan(mine, s_scan, &total);
  for (int b = b0; b < b1; ++b) {
    Row& r = row[b];
    const long long n = static_cast<long long>(r.copy) << 32 | r.need;
    r.need = static_cast<int>(at_row & 0xffffffffll);
    r.copy |= static_cast<int>(at_row >> 32) * 2;
    at_row += n;
  }
  const int wanted = static_cast<int>(total & 0xffffffffll);
  __syncthreads();
  cluster_wait();

  // One warp per piece of a row, so that few long rows spread over the cluster too.
  const long long pieces = (p.entries + kRowPiece - 1) / kRowPiece;
  const long long warps = kCtas * kWarpsPerCta, my_warp = rank * kWarpsPerCta + warp;
  for (long long w = my_warp; w < p.rows * pieces; w += warps) {
    const int r = static_cast<int>(pieces == 1 ? w : w / pieces);
    const int e0 = static_cast<int>(w - r * pieces) * kRowPiece;
#pragma unroll 4
    for (int e = e0 + lane; e < min(e0 + kRowPiece, p.entries); e += 32) {
      const int page = p.table[static_cast<size_t>(r) * p.entries + e];
      if (page >= 0 && page < p.num_pages) atomicSub(&p.new_refs[page], 1);
    }
  }
  for (long long w = my_warp; w < p.new_rows * pieces; w += warps) {
    const int b = static_cast<int>(pieces == 1 ? w : w / pieces);
    const int e0 = static_cast<int>(w - b * pieces) * kRowPiece;
    const Row r = row[b];
    const int full = p.by_page.quotient(r.len);
    const bool keeps = r.last >= 0 && !(r.copy & 1);
#pragma unroll 4
    for (int e = e0 + lane; e < min(e0 + kRowPiece, p.entries); e += 32) {
      int page = -1;
      if (e < full || (e == full && keeps)) {
        page = p.table[static_cast<size_t>(r.parent) * p.entries + e];
        if (page < 0 || page >= p.num_pages) page = -1;
        if (page >= 0) atomicAdd(&p.new_refs[page], 1);
      }
      p.new_table[static_cast<size_t>(b) * p.entries + e] = page;
    }
    if (lane == 0 && e0 == 0) {
      p.new_lens[b] = r.len;
      if (holds && (r.copy & 1) && p.refs[r.last] != 1) atomicAdd(&p.new_refs[r.last], kHold);
    }
  }
  cluster_sync_all();

  const Stretch pages(p.num_pages);
  int free_here = 0;
#pragma unroll 4
  for (int i = pages.begin + lane; i < pages.end; i += 32) {
    const int n = ld_fresh(&p.new_refs[i]);
    if (n < 0) p.new_refs[i] = 0;
    free_here += n <= 0;
  }
  cluster_share(block_sum(__reduce_add_sync(0xffffffffu, free_here), s_sum), s_free);
  cluster_sync_all();

  int at = 0, n_free = 0;
  for (int c = 0; c < kCtas; ++c) {
    if (c < rank) at += s_free[c];
    n_free += s_free[c];
  }
  at += warps_before(s_sum);
  for (int i0 = pages.begin; i0 < pages.end && at < wanted; i0 += 32 * kAtOnce) {
    int refs[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int page = i0 + u * 32 + lane;
      refs[u] = page < pages.end ? ld_fresh(&p.new_refs[page]) : 1;
    }
    for (int u = 0; u < kAtOnce; ++u) {
      const int page = i0 + u * 32 + lane;
      const bool free = refs[u] <= 0;
      const unsigned mask = __ballot_sync(0xffffffffu, free);
      const int k = at + __popc(mask & ((1u << lane) - 1));
      at += __popc(mask);
      if (!free || k >= wanted) continue;
      int lo = 0, hi = p.new_rows;  // the last row b with need <= k
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (row[mid].need <= k) lo = mid; else hi = mid;
      }
      const Row r = row[lo];
      const bool copies = r.copy & 1;
      const int j = k - r.need, full = p.by_page.quotient(r.len);
      const int e = full + j + (r.len > full * p.page_size && !copies);
      p.new_table[static_cast<size_t>(lo) * p.entries + e] = page;
      p.new_refs[page] = 1;
      if (copies && j == 0) {
        p.copies[r.copy >> 1] = r.last;
        p.copies[p.new_rows + (r.copy >> 1)] = page;
      }
    }
  }
  if (rank == 0) {  // the rows whose copy got its page are the first ones that copy
    int copies = 0;
    for (int b = tid; b - tid < p.new_rows; b += kThreads)
      copies += __syncthreads_count(b < p.new_rows && (row[b].copy & 1) && row[b].need < n_free);
    for (int i = copies + tid; i < p.new_rows; i += kThreads) p.copies[i] = p.copies[p.new_rows + i] = -1;
    if (tid == 0) {
      const int got = min(wanted, n_free);
      p.info[0] = n_free - got;
      p.info[1] = wanted - got;
      p.info[2] = copies;
    }
  }
  if (!holds) return;
  cluster_sync_all();
  for (int b = me; b < p.new_rows; b += all_threads) {
    const Row r = row[b];
    if (!(r.copy & 1) || p.refs[r.last] == 1) continue;
    const int left = atomicSub(&p.new_refs[r.last], kHold) - kHold;
    if (left > 0) continue;  // held still, or by rows that have yet to let go
    if (left < 0) p.new_refs[r.last] = 0;
    atomicAdd(&p.info[0], 1);
  }
}

struct CompactParams {
  const int32_t *table, *refs;
  int32_t *new_table, *new_refs, *moves, *index, *info;
  long long words;  // of the table
  int num_pages, max_moves;
};

// Grid: one cluster.  n live pages; the k-th free page below n receives the k-th
// live page at or above n.
__global__ void __launch_bounds__(kThreads) page_compact_kernel(const CompactParams p) {
  __shared__ int s_sum[kWarpsPerCta], s_warp[kWarpsPerCta], s_live[kCtas], s_low[kCtas];
  const int tid = threadIdx.x, lane = tid & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int all_threads = kCtas * kThreads, me = rank * kThreads + tid;
  pdl_launch_dependents();
  cluster_arrive();  // a CTA's shared memory may be written once it has started
  pdl_wait();
  const Stretch pages(p.num_pages);

  int mine = 0;
  for (int i = pages.begin + lane; i < pages.end; i += 32) mine += p.refs[i] > 0;
  cluster_wait();
  cluster_share(block_sum(__reduce_add_sync(0xffffffffu, mine), s_warp), s_live);
  cluster_sync_all();
  int at = 0, n = 0;  // live pages before this warp's, and all
  for (int c = 0; c < kCtas; ++c) {
    if (c < rank) at += s_live[c];
    n += s_live[c];
  }
  at += warps_before(s_warp);

  int low = 0;  // live pages below n
  for (int i = pages.begin + lane; i < min(pages.end, n); i += 32) low += p.refs[i] > 0;
  cluster_share(block_sum(__reduce_add_sync(0xffffffffu, low), s_sum), s_low);
  cluster_sync_all();
  low = 0;
  for (int c = 0; c < kCtas; ++c) low += s_low[c];
  const int moves = n - low;

  // Every page of the warp's stretch with its count and the live pages before it.
  auto walk = [&](auto&& visit) {
    int before = at;
    for (int i0 = pages.begin; i0 < pages.end; i0 += 32 * kAtOnce) {
      int refs[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int page = i0 + u * 32 + lane;
        refs[u] = page < pages.end ? p.refs[page] : 0;
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const unsigned mask = __ballot_sync(0xffffffffu, refs[u] > 0);
        const int page = i0 + u * 32 + lane;
        if (page < pages.end) visit(page, refs[u], before + __popc(mask & ((1u << lane) - 1)));
        before += __popc(mask);
      }
    }
  };
  walk([&](int page, int refs, int live_before) {
    if (page < n && refs > 0) {
      p.index[page] = page;
      p.new_refs[page] = refs;
    } else if (page < n) {
      p.index[page] = -1;
      p.moves[p.max_moves + page - live_before] = page;
    } else {
      p.new_refs[page] = 0;
      if (refs > 0)
        p.moves[live_before - low] = page;
      else
        p.index[page] = -1;
    }
  });
  for (int i = moves + me; i < p.max_moves; i += all_threads)
    p.moves[i] = p.moves[p.max_moves + i] = -1;
  if (me == 0) {
    p.info[0] = n;
    p.info[1] = moves;
  }
  cluster_sync_all();

  walk([&](int page, int refs, int live_before) {
    if (page < n || refs <= 0) return;
    const int to = ld_fresh(&p.moves[p.max_moves + live_before - low]);
    p.index[page] = to;
    p.new_refs[to] = refs;
  });
  cluster_sync_all();

#pragma unroll 4
  for (long long i = me; i < p.words; i += all_threads) {
    const int page = p.table[i];
    p.new_table[i] = page >= 0 && page < p.num_pages ? ld_fresh(&p.index[page]) : -1;
  }
}

// Copies of pages, in every slab of a pool.  Bound by HBM: each CTA moves pieces
// of up to 16 KB, four 16-byte words per thread in flight, on all SMs.
constexpr int kCopyThreads = 256;
constexpr int kPiece = kCopyThreads * 4;  // 16-byte words

struct CopyParams {
  uint4* pool;
  const int32_t* pages;  // [2][n]: from, to
  const int32_t* count;  // or null: n
  long long page_words;
  int n, slabs, num_pages, pieces;  // pieces of a page
};

__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const CopyParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int n = p.count != nullptr ? min(max(*p.count, 0), p.n) : p.n;
  const long long per_copy = static_cast<long long>(p.slabs) * p.pieces;
  for (long long w = blockIdx.x; w < n * per_copy; w += gridDim.x) {
    const int i = static_cast<int>(w / per_copy);
    const int rest = static_cast<int>(w - i * per_copy);
    const int slab = rest / p.pieces, piece = rest - slab * p.pieces;
    const int from = p.pages[i], to = p.pages[p.n + i];
    if (from == -1 && to == -1) continue;
    if (from < 0 || from >= p.num_pages || to < 0 || to >= p.num_pages) {
      if (threadIdx.x == 0) report_error(kDevErrBounds);
      continue;
    }
    const uint4* src = p.pool + (static_cast<long long>(slab) * p.num_pages + from) * p.page_words;
    uint4* dst = p.pool + (static_cast<long long>(slab) * p.num_pages + to) * p.page_words;
    const long long at = static_cast<long long>(piece) * kPiece + threadIdx.x;
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at + u * kCopyThreads < p.page_words) v[u] = __ldcg(src + at + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at + u * kCopyThreads < p.page_words) __stcg(dst + at + u * kCopyThreads, v[u]);
  }
}

}  // namespace
}  // namespace npu_b200

extern "C" int npu_b200_page_update(const int32_t* d_page_table, const int32_t* d_seq_lens,
                                    const int32_t* d_parents, const int32_t* d_capacity,
                                    const int32_t* d_page_refs, int32_t* d_new_table,
                                    int32_t* d_new_lens, int32_t* d_new_refs, int32_t* d_copies,
                                    int32_t* d_info, int rows, int new_rows, int table_entries,
                                    int page_size, int num_pages, void* stream) {
  using namespace npu_b200;
  clear_error();
  NPU_REQUIRE(d_page_table && d_seq_lens && d_parents && d_capacity && d_page_refs && d_new_table &&
                  d_new_lens && d_new_refs && d_copies && d_info,
              "page_update: null tensor pointer");
  NPU_REQUIRE(rows >= 1 && rows <= kMaxRows && new_rows >= 1 && new_rows <= kMaxRows,
              "page_update: %d rows to %d are not in [1, %d]", rows, new_rows, kMaxRows);
  int rc = check_pages("page_update", 1, 64, num_pages, page_size, table_entries);
  if (rc) return rc;
  NPU_REQUIRE(static_cast<long long>(new_rows) * table_entries < (1ll << 31),
              "page_update: %d rows of %d entries are too many", new_rows, table_entries);
  const size_t old_bytes = static_cast<size_t>(rows) * table_entries * 4;
  const size_t new_bytes = static_cast<size_t>(new_rows) * table_entries * 4;
  const size_t ref_bytes = static_cast<size_t>(num_pages) * 4;
  NPU_REQUIRE(!overlap(d_page_table, old_bytes, d_new_table, new_bytes) &&
                  !overlap(d_page_refs, ref_bytes, d_new_refs, ref_bytes) &&
                  !overlap(d_seq_lens, rows * size_t(4), d_new_lens, new_rows * size_t(4)),
              "page_update: the new table, lengths and counts must not overlap the old ones");
  UpdateParams p = {d_page_table, d_seq_lens, d_parents, d_capacity, d_page_refs,
                    d_new_table, d_new_lens, d_new_refs, d_copies, d_info,
                    rows, new_rows, table_entries, page_size, num_pages, Divisor::of(page_size)};
  const size_t smem = static_cast<size_t>(rows) * 4 + static_cast<size_t>(new_rows) * sizeof(Row);
  NPU_TRY_CUDA(cudaFuncSetAttribute(page_update_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kMaxRows * static_cast<int>(4 + sizeof(Row))));
  LaunchCfg cfg;
  cfg.grid = dim3(kCtas);
  cfg.block = dim3(kThreads);
  cfg.smem = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.pdl = true;
  cfg.cluster = kCtas;
  return launch(cfg, page_update_kernel, p);
}

extern "C" int npu_b200_page_compact(const int32_t* d_page_table, const int32_t* d_page_refs,
                                     int32_t* d_new_table, int32_t* d_new_refs, int32_t* d_moves,
                                     int32_t* d_index, int32_t* d_info, int rows, int table_entries,
                                     int num_pages, void* stream) {
  using namespace npu_b200;
  clear_error();
  NPU_REQUIRE(d_page_table && d_page_refs && d_new_table && d_new_refs && d_moves && d_index && d_info,
              "page_compact: null tensor pointer");
  NPU_REQUIRE(rows >= 1 && table_entries >= 1, "page_compact: table of %d x %d entries", rows,
              table_entries);
  NPU_REQUIRE(num_pages >= 1 && num_pages < 1 << 28, "page_compact: %d pages out of range", num_pages);
  CompactParams p;
  p.table = d_page_table;
  p.refs = d_page_refs;
  p.new_table = d_new_table;
  p.new_refs = d_new_refs;
  p.moves = d_moves;
  p.index = d_index;
  p.info = d_info;
  p.words = static_cast<long long>(rows) * table_entries;
  p.num_pages = num_pages;
  p.max_moves = num_pages / 2 > 0 ? num_pages / 2 : 1;
  const size_t ref_bytes = static_cast<size_t>(num_pages) * 4;
  NPU_REQUIRE(!overlap(d_page_table, p.words * 4, d_new_table, p.words * 4) &&
                  !overlap(d_page_refs, ref_bytes, d_new_refs, ref_bytes),
              "page_compact: the new table and counts must not overlap the old ones");
  LaunchCfg cfg;
  cfg.grid = dim3(kCtas);
  cfg.block = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.pdl = true;
  cfg.cluster = kCtas;
  return launch(cfg, page_compact_kernel, p);
}

extern "C" int npu_b200_page_copy(void* d_pool, const int32_t* d_pages, const int32_t* d_count, int n,
                                  int slabs, int num_pages, size_t page_bytes, void* stream) {
  using namespace npu_b200;
  clear_error();
  NPU_REQUIRE(d_pool && d_pages, "page_copy: null tensor pointer");
  NPU_REQUIRE(n >= 1 && slabs >= 1 && num_pages >= 1, "page_copy: %d copies, %d slabs of %d pages", n,
              slabs, num_pages);
  NPU_REQUIRE(page_bytes >= 16 && page_bytes % 16 == 0 && page_bytes <= size_t(1) << 32,
              "page_copy: pages of %zu bytes are not a multiple of 16 in [16, 2^32]", page_bytes);
  NPU_REQUIRE(aligned16(d_pool), "page_copy: the pool must be 16-byte aligned");
  CopyParams p;
  p.pool = static_cast<uint4*>(d_pool);
  p.pages = d_pages;
  p.count = d_count;
  p.page_words = static_cast<long long>(page_bytes / 16);
  p.n = n;
  p.slabs = slabs;
  p.num_pages = num_pages;
  p.pieces = static_cast<int>((p.page_words + kPiece - 1) / kPiece);
  NPU_REQUIRE(static_cast<long long>(slabs) * p.pieces < (1ll << 31),
              "page_copy: %d slabs of %d pieces are too many", slabs, p.pieces);
  const long long work = static_cast<long long>(n) * slabs * p.pieces;
  const long long most = 8ll * sm_count();
  LaunchCfg cfg;
  cfg.grid = dim3(static_cast<unsigned>(work < most ? work : most));
  cfg.block = dim3(kCopyThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.pdl = true;
  return launch(cfg, page_copy_kernel, p);
}
