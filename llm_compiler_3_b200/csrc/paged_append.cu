// New keys and values into the pages of a paged cache (paged.cuh): row i of
// sequence b goes to position starts[b] + i.  A copy, bound by HBM (or, for one
// row per sequence, by the launch): each thread moves 16 bytes of K and of V of
// four rows, all eight loads in flight before the first store.
#include "paged.cuh"

namespace npu_b200 {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAtOnce = 4;  // rows of a thread

struct AppendParams {
  const uint4* k;
  const uint4* v;
  uint4* k_pages;
  uint4* v_pages;
  const int32_t* table;
  const int32_t* starts;
  const int32_t* lens;  // or null: every row
  int kv_heads, rows;
  int entries, page_size, num_pages;
  Divisor by_rows, by_page;
};

// Grid (lines, sequence): a line is one row of one head, VECS 16-byte words.
template <int VECS>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
  constexpr int kLines = kAppendThreads / VECS;  // at a time
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y, x = threadIdx.x % VECS;
  const int n = p.lens != nullptr ? min(max(p.lens[b], 0), p.rows) : p.rows;
  const long long start = p.starts[b];
  const int lines = p.kv_heads * p.rows;
  const uint4* k = p.k + static_cast<size_t>(b) * lines * VECS;
  const uint4* v = p.v + static_cast<size_t>(b) * lines * VECS;
  const int32_t* table = p.table + static_cast<size_t>(b) * p.entries;
  for (int line0 = blockIdx.x * kLines * kAtOnce + threadIdx.x / VECS; line0 < lines;
       line0 += gridDim.x * kLines * kAtOnce) {
    uint4 kv[kAtOnce], vv[kAtOnce];
    size_t to[kAtOnce];
    bool ok[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int line = line0 + u * kLines;
      const int h = p.rows > 1 ? p.by_rows.quotient(line) : line, i = line - h * p.rows;
      ok[u] = line < lines && i < n;
      if (!ok[u]) continue;
      const size_t from = static_cast<size_t>(line) * VECS + x;
      kv[u] = __ldcs(k + from);
      vv[u] = __ldcs(v + from);
      const long long at = start + i;
      const bool inside = at >= 0 && at < static_cast<long long>(p.entries) * p.page_size;  // below 2^31
      const int pos = inside ? static_cast<int>(at) : 0, entry = p.by_page.quotient(pos);
      const int page = inside ? table[entry] : -1;
      ok[u] = page >= 0 && page < p.num_pages;
      if (!ok[u]) report_error(kDevErrBounds);
      to[u] = ((static_cast<size_t>(page) * p.kv_heads + h) * p.page_size + pos - entry * p.page_size) * VECS + x;
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (ok[u]) {
        p.k_pages[to[u]] = kv[u];
        p.v_pages[to[u]] = vv[u];
      }
  }
}

}  // namespace
}  // namespace npu_b200

extern "C" int npu_b200_paged_append(const void* d_k, const void* d_v, void* d_k_pages,
                                     void* d_v_pages, const int32_t* d_page_table,
                                     const int32_t* d_starts, const int32_t* d_lens, int batch,
                                     int kv_heads, int rows, int head_dim, int num_pages,
                                     int page_size, int table_entries, void* stream) {
  using namespace npu_b200;
  clear_error();
  NPU_REQUIRE(d_k && d_v && d_k_pages && d_v_pages && d_page_table && d_starts,
              "paged_append: null tensor pointer");
  int rc = check_pages("paged_append", kv_heads, head_dim, num_pages, page_size, table_entries);
  if (rc) return rc;
  NPU_REQUIRE(batch >= 1 && batch <= 65535, "paged_append: batch %d not in [1, 65535]", batch);
  NPU_REQUIRE(rows >= 1 && static_cast<long long>(rows) * kv_heads < (1ll << 30),
              "paged_append: %d rows out of range", rows);
  NPU_REQUIRE(aligned16(d_k) && aligned16(d_v) && aligned16(d_k_pages) && aligned16(d_v_pages),
              "paged_append: k, v and pages must be 16-byte aligned");
  const size_t bytes = static_cast<size_t>(batch) * kv_heads * rows * head_dim * 2;
  const size_t pool = static_cast<size_t>(num_pages) * kv_heads * page_size * head_dim * 2;
  NPU_REQUIRE(!overlap(d_k, bytes, d_k_pages, pool) && !overlap(d_v, bytes, d_v_pages, pool) &&
                  !overlap(d_k, bytes, d_v_pages, pool) && !overlap(d_v, bytes, d_k_pages, pool),
              "paged_append: k and v must not overlap the pages");
  AppendParams p;
  p.k = static_cast<const uint4*>(d_k);
  p.v = static_cast<const uint4*>(d_v);
  p.k_pages = static_cast<uint4*>(d_k_pages);
  p.v_pages = static_cast<uint4*>(d_v_pages);
  p.table = d_page_table;
  p.starts = d_starts;
  p.lens = d_lens;
  p.kv_heads = kv_heads;
  p.rows = rows;
  p.entries = table_entries;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.by_rows = Divisor::of(rows > 1 ? rows : 2);
  p.by_page = Divisor::of(page_size);
  const int vecs = head_dim / 8;
  const long long per_block = kAppendThreads / vecs * kAtOnce;
  const long long blocks = (static_cast<long long>(kv_heads) * rows + per_block - 1) / per_block;
  LaunchCfg cfg;
  cfg.grid = dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536), batch);
  cfg.block = dim3(kAppendThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.pdl = true;
  return head_dim == 128 ? launch(cfg, paged_append_kernel<16>, p) : launch(cfg, paged_append_kernel<8>, p);
}
