// New keys and values into the pages of a paged cache (paged.cuh): row i of
// sequence b goes to position starts[b] + i.  A copy, bound by HBM (or, for one
// row per sequence, by the launch): each thread moves 16 bytes of K and of V.
#include "paged.cuh"

namespace npu_b200 {
namespace {

constexpr int kAppendThreads = 256;

struct AppendParams {
  const uint4* k;
  const uint4* v;
  uint4* k_pages;
  uint4* v_pages;
  const int32_t* table;
  const int32_t* starts;
  const int32_t* lens;  // or null: every row
  int batch, kv_heads, rows, vecs;  // vecs: 16-byte words of a row
  int entries, page_size, num_pages;
};

// Grid (words of one sequence's new rows, sequence).
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y;
  const int n = p.lens != nullptr ? min(max(p.lens[b], 0), p.rows) : p.rows;
  const long long start = p.starts[b];
  const long long words = static_cast<long long>(p.kv_heads) * p.rows * p.vecs;
  for (long long w = blockIdx.x * static_cast<long long>(kAppendThreads) + threadIdx.x; w < words;
       w += static_cast<long long>(gridDim.x) * kAppendThreads) {
    const int row = static_cast<int>(w / p.vecs), x = static_cast<int>(w - static_cast<long long>(row) * p.vecs);
    const int h = row / p.rows, i = row - h * p.rows;
    if (i >= n) continue;
    const long long at = start + i;
    const long long entry = at / p.page_size;
    int page = -1;
    if (at >= 0 && entry < p.entries) page = p.table[static_cast<size_t>(b) * p.entries + entry];
    if (page < 0 || page >= p.num_pages) {
      report_error(kDevErrBounds);
      continue;
    }
    const size_t src = (static_cast<size_t>(b) * p.kv_heads * p.rows + row) * p.vecs + x;
    const size_t dst = ((static_cast<size_t>(page) * p.kv_heads + h) * p.page_size +
                        static_cast<int>(at - entry * p.page_size)) * p.vecs + x;
    p.k_pages[dst] = p.k[src];
    p.v_pages[dst] = p.v[src];
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
  NPU_REQUIRE(rows >= 1 && static_cast<long long>(rows) * kv_heads < (1ll << 31),
              "paged_append: %d rows out of range", rows);
  NPU_REQUIRE(aligned16(d_k) && aligned16(d_v) && aligned16(d_k_pages) && aligned16(d_v_pages),
              "paged_append: k, v and pages must be 16-byte aligned");
  AppendParams p;
  p.k = static_cast<const uint4*>(d_k);
  p.v = static_cast<const uint4*>(d_v);
  p.k_pages = static_cast<uint4*>(d_k_pages);
  p.v_pages = static_cast<uint4*>(d_v_pages);
  p.table = d_page_table;
  p.starts = d_starts;
  p.lens = d_lens;
  p.batch = batch;
  p.kv_heads = kv_heads;
  p.rows = rows;
  p.vecs = head_dim / 8;
  p.entries = table_entries;
  p.page_size = page_size;
  p.num_pages = num_pages;
  const long long words = static_cast<long long>(kv_heads) * rows * p.vecs;
  const long long blocks = (words + kAppendThreads - 1) / kAppendThreads;
  LaunchCfg cfg;
  cfg.grid = dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536), batch);
  cfg.block = dim3(kAppendThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.pdl = true;
  return launch(cfg, paged_append_kernel, p);
}
