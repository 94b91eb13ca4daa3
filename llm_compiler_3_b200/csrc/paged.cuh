// What the kernels over a paged key-value cache share: the page layout, the
// keys that a position sees under a sliding window with sinks, and the tiles
// that cover them.
//
// A pool of pages holds keys (and another one values) as [pages][kv heads][P][D]
// FP16; row j of a sequence is row j % P of page table[j / P].  The token at
// position p sees key j iff j <= p and (window == 0, or j > p - window, or
// j < sinks): with n = p + 1 keys, [0, s) and [lo, n) with lo = max(0, n - window)
// and s = min(sinks, lo).
#pragma once

#include "common.cuh"
#include "host.hpp"

namespace npu_b200 {

// The tiles of `T` keys that hold every key some position of [first, last] sees:
// tiles [0, n_sink) and [w0, w0 + n - n_sink) of the sequence.
template <int T>
struct TileRange {
  int n_sink, w0, n;
  // `lo`: the first key inside the window of the FIRST position, `len`: one past
  // the last key of the LAST; `sinks` as given.
  __device__ __forceinline__ void set(int lo, int len, int sinks) {
    const int s = min(sinks, lo);
    n_sink = (s + T - 1) / T;
    w0 = max(lo / T, n_sink);
    n = n_sink + max(0, (len + T - 1) / T - w0);
  }
  __device__ __forceinline__ int key0(int i) const { return (i < n_sink ? i : w0 + i - n_sink) * T; }
};

// Quotients by a number known at launch, d in [2, 2^31): with 2^l >= d > 2^(l-1) and
// m = floor(2^(31+l) / d) + 1, n / d = (n m) >> (31 + l) for every n < 2^31.
struct Divisor {
  uint32_t m, shift;
  static Divisor of(uint32_t d) {
    uint32_t l = 1;
    while ((1ull << l) < d) ++l;
    return {static_cast<uint32_t>((1ull << (31 + l)) / d + 1), l - 1};
  }
  __device__ __forceinline__ int quotient(int n) const {
    return static_cast<int>(__umulhi(static_cast<uint32_t>(n), m) >> shift);
  }
};

// Softmax weights, FP16 as the second product's operand, are relative to a reference 2^7 below
// the maximum that set it.  It moves once a weight would pass 2^15, so weights fit FP16, and
// those far below the maximum keep their bits down to 2^-21 of it (relative to the maximum
// itself they were gone at 2^-25, and with them all that thousands of such keys add up to).
constexpr float kBelowMax = 7.f;
constexpr float kMostLog2 = 15.f;

// Rows of the largest TMA box that never crosses a page: the largest power of
// two that divides P, at most `tile`.
inline int page_box(int page_size, int tile) {
  int box = 8;
  while (box * 2 <= tile && page_size % (box * 2) == 0) box *= 2;
  return box;
}

// Host checks that every operator over pages makes.
inline int check_pages(const char* what, int kv_heads, int head_dim, long long num_pages,
                       int page_size, int table_entries) {
  NPU_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim %d not in {64,128}", what, head_dim);
  NPU_REQUIRE(kv_heads >= 1 && kv_heads <= 65535, "%s: kv_heads %d out of range", what, kv_heads);
  NPU_REQUIRE(page_size >= 8 && page_size <= 65536 && page_size % 8 == 0,
              "%s: page_size %d is not a multiple of 8 in [8, 65536]", what, page_size);
  NPU_REQUIRE(num_pages >= 1 && num_pages * kv_heads * page_size < (1ll << 31),
              "%s: %lld pages of %d rows and %d heads are too many rows for 32-bit coordinates", what,
              num_pages, page_size, kv_heads);
  NPU_REQUIRE(table_entries >= 1 && static_cast<long long>(table_entries) * page_size < (1ll << 31) - 65536,
              "%s: %d table entries of %d rows are too many positions", what, table_entries, page_size);
  return NPU_B200_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace npu_b200
