// Attention of a chunk of new tokens per sequence over a paged key-value cache.
//
// Query i < q_lens[b] of sequence b sits at position p = seq_lens[b] - q_lens[b] + i
// and sees the keys of paged.cuh: causal, with an optional window and sinks.
//   out[b, h, i] = sum_j softmax_j(scale q[b, h, i] . k[j]) v[j]
// in one pass over the keys with a running reference m, sum l and output O (FP32).
// The weights are rounded to FP16 as the second product's operand (the values are
// FP16 too), the output is rounded once.  Rows that see no key, and rows past
// q_lens[b], are zero.
//
// Bound: the tensor cores, 4 D flops per visible (query, key) pair and head, and
// next to them the exponentials: an SM does 16 a clock, so 128 x 128 of them take
// as long as the tile's two products at D = 128.  Both run all the time only if two
// query tiles take turns: while one tile's scores become weights, the tensor cores
// do the other's P V and next Q K^T.
//
// One CTA per pair of query tiles; a tile is 128 rows, `hp` heads of one GQA group
// x `bm` queries, so that few queries still fill the rows and share one pass over
// K and V.
//   warps 0-3, 4-7  softmax of tile 0 / 1: thread r has row r (TMEM lane r)
//   warp 8          TMA: both Q tiles, then K and V tiles in one ring (K0 V0 K1 V1
//                   ...), one box per piece of a page, each lane one
//   warp 9          MMA issue: O_t += P_t V, then the next S_t = Q_t K^T
//   warp 10         V tiles with keys that not all of the CTA's queries see: clears the rows that
//                   none sees, takes infinite and NaN numbers out of the others
// When there are few query tiles, a cluster of up to 8 CTAs shares the keys of each pair;
// their O, references and sums meet in shared memory, each CTA joining a share of the dimensions.
// TMEM: S0, S1 (128 columns each), O0, O1 (D each); P_t, FP16, lies over the first
// half of S_t.  The tensor pipe works in order, so S_t(j + 1), issued after
// P_t(j) V, cannot overwrite weights that are still read, and its completion says
// that O_t is up to date.  A row's reference moves, and its O row is rescaled,
// only when a weight would pass 2^15 (paged.cuh).
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "paged.cuh"

namespace npu_b200 {

void prefill_blocking(int queries, int group, int* bm, int* hp);  // prefill_attention.cu

namespace {

constexpr int KT = 128;           // keys per tile
// A tile is four units of 32 keys, one after the other in the list of the units that hold
// visible keys: sinks and the window's ragged ends cost a unit, not a tile (a window of
// 1024 with 8 sinks, two chunks up to 2999 at head size 64, 128 queries to a tile: 87 -> 77
// us).
constexpr int kUnit = 32;
constexpr int kThreads = 352;
constexpr uint32_t kTmemCols = 512;
constexpr int kMaxSplits = 8;     // CTAs that share a tile pair's keys

template <int D>
struct PpShape {
  static constexpr int kRegions = D / 64;              // 128-byte swizzle regions of a row
  static constexpr int kRegion = 128 * 128;            // 128 rows of one region
  static constexpr int kTileBytes = kRegions * kRegion;  // a Q, K or V tile
  static constexpr int kStages = D == 128 ? 5 : 10;    // K and V tiles in the ring
  static constexpr int kRing = 2 * kTileBytes;
  static constexpr int kBars = kRing + kStages * kTileBytes;
  static constexpr int kNumBars = 1 + 3 * kStages + 6 + 1;
  static constexpr int kSmem = kBars + kNumBars * 8 + 16 + 1024;
  static_assert(kSmem <= 232448, "shared memory");
};
constexpr int kS = 0, kO = 2 * KT;  // TMEM columns; O_t at kO + t D

struct PpParams {
  const __half* v_pages;  // for values that are no numbers: tiles come through the tensor maps
  const int32_t* table;
  const int32_t* seq_lens;
  const int32_t* q_lens;  // or null: every query
  __half* out;
  int q_heads, kv_heads, queries, entries, page_size, box, num_pages, total_rows;
  int bm, hp, q_blocks, window, sinks, negate, splits;
  float scale_log2;  // > 0
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
      "[%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// A word whose first n bits are set.
__device__ __forceinline__ uint32_t first_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
}

// What the two query tiles of a CTA cover.
struct Span {
  int seq_len, q_len, first_pos;  // first_pos: position of query 0 of the chunk
  int lo, len, s;                 // keys that some of the CTA's queries see: [0, s) and [lo, len)
  int all_lo, all_len, sinks;     // that all at a position see: [0, sinks) and [all_lo, all_len)
  TileRange<kUnit> units;
  __device__ __forceinline__ bool sees(int j) const { return j < len && (j >= lo || j < s); }
  __device__ __forceinline__ bool sees_any(int j, int n) const { return j < len && (j + n > lo || j < s); }
  __device__ __forceinline__ bool seen_by_all(int j, int n) const {  // each key of [j, j + n)
    return j + n <= all_len && (j >= all_lo || j + n <= sinks);
  }
};

// Whether one of 8 numbers is infinite or NaN: times 0 they are NaN, all others 0.
__device__ __forceinline__ __half2 times_zero(const uint4& w, __half2 sum) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    sum = __hfma2(*reinterpret_cast<const __half2*>(&u[i]), __half2half2(__ushort_as_half(0)), sum);
  return sum;
}
__device__ __forceinline__ bool is_odd(__half2 sum) {
  return (*reinterpret_cast<const uint32_t*>(&sum) & 0x7c007c00u) != 0;
}
// Infinite and NaN numbers become 0.
__device__ __forceinline__ uint4 without_odd(const uint4& w) {
  uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t low = (u[i] & 0x7c00u) == 0x7c00u ? 0xffffu : 0u;
    const uint32_t high = (u[i] & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u;
    u[i] &= ~(low | high);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// The infinite and NaN values that tiles went without (warp 10), onto dimensions [d0, d1) of
// the rows of out that see them: any weight of such a value is that value.  One warp walks the
// keys [first, first + keys), its lanes over the dimensions, each with the places of the newest
// such values; lane r's row `at` sees the keys up to its turn's (none: a negative turn) from `lo`
// on, and the sinks.
template <int D>
__device__ __noinline__ void add_odd_values(const PpParams& p, int b, int hk, long long at, int turn, int lo,
                                            int first, int keys, int d0, int d1) {
  const int lane = threadIdx.x & 31;
  int nan[D / 32], high[D / 32], low[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) nan[e] = high[e] = low[e] = -1;
  __syncwarp();  // each lane has written its row
  for (int k0 = 0; k0 < keys; k0 += 32) {
    long long row = -1;  // of the pool
    if (k0 + lane < keys) {
      const int j = first + k0 + lane, page = p.table[static_cast<size_t>(b) * p.entries + j / p.page_size];
      if (page >= 0 && page < p.num_pages) row = (page * p.kv_heads + hk) * p.page_size + j % p.page_size;
    }
#pragma unroll 4
    for (int k = 0; k < 32; ++k) {
      const long long from = __shfl_sync(0xffffffffu, row, k);
      if (from >= 0) {
        const int j = first + k0 + k < p.sinks ? INT_MAX : first + k0 + k;
        const __half* v = p.v_pages + from * D + lane * (D / 32);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const float x = __half2float(v[e]);
          if (isnan(x)) nan[e] = max(nan[e], j);
          if (x == INFINITY) high[e] = max(high[e], j);
          if (x == -INFINITY) low[e] = max(low[e], j);
        }
      }
      for (unsigned todo = __ballot_sync(0xffffffffu, turn == k0 + k); todo != 0; todo &= todo - 1) {
        const int r = __ffs(todo) - 1, from_r = __shfl_sync(0xffffffffu, lo, r);
        __half* out = p.out + __shfl_sync(0xffffffffu, at, r) * D;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const int d = lane * (D / 32) + e;
          if (d < d0 || d >= d1 || max(nan[e], max(high[e], low[e])) < from_r) continue;
          const float x = (nan[e] >= from_r ? NAN : 0.f) + (high[e] >= from_r ? INFINITY : 0.f) +
                          (low[e] >= from_r ? -INFINITY : 0.f);
          out[d] = __float2half_rn(__half2float(out[d]) + x);
        }
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap qmap,
                         const __grid_constant__ CUtensorMap kmap,
                         const __grid_constant__ CUtensorMap vmap,
                         const __grid_constant__ PpParams p) {
  using S = PpShape<D>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const uint32_t sQ = smem_u32(smem), sRing = sQ + S::kRing;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* full = q_full + 1;         // [stages] a K or V tile is there
  uint64_t* raw = full + kStages;      // [stages] a V tile whose hidden rows are to be cleared is
  uint64_t* empty = raw + kStages;     // [stages] the MMAs have read it
  uint64_t* s_full = empty + kStages;  // [2] scores are there
  uint64_t* p_full = s_full + 2;       // [2] weights are there
  uint64_t* o_done = p_full + 2;       // [2] the last P V is done
  uint64_t* drain = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* odd_values = tmem_slot + 2;  // tiles went without some of V's (add_odd_values)
  // Over the ring at the end: O of a CTA that has a share of the keys, [tile][D / 4][row], and
  // its rows' maxima and sums.
  uint4* parts = reinterpret_cast<uint4*>(smem + S::kRing);
  float2* part_ml = reinterpret_cast<float2*>(parts + 2 * (D / 4) * 128);
  static_assert(2 * D * 512 + 2048 <= kStages * S::kTileBytes, "parts over the ring");

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int group = p.q_heads / p.kv_heads, subgroups = group / p.hp;
  const int n_units = p.q_blocks * subgroups;
  const int rank = static_cast<int>(blockIdx.x) % p.splits;  // in the cluster
  const int bh = static_cast<int>(blockIdx.x) / p.splits, hk = bh % p.kv_heads, b = bh / p.kv_heads;
  // Units (query block, head subgroup), last query blocks first; this CTA has
  // units u0 (tile 0) and u0 + 1 (tile 1, if there is one).
  const int u0 = 2 * static_cast<int>(blockIdx.y);
  const bool has1 = u0 + 1 < n_units;
  auto unit_m0 = [&](int u) { return (p.q_blocks - 1 - u / subgroups) * p.bm; };

  pdl_wait();
  Span span;
  span.seq_len = min(max(p.seq_lens[b], 0), p.entries * p.page_size);
  span.q_len = p.q_lens != nullptr ? min(max(p.q_lens[b], 0), p.queries) : p.queries;
  span.first_pos = span.seq_len - span.q_len;
  {
    const int m_lo = unit_m0(has1 ? u0 + 1 : u0);
    const int m_hi = min(unit_m0(u0) + p.bm, span.q_len);  // one past the last query
    const int first = max(0, span.first_pos + m_lo);
    span.len = m_hi > m_lo ? max(0, span.first_pos + m_hi) : 0;
    span.lo = p.window > 0 ? max(0, first - p.window + 1) : 0;
    span.s = min(p.sinks, span.lo);
    span.all_lo = p.window > 0 ? max(0, span.len - p.window) : 0;
    span.all_len = first + 1;
    span.sinks = p.sinks;
    span.units.set(span.lo, span.len, p.sinks);
    if (span.len == 0) span.units.n = 0;
  }
  // This CTA's tiles of keys: all, or its even share of them.
  const long long n_all = (span.units.n + KT / kUnit - 1) / (KT / kUnit);
  const int tile0 = static_cast<int>(n_all * rank / p.splits);
  const int n_tiles = static_cast<int>(n_all * (rank + 1) / p.splits) - tile0;
  // The key of row `row` of tile j (past the last unit: a hidden one), and whether all queries
  // see each key of the tile.
  auto key_of = [&](int j, int row) {
    return span.units.key0((tile0 + j) * (KT / kUnit) + row / kUnit) + row % kUnit;
  };
  auto whole = [&](int j) {
    bool all = true;
    for (int row = 0; row < KT; row += kUnit) all = all && span.seen_by_all(key_of(j, row), kUnit);
    return all;
  };

  // A lane of the TMA warp loads one box of each tile: rows of one page, one 64-dim region.
  const int my_region = lane % S::kRegions, my_row = lane / S::kRegions * p.box;
  const bool my_box = warp == 8 && lane < KT / p.box * S::kRegions;
  auto look_up = [&](int j) {  // the page of this lane's box of tile j; -2: nothing visible
    const int at = key_of(j, my_row);
    if (!my_box || !span.sees_any(at, p.box)) return -2;
    return p.table[static_cast<size_t>(b) * p.entries + at / p.page_size];
  };
  int page = n_tiles > 0 ? look_up(0) : -2;  // asked for before the barrier

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&raw[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *odd_values = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Not before: a dependent kernel's CTA that took this SM's TMEM first would wait for
  // this one to end, and this one for the TMEM.
  pdl_launch_dependents();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  // A softmax thread's row.
  const int tt = (warp >> 2) & 1, r = threadIdx.x & 127;
  const bool unit_ok = tt == 0 || has1;
  const int m0 = unit_ok ? unit_m0(u0 + tt) : 0, g = r / p.bm, i = r % p.bm;
  const bool row_ok = unit_ok && g < p.hp && m0 + i < p.queries;
  const long long at =  // of q and out
      (static_cast<long long>(b) * p.q_heads + hk * group + (u0 + tt) % subgroups * p.hp + g) * p.queries + m0 + i;
  // Keys of this row: j <= last and (j >= lo or j < sinks).
  const int last = row_ok && m0 + i < span.q_len ? span.first_pos + m0 + i : -1;
  const int lo = p.window > 0 ? max(0, last - p.window + 1) : 0;
  // The keys that some queries see and others do not: those before the last one's window, and
  // those after the first query.
  auto add_odd = [&](int d0, int d1) {
    const int from = max(span.lo, p.sinks), keys = min(span.all_lo, span.all_len) - from;
    add_odd_values<D>(p, b, hk, at, last >= 0 ? keys - 1 : -1, lo, from, keys, d0, d1);
    add_odd_values<D>(p, b, hk, at, last - span.all_len, lo, span.all_len, span.len - span.all_len, d0, d1);
  };

  if (warp == 8) {
    // ---------------- TMA producer ----------------
    if (n_tiles > 0) {
      if (lane == 0) {
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
        const int tiles_q = has1 ? 2 : 1;
        mbar_arrive_expect_tx(q_full, static_cast<uint32_t>(tiles_q * p.hp * S::kRegions * p.bm * 128));
        for (int t = 0; t < tiles_q; ++t) {
          const int u = u0 + t, m0 = unit_m0(u), gs = u % subgroups;
          for (int g = 0; g < p.hp; ++g) {
            const int plane = b * p.q_heads + hk * group + gs * p.hp + g;
            for (int a = 0; a < S::kRegions; ++a)
              tma_load_3d(sQ + t * S::kTileBytes + a * S::kRegion + g * p.bm * 128, &qmap, q_full,
                          a * 64, m0, plane);
          }
        }
      }
      bool ok = true;
      int issued = 0;
      uint32_t raw_uses = 0, was_raw = 0;  // bit s: raw[s] was used an odd number of times; last
      for (int j = 0; ok && j < n_tiles; ++j) {
        const int at = key_of(j, my_row);
        int row = p.total_rows;  // past the pool: the box is filled with zeros
        if (page >= 0 && page < p.num_pages)
          row = (page * p.kv_heads + hk) * p.page_size + at % p.page_size;
        else if (page != -2)
          report_error(kDevErrBounds);
        if (j + 1 < n_tiles) page = look_up(j + 1);
        for (int kv = 0; kv < 2; ++kv) {
          const int x = 2 * j + kv, s = x % kStages;
          if (x >= kStages)
            ok = __all_sync(0xffffffffu, wait_or_abort(&empty[s], ((x / kStages) - 1) & 1, abort_flag));
          if (!ok) break;
          const bool border = kv && !whole(j);
          uint64_t* bar = border ? &raw[s] : &full[s];
          was_raw = (was_raw & ~(1u << s)) | (border ? 1u << s : 0u);
          raw_uses ^= border ? 1u << s : 0u;
          if (lane == 0) mbar_arrive_expect_tx(bar, S::kTileBytes);
          __syncwarp();
          if (my_box)
            tma_load_2d(smem + S::kRing + s * S::kTileBytes + my_region * S::kRegion + my_row * 128,
                        kv ? &vmap : &kmap, bar, my_region * 64, row);
          issued = x + 1;
        }
      }
      // Leave no copy in flight into this CTA's shared memory.
      if (!ok) *abort_flag = 1;
      mbar_wait(q_full, 0, kDevErrTmaTimeout);
      for (int x = max(0, issued - kStages); x < issued; ++x) {
        const int s = x % kStages;
        const bool border = was_raw >> s & 1;
        mbar_wait(border ? &raw[s] : &full[s], border ? ~raw_uses >> s & 1 : (x / kStages) & 1, kDevErrTmaTimeout);
      }
    }
  } else if (warp == 9) {
    // ---------------- MMA issuer ----------------
    // What timing it taught: the whole warp runs along and one elected lane issues,
    // so that the compiler sees one value for all lanes and keeps descriptors in
    // uniform registers (behind `lane == 0` each MMA took 92 cycles to issue, more
    // than the 64 it runs); and little may stand between P_t's arrival and the first
    // MMA, as instructions that run once in a thousand cycles are fetched anew each
    // time: K and V are waited for before, and the next V's and K's places worked out.
    const uint32_t idesc_s = idesc_f16_f32(128, KT) | (p.negate ? 1u << 13 : 0u);
    constexpr uint32_t idesc_pv = idesc_f16_f32(128, D) | kIdescBMajorMN;
    const uint64_t dq = smem_desc_sw128(sQ), dk = smem_desc_sw128(sRing);
    const uint64_t dv = smem_desc_sw128_mn(sRing, S::kRegion, 1024);
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      return __all_sync(0xffffffffu, spin_or_abort(bar, phase, abort_flag)) != 0;
    };
    auto issue_s = [&](int t, uint64_t k) {  // by the elected lane
      const uint64_t q = dq + (t * S::kTileBytes >> 4);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = ((kk >> 2) * S::kRegion + (kk & 3) * 32) >> 4;
        tc_mma_f16(tmem + kS + t * KT, q + off, k + off, idesc_s, kk > 0 ? 1u : 0u);
      }
      tc_commit(&s_full[t]);
    };
    bool ok = n_tiles == 0 || (wait(q_full, 0) && wait(&full[0], 0));
    if (ok && n_tiles > 0) {
      tc_fence_after();
      if (elect_one()) {
        issue_s(0, dk);
        issue_s(1, dk);
        tc_commit(&empty[0]);
      }
    }
    int sv = 1 % kStages, sk = 2 % kStages;      // stages of V(j) and K(j + 1)
    uint32_t fv = 1 / kStages, fk = 2 / kStages;  // and their phases
    for (int j = 0; ok && j < n_tiles; ++j) {
      const bool more = j + 1 < n_tiles;
      ok = wait(&full[sv], fv) && (!more || wait(&full[sk], fk));
      if (!ok) break;
      const uint64_t v0 = dv + (sv * S::kTileBytes >> 4), k0 = dk + (sk * S::kTileBytes >> 4);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ok = wait(&p_full[t], j & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk)
            tc_mma_f16_tmem_a(tmem + kO + t * D, tmem + kS + t * KT + kk * 8, v0 + (kk * 2048 >> 4),
                              idesc_pv, j > 0 || kk > 0 ? 1u : 0u);
          if (more)
            issue_s(t, k0);
          else
            tc_commit(&o_done[t]);
          if (t == 1) {
            tc_commit(&empty[sv]);
            if (more) tc_commit(&empty[sk]);
          }
        }
        __syncwarp();
      }
      sv += 2;
      if (sv >= kStages) sv -= kStages, fv ^= 1;
      sk += 2;
      if (sk >= kStages) sk -= kStages, fk ^= 1;
    }
    if (!ok) {  // no MMA may write TMEM after it is released
      *abort_flag = 1;
      if (elect_one()) {
        tc_commit(drain);
        mbar_wait(drain, 0, kDevErrMmaTimeout);
      }
      __syncwarp();
    }
  } else if (warp == 10) {
    // ---------------- hidden rows of V ----------------
    // Rows that a query does not see may hold anything; its weights for them are 0, but 0 x inf
    // and 0 x NaN are NaN.  Rows that no query here sees are cleared; what is infinite or NaN in
    // rows that some see is, and comes back in add_odd_values.
    uint32_t raw_uses = 0;  // bit s: raw[s] was used an odd number of times
    for (int j = 0; j < n_tiles; ++j) {
      const int s = (2 * j + 1) % kStages;
      if (whole(j)) continue;
      if (!__all_sync(0xffffffffu, wait_or_abort(&raw[s], raw_uses >> s & 1, abort_flag))) break;
      raw_uses ^= 1u << s;
      for (int r = lane; r < KT; r += 32) {
        const int key = key_of(j, r);
        if (span.seen_by_all(key, 1)) continue;
        uint8_t* row = smem + S::kRing + s * S::kTileBytes + r * 128;
        auto chunk = [&](int x) {  // each lane begins at banks of its own
          return reinterpret_cast<uint4*>(row + (x >> 3) * S::kRegion + ((x + lane) & 7) * 16);
        };
        if (!span.sees(key)) {
          for (int x = 0; x < D / 8; ++x) *chunk(x) = make_uint4(0, 0, 0, 0);
          continue;
        }
        __half2 sum = __half2half2(__ushort_as_half(0));
#pragma unroll
        for (int x = 0; x < D / 8; ++x) sum = times_zero(*chunk(x), sum);
        if (is_odd(sum)) {
          for (int x = 0; x < D / 8; ++x) *chunk(x) = without_odd(*chunk(x));
          *odd_values = 1;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
    }
  } else {
    // ---------------- softmax warpgroups ----------------
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + kS + tt * KT, t_o = t_lane + kO + tt * D;
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      return __all_sync(0xffffffffu, wait_or_abort(bar, phase, abort_flag)) != 0;
    };
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      ok = wait(&s_full[tt], j & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[KT];
#pragma unroll
      for (int c = 0; c < KT; c += 32) tmem_ld32(t_s + c, sr + c);
      tmem_ld_wait();
      // Hidden keys, a unit to a word of bits (comparing key by key took 640 instructions).
      const int first_key = key_of(j, 0), last_key = key_of(j, KT - 1);
      if (!__all_sync(0xffffffffu, last_key <= last && (first_key >= lo || last_key < p.sinks))) {
#pragma unroll
        for (int c = 0; c < KT; c += 32) {
          const int key0 = key_of(j, c);
          const uint32_t seen = first_bits(last + 1 - key0) & (~first_bits(lo - key0) | first_bits(p.sinks - key0));
          if (__all_sync(0xffffffffu, seen == ~0u)) continue;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(seen >> e & 1)) sr[c + e] = 0xff800000u;  // -inf
        }
      }
      float top[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e] = __uint_as_float(sr[e]);
#pragma unroll
      for (int c = 4; c < KT - 4; c += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top[e] = max3(top[e], __uint_as_float(sr[c + e]), __uint_as_float(sr[c + 4 + e]));
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], __uint_as_float(sr[KT - 4 + e]));
      const float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]);
      const bool grow = __fmaf_rn(mx, p.scale_log2, -m_run) > kMostLog2;
      if (__any_sync(0xffffffffu, grow)) {
        float alpha = 1.f;
        if (grow) {
          const float m_tile = __fmaf_rn(mx, p.scale_log2, -kBelowMax);
          alpha = m_run == -INFINITY ? 0.f : fast_exp2(m_run - m_tile);
          l_run *= alpha;
          m_run = m_tile;
        }
        if (j > 0) {  // rescale this warp's O rows: with S_t(j) done, so is P_t(j - 1) V
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(t_o + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(t_o + c, o);
          }
        }
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run;  // no key seen yet: all -inf
      const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), minus2 = pack2(-m_use, -m_use);
      uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < KT; c += 64) {
        uint32_t pk[32];  // keys 2q, 2q + 1 in column q
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const uint64_t s2 = static_cast<uint64_t>(sr[c + e + 1]) << 32 | sr[c + e];
          const uint64_t x2 = fma2(s2, scale2, minus2);
          const float w0 = fast_exp2(lo2(x2)), w1 = fast_exp2(hi2(x2));
          sum2[(e >> 1) & 3] = add2(sum2[(e >> 1) & 3], pack2(w0, w1));
          pk[e >> 1] = pack_half2(w0, w1);
        }
        tmem_st32(t_s + c / 2, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[tt]);
      const uint64_t all2 = add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3]));
      l_run += lo2(all2) + hi2(all2);
    }
    if (ok && n_tiles > 0) ok = wait(&o_done[tt], 0);
    // Parts go over the ring, which the other tile's last product reads too.
    if (ok && n_tiles > 0 && p.splits > 1) ok = wait(&o_done[tt ^ 1], 0);
    if (!ok) {
      if (lane == 0) *abort_flag = 1;
    } else if (p.splits > 1) {
      tc_fence_after();
      if (n_tiles > 0) {
        uint32_t o[D];
#pragma unroll
        for (int c = 0; c < D; c += 32) tmem_ld32(t_o + c, o + c);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < D / 4; ++e)
          parts[(tt * (D / 4) + e) * 128 + r] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      }
      // Without a tile there is no part: a sum that none has.
      part_ml[tt * 128 + r] = make_float2(m_run, n_tiles > 0 ? l_run : -1.f);
    } else {
      tc_fence_after();
      const bool any = n_tiles > 0 && l_run != 0.f;
      const float inv = any ? 1.f / l_run : 0.f;
      uint4* row = reinterpret_cast<uint4*>(p.out + at * D);
      uint32_t o[D];
      if (n_tiles > 0) {
#pragma unroll
        for (int c = 0; c < D; c += 32) tmem_ld32(t_o + c, o + c);
        tmem_ld_wait();
      }
      if (row_ok) {
#pragma unroll
        for (int c = 0; c < D; c += 8) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = any ? __uint_as_float(o[c + e]) * inv : 0.f;
          row[c / 8] = make_uint4(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]),
                                  pack_half2(f[6], f[7]));
        }
      }
      if (n_tiles > 0 && *odd_values != 0) add_odd(0, D);
    }
  }

  if (p.splits > 1) {
    // ---------------- the cluster's parts of every row join ----------------
    // CTA `rank` takes its share of the dimensions; parts in the order of the CTAs.
    cluster_sync_all();
    if (warp < 8) {
      // Weight 0 is no reason to leave a part out: one whose scores are all NaN has no
      // maximum, one with a NaN among scores far below the others' weighs nothing, and both
      // have NaN as their sum.
      float w[kMaxSplits], l[kMaxSplits], top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int c = 0; c < kMaxSplits; ++c) {
        w[c] = -INFINITY;
        l[c] = -1.f;
        if (c >= p.splits) continue;
        const uint32_t ml = cluster_map(smem_u32(part_ml + tt * 128 + r), c);
        w[c] = ld_cluster_f32(ml);
        l[c] = ld_cluster_f32(ml + 4);
        top = fmaxf(top, w[c]);
      }
#pragma unroll
      for (int c = 0; c < kMaxSplits; ++c) {
        w[c] = w[c] == -INFINITY ? 0.f : fast_exp2(w[c] - top);
        if (!(l[c] < 0.f)) sum += w[c] * l[c];
      }
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      const int each = D / 4 / p.splits;  // groups of four dimensions
#pragma unroll 1
      for (int q = rank * each; q < (rank + 1) * each; q += 2) {
        float f[8] = {};
#pragma unroll
        for (int c = 0; c < kMaxSplits; ++c) {
          if (l[c] < 0.f) continue;
          const uint32_t from = cluster_map(smem_u32(parts + (tt * (D / 4) + q) * 128 + r), c);
          const float4 x = ld_cluster_v4(from), y = ld_cluster_v4(from + 128 * 16);
          f[0] += w[c] * x.x, f[1] += w[c] * x.y, f[2] += w[c] * x.z, f[3] += w[c] * x.w;
          f[4] += w[c] * y.x, f[5] += w[c] * y.y, f[6] += w[c] * y.z, f[7] += w[c] * y.w;
        }
        if (!row_ok) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = sum != 0.f ? f[e] * inv : 0.f;
        *reinterpret_cast<uint4*>(p.out + at * D + q * 4) = make_uint4(
            pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]), pack_half2(f[6], f[7]));
      }
      bool odd = false;
      for (int c = 0; c < p.splits; ++c)
        odd |= __float_as_uint(ld_cluster_f32(cluster_map(smem_u32(odd_values), c))) != 0;
      if (odd) add_odd(rank * each * 4, (rank + 1) * each * 4);
    }
    cluster_sync_all();  // nobody reads this CTA's parts any more
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <int D>
int launch_pp(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, PpParams& p,
              int batch, cudaStream_t stream) {
  using S = PpShape<D>;
  constexpr auto kern = paged_prefill_kernel<D>;
  NPU_TRY_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
  const int n_units = p.q_blocks * (p.q_heads / p.kv_heads / p.hp);
  // Few query tiles leave SMs idle: then a cluster of CTAs shares each pair's keys, as many
  // as run at once, and not more than the longest table has tiles.  A chunk of 40
  // tokens, 32 heads on 8: behind 16384 keys 289 -> 48 us, 4 of them behind 540 21.1 -> 18.2;
  // where the table has room for several tiles and the sequence is one, the cluster costs
  // 2 us (11.8 -> 14.0).
  const long long pairs = static_cast<long long>(batch) * p.kv_heads * ((n_units + 1) / 2);
  const long long keys = static_cast<long long>(p.entries) * p.page_size;
  long long most = (keys + KT - 1) / KT;
  if (p.window > 0) most = std::min(most, (static_cast<long long>(p.window) + 2 * p.bm + p.sinks) / KT + 2);
  p.splits = 1;
  while (p.splits < kMaxSplits && p.splits * 2 <= most &&
         pairs <= clusters_at_once<kern>(p.splits * 2, dim3(kThreads), S::kSmem))
    p.splits *= 2;
  LaunchCfg cfg;
  cfg.cluster = p.splits;
  cfg.grid = dim3(batch * p.kv_heads * p.splits, (n_units + 1) / 2);
  cfg.block = dim3(kThreads);
  cfg.smem = S::kSmem;
  cfg.stream = stream;
  cfg.pdl = true;
  return launch(cfg, kern, qm, km, vm, p);
}

}  // namespace
}  // namespace npu_b200

extern "C" int npu_b200_paged_prefill(const void* d_q, const void* d_k_pages, const void* d_v_pages,
                                      const int32_t* d_page_table, const int32_t* d_seq_lens,
                                      const int32_t* d_q_lens, void* d_out, int batch, int q_heads,
                                      int kv_heads, int head_dim, int queries, int num_pages,
                                      int page_size, int table_entries, int window, int sinks,
                                      float scale, void* stream) {
  using namespace npu_b200;
  clear_error();
  NPU_REQUIRE(d_q && d_k_pages && d_v_pages && d_page_table && d_seq_lens && d_out,
              "paged_prefill: null tensor pointer");
  int rc = check_pages("paged_prefill", kv_heads, head_dim, num_pages, page_size, table_entries);
  if (rc) return rc;
  NPU_REQUIRE(batch >= 1 && static_cast<long long>(batch) * kv_heads < (1ll << 31),
              "paged_prefill: batch %d x kv_heads %d out of range", batch, kv_heads);
  NPU_REQUIRE(q_heads >= kv_heads && q_heads % kv_heads == 0,
              "paged_prefill: q_heads %d is not a multiple of kv_heads %d", q_heads, kv_heads);
  NPU_REQUIRE(queries >= 1, "paged_prefill: queries %d", queries);
  NPU_REQUIRE(static_cast<long long>(batch) * q_heads < (1ll << 31),
              "paged_prefill: batch %d x q_heads %d is too large", batch, q_heads);
  NPU_REQUIRE(window >= 0 && sinks >= 0, "paged_prefill: window %d and sinks %d must not be negative",
              window, sinks);
  NPU_REQUIRE(std::isfinite(scale), "paged_prefill: scale is not finite");
  NPU_REQUIRE(aligned16(d_q) && aligned16(d_k_pages) && aligned16(d_v_pages) && aligned16(d_out),
              "paged_prefill: q, pages and out must be 16-byte aligned");
  PpParams p;
  p.v_pages = static_cast<const __half*>(d_v_pages);
  p.table = d_page_table;
  p.seq_lens = d_seq_lens;
  p.q_lens = d_q_lens;
  p.out = static_cast<__half*>(d_out);
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.queries = queries;
  p.entries = table_entries;
  p.page_size = page_size;
  p.box = page_box(page_size, window > 0 ? kUnit : KT);  // without a window units are in line
  p.num_pages = num_pages;
  const uint64_t rows = static_cast<uint64_t>(num_pages) * kv_heads * page_size;
  p.total_rows = static_cast<int>(rows);
  prefill_blocking(queries, q_heads / kv_heads, &p.bm, &p.hp);
  // Behind a window, more heads of fewer queries, which see fewer keys between them: 64
  // queries on 4 heads see 1087 of a window of 1024, 128 on 2 see 1151 (two chunks up to 2999
  // at head size 64: 77 -> 55 us).  Without one it only costs copies of Q (40 queries of 32
  // heads on 8 behind 16384 keys: 49 -> 52 us).
  while (window > 0 && p.bm > 16 && q_heads / kv_heads % (2 * p.hp) == 0) {
    p.bm /= 2;
    p.hp *= 2;
  }
  p.q_blocks = (queries + p.bm - 1) / p.bm;
  NPU_REQUIRE((static_cast<long long>(p.q_blocks) * (q_heads / kv_heads / p.hp) + 1) / 2 <= 65535,
              "paged_prefill: %d queries make too many query blocks", queries);
  p.window = window;
  p.sinks = sinks;
  // A negative scale negates Q inside the MMA; a scale of 0 is one so small that
  // every visible key weighs the same, while -inf stays -inf.
  p.negate = scale < 0.f;
  p.scale_log2 = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-30f);

  const size_t q_bytes = static_cast<size_t>(batch) * q_heads * queries * head_dim * 2;
  const size_t pool = rows * head_dim * 2;
  NPU_REQUIRE(!overlap(d_q, q_bytes, d_out, q_bytes) && !overlap(d_k_pages, pool, d_out, q_bytes) &&
                  !overlap(d_v_pages, pool, d_out, q_bytes),
              "paged_prefill: out must not overlap q or the pages");
  CUtensorMap qm, km, vm;
  rc = make_tensor_map_3d(&qm, d_q, head_dim, queries, static_cast<uint64_t>(batch) * q_heads,
                          static_cast<uint64_t>(queries) * head_dim * 2, p.bm, 64);
  if (rc) return rc;
  rc = make_tensor_map_2d(&km, d_k_pages, rows, head_dim, p.box, 64);
  if (rc) return rc;
  rc = make_tensor_map_2d(&vm, d_v_pages, rows, head_dim, p.box, 64);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return head_dim == 128 ? launch_pp<128>(qm, km, vm, p, batch, s)
                         : launch_pp<64>(qm, km, vm, p, batch, s);
}
