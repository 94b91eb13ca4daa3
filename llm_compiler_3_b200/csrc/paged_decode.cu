// Attention of one new token per sequence over a paged key-value cache.
//
// Per query head h with KV head h / group and n = seq_lens[b] keys:
//   out[b, h] = softmax_j(scale * q[b, h] . k[j]) v[j]  over the visible keys j
// (paged.cuh), with a running reference m, sum l and output O in FP32 per pass over
// the keys, joined as m = max m_i, l = sum l_i 2^(m_i - m), O = sum O_i 2^(m_i - m).
// The weights are rounded to FP16 as the second MMA's operand (the values are
// FP16 too); the output is rounded once.
//
// Bound: HBM, 4 D bytes per visible key and KV head, whatever the group.  So
// the keys are split by what there is to read, not by sequence: the 32-key
// tiles of every (sequence, KV head, block of 16 query heads) unit form one
// line of tiles, and each CTA (one per SM) takes an equal stretch of it.  Mixed
// lengths, empty slots and one long sequence then load every SM alike; the
// lengths are read on the device, so a captured call follows them.  A unit that
// lies in one stretch is written out at once; the parts of one that crosses a
// border go to the workspace and are joined by a second, dependent launch in
// the order of the stretches (no counters to clear, and no order that changes
// between runs).  Measured: 1.09 GB of ragged lengths up to 8192 in 187 us, 5.8
// TB/s.  What is left is that equal stretches do not take equal time (126 to 193
// us); dealing out the last three tenths in small stretches through a counter
// evened that out and still took as long (188 to 200 us), for the time that each
// change of stretch costs.
//
// Few short units go without the line: a cluster of up to 8 CTAs takes each, and
// joins its parts in distributed shared memory, so that one launch does it all (1 sequence of
// 1001 keys, 32 heads on 8: 6.7 us from call to call).
//
// Inside a stretch every warp takes each WARPS-th tile through its own TMA ring
// (K and V of 32 keys, 128-byte swizzle, one box per page piece: 32 rows, or
// fewer where the page ends inside a tile), running on across units, so that
// the ring stays full while the warps of a finished unit join in shared memory.
// Scores S^T = K Q^T and O^T += V^T P^T run on m16n8k16 MMAs with up to 16
// query heads as the N columns: one pass over K and V serves the whole group.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace npu_b200 {
namespace {

constexpr int kMaxShares = 8;  // CTAs of a cluster
constexpr int kFewTiles = 8;   // tiles of a warp, at most, where clusters take the units

template <int D, int NB>
struct PdShape {
  static constexpr int kTile = 32;                       // keys per warp stage
  // At D = 64 a tile is half the bytes for three quarters of the instructions: twice
  // the warps take it (48 -> 42 us); with 16 query heads their registers and join
  // buffer do not fit twice.
  static constexpr int kWarps = D == 64 && NB == 1 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kHeads = 8 * NB;                  // MMA columns: query heads of a unit
  static constexpr int kRegions = D / 64;                // 128-byte swizzle regions per row
  static constexpr int kRegionBytes = kTile * 128;
  static constexpr int kTileBytes = kTile * D * 2;       // K (or V) of one tile
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = D == 64 && NB == 2 ? 6 : 3;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kJoinFloats = kWarps * kHeads * (D + 3) + 2 * kHeads;
  static constexpr int kBars = kRing + ((kJoinFloats * 4 + 15) & ~15);
  static constexpr size_t kSmem = 1024 + kBars + kWarps * kStages * 8;
};

struct PdParams {
  const __half* q;
  const int32_t* table;
  const int32_t* lens;
  __half* out;
  float* part;      // [CTAs][2][pitch]
  int4* joins;      // [CTAs]: the unit that starts in a CTA's stretch and goes on in the next
  int batch, q_heads, kv_heads, group, chunks;  // chunks: blocks of 8 NB query heads per KV head
  int entries, page_size, box, num_pages, total_rows;
  int window, sinks, pitch;
  int shares;       // CTAs of a cluster that share one unit; 0: stretches of the line
  Divisor by_page;
  float scale_log2;
};

// One sequence's keys, in tiles of T.
template <int T>
struct Keys {
  int len, lo, s;
  TileRange<T> tiles;
  __device__ __forceinline__ void set(const PdParams& p, int b) {
    len = min(max(p.lens[b], 0), p.entries * p.page_size);
    lo = p.window > 0 ? max(0, len - p.window) : 0;
    s = min(p.sinks, lo);
    tiles.set(lo, len, p.sinks);
    tiles.n = max(tiles.n, 1);  // an empty sequence is a tile without visible keys: a zero row
  }
  __device__ __forceinline__ bool sees(int j) const { return j < len && (j >= lo || j < s); }
  // Some key of [j, j + n) is visible / all are.
  __device__ __forceinline__ bool sees_any(int j, int n) const {
    return j < len && (j + n > lo || j < s);
  }
  __device__ __forceinline__ bool sees_all(int j, int n) const {
    return j + n <= len && (j >= lo || j + n <= s);
  }
};

// A place in the line of tiles: tile i of (sequence b, KV head h, block c of its
// query heads).
template <int T>
struct Place {
  int b, h, c, i;
  Keys<T> keys;
  __device__ __forceinline__ void forward(const PdParams& p, int step) {
    i += step;
    while (i >= keys.tiles.n) {
      i -= keys.tiles.n;
      if (++c < p.chunks) continue;
      c = 0;
      if (++h < p.kv_heads) continue;
      h = 0;
      if (++b >= p.batch) return;
      keys.set(p, b);
    }
  }
};

// ldmatrix at a constant distance from an address.
template <int OFF>
__device__ __forceinline__ void ldmatrix_x4_at(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(OFF));
}
template <int OFF>
__device__ __forceinline__ void ldmatrix_x4_trans_at(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(OFF));
}

// A loop whose index is a constant in its body.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<N, I + 1>(f);
  }
}

template <int D, int NB>
__global__ void __launch_bounds__(PdShape<D, NB>::kThreads, 1)
    paged_decode_kernel(const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const PdParams p) {
  using S = PdShape<D, NB>;
  constexpr int KSTEPS = D / 16, DBLK = D / 16, kWarps = S::kWarps;
  constexpr int kTile = S::kTile, MT = kTile / 16;  // 16-key blocks of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* co = reinterpret_cast<float*>(smem + S::kRing);   // [warps][heads][D]
  float* cm = co + kWarps * S::kHeads * D;                 // [warps][heads] maxima
  float* cl = cm + kWarps * S::kHeads;                     // [warps][heads] sums
  float* cw = cl + kWarps * S::kHeads;                     // [warps][heads] weights
  float* cM = cw + kWarps * S::kHeads;                     // [heads]
  float* cL = cM + S::kHeads;                              // [heads]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  // A share's part, O [heads][D] and the heads' maxima and sums, over the ring at the end.
  float* share = reinterpret_cast<float*>(smem);
  __shared__ long long s_sum[kWarps];
  __shared__ long long s_base;
  __shared__ int s_b;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  uint8_t* my_stages = smem + warp * S::kStages * S::kStageBytes;
  uint64_t* my_bars = bars + warp * S::kStages;
  if (lane == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    for (int s = 0; s < S::kStages; ++s) mbar_init(&my_bars[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's stretch [t0, t1) of the line, and where it begins ----
  Place<kTile> at;
  long long t0, t1, per = 1;
  const int units = p.kv_heads * p.chunks;
  if (p.shares > 0) {  // or its share of one unit's tiles
    const int unit = static_cast<int>(blockIdx.x) / p.shares, rank = static_cast<int>(blockIdx.x) % p.shares;
    at.b = unit / units;
    at.h = (unit - at.b * units) / p.chunks;
    at.c = unit - at.b * units - at.h * p.chunks;
    at.keys.set(p, at.b);
    t0 = static_cast<long long>(at.keys.tiles.n) * rank / p.shares;
    t1 = static_cast<long long>(at.keys.tiles.n) * (rank + 1) / p.shares;
    at.i = static_cast<int>(t0);
  } else {
    const int each = (p.batch + kWarps * 32 - 1) / (kWarps * 32);  // sequences per thread
    const int b_first = min(static_cast<int>(threadIdx.x) * each, p.batch);
    const int b_end = min(b_first + each, p.batch);
    long long mine = 0;
    for (int b = b_first; b < b_end; ++b) {
      at.keys.set(p, b);
      mine += static_cast<long long>(at.keys.tiles.n) * units;
    }
    long long upto = mine;  // inclusive scan over the threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += s_sum[w];
      total += s_sum[w];
    }
    per = (total + gridDim.x - 1) / gridDim.x;
    per = max(per, static_cast<long long>(kWarps));  // no warp without a tile
    t0 = blockIdx.x * per;
    t1 = min(total, t0 + per);
    if (threadIdx.x == 0) p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
    if (t0 >= t1) return;
    if (t0 >= upto - mine && t0 < upto) {  // exactly one thread
      long long base = upto - mine;
      for (int b = b_first; b < b_end; ++b) {
        at.keys.set(p, b);
        const long long n = static_cast<long long>(at.keys.tiles.n) * units;
        if (t0 < base + n) {
          s_b = b;
          s_base = base;
          break;
        }
        base += n;
      }
    }
    __syncthreads();
    at.b = s_b;
    at.keys.set(p, at.b);
    {
      const long long rem = t0 - s_base;
      const int unit = static_cast<int>(rem / at.keys.tiles.n);
      at.i = static_cast<int>(rem - static_cast<long long>(unit) * at.keys.tiles.n);
      at.h = unit / p.chunks;
      at.c = unit - at.h * p.chunks;
    }
  }
  const int n_mine = static_cast<int>(t1 - t0);
  const int my_tiles = n_mine > warp ? (n_mine - warp + kWarps - 1) / kWarps : 0;

  // ---- the ring: each lane issues one box of K or V ----
  const int boxes = kTile / p.box;
  const int combos = boxes * S::kRegions * 2;
  const int my_box = lane / (S::kRegions * 2), my_region = (lane >> 1) % S::kRegions;
  const bool my_v = lane & 1;
  Place<kTile> ahead = at;
  ahead.forward(p, warp);
  // This lane's box of the tile at `ahead`: its page (-2: no visible key in it), and
  // its row from the page's first.
  int page = -2, row_in_page = 0;
  const int page_rows = p.kv_heads * p.page_size;
  auto look_up = [&]() {
    const int j = ahead.keys.tiles.key0(ahead.i) + my_box * p.box;
    const int entry = p.by_page.quotient(j);
    row_in_page = ahead.h * p.page_size + j - entry * p.page_size;
    page = -2;
    if (lane < combos && ahead.keys.sees_any(j, p.box))
      page = p.table[static_cast<size_t>(ahead.b) * p.entries + entry];
  };
  auto issue = [&](int k, int st) {
    if (lane == 0) mbar_arrive_expect_tx(&my_bars[st], S::kStageBytes);
    __syncwarp();
    if (lane < combos) {
      int row = p.total_rows;  // past the pool: the box is filled with zeros
      if (page >= 0 && page < p.num_pages)
        row = page * page_rows + row_in_page;
      else if (page != -2)
        report_error(kDevErrBounds);
      uint8_t* dst = my_stages + st * S::kStageBytes + (my_v ? S::kTileBytes : 0) +
                     my_region * S::kRegionBytes + my_box * p.box * 128;
      tma_load_2d(dst, my_v ? &vmap : &kmap, &my_bars[st], my_region * 64, row);
    }
    if (k + 1 < my_tiles) {
      ahead.forward(p, kWarps);
      look_up();
    }
  };
  if (my_tiles > 0) look_up();
  int issued = 0;
  for (; issued < my_tiles && issued < S::kStages; ++issued) issue(issued, issued);

  // This lane's part of the ldmatrix addresses: chunk x of row r lies at x ^ (r % 8).
  uint32_t k_at[4], v_at[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int k_row = lane & 15, v_row = (lane & 7) + ((lane >> 4) << 3);
    k_at[x] = k_row * 128 + (((2 * x + (lane >> 4)) ^ (k_row & 7)) << 4);
    v_at[x] = v_row * 128 + (((2 * x + ((lane >> 3) & 1)) ^ (v_row & 7)) << 4);
  }

  // ---- the stretch, unit by unit ----
  int k = 0;  // this warp's next tile, in stage `st` at its `phase`-th turn
  int st = 0;
  uint32_t phase = 0;
  bool bad = false;
  for (int done = 0; done < n_mine;) {
    const int here = min(at.keys.tiles.n - at.i, n_mine - done);  // tiles of this unit
    const int heads = min(S::kHeads, p.group - at.c * S::kHeads);
    const size_t q_row = static_cast<size_t>(at.b) * p.q_heads + at.h * p.group + at.c * S::kHeads;

    // Q^T fragments: column n = query head n of the block, zero past it.
    uint32_t qf[NB][KSTEPS][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const __half* qh = p.q + (q_row + nb * 8 + g) * D;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        const bool ok = nb * 8 + g < heads;
        qf[nb][s][0] = ok ? *reinterpret_cast<const uint32_t*>(qh + 16 * s + 2 * c) : 0u;
        qf[nb][s][1] = ok ? *reinterpret_cast<const uint32_t*>(qh + 16 * s + 2 * c + 8) : 0u;
      }
    }
    float m_run[NB][2], l_run[NB][2], o[NB][DBLK][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m_run[nb][0] = m_run[nb][1] = -INFINITY;
      l_run[nb][0] = l_run[nb][1] = 0.f;
#pragma unroll
      for (int d = 0; d < DBLK; ++d) o[nb][d][0] = o[nb][d][1] = o[nb][d][2] = o[nb][d][3] = 0.f;
    }

    for (; !bad && k * kWarps + warp < done + here; ++k) {
      if (!__all_sync(0xffffffffu, mbar_wait(&my_bars[st], phase, kDevErrTmaTimeout))) {
        bad = true;
        break;
      }
      const int key0 = at.keys.tiles.key0(at.i + k * kWarps + warp - done);
      const bool whole = at.keys.sees_all(key0, kTile);
      uint8_t* kst = my_stages + st * S::kStageBytes;
      const uint32_t kbase = smem_u32(kst), vbase = kbase + S::kTileBytes;
      if (!whole) {
        // A hidden row may hold anything; its weight is 0, but 0 * NaN is NaN.
        for (int row = lane; row < kTile; row += 32)
          if (!at.keys.sees(key0 + row)) {
#pragma unroll
            for (int r = 0; r < S::kRegions; ++r)
              for (int x = 0; x < 128; x += 16)
                *reinterpret_cast<uint4*>(kst + S::kTileBytes + r * S::kRegionBytes + row * 128 + x) =
                    make_uint4(0, 0, 0, 0);
          }
        __syncwarp();
      }

      // scores S^T[key, head] of the 16-key blocks
      float sv[MT][NB][4] = {};
      unrolled<MT>([&](auto mt) {
        unrolled<KSTEPS>([&](auto s) {
          uint32_t a[4];
          ldmatrix_x4_at<(s / 4) * S::kRegionBytes + mt * 2048>(a, kbase + k_at[s % 4]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            mma_16816(sv[mt][nb], a[0], a[1], a[2], a[3], qf[nb][s][0], qf[nb][s][1]);
        });
      });
      // Online softmax, in the base-2 logarithm's domain.  A column's reference moves only
      // when a weight would pass 2^15: then, and only then, the lanes of a column compare notes
      // and O is rescaled.
      bool grows = false;
      float most[NB][2];  // scores that need no other reference
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          most[nb][j] = m_run[nb][j] + kMostLog2;
          if (most[nb][j] - m_run[nb][j] > kMostLog2) most[nb][j] = m_run[nb][j];  // rounded up
        }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = sv[mt][nb][r] * p.scale_log2;
            if (!whole && !at.keys.sees(key0 + mt * 16 + g + ((r & 2) ? 8 : 0))) v = -INFINITY;
            sv[mt][nb][r] = v;
            grows |= v > most[nb][r & 1];
          }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float alpha[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) top = max3(top, sv[mt][nb][j], sv[mt][nb][2 + j]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            alpha[j] = 1.f;
            if (top > most[nb][j]) {
              top -= kBelowMax;
              alpha[j] = m_run[nb][j] == -INFINITY ? 0.f : fast_exp2(m_run[nb][j] - top);
              m_run[nb][j] = top;
              l_run[nb][j] *= alpha[j];
            }
          }
#pragma unroll
          for (int d = 0; d < DBLK; ++d) {
            o[nb][d][0] *= alpha[0];
            o[nb][d][1] *= alpha[1];
            o[nb][d][2] *= alpha[0];
            o[nb][d][3] *= alpha[1];
          }
        }
      }
      uint32_t pb[MT][NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float m_use[2];  // no key seen yet: all scores are -inf
#pragma unroll
        for (int j = 0; j < 2; ++j) m_use[j] = m_run[nb][j] == -INFINITY ? 0.f : m_run[nb][j];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            w[r] = fast_exp2(sv[mt][nb][r] - m_use[r & 1]);
            l_run[nb][r & 1] += w[r];
          }
          pb[mt][nb][0] = movmatrix_trans(pack_half2(w[0], w[1]));
          pb[mt][nb][1] = movmatrix_trans(pack_half2(w[2], w[3]));
        }
      }
      // O^T[dim, head] += V^T P^T
      unrolled<MT>([&](auto mt) {
        unrolled<DBLK>([&](auto d) {
          uint32_t a[4];
          ldmatrix_x4_trans_at<(d / 4) * S::kRegionBytes + mt * 2048>(a, vbase + v_at[d % 4]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            mma_16816(o[nb][d], a[0], a[1], a[2], a[3], pb[mt][nb][0], pb[mt][nb][1]);
        });
      });
      __syncwarp();
      if (issued < my_tiles) {
        if (!whole) fence_proxy_async_smem();  // the zero-fill precedes the next TMA write
        issue(issued++, st);
      }
      if (++st == S::kStages) {
        st = 0;
        phase ^= 1;
      }
    }

    // ---- the warps' parts of this unit join ----
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = l_run[nb][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int head = nb * 8 + 2 * c + j;
        if (g == 0) {
          cm[warp * S::kHeads + head] = m_run[nb][j];
          cl[warp * S::kHeads + head] = l;
        }
        float* oh = co + (warp * S::kHeads + head) * D;
#pragma unroll
        for (int d = 0; d < DBLK; ++d) {
          oh[16 * d + g] = o[nb][d][j];
          oh[16 * d + g + 8] = o[nb][d][2 + j];
        }
      }
    bad = __syncthreads_or(bad);
    if (bad) break;
    if (threadIdx.x < heads) {
      const int head = threadIdx.x;
      float mx = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, cm[w * S::kHeads + head]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = cm[w * S::kHeads + head];
        const float wt = mw == -INFINITY ? 0.f : fast_exp2(mw - mx);
        cw[w * S::kHeads + head] = wt;
        L += cl[w * S::kHeads + head] * wt;
      }
      cM[head] = mx;
      cL[head] = L;
    }
    __syncthreads();
    const bool alone = p.shares < 2 && at.i == 0 && here == at.keys.tiles.n;
    float* slot = p.shares > 0 ? share : p.part + (static_cast<size_t>(blockIdx.x) * 2 + (done == 0 ? 0 : 1)) * p.pitch;
    for (int x = threadIdx.x; x < heads * D / 4; x += kWarps * 32) {
      const int head = x * 4 / D, dim = x * 4 - head * D;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float wt = cw[w * S::kHeads + head];
        const float4 v = *reinterpret_cast<const float4*>(co + (w * S::kHeads + head) * D + dim);
        O.x += v.x * wt;
        O.y += v.y * wt;
        O.z += v.z * wt;
        O.w += v.w * wt;
      }
      if (alone) {
        const float L = cL[head], inv = L == 0.f ? 0.f : 1.f / L;
        *reinterpret_cast<uint2*>(p.out + (q_row + head) * D + dim) =
            make_uint2(pack_half2(O.x * inv, O.y * inv), pack_half2(O.z * inv, O.w * inv));
      } else {
        *reinterpret_cast<float4*>(slot + head * D + dim) = O;
        if (dim == 0) {
          slot[S::kHeads * D + head] = cM[head];
          slot[S::kHeads * D + S::kHeads + head] = cL[head];
        }
      }
    }
    // A unit that begins here and goes on in the next stretches: its parts are
    // this slot and the first slots of the CTAs that follow.
    if (threadIdx.x == 0 && at.i == 0 && here < at.keys.tiles.n && p.shares == 0) {
      const int others = static_cast<int>((at.keys.tiles.n - here + per - 1) / per);
      p.joins[blockIdx.x] = make_int4(1 + others, static_cast<int>(q_row), heads, done == 0 ? 0 : 1);
    }
    done += here;
    if (p.shares > 0) break;
    at.forward(p, here);
    __syncthreads();  // the join buffer is free again
  }
  if (p.shares > 1) {
    // ---- the cluster's parts of the unit join, each CTA's share of the output ----
    const int heads = min(S::kHeads, p.group - at.c * S::kHeads);
    if (n_mine == 0 && threadIdx.x < S::kHeads) {  // no part: a sum that none has
      share[S::kHeads * D + threadIdx.x] = -INFINITY;
      share[S::kHeads * D + S::kHeads + threadIdx.x] = -1.f;
    }
    cluster_sync_all();
    const int rank = static_cast<int>(blockIdx.x) % p.shares;
    const size_t q_row = static_cast<size_t>(at.b) * p.q_heads + at.h * p.group + at.c * S::kHeads;
    for (int x = rank * S::kThreads + threadIdx.x; x < heads * D / 4; x += p.shares * S::kThreads) {
      const int head = x * 4 / D, dim = x * 4 - head * D;
      float m[kMaxShares], l[kMaxShares], mx = -INFINITY, L = 0.f;
      float4 v[kMaxShares], O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kMaxShares; ++c) {  // all loads in flight together
        m[c] = -INFINITY;
        l[c] = -1.f;
        if (c >= p.shares) continue;
        const uint32_t ml = cluster_map(smem_u32(share + S::kHeads * D + head), c);
        m[c] = ld_cluster_f32(ml);
        l[c] = ld_cluster_f32(ml + S::kHeads * 4);
        v[c] = ld_cluster_v4(cluster_map(smem_u32(share + head * D + dim), c));
        mx = fmaxf(mx, m[c]);
      }
#pragma unroll
      for (int c = 0; c < kMaxShares; ++c) {
        if (l[c] < 0.f) continue;
        // Weight 0 is no reason to leave a part out: one whose scores are all NaN has no
        // maximum either, and its sum and O are NaN.
        const float wt = m[c] == -INFINITY ? 0.f : fast_exp2(m[c] - mx);
        L += wt * l[c];
        O.x += v[c].x * wt;
        O.y += v[c].y * wt;
        O.z += v[c].z * wt;
        O.w += v[c].w * wt;
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      *reinterpret_cast<uint2*>(p.out + (q_row + head) * D + dim) =
          make_uint2(pack_half2(O.x * inv, O.y * inv), pack_half2(O.z * inv, O.w * inv));
    }
    cluster_sync_all();  // nobody reads this CTA's part any more
  }
  if (bad) {  // leave no copy in flight into this CTA's shared memory
    for (; k < issued; ++k)
      mbar_wait(&my_bars[k % S::kStages], (k / S::kStages) & 1, kDevErrTmaTimeout);
  }
}

// Block (x, y): head y of the unit that begins in stretch x and goes on after
// it.  Thread d sums dimension d over the parts, in the order of the stretches.
template <int D, int NB>
__global__ void __launch_bounds__(D) paged_decode_join_kernel(const PdParams p) {
  constexpr int kHeads = 8 * NB;
  pdl_launch_dependents();
  pdl_wait();
  const int4 join = p.joins[blockIdx.x];
  const int parts = join.x, head = blockIdx.y;
  if (parts == 0 || head >= join.z) return;
  const float* first = p.part + (static_cast<size_t>(blockIdx.x) * 2 + join.w) * p.pitch;
  const float* next = p.part + (static_cast<size_t>(blockIdx.x) + 1) * 2 * p.pitch;
  auto part = [&](int i) { return i == 0 ? first : next + static_cast<size_t>(i - 1) * 2 * p.pitch; };
  float mx = -INFINITY;
  for (int i = 0; i < parts; ++i) mx = fmaxf(mx, part(i)[kHeads * D + head]);
  float L = 0.f, O = 0.f;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float* s = part(i);
    const float m = s[kHeads * D + head];
    const float wt = m == -INFINITY ? 0.f : fast_exp2(m - mx);
    L += wt * s[kHeads * D + kHeads + head];
    O += wt * s[head * D + threadIdx.x];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  p.out[(static_cast<size_t>(join.y) + head) * D + threadIdx.x] = __float2half_rn(O * inv);
}

template <int D, int NB>
int launch_pd(const CUtensorMap& km, const CUtensorMap& vm, PdParams& p, long long most, cudaStream_t stream) {
  using S = PdShape<D, NB>;
  constexpr auto kern = paged_decode_kernel<D, NB>;
  NPU_TRY_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(S::kSmem)));
  LaunchCfg cfg;
  cfg.block = dim3(S::kThreads);
  cfg.smem = S::kSmem;
  cfg.stream = stream;
  cfg.pdl = true;
  // Few units of few tiles: a cluster to each, its CTAs sharing the keys and joining
  // through distributed shared memory, in one launch.  32 heads on 8, 1 sequence of 1000
  // keys 7.5 -> 6.3 us, of 4000 12.8 -> 9.3, 16 of up to 500 16.0 -> 8.3; the line is the
  // faster one again from some 8 tiles a warp (12000 keys: 17.1, with clusters 19.3), where
  // its even stretches and all SMs are worth a second launch.
  const long long units = static_cast<long long>(p.batch) * p.kv_heads * p.chunks;
  int shares = 1;
  while (shares < kMaxShares && shares * S::kWarps < most &&
         units <= clusters_at_once<kern>(shares * 2, cfg.block, cfg.smem))
    shares *= 2;
  if (units <= sm_count() && most <= static_cast<long long>(kFewTiles) * S::kWarps * shares) {
    p.shares = shares;
    cfg.grid = dim3(static_cast<unsigned>(units) * shares);
    cfg.cluster = shares;
    return launch(cfg, kern, km, vm, p);
  }
  p.shares = 0;
  const int ctas = static_cast<int>(std::min<long long>(sm_count(), (most * units + S::kWarps - 1) / S::kWarps));
  cfg.grid = dim3(ctas);
  int rc = launch(cfg, kern, km, vm, p);
  if (rc) return rc;
  LaunchCfg join;
  join.grid = dim3(ctas, p.group < S::kHeads ? p.group : S::kHeads);
  join.block = dim3(D);
  join.stream = stream;
  join.pdl = true;
  return launch(join, paged_decode_join_kernel<D, NB>, p);
}

// Floats of one part: O [heads][D], m [heads], l [heads].
int pd_pitch(int group, int head_dim) {
  const int heads = group <= 8 ? 8 : 16;
  return heads * (head_dim + 2);
}

}  // namespace

size_t paged_decode_workspace(int q_heads, int kv_heads, int head_dim) {
  if (kv_heads < 1 || q_heads < kv_heads || head_dim < 1) return 0;
  const size_t ctas = static_cast<size_t>(sm_count());
  return ctas * (sizeof(int4) + 2 * sizeof(float) * pd_pitch(q_heads / kv_heads, head_dim));
}

}  // namespace npu_b200

extern "C" size_t npu_b200_paged_decode_workspace_size(int q_heads, int kv_heads, int head_dim) {
  return npu_b200::paged_decode_workspace(q_heads, kv_heads, head_dim);
}

extern "C" int npu_b200_paged_decode(const void* d_q, const void* d_k_pages, const void* d_v_pages,
                                     const int32_t* d_page_table, const int32_t* d_seq_lens,
                                     void* d_out, int batch, int q_heads, int kv_heads,
                                     int head_dim, int num_pages, int page_size, int table_entries,
                                     int window, int sinks, float scale, void* d_workspace,
                                     size_t workspace_bytes, void* stream) {
  using namespace npu_b200;
  clear_error();
  NPU_REQUIRE(d_q && d_k_pages && d_v_pages && d_page_table && d_seq_lens && d_out,
              "paged_decode: null tensor pointer");
  int rc = check_pages("paged_decode", kv_heads, head_dim, num_pages, page_size, table_entries);
  if (rc) return rc;
  NPU_REQUIRE(batch >= 1 && batch <= 1 << 20, "paged_decode: batch %d out of range", batch);
  NPU_REQUIRE(q_heads >= kv_heads && q_heads % kv_heads == 0,
              "paged_decode: q_heads %d is not a multiple of kv_heads %d", q_heads, kv_heads);
  NPU_REQUIRE(static_cast<long long>(batch) * q_heads < (1ll << 31),
              "paged_decode: batch %d x q_heads %d is too large", batch, q_heads);
  NPU_REQUIRE(window >= 0 && sinks >= 0, "paged_decode: window %d and sinks %d must not be negative",
              window, sinks);
  NPU_REQUIRE(std::isfinite(scale), "paged_decode: scale is not finite");
  NPU_REQUIRE(aligned16(d_q) && aligned16(d_k_pages) && aligned16(d_v_pages) && aligned16(d_out) &&
                  aligned16(d_workspace),
              "paged_decode: q, pages, out and workspace must be 16-byte aligned");
  const size_t need = paged_decode_workspace(q_heads, kv_heads, head_dim);
  NPU_REQUIRE(d_workspace && workspace_bytes >= need,
              "paged_decode: workspace of %zu bytes needed, %zu given", need, workspace_bytes);

  const size_t q_bytes = static_cast<size_t>(batch) * q_heads * head_dim * 2;
  const uint64_t rows = static_cast<uint64_t>(num_pages) * kv_heads * page_size;
  const size_t pool = rows * head_dim * 2;
  NPU_REQUIRE(!overlap(d_q, q_bytes, d_out, q_bytes) && !overlap(d_k_pages, pool, d_out, q_bytes) &&
                  !overlap(d_v_pages, pool, d_out, q_bytes),
              "paged_decode: out must not overlap q or the pages");

  const int tile = head_dim == 128 ? PdShape<128, 1>::kTile : PdShape<64, 1>::kTile;
  const int box = page_box(page_size, tile);
  CUtensorMap km, vm;
  rc = make_tensor_map_2d(&km, d_k_pages, rows, head_dim, box, 64);
  if (rc) return rc;
  rc = make_tensor_map_2d(&vm, d_v_pages, rows, head_dim, box, 64);
  if (rc) return rc;

  PdParams p;
  p.q = static_cast<const __half*>(d_q);
  p.table = d_page_table;
  p.lens = d_seq_lens;
  p.out = static_cast<__half*>(d_out);
  p.batch = batch;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads;
  const int heads = p.group <= 8 ? 8 : 16;
  p.chunks = (p.group + heads - 1) / heads;
  p.entries = table_entries;
  p.page_size = page_size;
  p.by_page = Divisor::of(page_size);
  p.box = box;
  p.num_pages = num_pages;
  p.total_rows = static_cast<int>(rows);
  p.window = window;
  p.sinks = sinks;
  p.pitch = pd_pitch(p.group, head_dim);
  p.scale_log2 = scale * 1.4426950408889634f;
  // No more CTAs than the longest table could keep busy.
  long long most = (static_cast<long long>(table_entries) * page_size + tile - 1) / tile;
  if (window > 0)
    most = std::min(most, static_cast<long long>(window) / tile + sinks / tile + 4);
  NPU_REQUIRE(most * batch * kv_heads * p.chunks < 1ll << 36,
              "paged_decode: a batch of %d over tables of %d entries is too large", batch, table_entries);
  p.joins = static_cast<int4*>(d_workspace);
  p.part = reinterpret_cast<float*>(p.joins + sm_count());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    return heads == 8 ? launch_pd<128, 1>(km, vm, p, most, s) : launch_pd<128, 2>(km, vm, p, most, s);
  return heads == 8 ? launch_pd<64, 1>(km, vm, p, most, s) : launch_pd<64, 2>(km, vm, p, most, s);
}
