// Beam search: the choice of the next beams over beams x vocabulary, and the
// reordering of per-beam states.
//
// With x[w, t] the logits of beam w, M = max_t x and S = sum_t e^(x - M), token t
// of beam w is worth ((x - M) - ln S) + score[w]; a finished beam is worth its
// score, as the end token.  The `width` largest are chosen over all beams of a
// sequence, the lowest w * vocab + t among equals.
//
// Bound: one pass over the logits (HBM); next to it the exponentials, of which
// an SM does 16 a clock against the ~12 FP16 logits a clock that HBM brings it.
// So one pass does both: each warp streams its part of a row, 16 bytes per lane,
// keeps the sum relative to its running maximum, and holds its `width` best logits
// sorted across its lanes.  A logit is looked at only if it is a new maximum or
// reaches a floor that `width` others are known to reach: at first the width-th
// largest of the CTA's lanes' maxima over their first words, then the worst kept one
// of any warp.  So maximum and selection cost one comparison per 8 logits and a few
// insertions (with floors that each warp knew alone they cost twice the rest).  A second, dependent launch joins the stretches.
//
// Which of two candidates is larger decides whole beams, so what follows the
// stretches (the sum over them, its logarithm, the candidates' worth) is in FP64;
// within a stretch the FP32 sum of up to 2^-22-exact exponentials leaves ln S
// some 1e-7 off.
#include <float.h>
#include <limits.h>

#include <algorithm>

#include "common.cuh"
#include "host.hpp"

namespace npu_b200 {
namespace {

constexpr int kMaxWidth = 32;   // candidates kept: one per lane
constexpr int kMaxBeams = 32;   // beams of a sequence: one per lane in the join
constexpr int kMaxSplits = 128; // stretches of a row
constexpr int kStaged = 512;    // entries of a row's lists that the join keeps in shared memory
constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamParams {
  const void* logits;
  const float* scores;
  const uint8_t* done;  // or null
  float* out_scores;
  int32_t* out_tokens;
  int32_t* out_parents;
  uint8_t* out_done;    // or null
  // Stretch s of row r: maximum, sum, and the best logits with their tokens.
  float* part_max;      // [rows][splits]
  float* part_sum;
  float* part_val;      // [rows][splits][width]
  int32_t* part_idx;
  int beams, vocab, width, splits, words;  // words: 16-byte words of a stretch
  int eos;
  long long total;      // logits of the tensor
};

// The best logits of a warp, in falling order across its lanes: larger first,
// lower token among equals.  Lanes past `width` hold what fell out.
struct Best {
  float val = -INFINITY;
  int idx = INT_MAX;
  float floor = -INFINITY;  // the worst kept: lane width - 1, in every lane
  int floor_idx = INT_MAX;
  __device__ __forceinline__ bool takes(float v, int i) const {
    return v > floor || (v == floor && i < floor_idx && v > -INFINITY);
  }
  // One candidate, the same in every lane.
  __device__ __forceinline__ void put(float v, int i, int width) {
    const int lane = threadIdx.x & 31;
    const bool before = val > v || (val == v && idx < i);
    const int at = __popc(__ballot_sync(0xffffffffu, before));
    const float up_v = __shfl_up_sync(0xffffffffu, val, 1);
    const int up_i = __shfl_up_sync(0xffffffffu, idx, 1);
    if (lane > at) {
      val = up_v;
      idx = up_i;
    } else if (lane == at) {
      val = v;
      idx = i;
    }
    floor = __shfl_sync(0xffffffffu, val, width - 1);
    floor_idx = __shfl_sync(0xffffffffu, idx, width - 1);
  }
  // Each lane offers one.
  __device__ __forceinline__ void offer(float v, int i, int width) {
    unsigned mask = __ballot_sync(0xffffffffu, takes(v, i));
    while (mask) {
      const int src = __ffs(mask) - 1;
      put(__shfl_sync(0xffffffffu, v, src), __shfl_sync(0xffffffffu, i, src), width);
      mask = __ballot_sync(0xffffffffu, takes(v, i)) & ~((2u << src) - 1);
    }
  }
};

// Whole numbers in the order of the floating ones (-0 as 0).
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The `width` largest of the lanes' values in falling order (equal ones each):
// lane k < width returns the k-th.
__device__ __forceinline__ float best_of_lanes(float v, int width) {
  const int lane = threadIdx.x & 31;
  uint32_t k = order_of(v), mine = order_of(-INFINITY);
  for (int i = 0; i < width; ++i) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, k);
    const unsigned who = __ballot_sync(0xffffffffu, k == top);
    if (lane == __ffs(who) - 1) k = 0;
    if (lane == i) mine = top;
  }
  return of_order(mine);
}

// The `width` best of `lists` lists in falling order, one to a lane (list l of lane
// l, l + 32, ...): `width` times the best head is taken.  val(l, i) and idx(l, i) are
// read as the heads move; a list ends at -inf or at `width`.  Lane k returns the k-th.
template <typename Val, typename Idx>
__device__ __forceinline__ void merge_lists(int lists, int width, Val val, Idx idx, float* out_v,
                                            int* out_i) {
  const int lane = threadIdx.x & 31;
  float v = -INFINITY;
  int t = INT_MAX, from = 0;  // this lane's best head
  int at[kMaxSplits / 32] = {};
  auto refill = [&]() {
    v = -INFINITY;
    t = INT_MAX;
#pragma unroll
    for (int u = 0; u < kMaxSplits / 32; ++u) {
      const int l = lane + 32 * u;
      if (l < lists && at[u] < width) {
        const float hv = val(l, at[u]);
        const int hi = idx(l, at[u]);
        if (hv > v || (hv == v && hi < t)) {
          v = hv;
          t = hi;
          from = u;
        }
      }
    }
  };
  refill();
  *out_v = -INFINITY;
  *out_i = INT_MAX;
  for (int k = 0; k < width; ++k) {
    const uint32_t key = order_of(v);
    const uint32_t top = __reduce_max_sync(0xffffffffu, key);
    const int low = __reduce_min_sync(0xffffffffu, key == top ? t : INT_MAX);
    if (lane == k) {
      *out_v = of_order(top);
      *out_i = low;
    }
    if (key == top && t == low && v > -INFINITY) {
#pragma unroll
      for (int u = 0; u < kMaxSplits / 32; ++u)
        if (u == from) ++at[u];
      refill();
    }
  }
}

// NaN counts as -inf, +inf as the largest number of the type.
__device__ __forceinline__ void widen(const uint4& w, float (&x)[8], const __half*) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  const __half2 low = __half2half2(__ushort_as_half(0xfc00)), high = __half2half2(__ushort_as_half(0x7bff));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(__hmin2(__hmax2(*reinterpret_cast<const __half2*>(&u[i]), low), high));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void widen(const uint4& w, float (&x)[4], const float*) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fminf(fmaxf(__uint_as_float(u[i]), -INFINITY), FLT_MAX);
}

// The 16-byte word `w` of a tensor of `total` logits; the last one may reach past
// its end and is then put together one by one, zero behind it.
template <typename T>
__device__ __forceinline__ uint4 tensor_word(const T* logits, long long w, long long total) {
  constexpr int L = 16 / sizeof(T);
  uint4 v = make_uint4(0, 0, 0, 0);
  if ((w + 1) * L <= total) {
    v = __ldg(reinterpret_cast<const uint4*>(logits) + w);
  } else {
    T part[L];
#pragma unroll
    for (int i = 0; i < L; ++i) part[i] = w * L + i < total ? logits[w * L + i] : T(0.f);
    memcpy(&v, part, 16);
  }
  return v;
}

// 16 bytes from byte 2 `halves` of the 32 bytes a, b (the same in every lane).
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int halves) {
  uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (halves & 4) {
#pragma unroll
    for (int i = 0; i < 6; ++i) u[i] = u[i + 2];
  }
  if (halves & 2) {
#pragma unroll
    for (int i = 0; i < 5; ++i) u[i] = u[i + 1];
  }
  if (halves & 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __funnelshift_r(u[i], u[i + 1], 16);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// Block (s, row): stretch s of row `row`, a piece per warp.
template <typename T>
__global__ void __launch_bounds__(kSelThreads, 4) beam_stretch_kernel(const BeamParams p) {
  constexpr int L = 16 / sizeof(T);  // logits of a word
  __shared__ float s_val[kSelWarps][32], s_max[kSelWarps], s_sum[kSelWarps];
  __shared__ int s_idx[kSelWarps][32];
  __shared__ uint32_t s_floor;  // order_of() of what `width` logits of the row reach
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.y;
  if (threadIdx.x == 0) s_floor = 0;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  if (p.done != nullptr && p.done[row]) return;  // the join does not look at its stretches
  const T* logits = static_cast<const T*>(p.logits);
  // Which lane adds which token goes by the token alone, so that equal rows have
  // equal sums to the last bit, and their continuations tie.  A row that does not
  // begin on a 16-byte border takes each of its words from two.
  const long long first = row * p.vocab / L;
  const int lead = static_cast<int>(row * p.vocab - first * L);
  const int words = (p.vocab + L - 1) / L;
  const int w_begin = min(static_cast<int>(blockIdx.x) * p.words, words);
  const int w_end = min(w_begin + p.words, words);

  Best best;
  float m = -FLT_MAX, sum = 0.f;  // of the warp, and the lane's share
  constexpr int kAhead = 4;
  constexpr int kTurn = 32 * kAhead;  // words that a warp loads together
  const int turns = (w_end - w_begin + kSelWarps * kTurn - 1) / (kSelWarps * kTurn);
  for (int turn = 0; turn < turns; ++turn) {  // every warp takes every turn
    const int w0 = w_begin + (turn * kSelWarps + warp) * kTurn;
    // A turn inside the stretch, the row and the tensor needs no checks.
    const bool inside = w0 + kTurn <= w_end && (w0 + kTurn) * L <= p.vocab;
    uint4 raw[kAhead];
    if (inside) {
      const uint4* src = reinterpret_cast<const uint4*>(logits) + first + w0 + lane;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) raw[u] = __ldg(src + u * 32);
    } else {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        raw[u] = tensor_word(logits, first + min(w0 + u * 32 + lane, w_end - 1), p.total);
    }
    if (lead != 0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        raw[u] = shifted(raw[u], tensor_word(logits, first + min(w0 + u * 32 + lane, w_end - 1) + 1, p.total),
                         lead * static_cast<int>(sizeof(T)) / 2);
    }
    auto logits_of = [&](int u, float(&x)[L]) {
      widen(raw[u], x, logits);
      if (!inside) {
        const int n = w0 + u * 32 + lane < w_end ? p.vocab - (w0 + u * 32 + lane) * L : 0;
#pragma unroll
        for (int i = 0; i < L; ++i)
          if (i >= n) x[i] = -INFINITY;
      }
      float top = max3(x[0], x[1], max3(x[2], x[3], x[L - 1]));
      if (L == 8) top = max3(top, x[4 % L], max3(x[5 % L], x[6 % L], top));
      return top;
    };
    if (turn == 0) {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        float x[L];
        top = fmaxf(top, logits_of(u, x));
      }
      m = fmaxf(m, of_order(__reduce_max_sync(0xffffffffu, order_of(top))));
      s_val[warp][lane] = best_of_lanes(top, p.width);
      __syncthreads();
      if (warp == 0) {  // the warps' lists into one: its last is the first floor
        float val;
        int idx;
        merge_lists(kSelWarps, p.width, [&](int l, int i) { return s_val[l][i]; },
                    [&](int l, int) { return l; }, &val, &idx);
        val = __shfl_sync(0xffffffffu, val, p.width - 1);
        if (lane == 0) s_floor = order_of(val);
      }
      __syncthreads();
    }
    float floor = of_order(max(order_of(best.floor), *const_cast<volatile uint32_t*>(&s_floor)));
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float x[L];
      const float top = logits_of(u, x);
      if (__any_sync(0xffffffffu, top >= floor || top > m)) {
        const float m_new = fmaxf(m, of_order(__reduce_max_sync(0xffffffffu, order_of(top))));
        sum *= fast_exp2((m - m_new) * kLog2e);
        m = m_new;
        const int t0 = (w0 + u * 32 + lane) * L;  // token of the word's first logit
#pragma unroll
        for (int i = 0; i < L; ++i) best.offer(x[i] >= floor ? x[i] : -INFINITY, t0 + i, p.width);
        if (best.floor > floor) {
          floor = best.floor;
          if (lane == 0) atomicMax(&s_floor, order_of(floor));
        }
      }
      const uint64_t minus2 = pack2(-m, -m), log2e2 = pack2(kLog2e, kLog2e);
      uint64_t s2 = 0;
#pragma unroll
      for (int i = 0; i < L; i += 2) {
        const uint64_t d2 = mul2(add2(pack2(x[i], x[i + 1]), minus2), log2e2);
        s2 = add2(s2, pack2(fast_exp2(lo2(d2)), fast_exp2(hi2(d2))));
      }
      sum += lo2(s2) + hi2(s2);
    }
  }
  // The lanes' sums, then the warps'.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  s_val[warp][lane] = best.val;
  s_idx[warp][lane] = best.idx;
  if (lane == 0) {
    s_max[warp] = m;
    s_sum[warp] = sum;
  }
  __syncthreads();
  if (warp != 0) return;
  float m_all = -FLT_MAX, sum_all = 0.f;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) m_all = fmaxf(m_all, s_max[w]);
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) sum_all += s_sum[w] * fast_exp2((s_max[w] - m_all) * kLog2e);
  float val;
  int idx;
  merge_lists(kSelWarps, p.width, [&](int l, int i) { return s_val[l][i]; },
              [&](int l, int i) { return s_idx[l][i]; }, &val, &idx);
  const long long at = row * p.splits + blockIdx.x;
  if (lane == 0) {
    p.part_max[at] = m_all;
    p.part_sum[at] = sum_all;
  }
  if (lane < p.width) {
    p.part_val[at * p.width + lane] = val;
    p.part_idx[at * p.width + lane] = idx;
  }
}

// One CTA per sequence: warp w joins the stretches of beams w, w + warps, ...;
// then warp 0 takes the largest of the beams' heads, `width` times.
__global__ void __launch_bounds__(kSelThreads) beam_join_kernel(const BeamParams p) {
  __shared__ double s_worth[kMaxBeams][kMaxWidth];
  __shared__ int s_token[kMaxBeams][kMaxWidth];
  __shared__ float s_val[kSelWarps][kStaged];
  __shared__ int s_idx[kSelWarps][kStaged];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long seq = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  for (int w = warp; w < p.beams; w += kSelWarps) {
    const long long row = seq * p.beams + w;
    const double score = p.scores[row];
    double worth = -INFINITY;
    int token = INT_MAX;
    if (p.done != nullptr && p.done[row]) {
      if (lane == 0) {
        worth = score;
        token = p.eos;
      }
    } else {
      const int n = p.splits * p.width;
      const float* val = p.part_val + row * n;
      const int* idx = p.part_idx + row * n;
      if (n <= kStaged) {
        for (int i = lane; i < n; i += 32) {
          s_val[warp][i] = val[i];
          s_idx[warp][i] = idx[i];
        }
        val = s_val[warp];
        idx = s_idx[warp];
      }
      float m = -FLT_MAX;
      for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, p.part_max[row * p.splits + s]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      double sum = 0.0;
      for (int s = lane; s < p.splits; s += 32) {
        const float d = p.part_max[row * p.splits + s] - m;
        sum += static_cast<double>(p.part_sum[row * p.splits + s]) * exp(static_cast<double>(d));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncwarp();
      float best;
      merge_lists(p.splits, p.width, [&](int l, int i) { return val[l * p.width + i]; },
                  [&](int l, int i) { return idx[l * p.width + i]; }, &best, &token);
      if (best > -INFINITY)
        worth = ((static_cast<double>(best) - static_cast<double>(m)) - log(sum)) + score;
    }
    if (!(worth > -INFINITY)) worth = -INFINITY;  // NaN scores choose nothing
    s_worth[w][lane] = worth;
    s_token[w][lane] = token;
  }
  __syncthreads();
  if (warp != 0) return;
  int head = 0;  // lane w: the next candidate of beam w
  for (int k = 0; k < p.width; ++k) {
    double worth = -INFINITY;
    int token = INT_MAX;
    if (lane < p.beams && head < p.width) {
      worth = s_worth[lane][head];
      token = s_token[lane][head];
    }
    // The largest, the lowest lane (beam) among equals: FP64 in the order of whole
    // numbers, half by half.
    const long long bits = __double_as_longlong(worth + 0.0);
    const unsigned long long key = bits ^ ((bits >> 63) | (1ll << 63));
    const uint32_t high = static_cast<uint32_t>(key >> 32);
    const uint32_t top = __reduce_max_sync(0xffffffffu, high);
    const uint32_t low = high == top ? static_cast<uint32_t>(key) : 0u;
    const uint32_t top_low = __reduce_max_sync(0xffffffffu, low);
    const int beam = __ffs(__ballot_sync(0xffffffffu, high == top && low == top_low)) - 1;
    worth = __shfl_sync(0xffffffffu, worth, beam);
    token = __shfl_sync(0xffffffffu, token, beam);
    const bool none = worth == -INFINITY;
    if (!none && lane == beam) ++head;
    if (lane == 0) {
      const long long at = seq * p.width + k;
      const long long row = seq * p.beams + beam;
      p.out_scores[at] = none ? -INFINITY : static_cast<float>(worth);
      p.out_tokens[at] = none ? -1 : token;
      p.out_parents[at] = none ? -1 : static_cast<int32_t>(row);
      if (p.out_done != nullptr)
        p.out_done[at] = !none && ((p.done != nullptr && p.done[row]) || token == p.eos);
    }
  }
}

// Rows of a state in their new order; -1 gives a zero row.
struct ReorderParams {
  const void* state;
  void* out;
  const int32_t* parents;
  long long row_words;  // of the kernel's word
  int rows, new_rows;
};

template <typename V>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const V* state = static_cast<const V*>(p.state);
  V* out = static_cast<V*>(p.out);
  for (int r = blockIdx.y; r < p.new_rows; r += gridDim.y) {
    const int from = p.parents[r];
    const bool ok = from >= 0 && from < p.rows;
    if (!ok && from != -1 && blockIdx.x == 0 && threadIdx.x == 0) report_error(kDevErrBounds);
    const long long step = static_cast<long long>(gridDim.x) * 256;
#pragma unroll 4
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < p.row_words; i += step)
      out[r * p.row_words + i] = ok ? state[from * p.row_words + i] : V{};
  }
}

template <typename V>
int launch_reorder(ReorderParams p, long long row_bytes, cudaStream_t stream) {
  p.row_words = row_bytes / static_cast<long long>(sizeof(V));
  long long x = (p.row_words + 1023) / 1024;
  const long long most = 16ll * sm_count() / p.new_rows + 1;
  if (x > most) x = most;
  LaunchCfg cfg;
  cfg.grid = dim3(static_cast<unsigned>(x), static_cast<unsigned>(p.new_rows < 65535 ? p.new_rows : 65535));
  cfg.block = dim3(256);
  cfg.stream = stream;
  cfg.pdl = true;
  return launch(cfg, beam_reorder_kernel<V>, p);
}

// Stretches of a row: enough CTAs to fill the SMs a few times over, none shorter
// than half a turn of its warps, none over 2^17 logits (a lane then adds at most 64
// words' sums in FP32).
int beam_splits(long long rows, int vocab) {
  const long long want = (8ll * sm_count() + rows - 1) / rows;
  const long long most = (vocab + kSelThreads * 16 - 1) / (kSelThreads * 16);
  const long long least = (vocab + (1 << 17) - 1) / (1 << 17);
  const long long s = std::max(std::min(want, most), least);
  return static_cast<int>(std::min<long long>(s, kMaxSplits));
}

size_t beam_workspace(int batch, int beams, int vocab, int width) {
  if (batch < 1 || beams < 1 || vocab < 1 || width < 1) return 0;
  const size_t rows = static_cast<size_t>(batch) * beams;
  return rows * beam_splits(rows, vocab) * (8 + 8 * static_cast<size_t>(width));
}

}  // namespace
}  // namespace npu_b200

extern "C" size_t npu_b200_beam_select_workspace_size(int batch, int beams, int vocab, int width) {
  return npu_b200::beam_workspace(batch, beams, vocab, width);
}

extern "C" int npu_b200_beam_select(const void* d_logits, int logits_f32, const float* d_scores,
                                    const uint8_t* d_done, float* d_out_scores,
                                    int32_t* d_out_tokens, int32_t* d_out_parents,
                                    uint8_t* d_out_done, int batch, int beams, int vocab, int width,
                                    int eos, void* d_workspace, size_t workspace_bytes,
                                    void* stream) {
  using namespace npu_b200;
  clear_error();
  NPU_REQUIRE(d_logits && d_scores && d_out_scores && d_out_tokens && d_out_parents,
              "beam_select: null tensor pointer");
  NPU_REQUIRE(beams >= 1 && beams <= kMaxBeams, "beam_select: beams %d not in [1, %d]", beams, kMaxBeams);
  NPU_REQUIRE(width >= 1 && width <= kMaxWidth, "beam_select: width %d not in [1, %d]", width, kMaxWidth);
  NPU_REQUIRE(vocab >= 1 && vocab <= 1 << 24, "beam_select: vocab %d not in [1, 2^24]", vocab);
  NPU_REQUIRE(batch >= 1 && static_cast<long long>(batch) * beams <= 65535,
              "beam_select: batch %d x beams %d not in [1, 65535]", batch, beams);
  NPU_REQUIRE(eos >= -1 && eos < vocab, "beam_select: end token %d not in [-1, %d)", eos, vocab);
  NPU_REQUIRE(d_done == nullptr || eos >= 0, "beam_select: finished beams need an end token");
  NPU_REQUIRE((reinterpret_cast<uintptr_t>(d_logits) & 15) == 0,
              "beam_select: logits must be 16-byte aligned");
  const size_t need = beam_workspace(batch, beams, vocab, width);
  NPU_REQUIRE(d_workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(d_workspace) & 15) == 0,
              "beam_select: workspace of %zu bytes (16-byte aligned) needed, %zu given", need,
              workspace_bytes);
  const long long rows = static_cast<long long>(batch) * beams;
  BeamParams p;
  p.logits = d_logits;
  p.scores = d_scores;
  p.done = d_done;
  p.out_scores = d_out_scores;
  p.out_tokens = d_out_tokens;
  p.out_parents = d_out_parents;
  p.out_done = d_out_done;
  p.beams = beams;
  p.vocab = vocab;
  p.width = width;
  p.eos = eos;
  p.total = rows * vocab;
  p.splits = beam_splits(rows, vocab);
  const int per_word = logits_f32 ? 4 : 8;
  const int words = (vocab + per_word - 1) / per_word;
  p.words = (words + p.splits - 1) / p.splits;
  p.part_max = static_cast<float*>(d_workspace);
  p.part_sum = p.part_max + rows * p.splits;
  p.part_val = p.part_sum + rows * p.splits;
  p.part_idx = reinterpret_cast<int32_t*>(p.part_val + rows * p.splits * width);
  LaunchCfg cfg;
  cfg.grid = dim3(p.splits, static_cast<unsigned>(rows));
  cfg.block = dim3(kSelThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.pdl = true;
  int rc = logits_f32 ? launch(cfg, beam_stretch_kernel<float>, p) : launch(cfg, beam_stretch_kernel<__half>, p);
  if (rc) return rc;
  cfg.grid = dim3(batch);
  return launch(cfg, beam_join_kernel, p);
}

extern "C" int npu_b200_beam_reorder(const void* d_state, const int32_t* d_parents, void* d_out,
                                     int rows, int new_rows, size_t row_bytes, void* stream) {
  using namespace npu_b200;
  clear_error();
  NPU_REQUIRE(d_state && d_parents && d_out, "beam_reorder: null tensor pointer");
  NPU_REQUIRE(rows >= 1 && new_rows >= 1 && row_bytes >= 1 && row_bytes < size_t(1) << 40,
              "beam_reorder: %d rows to %d of %zu bytes", rows, new_rows, row_bytes);
  const uintptr_t a = reinterpret_cast<uintptr_t>(d_state), b = reinterpret_cast<uintptr_t>(d_out);
  NPU_REQUIRE(a >= b + row_bytes * new_rows || b >= a + row_bytes * rows,
              "beam_reorder: the output must not overlap the state");
  ReorderParams p = {d_state, d_out, d_parents, 0, rows, new_rows};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uintptr_t all = a | b | row_bytes;
  if ((all & 15) == 0) return launch_reorder<uint4>(p, row_bytes, s);
  if ((all & 3) == 0) return launch_reorder<uint32_t>(p, row_bytes, s);
  return launch_reorder<uint8_t>(p, row_bytes, s);
}
