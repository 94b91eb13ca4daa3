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
// keeps the sum relative to its running maximum, and lists the logits that reach a
// floor which `width` logits of the CTA are known to reach: the width-th largest of
// its lanes' maxima over their first words, then, each time twice as much has been
// read, the width-th best candidate.  That leaves some width x log2(length / 4096)
// candidates of a stretch, so the selection costs one comparison per 8 logits (sorted
// lists that each warp kept for itself cost twice the rest; rows whose logits nearly all equal
// the floor, as under a mask of the type's lowest number, cost 17 times as much).  A warp whose list runs
// full, on rising logits, keeps its `width` best and raises the floor.  A second,
// dependent launch joins the stretches.
//
// Which of two candidates is larger decides whole beams, so what follows the
// stretches (the sum over them, its logarithm, the candidates' worth) is in FP64;
// within a stretch the FP32 sum of exponentials exact to 2^-22 leaves ln S some 1e-7
// off.
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
constexpr int kList = 320;      // candidates of a warp; one word of each lane adds at most 256
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = static_cast<float>(1.4426950408889634 - static_cast<double>(kLog2e));
constexpr double kLn2 = 0.69314718055994530942;
constexpr float kNothing = -FLT_MAX;  // the reference of a stretch without a logit above -inf

struct BeamParams {
  const void* logits;
  const float* scores;
  const uint8_t* done;  // or null
  float* out_scores;
  int32_t* out_tokens;
  int32_t* out_parents;
  uint8_t* out_done;    // or null
  // Stretch s of row r: reference, sum, and the best logits with their tokens.
  float* part_ref;      // [rows][splits]
  float* part_sum;
  float* part_val;      // [rows][splits][width]
  int32_t* part_idx;
  int beams, vocab, width, splits, words;  // words: 16-byte words of a stretch
  int eos, f32;
  long long total;      // logits of the tensor
};

// Whole numbers in the order of the floating ones (-0 as 0).
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// One warp's candidates.
struct Candidates {
  float val[kList];
  int idx[kList];
  int n;
};

// The `width` best of a list's candidates, larger first, lower token among equals:
// lane k returns the k-th.  Each turn takes the best that comes after the last one.
__device__ __forceinline__ void take_best(const Candidates& list, int width, float* out_v, int* out_i) {
  const int lane = threadIdx.x & 31;
  uint32_t last = 0xffffffffu;
  int last_i = -1;
  *out_v = -INFINITY;
  *out_i = INT_MAX;
  for (int k = 0; k < width; ++k) {
    uint32_t best = 0;
    int best_i = INT_MAX;
    for (int e = lane; e < list.n; e += 32) {
      const uint32_t v = order_of(list.val[e]);
      const int i = list.idx[e];
      const bool after = v < last || (v == last && i > last_i);
      if (after && (v > best || (v == best && i < best_i))) {
        best = v;
        best_i = i;
      }
    }
    last = __reduce_max_sync(0xffffffffu, best);
    if (last == 0) break;  // no more
    last_i = __reduce_min_sync(0xffffffffu, best == last ? best_i : INT_MAX);
    if (lane == k) {
      *out_v = of_order(last);
      *out_i = last_i;
    }
  }
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

// What differs between FP16 and FP32 logits.  Sums are relative to a reference: for
// FP16 a power of two 2^r, so that e^x / 2^r = 2^(x log2 e - r) takes two FMAs whose
// roundings are relative to the result, and a new reference costs no rounding; for
// FP32, whose x log2 e may overflow, e^m.
// NaN counts as -inf, +inf as the largest number of the type.
template <typename T>
struct Kind;
template <>
struct Kind<__half> {
  static constexpr int kLogits = 8;
  static constexpr float kMost = 65504.f;
  // The largest logit of a word, NaN if there is one.
  static __device__ __forceinline__ float top(const uint4& w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __half2*>(&u[i]);
    const __half2 t = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __half2float(__hmax_nan(__low2half(t), __high2half(t)));
  }
  // The word with its first n logits made ordinary, and -inf after them.
  static __device__ __forceinline__ uint4 clean(const uint4& w, int n) {
    uint32_t u[4] = {w.x, w.y, w.z, w.w};
    const __half2 low = __half2half2(__ushort_as_half(0xfc00)), high = __half2half2(__ushort_as_half(0x7bff));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __hmin2(__hmax2(*reinterpret_cast<const __half2*>(&u[i]), low), high);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
      if (2 * i + 1 >= n) u[i] = 2 * i >= n ? 0xfc00fc00u : (u[i] & 0xffffu) | 0xfc000000u;
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ void widen(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float reference(float m) { return ceilf(m * kLog2e); }
  // The exponents (base 2) of x0, x1 relative to the reference.
  static __device__ __forceinline__ uint64_t exponents(float x0, float x1, float ref) {
    const uint64_t x = pack2(x0, x1);
    return fma2(x, pack2(kLog2eLow, kLog2eLow), fma2(x, pack2(kLog2e, kLog2e), pack2(-ref, -ref)));
  }
  static __device__ __forceinline__ float ratio(float from, float to) { return fast_exp2(from - to); }
};
template <>
struct Kind<float> {
  static constexpr int kLogits = 4;
  static constexpr float kMost = FLT_MAX;
  static __device__ __forceinline__ float top(const uint4& w) {
    float a, b;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(__uint_as_float(w.x)), "f"(__uint_as_float(w.y)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(__uint_as_float(w.z)), "f"(__uint_as_float(w.w)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(b));
    return a;
  }
  static __device__ __forceinline__ uint4 clean(const uint4& w, int n) {
    uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = i >= n ? 0xff800000u
                    : __float_as_uint(fminf(fmaxf(__uint_as_float(u[i]), -INFINITY), kMost));
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ void widen(const uint4& w, float (&x)[4]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(u[i]);
  }
  static __device__ __forceinline__ float reference(float m) { return m; }
  static __device__ __forceinline__ uint64_t exponents(float x0, float x1, float ref) {
    return mul2(add2(pack2(x0, x1), pack2(-ref, -ref)), pack2(kLog2e, kLog2e));
  }
  static __device__ __forceinline__ float ratio(float from, float to) {
    return fast_exp2((from - to) * kLog2e);
  }
};

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

__device__ __forceinline__ float warp_max(float v) {
  return of_order(__reduce_max_sync(0xffffffffu, order_of(v)));
}

// The `width` best of up to 256 candidates in one warp's registers (order_of() keys, 0:
// none), larger first, lower token among equals: take(k, key, token) in every lane.
// (Ranking each candidate among all, by a thread of its own, is quadratic in their
// number: 64 x 8 rows of 128256 took 72 us instead of 57.)
constexpr int kPerLane = kSelThreads / 32;
template <typename Take>
__device__ __forceinline__ void best_of(uint32_t (&key)[kPerLane], const int (&token)[kPerLane], int width,
                                        Take take) {
  for (int k = 0; k < width; ++k) {
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < kPerLane; ++u) most = max(most, key[u]);
    most = __reduce_max_sync(0xffffffffu, most);
    if (most == 0) break;
    int low = INT_MAX;
#pragma unroll
    for (int u = 0; u < kPerLane; ++u)
      if (key[u] == most) low = min(low, token[u]);
    low = __reduce_min_sync(0xffffffffu, low);
    take(k, most, low);
#pragma unroll
    for (int u = 0; u < kPerLane; ++u)
      if (key[u] == most && token[u] == low) key[u] = 0;
  }
}

// All lists' candidates, at most 256, to one warp's registers.
__device__ __forceinline__ void gather(const Candidates* lists, uint32_t (&key)[kPerLane], int (&token)[kPerLane]) {
  int from[kSelWarps];  // of the lists, one behind the other
  int n = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    from[w] = n;
    n += lists[w].n;
  }
#pragma unroll
  for (int u = 0; u < kPerLane; ++u) {
    const int e = (threadIdx.x & 31) + 32 * u;
    key[u] = 0;
    token[u] = INT_MAX;
    if (e >= n) continue;
    int w = 0, first = 0;
#pragma unroll
    for (int v = 1; v < kSelWarps; ++v)
      if (e >= from[v]) {
        w = v;
        first = from[v];
      }
    key[u] = order_of(lists[w].val[e - first]);
    token[u] = lists[w].idx[e - first];
  }
}
__device__ __forceinline__ int candidates(const Candidates* lists) {
  int n = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) n += lists[w].n;
  return n;
}

// What a warp carries along its part of a stretch: its maximum and reference, the
// lane's share of the sum; no logit below `floor` is a candidate, none below `gate`
// a candidate or a new maximum.
struct Running {
  float m = -INFINITY, ref = 0.f, sum = 0.f;
  float floor = -INFINITY, gate = -INFINITY;
};

// One turn of a warp: the lane's words w, w + 32, ...  Nearly always nothing in them
// reaches the gate (one vote), and what is left is a straight run of exponentials.
template <typename T, int N>
__device__ __forceinline__ void take_turn(uint4 (&raw)[N], int w, int width, Candidates& list,
                                          uint32_t* s_floor, Running& r) {
  using Kd = Kind<T>;
  constexpr int L = Kd::kLogits;
  const int lane = threadIdx.x & 31;
  float top[N];
  bool pass = false;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    top[u] = Kd::top(raw[u]);
    pass |= !(top[u] < r.gate);
  }
  if (__any_sync(0xffffffffu, pass)) {
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (!(top[u] <= Kd::kMost)) {
        raw[u] = Kd::clean(raw[u], L);
        top[u] = Kd::top(raw[u]);
      }
      most = fmaxf(most, top[u]);
    }
    if (__any_sync(0xffffffffu, most > r.m)) {
      r.m = warp_max(most);
      const float to = Kd::reference(r.m);
      r.sum = r.sum > 0.f ? r.sum * Kd::ratio(r.ref, to) : 0.f;
      r.ref = to;
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (!__any_sync(0xffffffffu, top[u] >= r.floor && top[u] > -INFINITY)) continue;
      if (list.n > kList - 32 * L) {  // no room for the most that may come
        __syncwarp();
        float val;
        int idx;
        take_best(list, width, &val, &idx);
        __syncwarp();
        if (lane < width) {
          list.val[lane] = val;
          list.idx[lane] = idx;
        }
        if (lane == 0) list.n = width;
        r.floor = fmaxf(r.floor, __shfl_sync(0xffffffffu, val, width - 1));
        if (lane == 0) atomicMax(s_floor, order_of(r.floor));
        __syncwarp();
      }
      if (top[u] >= r.floor && top[u] > -INFINITY) {
        float x[L];
        Kd::widen(raw[u], x);
#pragma unroll
        for (int i = 0; i < L; ++i)
          if (x[i] >= r.floor && x[i] > -INFINITY) {
            const int at = atomicAdd(&list.n, 1);
            list.val[at] = x[i];
            list.idx[at] = (w + u * 32) * L + i;
          }
      }
      __syncwarp();
    }
  }
  uint64_t s2[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float x[L];
    Kd::widen(raw[u], x);
#pragma unroll
    for (int i = 0; i < L; i += 2) {
      const uint64_t e2 = Kd::exponents(x[i], x[i + 1], r.ref);
      s2[(i >> 1) & 1] = add2(s2[(i >> 1) & 1], pack2(fast_exp2(lo2(e2)), fast_exp2(hi2(e2))));
    }
  }
  const uint64_t all2 = add2(s2[0], s2[1]);
  r.sum += lo2(all2) + hi2(all2);
}

// Block (s, row): stretch s of row `row`, a piece per warp.  CTAS to an SM: registers for
// three, or fewer for four.
template <typename T, int CTAS>
__global__ void __launch_bounds__(kSelThreads, CTAS) beam_stretch_kernel(const BeamParams p) {
  using Kd = Kind<T>;
  constexpr int L = Kd::kLogits;
  __shared__ float s_ref[kSelWarps], s_sum[kSelWarps];
  __shared__ Candidates s_list[kSelWarps];
  __shared__ uint32_t s_top[kSelThreads];  // the lanes' best first logits
  __shared__ uint32_t s_floor;  // order_of() of what `width` logits of the CTA reach
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.y;
  if (lane == 0) s_list[warp].n = 0;
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
  Candidates& list = s_list[warp];
  Running r;
  constexpr int kAhead = 4;
  constexpr int kTurn = 32 * kAhead;  // words that a warp loads together
  const int turns = (w_end - w_begin + kSelWarps * kTurn - 1) / (kSelWarps * kTurn);
  uint4 next[kAhead];
  auto load = [&](int turn) {  // a turn inside the stretch, the row and the tensor needs no checks
    const int w0 = w_begin + (turn * kSelWarps + warp) * kTurn;
    if (w0 + kTurn <= w_end && (w0 + kTurn) * L <= p.vocab) {
      const uint4* src = reinterpret_cast<const uint4*>(logits) + first + w0 + lane;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) next[u] = __ldg(src + u * 32);
    } else {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        next[u] = tensor_word(logits, first + min(w0 + u * 32 + lane, w_end - 1), p.total);
    }
  };
  if (turns > 0) load(0);
  for (int turn = 0; turn < turns; ++turn) {  // every warp takes every turn
    const int w0 = w_begin + (turn * kSelWarps + warp) * kTurn, w = w0 + lane;
    uint4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) raw[u] = next[u];
    if (lead != 0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        raw[u] = shifted(raw[u], tensor_word(logits, first + min(w + u * 32, w_end - 1) + 1, p.total),
                         lead * static_cast<int>(sizeof(T)) / 2);
    }
    if (turn + 1 < turns) load(turn + 1);
    if (w0 + kTurn > w_end || (w0 + kTurn) * L > p.vocab) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        raw[u] = Kd::clean(raw[u], w + u * 32 < w_end ? p.vocab - (w + u * 32) * L : 0);
    }
    if (turn == 0) {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        float t = Kd::top(raw[u]);
        if (!(t <= Kd::kMost)) t = Kd::top(Kd::clean(raw[u], L));
        top = fmaxf(top, t);
      }
      r.m = fmaxf(r.m, warp_max(top));
      if (r.m > -INFINITY) r.ref = Kd::reference(r.m);
      s_top[threadIdx.x] = order_of(top);
      __syncthreads();
      if (warp == 0) {  // the width-th of all is the floor
        uint32_t key[kPerLane];
        int at[kPerLane];
#pragma unroll
        for (int u = 0; u < kPerLane; ++u) key[u] = s_top[at[u] = lane + 32 * u];
        best_of(key, at, p.width, [&](int k, uint32_t v, int) {
          if (k == p.width - 1) s_floor = v;
        });
      }
      __syncthreads();
    }
    if (turn > 0 && (turn & (turn - 1)) == 0) {  // read twice as much as at the last floor
      __syncthreads();
      if (warp == 0 && candidates(s_list) <= kSelThreads) {
        uint32_t key[kPerLane];
        int token[kPerLane];
        gather(s_list, key, token);
        best_of(key, token, p.width, [&](int k, uint32_t v, int) {
          if (k == p.width - 1) atomicMax(&s_floor, v);
        });
      }
      __syncthreads();
    }
    r.floor = fmaxf(r.floor, of_order(*const_cast<volatile uint32_t*>(&s_floor)));
    r.gate = fminf(r.floor, fmaxf(r.m, -FLT_MAX));
    take_turn<T>(raw, w, p.width, list, &s_floor, r);
  }
  // The lanes' sums, then the warps'.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
  if (lane == 0) {
    s_ref[warp] = r.m > -INFINITY ? r.ref : kNothing;
    s_sum[warp] = r.sum;
  }
  __syncthreads();
  // Of more candidates than one warp's registers take, `width` of each warp are enough.
  if (candidates(s_list) > kSelThreads) {  // the same in every thread
    float val;
    int idx;
    take_best(list, p.width, &val, &idx);
    __syncthreads();
    if (lane < p.width) {
      list.val[lane] = val;
      list.idx[lane] = idx;
    }
    if (lane == 0) list.n = min(list.n, p.width);
    __syncthreads();
  }
  if (warp != 0) return;
  const long long at = row * p.splits + blockIdx.x;
  uint32_t key[kPerLane], value = order_of(-INFINITY);
  int tokens[kPerLane], token = INT_MAX;
  gather(s_list, key, tokens);
  best_of(key, tokens, p.width, [&](int k, uint32_t v, int t) {
    if (lane == k) {
      value = v;
      token = t;
    }
  });
  if (lane < p.width) {
    p.part_val[at * p.width + lane] = of_order(value);
    p.part_idx[at * p.width + lane] = token;
  }
  float ref_all = kNothing, sum_all = 0.f;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) ref_all = fmaxf(ref_all, s_ref[w]);
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) sum_all += s_sum[w] * Kd::ratio(s_ref[w], ref_all);
  if (lane == 0) {
    p.part_ref[at] = ref_all;
    p.part_sum[at] = sum_all;
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
      float m = kNothing;  // the stretches' largest reference
      for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, p.part_ref[row * p.splits + s]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      double sum = 0.0;
      for (int s = lane; s < p.splits; s += 32) {
        const double d = static_cast<double>(p.part_ref[row * p.splits + s]) - m;
        sum += static_cast<double>(p.part_sum[row * p.splits + s]) * (p.f32 ? exp(d) : exp2(d));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncwarp();
      float best;
      merge_lists(p.splits, p.width, [&](int l, int i) { return val[l * p.width + i]; },
                  [&](int l, int i) { return idx[l * p.width + i]; }, &best, &token);
      if (best > -INFINITY)
        worth = ((best - (p.f32 ? 1.0 : kLn2) * m) - log(sum)) + score;
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

// Stretches of a row: as many as keep all CTAs resident at once (3 an SM), since each CTA pays
// for its floor and its last choice; none shorter than half a turn of its
// warps, none over 2^17 logits (a lane then adds at most 64 words' sums in FP32).
int beam_splits(long long rows, int vocab) {
  const long long want = 3ll * sm_count() / rows;
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
  const size_t chosen = static_cast<size_t>(batch) * width;
  NPU_REQUIRE(!overlap(d_scores, rows * 4, d_out_scores, chosen * 4) &&
                  !(d_done != nullptr && d_out_done != nullptr && overlap(d_done, rows, d_out_done, chosen)),
              "beam_select: the new scores and flags must not overlap the old ones");
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
  p.f32 = logits_f32 != 0;
  p.total = rows * vocab;
  p.splits = beam_splits(rows, vocab);
  const int per_word = logits_f32 ? 4 : 8;
  const int words = (vocab + per_word - 1) / per_word;
  p.words = (words + p.splits - 1) / p.splits;
  p.part_ref = static_cast<float*>(d_workspace);
  p.part_sum = p.part_ref + rows * p.splits;
  p.part_val = p.part_sum + rows * p.splits;
  p.part_idx = reinterpret_cast<int32_t*>(p.part_val + rows * p.splits * width);
  LaunchCfg cfg;
  cfg.grid = dim3(p.splits, static_cast<unsigned>(rows));
  cfg.block = dim3(kSelThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.pdl = true;
  // Where three CTAs an SM do not hold all rows at once, four do with some spilled registers
  // (64 x 8 rows of 128256 tokens 57 -> 46 us; 100 x 4 of 32000, which three hold, 15.9 ->
  // 18).  Not with finished beams, whose CTAs end at once: the places they leave go to the
  // rows that wait (a fifth of them finished: 43 us, with four 49); flags of which few are set
  // pay for it (none of them: 68 us instead of 53, cold caches).
  const bool four = rows * p.splits > 3ll * sm_count() && d_done == nullptr;
  const auto stretch = logits_f32 ? (four ? beam_stretch_kernel<float, 4> : beam_stretch_kernel<float, 3>)
                                  : (four ? beam_stretch_kernel<__half, 4> : beam_stretch_kernel<__half, 3>);
  int rc = launch(cfg, stretch, p);
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
  NPU_REQUIRE(!overlap(d_state, row_bytes * rows, d_out, row_bytes * new_rows) &&
                  !overlap(d_parents, new_rows * size_t(4), d_out, row_bytes * new_rows),
              "beam_reorder: the output must not overlap the state or the parents");
  ReorderParams p = {d_state, d_out, d_parents, 0, rows, new_rows};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uintptr_t all = a | b | row_bytes;
  if ((all & 15) == 0) return launch_reorder<uint4>(p, row_bytes, s);
  if ((all & 3) == 0) return launch_reorder<uint32_t>(p, row_bytes, s);
  return launch_reorder<uint8_t>(p, row_bytes, s);
}
