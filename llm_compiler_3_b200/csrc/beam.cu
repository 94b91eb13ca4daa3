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
// So one pass does both: each warp streams a stretch of a row, 16 bytes per lane,
// keeps per lane the running maximum and sum (rescaled once per 8 logits), and
// holds its `width` best logits sorted across its lanes.  After the first few
// words hardly any logit passes the warp's worst kept one, so the selection costs
// one comparison per 8 logits.  A second, dependent launch joins the stretches.
//
// Which of two candidates is larger decides whole beams, so what follows the
// stretches (the sum over them, its logarithm, the candidates' worth) is in FP64;
// within a stretch the FP32 sum of up to 2^-22-exact exponentials leaves ln S
// some 1e-7 off.
#include <float.h>
#include <limits.h>

#include "common.cuh"
#include "host.hpp"

namespace npu_b200 {
namespace {

constexpr int kMaxWidth = 32;   // candidates kept: one per lane
constexpr int kMaxBeams = 32;   // beams of a sequence: one per lane in the join
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
  // Each lane may offer one.
  __device__ __forceinline__ void offer(float v, int i, bool has, int width) {
    unsigned mask = __ballot_sync(0xffffffffu, has && takes(v, i));
    while (mask) {
      const int src = __ffs(mask) - 1;
      put(__shfl_sync(0xffffffffu, v, src), __shfl_sync(0xffffffffu, i, src), width);
      mask = __ballot_sync(0xffffffffu, has && takes(v, i)) & ~((2u << src) - 1);
    }
  }
};

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
__global__ void __launch_bounds__(kSelThreads) beam_stretch_kernel(const BeamParams p) {
  constexpr int L = 16 / sizeof(T);  // logits of a word
  __shared__ float s_val[kSelWarps][32], s_max[kSelWarps], s_sum[kSelWarps];
  __shared__ int s_idx[kSelWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.y;
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
  const int each = ((w_end - w_begin + kSelWarps - 1) / kSelWarps + 31) & ~31;
  const int my_begin = min(w_begin + warp * each, w_end), my_end = min(my_begin + each, w_end);

  Best best;
  float m = -FLT_MAX, sum = 0.f;
  constexpr int kAhead = 4;
  for (int w0 = my_begin; w0 < my_end; w0 += 32 * kAhead) {
    uint4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int w = min(w0 + u * 32 + lane, my_end - 1);
      raw[u] = tensor_word(logits, first + w, p.total);
    }
    if (lead != 0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int w = min(w0 + u * 32 + lane, my_end - 1);
        raw[u] = shifted(raw[u], tensor_word(logits, first + w + 1, p.total),
                         lead * static_cast<int>(sizeof(T)) / 2);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int w = w0 + u * 32 + lane;
      const int t0 = w * L;  // token of the word's first logit
      float x[L];
      widen(raw[u], x, logits);
      if (w >= my_end || t0 + L > p.vocab) {
#pragma unroll
        for (int i = 0; i < L; ++i)
          if (w >= my_end || t0 + i >= p.vocab) x[i] = -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < L; ++i) top = fmaxf(top, x[i]);
      const float m_new = fmaxf(m, top);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < L; ++i) s += fast_exp2((x[i] - m_new) * kLog2e);
      sum = sum * fast_exp2((m - m_new) * kLog2e) + s;
      m = m_new;
      if (__any_sync(0xffffffffu, top >= best.floor && top > -INFINITY)) {
#pragma unroll
        for (int i = 0; i < L; ++i) best.offer(x[i], t0 + i, true, p.width);
      }
    }
  }
  // The lanes' maxima and sums, then the warps'.
  const float m_warp = [&] {
    float v = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }();
  sum *= fast_exp2((m - m_warp) * kLog2e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  s_val[warp][lane] = best.val;
  s_idx[warp][lane] = best.idx;
  if (lane == 0) {
    s_max[warp] = m_warp;
    s_sum[warp] = sum;
  }
  __syncthreads();
  if (warp != 0) return;
  float m_all = -FLT_MAX, sum_all = 0.f;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) m_all = fmaxf(m_all, s_max[w]);
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) sum_all += s_sum[w] * fast_exp2((s_max[w] - m_all) * kLog2e);
  for (int w = 1; w < kSelWarps; ++w)
    best.offer(s_val[w][lane], s_idx[w][lane], lane < p.width, p.width);
  const long long at = row * p.splits + blockIdx.x;
  if (lane == 0) {
    p.part_max[at] = m_all;
    p.part_sum[at] = sum_all;
  }
  if (lane < p.width) {
    p.part_val[at * p.width + lane] = best.val;
    p.part_idx[at * p.width + lane] = best.idx;
  }
}

// One CTA per sequence: warp w joins the stretches of beams w, w + warps, ...;
// then warp 0 takes the largest of the beams' heads, `width` times.
__global__ void __launch_bounds__(kSelThreads) beam_join_kernel(const BeamParams p) {
  __shared__ double s_worth[kMaxBeams][kMaxWidth];
  __shared__ int s_token[kMaxBeams][kMaxWidth];
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
      Best best;
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
      const int n = p.splits * p.width;
      for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + lane;
        const float v = i < n ? p.part_val[row * n + i] : -INFINITY;
        const int t = i < n ? p.part_idx[row * n + i] : INT_MAX;
        best.offer(v, t, i < n, p.width);
      }
      if (lane < p.width && best.val > -INFINITY) {
        worth = ((static_cast<double>(best.val) - static_cast<double>(m)) - log(sum)) + score;
        token = best.idx;
      }
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
    int beam = INT_MAX, token = INT_MAX;
    if (lane < p.beams && head < p.width) {
      worth = s_worth[lane][head];
      token = s_token[lane][head];
      beam = lane;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ow = __shfl_xor_sync(0xffffffffu, worth, o);
      const int ob = __shfl_xor_sync(0xffffffffu, beam, o);
      const int ot = __shfl_xor_sync(0xffffffffu, token, o);
      if (ow > worth || (ow == worth && ob < beam)) {
        worth = ow;
        beam = ob;
        token = ot;
      }
    }
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
// than one turn of its warps, none over 2^17 logits (a lane then adds at most 64
// words' sums in FP32).
int beam_splits(long long rows, int vocab) {
  const long long want = (8ll * sm_count() + rows - 1) / rows;
  const long long most = (vocab + kSelThreads * 32 - 1) / (kSelThreads * 32);
  const long long least = (vocab + (1 << 17) - 1) / (1 << 17);
  const long long s = want < most ? want : most;
  return static_cast<int>(s < least ? least : s);
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
  NPU_REQUIRE(vocab >= 1 && vocab <= 1 << 26, "beam_select: vocab %d not in [1, 2^26]", vocab);
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
