// Host-side helpers shared by the C-ABI translation units of libnpu_b200.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <string>

#include "../../include/npu_b200.h"

namespace npu_b200 {

// Thread-local error message behind npu_b200_last_error().
int set_error(int code, const char* fmt, ...);
void clear_error();

// Returns NPU_B200_E_CUDA with a message if `e` is an error.
int check_cuda(cudaError_t e, const char* what);

#define NPU_TRY_CUDA(expr)                                   \
  do {                                                       \
    int _rc = ::npu_b200::check_cuda((expr), #expr);         \
    if (_rc != NPU_B200_OK) return _rc;                      \
  } while (0)

#define NPU_REQUIRE(cond, ...)                                       \
  do {                                                               \
    if (!(cond)) return ::npu_b200::set_error(NPU_B200_E_INVALID, __VA_ARGS__); \
  } while (0)

// Number of SMs of the current device (cached per device).
int sm_count();

// 2-D tensor map over a row-major FP16 matrix [rows, cols] with a box of
// box_cols x box_rows elements and the 128-byte swizzle.  box_cols * 2 must be
// <= 128.  The base must be 16-byte aligned and cols * 2 a multiple of 16.
int make_tensor_map_2d(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols,
                       uint32_t box_rows, uint32_t box_cols);

// 3-D tensor map over `planes` row-major FP16 matrices [rows, cols], plane_bytes
// apart, box box_cols x box_rows x 1, 128-byte swizzle.  Elements past `rows`
// in a plane (or past the last plane) load as zero.
int make_tensor_map_3d(CUtensorMap* map, const void* base, uint64_t cols, uint64_t rows,
                       uint64_t planes, uint64_t plane_bytes, uint32_t box_rows,
                       uint32_t box_cols);

// Graph plans (graph.cu): the state a context holds once npu_b200_load_graph
// succeeded, freed by graph_free; runtime.cu owns the context and exposes its
// device and graph slot.
struct GraphState;
void graph_free(GraphState* g);
int ctx_device(const npu_b200_ctx* c);
GraphState*& ctx_graph(npu_b200_ctx* c);

// Whether two ranges of memory have a byte in common.
inline bool overlap(const void* a, size_t an, const void* b, size_t bn) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + bn && y < x + an;
}

// Launch helper: enables programmatic dependent launch when `pdl` is set.
struct LaunchCfg {
  dim3 grid, block;
  size_t smem = 0;
  cudaStream_t stream = nullptr;
  bool pdl = false;
  int cluster = 1;  // thread-block cluster size along x (1 = no cluster)
};

template <typename... KArgs, typename... Args>
int launch(const LaunchCfg& c, void (*kernel)(KArgs...), Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = c.grid;
  cfg.blockDim = c.block;
  cfg.dynamicSmemBytes = c.smem;
  cfg.stream = c.stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (c.pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  if (c.cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = c.cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = n ? attr : nullptr;
  cfg.numAttrs = n;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...),
                    "cudaLaunchKernelEx");
}

// A number that one device answers the same to every asker (not 0), kept from its first answer on;
// host threads may ask at once.  A question that failed (0) is asked again by the next call.
class AskedOnce {
 public:
  template <typename Ask>
  int get(Ask ask) {
    int n = answer_.load(std::memory_order_relaxed);
    if (n == 0 && (n = ask()) != 0) answer_.store(n, std::memory_order_relaxed);
    return n;
  }

 private:
  std::atomic<int> answer_{0};
};

// How many clusters of `size` CTAs (2, 4 or 8; `size` 1: CTAs) of KERNEL run at once on the
// current device: clusters of 8 that fill an SM each leave 28 of 148 SMs idle.  None, if that
// cannot be told.
template <auto KERNEL>
int clusters_at_once(int size, dim3 block, size_t smem) {
  static AskedOnce asked[64][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || size > 8) return 0;
  const int n = asked[dev][size].get([&] {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = size;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, KERNEL, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return clusters > 0 ? clusters : -1;
  });
  return n > 0 ? n : 0;
}

}  // namespace npu_b200
