// Host-side helpers shared by the C-ABI translation units: thread-local error
// text, argument checks, and TMA tensor-map encoding through the driver entry
// point (so the library needs no link-time dependency on libcuda).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <utility>

#include "../../include/kotflash_b200.h"

namespace kf {

int set_error(int code, const char* fmt, ...);

// Returns KF_ERR_CUDA (and records the message) if the last launch failed.
int check_launch(const char* what);

// Encode a 4-D tiled TMA descriptor over a 16-bit [n0,n1,n2,n3] view whose
// innermost dimension (n3) is contiguous.  The box is (box_inner along n3,
// box_rows along n2, 1, 1) with 128-byte swizzle; out-of-range elements read
// as zero.  Returns KF_OK or an error code with the message recorded.
int encode_tmap_4d(CUtensorMap* map, const kf_tensor4* t, int box_inner, int box_rows);

// Encode a 5-D tiled TMA descriptor over a 16-bit pool of pages [n0 pages, n1
// heads, n2 rows, n3 columns] whose innermost dimension is contiguous, with
// coordinates (column, row, panel, head, page).  panels == 1: columns are n3,
// the box is (cols, rows).  panels > 1: n3 = panels * cols, columns run within
// a panel and the box holds its rows of all panels, panel after panel.
// Swizzle over the panel's 32, 64 or 128 bytes, or none; out-of-range elements
// read as zero.
int encode_tmap_pages(CUtensorMap* map, const kf_tensor4* t, int cols, int rows, int panels, bool swizzle);

// Encode a 2-D tiled TMA descriptor over a row-major fp32 matrix
// [rows][cols] (cols contiguous) with a (box_cols x box_rows) box and 128-byte
// swizzle (box_cols * 4 must be <= 128).
int encode_tmap_2d_f32(CUtensorMap* map, void* ptr, int64_t rows, int64_t cols, int box_cols,
                       int box_rows);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int sm_count_current_device();

// Multiplier and shift of the division by d in [1, 2^31): x / d = x * mul >>
// shift in 64 bits for every x < 2^31.  With 2^(s-1) < d <= 2^s and mul =
// ceil(2^(31+s) / d): mul < 2^32, and mul * d exceeds 2^(31+s) by less than
// 2^s, so the error of x * mul / 2^(31+s) stays below 1 / d.
inline void division(int64_t d, uint32_t* mul, uint32_t* shift) {
  int s = 0;
  while (((int64_t)1 << s) < d) ++s;
  *mul = (uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d);
  *shift = (uint32_t)(31 + s);
}

// Makes the GPU that owns `ptr` the current device for the guard's lifetime
// and restores the caller's device afterwards, so an entry point launches,
// encodes tensor maps and reads device properties on the tensor's own GPU
// whatever device the calling thread has current (the C-ABI counterpart of
// the reference extension's c10::cuda::CUDAGuard on its cache tensor,
// kotflash/csrc/kv_append_cuda.cu:77).  A pointer the runtime does not know
// (host memory, null) leaves the current device alone.  status() is KF_OK or
// KF_ERR_CUDA with the message recorded.
class DeviceGuard {
 public:
  explicit DeviceGuard(const void* ptr);
  ~DeviceGuard();
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
  int status() const { return rc_; }

 private:
  int prev_ = -1;
  bool switched_ = false;
  int rc_ = 0;
};

// Launch with programmatic stream serialization: the kernel may be scheduled
// before the previous kernel in the stream finishes and orders itself with
// griddepcontrol.wait, hiding launch latency between back-to-back kernels
// (split -> merge, and one decode step -> the next).  `cluster` > 1 groups
// that many consecutive blocks (at most 8) of a one-dimensional grid.
template <typename... KArgs, typename... Args>
int launch_dependent_cluster(void (*kern)(KArgs...), unsigned cluster, dim3 grid, dim3 block, size_t smem,
                             cudaStream_t st, const char* what, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...) != cudaSuccess) {
    (void)cudaGetLastError();
    return set_error(KF_ERR_CUDA, "%s: launch failed", what);
  }
  return check_launch(what);
}

template <typename... KArgs, typename... Args>
int launch_dependent(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                     const char* what, Args&&... args) {
  return launch_dependent_cluster(kern, 1, grid, block, smem, st, what, std::forward<Args>(args)...);
}

}  // namespace kf
