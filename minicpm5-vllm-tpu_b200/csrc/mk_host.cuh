// Host-side helpers shared by the library's translation units: status macros, kernel launches and the
// per-device state that mk_api.cu sets up.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <utility>

#include "../../include/minicpm5_mk.h"

#define MK_CUDA(x)                                   \
  do {                                               \
    cudaError_t e_ = (x);                            \
    if (e_ != cudaSuccess) return MK_ERR_CUDA;       \
  } while (0)
#define MK_TRY(x)                \
  do {                           \
    mk_status s_ = (x);          \
    if (s_ != MK_OK) return s_;  \
  } while (0)

namespace mk {

typedef CUresult (*PFN_encodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline mk_status cuda_status(cudaError_t e) { return e == cudaSuccess ? MK_OK : MK_ERR_CUDA; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch `k` on `st`; with `pdl` the launch carries programmatic stream serialization, so the kernel may
// begin while the previous kernel of the stream drains (every kernel of the forward calls pdl_wait()
// before touching memory an earlier kernel uses).
template <typename... KArgs, typename... Args>
mk_status launch_k(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl,
                   Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k, std::forward<Args>(args)...) == cudaSuccess ? MK_OK : MK_ERR_CUDA;
}

// The same with clusters of `size` CTAs along x (grid.x a multiple of it).
template <typename... KArgs, typename... Args>
mk_status launch_k_cluster(int size, void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl,
                           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = size;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k, std::forward<Args>(args)...) == cudaSuccess ? MK_OK : MK_ERR_CUDA;
}
// Clusters of two CTAs.
template <typename... KArgs, typename... Args>
mk_status launch_k_pair(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl,
                        Args&&... args) {
  return launch_k_cluster(2, k, grid, block, smem, st, pdl, std::forward<Args>(args)...);
}

// What a kernel launch needs to know of the current device (mk_api.cu): the number of SMs, the device
// error word (first error wins, read by mk_get_error) and the driver's tensor-map encoder.
struct HostDevice {
  int sm_count = 0;
  int* err = nullptr;
  PFN_encodeTiled encode = nullptr;
};
mk_status host_device(HostDevice* out);

}  // namespace mk
