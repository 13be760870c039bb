// Launches of the selective scan's forward and gradient.
#pragma once

#include "scan_common.cuh"

namespace gru {
namespace scan {

// CTAs that share a sequence's tile of channels as a cluster: as many as fill
// the GPU's places for CTAs (`resident` an SM) and have a block each.
inline int sharing(const Problem& p, int blocks, int resident) {
  const long units = (long)p.B * p.tiles, places = 148L * resident;
  int q = 1;
  while (q < 8 && units * q * 2 <= places && q * 2 <= blocks) q *= 2;
  return q;
}

template <typename Kernel>
int launch_shared(Kernel kernel, const Problem& p, int q, int threads, size_t smem, cudaStream_t stream) {
  GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)q, at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((long)p.B * p.tiles * q));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &at;
  cfg.numAttrs = q > 1 ? 1 : 0;
  GRU_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return GRU_OK;
}

int forward(const Problem& p, int dtype, cudaStream_t stream);
int backward(const Problem& p, int dtype, cudaStream_t stream);
int backward_sharing(const Problem& p);  // CTAs of a tile, each with sums of its own

}  // namespace scan
}  // namespace gru
