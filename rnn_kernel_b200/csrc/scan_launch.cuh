// Launches of the selective scan's forward and gradient.
#pragma once

#include "scan_common.cuh"

namespace gru {
namespace scan {

// Warps of a CTA of either pass, for this many states.
int forward_warps(int np);
int backward_warps(int np);
int forward(const Problem& p, int dtype, cudaStream_t stream);
int backward(const Problem& p, int dtype, cudaStream_t stream);

}  // namespace scan
}  // namespace gru
