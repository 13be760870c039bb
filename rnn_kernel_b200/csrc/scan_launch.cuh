// Launches of the selective scan's forward and gradient.
#pragma once

#include "scan_common.cuh"

namespace gru {
namespace scan {

struct Fit {
  int warps, resident;  // of a CTA, and CTAs of an SM
};
Fit forward_fit(int np);  // np: the states rounded up to a multiple of four
Fit backward_fit(int np);
int forward(const Problem& p, int dtype, cudaStream_t stream);
int backward(const Problem& p, int dtype, cudaStream_t stream);

}  // namespace scan
}  // namespace gru
