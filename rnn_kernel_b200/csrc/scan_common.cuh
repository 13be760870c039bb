// The selective state space scan: what its kernels share (contract in
// include/rnn_kernel_b200.h).
#pragma once

#include "row_ops.cuh"

namespace gru {
namespace scan {

constexpr int kMaxStates = 64;
constexpr int kGroup = 4;        // states a lane works on at a time
constexpr int kLanes = 32;       // channels of a CTA, one a lane
constexpr int kMark = 64;        // tokens between two states that the forward keeps for the gradient

struct Problem {
  const void *x, *dt, *b, *c, *z;
  const float *a, *skip, *bias, *s0;
  long xs[2], dts[2], zs[2], bs[3], cs[3];  // batch, token (, group)
  void* out;
  float* last;
  float* marks;  // [B][tiles][mark][state group][32] float4: states at the tokens 0, kMark, ...
  // gradient
  const void* dout;
  const float* dlast;
  void *dx, *ddt, *dz, *db, *dc;
  float *da, *dskip, *dbias, *ds0;
  float* part_bc;  // [B][tiles][T][2][padded N]
  float* part_a;   // [B][D][N]
  float* part_ch;  // [B][2][D]: of skip and dt_bias
  int B, T, D, N, G, R;  // R: channels of a group
  int softplus;
  int per_group, tiles;  // tiles of 32 channels in a group, and in all
  int ng;                // groups of states: ceil(N / 4)
  int nmarks;
};

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A in powers of two, kept finite: a token that is not there has dt = 0, and
// 0 * infinity would make its decay NaN, not 1.
__device__ __forceinline__ float decay_rate(float a) {
  const float r = a * 1.4426950408889634f;
  return r < -3.0e38f ? -3.0e38f : r > 3.0e38f ? 3.0e38f : r;
}

// log(1 + e^x): e^x (1 - e^x / 2) below -8 by log1p, x above 20.
__device__ __forceinline__ float softplus_of(float x) { return x > 20.0f ? x : log1pf(expf(x)); }

// The step size of a raw value.
__device__ __forceinline__ float step_of(const Problem& p, float raw, float bias) {
  raw += bias;
  return p.softplus ? softplus_of(raw) : raw;
}

}  // namespace scan
}  // namespace gru
