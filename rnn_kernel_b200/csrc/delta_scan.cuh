// What the gated delta rule's forward and backward scans share: a warp's part
// of the products with the state and with a chunk's 64 x 64 tiles.
#pragma once

#include "delta_common.cuh"

namespace gru {
namespace delta {

// The quarter of the tokens (and of the key columns) of a scan's warp, among the
// four of its value columns.  The second four take them the other way around:
// quarters have 1 to 4 steps of a triangular product, and warps 4 apart share an
// SM's quarter.
__device__ __forceinline__ int quarter_of(int thread) {
  const int warp = thread >> 5;
  return (warp & 4 ? ~warp : warp) & 3;
}

// Barriers of the four warps that share value columns: what one group writes the
// other never reads, and groups apart from one another use the SM's pipes in turn.
__device__ __forceinline__ void group_sync(int pair) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(pair + 1) : "memory"); }
__device__ __forceinline__ bool group_sync_or(int pair, bool x) {
  int y;
  asm volatile(
      "{\n.reg .pred p, q;\n"
      "setp.ne.s32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, %2, 128, p;\n"
      "selp.s32 %0, 1, 0, q;\n}"
      : "=r"(y)
      : "r"((int)x), "r"(pair + 1)
      : "memory");
  return y != 0;
}

// x (16 tokens x 16 columns) = K S of this warp's tokens; S as planes with a
// scale for each quarter of its rows.
template <int NP, int DK>
__device__ __forceinline__ void times_state(float (&x)[2][4], const f16* kp, int m8, const f16* sp, const float* scale) {
  constexpr int per = DK / 64;  // steps to a quarter
  zero(x);
  const uint32_t pa = addr_a<DK, false>(kp, m8, 0), pb = addr_b<kGroup, true>(sp, 0, 0);
#pragma unroll
  for (int kk = 0; kk < DK / 16; kk += 2) {
    float t[2][2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t fa[NP][4], fb[2][2][2];
#pragma unroll
      for (int p = 0; p < NP; ++p) ldm4<false>(fa[p], pa + (kk + h) * 256 + p * kC * DK * 2);
      load_b<2, 2, true>(fb, pb + (kk + h) * 512, 0, 2 * kGroup * DK * 2);
      mma_terms<NP, 2, 2>(t[h], fa, fb);
    }
    const float f0 = scale[kk / per], f1 = scale[(kk + 1) / per];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] += f0 * t[0][n][e] + f1 * t[1][n][e];
  }
}

// x += A B over steps [k0, k1): A a 64 x 64 tile (16 rows at m8, or transposed),
// B 64 tokens x 16 columns as NB planes (`plane` bytes apart) with a scale for
// each step.
template <int NA, int NB, bool TA>
__device__ __forceinline__ void times_tokens(float (&x)[2][4], const f16* A, int m8, const f16* B, int plane,
                                             const float* scale, float factor, int k0, int k1) {
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (kk < k0 || kk >= k1) continue;
    uint32_t fa[NA][4], fb[NB][2][2];
    const uint32_t pa = addr_a<kC, TA>(A, m8, 2 * kk);
#pragma unroll
    for (int p = 0; p < NA; ++p) ldm4<TA>(fa[p], pa + p * kTile * 2);
    load_b<NB, 2, true>(fb, addr_b<kGroup, true>(B, 2 * kk, 0), 0, plane);
    float t[2][4];
    mma_terms<NA, NB, 2>(t, fa, fb);
    const float f = factor * scale[kk];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] += f * t[n][e];
  }
}

// s (this warp's quarter of the key columns x 16) += K^T X, X 64 tokens x 16
// columns as two planes with a scale for each 16 tokens.
template <int NP, int DK>
__device__ __forceinline__ void add_to_state(float (&s)[DK / 64][2][4], const f16* kp, int quarter, const f16* X,
                                             const float* scale, float factor) {
  constexpr int MT = DK / 64;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    uint32_t fb[2][2][2];
    load_b<2, 2, true>(fb, addr_b<kGroup, true>(X, 2 * kk, 0), 0, 2 * kGroup * kC * 2);
    const float f = factor * scale[kk];
    float t[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t fa[NP][4];
      const uint32_t pa = addr_a<DK, true>(kp, (quarter * MT + m) * 2, 2 * kk);
#pragma unroll
      for (int p = 0; p < NP; ++p) ldm4<true>(fa[p], pa + p * kC * DK * 2);
      mma_terms<NP, 2, 2>(t[m], fa, fb);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[m][n][e] += f * t[m][n][e];
  }
}

// Planes of this warp's quarter of the state into shared memory, and into `out`,
// if any.
template <int DK>
__device__ __forceinline__ void put_state(const float (&s)[DK / 64][2][4], int quarter, f16* sp, float* scale, f16* out,
                                          float* out_scale) {
  constexpr int MT = DK / 64;
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = max_mag(m, s[i][n][e]);
  m = warp_largest(m);
  if (!finite(m)) {
    m = 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max_finite(m, s[i][n][e]);
    m = warp_largest(m);
  }
  const float inv = plane_inv(m);
  if ((threadIdx.x & 31) == 0) {
    scale[quarter] = plane_scale(inv);
    if (out) out_scale[quarter] = plane_scale(inv);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
    store_rows<2>(sp, 2 * kGroup * DK, (quarter * MT + i) * 2, s[i], inv, out, kGroup * DK);
}

}  // namespace delta
}  // namespace gru
