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

// x += sign A B (UP: A^T B) for the 16 tokens of `quarter`, over the tokens up to
// (from) them: A a lower 64 x 64 tile as planes; B 64 tokens x 16 columns as NB
// planes, with the tokens' weights.  `own`: exponents of the lane's rows, A's Row (UP:
// Column); w: of its rows as tokens of B, if they are not `narrow`.  STRICT: A's
// diagonal is zero.
template <int NB, bool UP, bool STRICT>
__device__ __forceinline__ void times_tokens(float (&x)[2][4], const f16* A, const int (&own)[2], int quarter, const f16* B,
                                             const int (&w)[2], bool narrow, const __half* factor, const int* top, float sign) {
  constexpr int plane = 2 * kGroup * kC * 2;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (UP ? kk < quarter : kk > quarter) continue;
    const Weights f = kk == quarter && !narrow ? diagonal_weights<UP, STRICT>(w) : get_weights(kk, factor, top);
    uint32_t fa[2][4], fb[NB][2][2];
    const uint32_t pa = addr_a<kC, UP>(A, quarter * 2, 2 * kk);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      ldm4<UP>(fa[p], pa + p * kTile * 2);
      weigh(fa[p], f);
    }
    load_b<NB, 2, true>(fb, addr_b<kGroup, true>(B, 2 * kk, 0), 0, plane);
    float t[2][4];
    mma_terms<2, NB, 2>(t, fa, fb);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float g = sign * power_of(f.top[e] + own[e]);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        x[n][2 * e] += g * t[n][2 * e];
        x[n][2 * e + 1] += g * t[n][2 * e + 1];
      }
    }
  }
}

// A warp's 16 tokens x 16 columns as NP planes with a scale for each token, in shared
// memory and, if given, in `out`; the exponents of the lane's scales.
template <int NP>
__device__ __forceinline__ void put_tokens(const float (&x)[2][4], int quarter, f16* tile, int (&exponent)[2], f16* out,
                                           float* out_scale) {
  float m[2];
  bool all_finite;
  row_max(x, m, all_finite);
  const float inv[2] = {plane_inv(m[0]), plane_inv(m[1])};
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float s = plane_scale(inv[e]);
    exponent[e] = exponent_of(s);
    // below zero: the 16 tokens hold something that is not finite
    if (out_scale && (lane & 3) == 0) out_scale[quarter * 16 + (lane >> 2) + 8 * e] = all_finite ? s : -s;
  }
  store_rows<NP>(tile, 2 * kGroup * kC, quarter * 2, x, inv, out, kGroup * kC);
}

// The same with one scale, for a sum over all of a chunk's tokens.
__device__ __forceinline__ void put_sum(const float (&x)[2][4], int quarter, f16* tile, float* scale) {
  const float i = plane_inv(warp_max(x)), inv[2] = {i, i};
  if ((threadIdx.x & 31) == 0) scale[quarter] = plane_scale(i);
  store_rows<2>(tile, 2 * kGroup * kC, quarter * 2, x, inv, nullptr, 0);
}

// s (this warp's quarter of the key columns x 16) += K^T X, X 64 tokens x 16
// columns, with K's scales in it, as two planes with a scale for each 16 tokens.
template <int NP, int DK>
__device__ __forceinline__ void add_to_state(float (&s)[DK / 64][2][4], const f16* kp, int quarter, const f16* X,
                                             const float* scale) {
  constexpr int MT = DK / 64;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    uint32_t fb[2][2][2];
    load_b<2, 2, true>(fb, addr_b<kGroup, true>(X, 2 * kk, 0), 0, 2 * kGroup * kC * 2);
    const float f = scale[kk];
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
  const float i0 = plane_inv(m), inv[2] = {i0, i0};
  if ((threadIdx.x & 31) == 0) {
    scale[quarter] = plane_scale(i0);
    if (out) out_scale[quarter] = plane_scale(i0);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
    store_rows<2>(sp, 2 * kGroup * DK, (quarter * MT + i) * 2, s[i], inv, out, kGroup * DK);
}

}  // namespace delta
}  // namespace gru
