// The gated delta rule over chunks of 64 tokens: forward.
//
// With G_i the sum of the log decays of a chunk's tokens up to i, D_ij =
// e^(G_i - G_j), B = diag(beta), S0 the state before the chunk (kernels and
// comments use u_i = beta_i e_i, e_i the delta rule's prediction error):
//
//   N = strict_lower(K K^T o D)          W = (I + N B)^-1 N
//   R = V - diag(e^G) K S0               E = R - W (B R)       U = B E
//   O = scale diag(e^G) Q S0 + P U,      P = scale lower(Q K^T o D)
//   S1 = e^G_end S0 + (diag(e^(G_end - G)) K)^T U
//
// W holds both inverses that forward and gradient need, without a division by
// beta: (I + N B)^-1 = I - W B and (I + B N)^-1 = I - B W.
//
// Three launches.  `prepare` (all chunks at once) computes W and P.  `scan` is
// the only sequential part.  `output` (all chunks at once) computes O from the
// states and errors that the scan leaves.

#include <algorithm>
#include <string>

#include "delta_scan.cuh"

namespace gru {
namespace delta {
namespace {

// The chunks of every sequence that a launch works on; `parts`: CTAs of prepare
// that share a key head's value heads.
struct Range {
  int first, n, parts;
};

// ---------------------------------------------------------------------------
// prepare: one CTA per (batch, key head, chunk), over the head's value heads; in
// a small grid one for each of those.
// Latency-bound (a chain of small products between barriers), so it keeps its
// shared memory small enough for several CTAs on an SM (2048 chunks of heads of
// 128, two to a key head: 64 us).
// ---------------------------------------------------------------------------

constexpr int kLd = 68;  // row length of the FP32 64 x 64 tiles: a multiple of 4, not of 32
constexpr int kLx = 36;

template <typename T, int DK>
struct PrepareSmem {
  static constexpr int NP = Planes<T>::n;
  static constexpr int planes = 2 * NP * kC * DK * 2;
  static constexpr int tiles = (2 * kC * kLd + kC * kLx) * 4;  // N, W and X, over the planes once those are used up
  static constexpr int main = planes > tiles ? planes : tiles;
  static constexpr int bytes = main + 2 * kGates * kC * 4 + kC * 4 + 64 * 4;
};

// acc += A B of FP32 tiles in shared memory, 16 rows from m0 and 8 columns
// from n0, A's columns times colscale[k] (SCALED): operands as three bf16
// planes, which need no scale.  k0, k1: a range of k in multiples of 16.
template <bool SCALED>
__device__ __forceinline__ void mma_f32(float (&acc)[4], const float* A, int lda, int m0, const float* B, int ldb, int n0,
                                        int k0, int k1, const float* colscale) {
  const int g = (threadIdx.x & 31) >> 2, c = (threadIdx.x & 3) * 2;
  auto planes = [](float x, float y, uint32_t (&w)[3]) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      w[p] = *reinterpret_cast<const uint32_t*>(&h);
      x -= __uint_as_float(w[p] << 16);
      y -= __uint_as_float(w[p] & 0xffff0000u);
    }
  };
#pragma unroll 1
  for (int k = k0; k < k1; k += 16) {
    uint32_t fa[3][4], fb[2][3];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int kk = k + c + 8 * (j >> 1);
      float2 x = *reinterpret_cast<const float2*>(A + (m0 + g + 8 * (j & 1)) * lda + kk);
      if (SCALED) x.x *= colscale[kk], x.y *= colscale[kk + 1];
      uint32_t w[3];
      planes(x.x, x.y, w);
#pragma unroll
      for (int p = 0; p < 3; ++p) fa[p][j] = w[p];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float* q = B + (k + c + 8 * j) * ldb + n0 + g;
      planes(q[0], q[ldb], fb[j]);
    }
    // two chains: the larger products apart from the smaller
    float t[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    mma_bf16(t, fa[0], fb[0][2], fb[1][2]);
    mma_bf16(u, fa[0], fb[0][1], fb[1][1]);
    mma_bf16(t, fa[1], fb[0][1], fb[1][1]);
    mma_bf16(u, fa[1], fb[0][0], fb[1][0]);
    mma_bf16(t, fa[2], fb[0][0], fb[1][0]);
    mma_bf16(u, fa[0], fb[0][0], fb[1][0]);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += t[e] + u[e];
  }
}

// One doubling of W's diagonal blocks: with the blocks W0 (rows and columns o
// to s) and W1 (from s on) done, the block of W1's rows and W0's columns is X - W1
// (B1 X), X = N10 - (N10 B0) W0.  A warp does 16 rows (from m0) x 8 columns (from
// o + n0) of it: first X, into `x`, and B1 X into shared memory, then the block.
__device__ __forceinline__ void join_first(float (&x)[4], const float* N, const float* W, float* X, int m0, int o, int s,
                                           int n0, const float* beta) {
  float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  mma_f32<true>(t, N, kLd, m0, W, kLd, o + n0, o, s, beta);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = frag_row(m0, e), c = frag_col(n0);
    const float2 f = *reinterpret_cast<const float2*>(N + r * kLd + o + c);
    x[2 * e] = f.x - t[2 * e];
    x[2 * e + 1] = f.y - t[2 * e + 1];
    *reinterpret_cast<float2*>(X + r * kLx + c) = make_float2(beta[r] * x[2 * e], beta[r] * x[2 * e + 1]);
  }
}
__device__ __forceinline__ void join_second(const float (&x)[4], float* W, const float* X, int m0, int o, int s, int n0) {
  float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  mma_f32<false>(t, W, kLd, m0, X, kLx, n0, s, m0 + 16, nullptr);
#pragma unroll
  for (int e = 0; e < 2; ++e)
    *reinterpret_cast<float2*>(W + frag_row(m0, e) * kLd + o + frag_col(n0)) =
        make_float2(x[2 * e] - t[2 * e], x[2 * e + 1] - t[2 * e + 1]);
}

// The gates of one value head's chunk, by one warp.  `bad`: tokens whose key is
// not finite.
__device__ __forceinline__ void chunk_gates(const Problem& a, int b, int hv, int t0, int rows, const int* bad, float* gates) {
  const int lane = threadIdx.x & 31;
  // sums of log decays in FP64: differences of neighbours stay exact to FP32
  // where the sums are large
  double x[2];
  float be[2];
  unsigned lost[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e, t = t0 + min(i, rows - 1);
    float gv = a.g[b * a.sg[0] + t * a.sg[1] + hv * a.sg[2]];
    be[e] = a.beta[b * a.sb[0] + t * a.sb[1] + hv * a.sb[2]];
    if (i >= rows) gv = be[e] = 0.0f;
    const bool off = bad[i] != 0 || !(gv <= 3.4028235e38f) || !finite(be[e]);
    lost[e] = __ballot_sync(0xffffffffu, off);
    if (!(gv <= 3.4028235e38f)) gv = 0.0f;
    if (!finite(be[e])) be[e] = 0.0f;
    if (gv < kNoDecay) gv = kNoDecay;
    x[e] = gv;
  }
  // The first token with a key, decay or strength that is not finite: it and
  // those after it get NaN through e^G, those before it nothing.
  const int first = min(lost[0] ? 2 * (__ffs(lost[0]) - 1) : kC, lost[1] ? 2 * (__ffs(lost[1]) - 1) + 1 : kC);
  double s = x[0] + x[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  const double end = __shfl_sync(0xffffffffu, s, 31);
  const float top = warp_largest(fmaxf(fabsf(be[0]), fabsf(be[1])));
  if (lane == 0) gates[5 * kC + 4] = plane_scale(plane_inv(top)) * 32768.0f;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    const double gi = e ? s : s - x[1];
    gates[i] = i < first ? expf((float)gi) : __uint_as_float(0x7fffffffu);
    gates[kC + i] = expf((float)(end - gi));
    gates[2 * kC + i] = be[e];
    const double g2 = gi * 1.4426950408889634;
    gates[3 * kC + i] = (float)g2;
    gates[4 * kC + i] = (float)(g2 - (double)(float)g2);
  }
}

// The largest of a value over the CTA (after a barrier).
__device__ __forceinline__ void put_max(float* red, float m) {
  const unsigned u = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(u);
}
__device__ __forceinline__ float get_max(const float* red) {
  float m = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) m = fmaxf(m, red[w]);
  return m;
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads, sizeof(T) * DK > 256 ? 2 : 3) delta_prepare_kernel(const Problem a, const Range range) {
  constexpr int NP = Planes<T>::n;
  constexpr int NQ = kC * DK / 4 / kThreads;
  extern __shared__ __align__(16) unsigned char smem[];
  using L = PrepareSmem<T, DK>;
  f16* ks = reinterpret_cast<f16*>(smem);
  f16* qs = ks + NP * kC * DK;
  float* N = reinterpret_cast<float*>(smem);  // over the planes
  float* W = N + kC * kLd;
  float* X = W + kC * kLd;
  float* gates2 = reinterpret_cast<float*>(smem + L::main);   // of this value head and of the next
  int* bad = reinterpret_cast<int*>(gates2 + 2 * kGates * kC);  // tokens whose key is not finite
  float* red = reinterpret_cast<float*>(bad + kC);         // [4][8] and scales

  let_next_start();
  const int part = blockIdx.x % range.parts, block = blockIdx.x / range.parts;
  const int chunk = range.first + block % range.n, bh = block / range.n;
  const int h = bh % a.Hk, b = bh / a.Hk;
  const int r0 = part * (a.rep / range.parts), r1 = r0 + a.rep / range.parts;
  const long nk = (long)bh * a.nc + chunk;
  const int t0 = chunk * kC, rows = min(kC, a.T - t0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* q = static_cast<const T*>(a.q) + b * a.sq[0] + t0 * a.sq[1] + h * a.sq[2];
  const T* k = static_cast<const T*>(a.k) + b * a.sk[0] + t0 * a.sk[1] + h * a.sk[2];
  constexpr int am = 4 * sizeof(T) - 1;  // 4-element accesses
  const bool vq = ((reinterpret_cast<uintptr_t>(q) | (a.sq[1] * sizeof(T))) & am) == 0;
  const bool vk = ((reinterpret_cast<uintptr_t>(k) | (a.sk[1] * sizeof(T))) & am) == 0;
  if (threadIdx.x < kC) bad[threadIdx.x] = 0;
  __syncthreads();
  {
    // A thread's four elements are half a row of a block: item j is elements
    // [4 j, 4 j + 4) of the tile as it lies in memory.  They stay as loaded until
    // all are there: a conversion in between would wait for each.
    typedef typename Quad<T>::type Raw;
    Raw kr[NQ], qr[NQ];
    auto place = [&](int x, int& r, int& c) {
      const int j = threadIdx.x + x * kThreads, blk = j >> 4;
      r = (blk / (DK / 8)) * 8 + ((j >> 1) & 7), c = (blk % (DK / 8)) * 8 + (j & 1) * 4;
    };
    if (vq && vk && a.dk % 4 == 0) {
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        int r, c;
        place(x, r, c);
        const bool in = r < rows && c < a.dk;
        kr[x] = *reinterpret_cast<const Raw*>(in ? k + r * a.sk[1] + c : k);
        qr[x] = *reinterpret_cast<const Raw*>(in ? q + r * a.sq[1] + c : q);
      }
    } else {
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        int r, c;
        place(x, r, c);
        auto some = [&](const T* p, long stride) {
          const T* row = p + min(r, rows - 1) * stride;
          const int last = a.dk - 1;
          return Quad<T>::make(row[min(c, last)], row[min(c + 1, last)], row[min(c + 2, last)], row[min(c + 3, last)]);
        };
        kr[x] = some(k, a.sk[1]);
        qr[x] = some(q, a.sq[1]);
      }
    }
    const bool whole = rows == kC && a.dk == DK;
    auto value = [&](const Raw& raw, int x) {
      float4 f = Quad<T>::get(raw);
      if (whole) return f;
      int r, c;
      place(x, r, c);
      const int left = r < rows ? a.dk - c : 0;
      f.x = left > 0 ? f.x : 0.0f, f.y = left > 1 ? f.y : 0.0f, f.z = left > 2 ? f.z : 0.0f, f.w = left > 3 ? f.w : 0.0f;
      return f;
    };
    float mk = 0.0f, mq = 0.0f;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const float4 f = value(kr[x], x), g = value(qr[x], x);
      mk = max_mag(max_mag(max_mag(max_mag(mk, f.x), f.y), f.z), f.w);
      mq = max_mag(max_mag(max_mag(max_mag(mq, g.x), g.y), g.z), g.w);
    }
    // A key that is not finite spoils its own token and the later ones (see the
    // gates); inside the products it would reach earlier ones too, so there it
    // counts as zero.
    const bool lost = !finite(mk);
    if (lost) {
      mk = 0.0f;
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        const float4 f = value(kr[x], x);
        mk = max_finite(max_finite(max_finite(max_finite(mk, f.x), f.y), f.z), f.w);
        int r, c;
        place(x, r, c);
        if (!(finite(f.x) && finite(f.y) && finite(f.z) && finite(f.w))) bad[r] = 1;
      }
    }
    if (!finite(mq)) {
      mq = 0.0f;
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        const float4 f = value(qr[x], x);
        mq = max_finite(max_finite(max_finite(max_finite(mq, f.x), f.y), f.z), f.w);
      }
    }
    put_max(red, mk);
    put_max(red + 8, mq);
    __syncthreads();
    const float ik = plane_inv(get_max(red)), iq = plane_inv(get_max(red + 8));
    if (threadIdx.x == 0) {
      red[32] = plane_scale(ik);
      red[33] = plane_scale(iq);
    }
    f16* ko = a.kp + nk * NP * kC * DK;
    f16* qo = a.qp + nk * NP * kC * DK;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int at = (threadIdx.x + x * kThreads) * 4;
      float4 f = value(kr[x], x);
      if (lost) {
        f.x = finite(f.x) ? f.x : 0.0f, f.y = finite(f.y) ? f.y : 0.0f;
        f.z = finite(f.z) ? f.z : 0.0f, f.w = finite(f.w) ? f.w : 0.0f;
      }
      uint32_t w0[NP], w1[NP];
      split2<NP>(f.x, f.y, ik, w0);
      split2<NP>(f.z, f.w, ik, w1);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        *reinterpret_cast<uint2*>(ks + p * kC * DK + at) = make_uint2(w0[p], w1[p]);
        if (part == 0) *reinterpret_cast<uint2*>(ko + p * kC * DK + at) = make_uint2(w0[p], w1[p]);
      }
      f = value(qr[x], x);
      split2<NP>(f.x, f.y, iq, w0);
      split2<NP>(f.z, f.w, iq, w1);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        *reinterpret_cast<uint2*>(qs + p * kC * DK + at) = make_uint2(w0[p], w1[p]);
        if (part == 0) *reinterpret_cast<uint2*>(qo + p * kC * DK + at) = make_uint2(w0[p], w1[p]);
      }
    }
  }
  __syncthreads();

  // this warp's 16 x 32 of K K^T and Q K^T
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 32;
  float ak[4][4], aq[4][4];
  zero(ak);
  zero(aq);
  // warp 1's tiles are above the diagonal: it makes the first gates meanwhile
  if (warp == 1) chunk_gates(a, b, h * a.rep + r0, t0, rows, bad, gates2 + (r0 & 1) * kGates * kC);
  if (n0 <= m0) {
    const uint32_t pk = addr_a<DK, false>(ks, m0 / 8, 0), pq = addr_a<DK, false>(qs, m0 / 8, 0);
    const uint32_t pb = addr_b<DK, false>(ks, 0, n0 / 8);
    // rolled, like the joins' steps: unrolled, a tenth of the stalls are for instructions
#pragma unroll 1
    for (int kk = 0; kk < DK / 16; ++kk) {
      uint32_t fk[NP][4], fq[NP][4], fb[NP][4][2];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        ldm4<false>(fk[p], pk + kk * 256 + p * kC * DK * 2);
        ldm4<false>(fq[p], pq + kk * 256 + p * kC * DK * 2);
      }
      load_b<NP, 4, false>(fb, pb + kk * 256, 32 * DK, kC * DK * 2);
      float t[4][4], u[4][4];
      mma_terms<NP, NP, 4>(t, fk, fb);
      mma_terms<NP, NP, 4>(u, fq, fb);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ak[n][e] += t[n][e];
          aq[n][e] += u[n][e];
        }
    }
  }
  const float sk = red[32], sq = red[33];
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ak[n][e] *= sk * sk;
      aq[n][e] *= sq * sk;
    }
  __syncthreads();
  for (int x = threadIdx.x; x < kC * kLd; x += kThreads) W[x] = 0.0f;  // above its diagonal blocks it stays zero

  for (int r = r0; r < r1; ++r) {
    const int hv = h * a.rep + r;
    const long nv = ((long)b * a.Hv + hv) * a.nc + chunk;
    const float* gates = gates2 + (r & 1) * kGates * kC;
    __syncthreads();
    float mp = 0.0f;
    float pv[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = frag_row(m0, e), j = frag_col(n0 + n * 8);
        float nn[2];
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          const float d = j + l <= i ? decay_between(gates, i, j + l) : 0.0f;
          nn[l] = j + l < i ? ak[n][2 * e + l] * d : 0.0f;
          pv[n][2 * e + l] = j + l <= i ? aq[n][2 * e + l] * (d * a.scale) : 0.0f;
          mp = max_finite(mp, pv[n][2 * e + l]);
        }
        *reinterpret_cast<float2*>(N + i * kLd + j) = make_float2(nn[0], nn[1]);
      }
    put_max(red, mp);
    __syncthreads();
    const float ip = plane_inv(get_max(red));
    f16* pp = a.pp + nv * 2 * kTile;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t w[2];
        split2<2>(pv[n][2 * e], pv[n][2 * e + 1], ip, w);
        const int at = ((m0 / 8 + e) * (kC / 8) + n0 / 8 + n) * 32 + lane;
        reinterpret_cast<uint32_t*>(pp)[at] = w[0];
        reinterpret_cast<uint32_t*>(pp + kTile)[at] = w[1];
      }
    // W's 16 x 16 diagonal blocks, a thread per column: W_ic = N_ic - sum_j
    // N_ij beta_j W_jc, every row's term taken off as soon as it is known
    if (threadIdx.x < kC) {
      const int o = threadIdx.x & ~15, c = threadIdx.x & 15;
      float w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = N[(o + i) * kLd + o + c];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        W[(o + i) * kLd + o + c] = w[i];
        const float u = w[i] * gates[2 * kC + o + i];
#pragma unroll
        for (int j = i + 1; j < 16; ++j) w[j] -= N[(o + j) * kLd + o + i] * u;
      }
    }
    __syncthreads();
    const float* beta = gates + 2 * kC;
    float jx[4];
    // 16 -> 32: two blocks, two column tiles each; the last warp makes the
    // next value head's gates meanwhile
    const int o1 = (warp >> 1) * 32, n1 = (warp & 1) * 8;
    if (warp < 4) join_first(jx, N, W, X, o1 + 16, o1, o1 + 16, n1, beta);
    if (warp == 7 && r + 1 < r1)
      chunk_gates(a, b, hv + 1, t0, rows, bad, gates2 + ((r + 1) & 1) * kGates * kC);
    __syncthreads();
    if (warp < 4) join_second(jx, W, X, o1 + 16, o1, o1 + 16, n1);
    __syncthreads();
    // 32 -> 64: two row tiles, four column tiles
    const int m2 = 32 + (warp >> 2) * 16, n2 = (warp & 3) * 8;
    join_first(jx, N, W, X, m2, 0, 32, n2, beta);
    __syncthreads();
    join_second(jx, W, X, m2, 0, 32, n2);
    __syncthreads();
    // W's planes: a thread takes two rows of eight elements of the tile's blocks
    float4 wx[2][2];
    float mw = 0.0f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int j = threadIdx.x + x * kThreads, blk = j >> 3;
      const float* f = W + ((blk / 8) * 8 + (j & 7)) * kLd + (blk % 8) * 8;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        wx[x][y] = *reinterpret_cast<const float4*>(f + 4 * y);
        const float m = max_finite(max_finite(mw, wx[x][y].x), wx[x][y].y);
        mw = max_finite(max_finite(m, wx[x][y].z), wx[x][y].w);
      }
    }
    put_max(red + 8, mw);
    __syncthreads();
    const float iw = plane_inv(get_max(red + 8));
    f16* wp = a.wp + nv * 2 * kTile;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t w[4][2];
      split2<2>(wx[x][0].x, wx[x][0].y, iw, w[0]);
      split2<2>(wx[x][0].z, wx[x][0].w, iw, w[1]);
      split2<2>(wx[x][1].x, wx[x][1].y, iw, w[2]);
      split2<2>(wx[x][1].z, wx[x][1].w, iw, w[3]);
#pragma unroll
      for (int p = 0; p < 2; ++p)
        reinterpret_cast<uint4*>(wp + p * kTile)[threadIdx.x + x * kThreads] =
            make_uint4(w[0][p], w[1][p], w[2][p], w[3][p]);
    }
    for (int x = threadIdx.x; x < 5 * kC; x += kThreads) a.gates[nv * kGates * kC + x] = gates[x];
    if (threadIdx.x < 5) {
      const float v[5] = {plane_scale(iw), plane_scale(ip), red[32], red[33], gates[5 * kC + 4]};
      a.gates[nv * kGates * kC + 5 * kC + threadIdx.x] = v[threadIdx.x];
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// scan: one CTA per (batch, value head, 32 value columns), chunk after chunk
// (columns do not interact).
//
// Eight warps: four quarters of the rows (tokens, or key columns of the state)
// x two groups of 16 columns.  The state stays in registers as FP32
// accumulators; its planes, those of B R and of U go through shared memory
// between three barriers a chunk (two of them among a group's four warps only),
// every warp's quarter with its own scale, so that no scale needs an exchange of
// its own.  K, W and the gates are loaded a
// chunk ahead; so are the warp's values of V, into registers.
//
// Bound by the chain of three dependent products a chunk (2.6 us at 128 x 128,
// of which the tensor pipe is busy a quarter).  (With a warp to 16
// columns that keeps its whole state in registers and needs no barrier, the
// same work took 6.6 us a chunk at 128 x 128: one warp a scheduler hides none
// of its 3200 instructions' latencies.)
// ---------------------------------------------------------------------------

template <int NP, int DK>
struct ScanSmem {
  static constexpr int k = NP * kC * DK, w = 2 * kTile;  // elements
  static constexpr int stage = (k + w) * 2 + kGates * kC * 4;
  static constexpr int s = 4 * kGroup * DK, x = 4 * kGroup * kC;  // two planes of two groups
  static constexpr int bytes = 2 * stage + (s + 2 * x) * 2 + 3 * 8 * 4 + kSlice * 4;
};

template <int NP, int DK>
__device__ __forceinline__ void scan_load(unsigned char* stage, const Problem& a, long nk, long nv) {
  using L = ScanSmem<NP, DK>;
  f16* k = reinterpret_cast<f16*>(stage);
  copy_async<L::k * 2, kThreads>(k, a.kp + nk * L::k);
  copy_async<L::w * 2, kThreads>(k + L::k, a.wp + nv * L::w);
  copy_async<kGates * kC * 4, kThreads>(k + L::k + L::w, a.gates + nv * kGates * kC);
  cp_async_commit();
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads, 2) delta_scan_kernel(const Problem a, const Range range) {
  constexpr int NP = Planes<T>::n, MT = DK / 64;
  using L = ScanSmem<NP, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int slices = a.dvp / kSlice, groups = a.dvp / kGroup;
  const int bh = blockIdx.x / slices, hv = bh % a.Hv, b = bh / a.Hv;
  const int lane = threadIdx.x & 31, pair = threadIdx.x >> 7, quarter = quarter_of(threadIdx.x);
  const int group = (blockIdx.x % slices) * 2 + pair, c0 = group * kGroup;
  const long nv0 = (long)bh * a.nc, nk0 = ((long)b * a.Hk + hv / a.rep) * a.nc;
  f16* base = reinterpret_cast<f16*>(smem + 2 * L::stage);
  f16* sp = base + pair * kGroup * DK;  // this group's first planes; the second are two groups on
  f16* xp = base + L::s + pair * kGroup * kC;
  f16* yp = xp + L::x;
  float* scales = reinterpret_cast<float*>(base + L::s + 2 * L::x);
  float* ssc = scales + pair * 4;
  float* xsc = scales + 8 + pair * 4;
  float* ysc = scales + 16 + pair * 4;
  int* first = reinterpret_cast<int*>(scales + 24);  // of each column, the first token that is not finite

  float s[MT][2][4];
  // a later range goes on from what the one before it left
  const float* from = range.first ? a.s_out : a.s0;
  const float* s0 = from ? from + (long)bh * a.dk * a.dv : nullptr;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = frag_row((quarter * MT + m) * 16, e >> 1), c = c0 + frag_col(n * 8) + (e & 1);
        s[m][n][e] = s0 && r < a.dk && c < a.dv ? s0[(long)r * a.dv + c] : 0.0f;
      }
  const T* v = static_cast<const T*>(a.v) + b * a.sv[0] + hv * a.sv[2] + c0;
  const bool vec = pairs_ok<T>(a.v, a.sv[0], a.sv[1], a.sv[2], a.dv);
  Columns<T, 2> vt;
  auto load_v = [&](int chunk) {
    const int t = chunk * kC + quarter * 16;
    vt.start(v + t * a.sv[1], a.sv[1], a.T - t, a.dv - c0, vec);
  };
  auto state_out = [&](int chunk) {
    const long nv = nv0 + chunk;
    put_state<DK>(s, quarter, sp, ssc, chunk < range.first + range.n ? a.states + (nv * groups + group) * 2 * kGroup * DK : nullptr,
                  a.sscale + (nv * groups + group) * 4);
  };
  const int end = range.first + range.n;
  load_v(range.first);
  wait_for_before();
  let_next_start();
  scan_load<NP, DK>(smem + (range.first & 1) * L::stage, a, nk0 + range.first, nv0 + range.first);
  if (threadIdx.x < kSlice) first[threadIdx.x] = kC;
  state_out(range.first);
  for (int chunk = range.first; chunk < end; ++chunk) {
    const f16* kp = reinterpret_cast<const f16*>(smem + (chunk & 1) * L::stage);
    const f16* wp = kp + L::k;
    const float* gate = reinterpret_cast<const float*>(wp + L::w);
    const long nv = nv0 + chunk;
    cp_async_wait<0>();
    __syncthreads();
    if (chunk + 1 < end) scan_load<NP, DK>(smem + ((chunk + 1) & 1) * L::stage, a, nk0 + chunk + 1, nv + 1);
    const float sw = gate[5 * kC], sk = gate[5 * kC + 2];
    const int row[2] = {frag_row(quarter * 16, 0), frag_row(quarter * 16, 1)};  // this lane's tokens

    float x[2][4];
    times_state<NP, DK>(x, kp, quarter * 2, sp, ssc);
    // R, and the planes of B R
    bool off = false;
    {
      float y[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float eg = gate[row[e]] * sk, be = gate[2 * kC + row[e]];
          const float2 vv = vt.get(n, e);
          x[n][2 * e] = vv.x - eg * x[n][2 * e];
          x[n][2 * e + 1] = vv.y - eg * x[n][2 * e + 1];
          y[n][2 * e] = be * x[n][2 * e];
          y[n][2 * e + 1] = be * x[n][2 * e + 1];
        }
      if (chunk + 1 < end) load_v(chunk + 1);
      bool all_finite;
      const float inv = plane_inv(warp_max(y, all_finite));
      if (lane == 0) xsc[quarter] = plane_scale(inv);
      if (!all_finite) {
        // What is not finite is left out, since a zero of W times it would
        // reach earlier tokens, and put back below.
        off = true;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[n][e] = finite(y[n][e]) && finite(x[n][e]) ? y[n][e] : 0.0f;
      }
      store_rows<2>(xp, 2 * kGroup * kC, quarter * 2, y, inv, nullptr, 0);
    }
    off = group_sync_or(pair, off);
    if (off) {  // rare, and the same for the whole group
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!finite(x[n][e])) atomicMin(first + pair * kGroup + frag_col(n * 8) + (e & 1), row[e >> 1]);
      group_sync(pair);
    }
    // E
    times_tokens<2, 2, false>(x, wp, quarter * 2, xp, 2 * kGroup * kC * 2, xsc, -sw, 0, quarter + 1);
    if (off) {
      // a later token's error holds every earlier one's
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (row[e >> 1] > first[pair * kGroup + frag_col(n * 8) + (e & 1)]) x[n][e] = __uint_as_float(0x7fffffffu);
    }
    {
      bool all_finite;
      const float inv = plane_inv(warp_max(x, all_finite));
      // a scale below zero marks a quarter that holds something not finite
      if (lane == 0) a.escale[(nv * groups + group) * 4 + quarter] = all_finite ? plane_scale(inv) : -plane_scale(inv);
      f16* out = a.e + (nv * groups + group) * 2 * kGroup * kC;
      store_rows<2>(yp, 2 * kGroup * kC, quarter * 2, x, inv, out, kGroup * kC);  // yp: on the way only
    }
    // S <- e^G S + K^T (e^(G_end - G) U)
    {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] *= gate[kC + row[e >> 1]] * gate[2 * kC + row[e >> 1]];
      const float inv = plane_inv(warp_max(x));
      if (lane == 0) ysc[quarter] = plane_scale(inv);
      __syncwarp();
      store_rows<2>(yp, 2 * kGroup * kC, quarter * 2, x, inv, nullptr, 0);
    }
    group_sync(pair);
    if (off && (threadIdx.x & 127) < kGroup) first[pair * kGroup + (threadIdx.x & 127)] = kC;
    const float decay = gate[kC - 1];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[m][n][e] *= decay;
    add_to_state<NP, DK>(s, kp, quarter, yp, ysc, sk);
    state_out(chunk + 1);
  }
  float* last = a.s_out + (long)bh * a.dk * a.dv;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = frag_row((quarter * MT + m) * 16, e >> 1), c = c0 + frag_col(n * 8) + (e & 1);
        if (r < a.dk && c < a.dv) last[(long)r * a.dv + c] = s[m][n][e];
      }
}

// ---------------------------------------------------------------------------
// output: one CTA per (batch, value head, chunk), 64 value columns at a time; a
// warp takes 16 tokens x 32 columns.  Every operand keeps both planes, whatever
// the output's type: an FP32 result is rounded once, when it is stored (one
// plane of each, 2^-12 of the operands' size, moved a tenth of the bf16 outputs
// by their last bit).  Bound by the latency of its loads.
// ---------------------------------------------------------------------------

template <typename T, int DK>
struct OutputSmem {
  static constexpr int cols = 64;
  static constexpr int q = Planes<T>::n * kC * DK, p = 2 * kTile;  // elements
  static constexpr int s = 2 * cols * DK, e = 2 * cols * kC;
  static constexpr int slice = s + e + 2 * 32;  // and the scales of S and E, four groups and quarters
  static constexpr int buffers = (q + p + 2 * slice) * 2 > 96 * 1024 ? 1 : 2;
  static constexpr int bytes = (q + p + buffers * slice) * 2 + kGates * kC * 4;
};

template <typename T, int DK>
__device__ __forceinline__ void output_load(f16* dst, const Problem& a, long nv, int c0) {
  using L = OutputSmem<T, DK>;
  const long first = nv * (a.dvp / kGroup) + c0 / kGroup;
#pragma unroll
  for (int g = 0; g < L::cols / kGroup; ++g) {
    if (c0 + g * kGroup >= a.dvp) break;
    copy_async<2 * kGroup * DK * 2, kThreads>(dst + g * 2 * kGroup * DK, a.states + (first + g) * 2 * kGroup * DK);
    copy_async<2 * kGroup * kC * 2, kThreads>(dst + L::s + g * 2 * kGroup * kC, a.e + (first + g) * 2 * kGroup * kC);
  }
  if (threadIdx.x < 8) {
    const int g = threadIdx.x & 3;
    if (c0 + g * kGroup < a.dvp)
      cp_async16(dst + L::s + L::e + threadIdx.x * 8, (threadIdx.x < 4 ? a.sscale : a.escale) + (first + g) * 4);
  }
  cp_async_commit();
}

// acc (two groups of 16 columns) += A B, one step of 16; both groups' scales are
// scale[0] and scale[4].
template <int NA, int TILE>
__device__ __forceinline__ void output_step(float (&acc)[4][4], const uint32_t (&fa)[NA][4], uint32_t pb, const float* scale) {
  uint32_t fb[2][4][2];
  load_b<2, 4, true>(fb, pb, 2 * TILE * 2, TILE * 2);
  float t[4][4];
  mma_terms<NA, 2, 4>(t, fa, fb);
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float f = scale[(n >> 1) * 4];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] += f * t[n][e];
  }
}

// An element of P U (without the scales of P and B), for a chunk with an error that is not
// finite: the zeros of P above its diagonal would spread it to earlier tokens.
__device__ __noinline__ float output_element(const f16* pp, const f16* ep, int plane, const float* scale,
                                             int i, int c) {
  float sum = 0.0f;
  for (int j = 0; j <= i; ++j) {
    const int ip = ((i >> 3) * 8 + (j >> 3)) * 64 + (i & 7) * 8 + (j & 7);
    const int ie = ((j >> 3) * 2 + (c >> 3)) * 64 + (j & 7) * 8 + (c & 7);
    float u = 0.0f, w = 0.0f;
    for (int p = 0; p < 2; ++p) {
      u += __half2float(pp[p * kTile + ip]);
      w += __half2float(ep[p * plane + ie]);
    }
    sum += fabsf(scale[j >> 4]) * (u * w);
  }
  return sum;
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads) delta_output_kernel(const Problem a, const Range range) {
  constexpr int NP = Planes<T>::n;
  using L = OutputSmem<T, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  f16* qp = reinterpret_cast<f16*>(smem);
  f16* pp = qp + L::q;
  f16* slices = pp + L::p;
  float* gate = reinterpret_cast<float*>(slices + L::buffers * L::slice);

  const int chunk = range.first + blockIdx.x % range.n, bh = blockIdx.x / range.n;
  const int hv = bh % a.Hv, b = bh / a.Hv;
  const long nv = (long)bh * a.nc + chunk, nk = ((long)b * a.Hk + hv / a.rep) * a.nc + chunk;
  wait_for_before();
  copy_async<L::q * 2, kThreads>(qp, a.qp + nk * L::q);
  copy_async<L::p * 2, kThreads>(pp, a.pp + nv * L::p);
  copy_async<kGates * kC * 4, kThreads>(gate, a.gates + nv * kGates * kC);
  output_load<T, DK>(slices, a, nv, 0);
  const int warp = threadIdx.x >> 5;
  // rows of 1 and 4 steps of P to two of the SM's quarters, of 2 and 3 to the others
  const int m0 = (warp >> 1 ^ warp >> 2) * 16, half = warp & 1;
  T* o = static_cast<T*>(a.o) + (((long)b * a.T + (long)chunk * kC) * a.Hv + hv) * a.dv;
  const int rows = a.T - chunk * kC;
  const bool vec = a.dv % 2 == 0 && (reinterpret_cast<uintptr_t>(o) & (2 * sizeof(T) - 1)) == 0;
  const bool whole = a.dv % 8 == 0 && (reinterpret_cast<uintptr_t>(a.o) & 15) == 0;
  for (int c0 = 0, buf = 0; c0 < a.dvp; c0 += L::cols) {
    cp_async_wait<0>();
    __syncthreads();
    if (c0 == 0) {
      // P -> P B in place, eight columns at a time
      const float ib = 1.0f / gate[5 * kC + 4];  // a power of two
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = threadIdx.x + i * kThreads;  // of 8 elements
        const float* be = gate + 2 * kC + ((row >> 3) & 7) * 8;
        uint32_t r[2][4];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint4 u = reinterpret_cast<const uint4*>(pp + p * kTile)[row];
          r[p][0] = u.x, r[p][1] = u.y, r[p][2] = u.z, r[p][3] = u.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = pair(r[0][j], r[1][j]);
          uint32_t w[2];
          split2<2>(f.x * be[2 * j], f.y * be[2 * j + 1], ib, w);
          r[0][j] = w[0], r[1][j] = w[1];
        }
#pragma unroll
        for (int p = 0; p < 2; ++p)
          reinterpret_cast<uint4*>(pp + p * kTile)[row] = make_uint4(r[p][0], r[p][1], r[p][2], r[p][3]);
      }
      __syncthreads();
    }
    const f16* sp = slices + buf * L::slice;
    const f16* ep = sp + L::s;
    if (L::buffers == 2 && c0 + L::cols < a.dvp) {
      buf ^= 1;
      output_load<T, DK>(slices + buf * L::slice, a, nv, c0 + L::cols);
    }
    const int cw = c0 + half * 32;  // this warp's columns; those it has are whole slices
    if (cw < a.dvp) {
      const float* fs = reinterpret_cast<const float*>(ep + L::e) + half * 8;
      const float* fe = fs + 16;
      const f16* sg = sp + half * 4 * kGroup * DK;
      const f16* eg = ep + half * 4 * kGroup * kC;
      float x[4][4], y[4][4];
      zero(x);
      zero(y);
      {
        const uint32_t pa = addr_a<DK, false>(qp, m0 / 8, 0), pb = addr_b<kGroup, true>(sg, 0, 0);
        constexpr int per = DK / 64;  // steps to a scale
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
          uint32_t fa[NP][4];
#pragma unroll
          for (int p = 0; p < NP; ++p) ldm4<false>(fa[p], pa + kk * 256 + p * kC * DK * 2);
          output_step<NP, kGroup * DK>(x, fa, pb + kk * 512, fs + kk / per);
        }
      }
      bool lost = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) lost |= fe[i] < 0.0f;
      const float fy = gate[5 * kC + 1] * gate[5 * kC + 4];
      if (lost) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            y[n][e] = output_element(pp, eg + (n >> 1) * 2 * kGroup * kC, kGroup * kC, fe + (n >> 1) * 4,
                                         frag_row(m0, e >> 1), frag_col((n & 1) * 8) + (e & 1));
      } else {
        const uint32_t pa = addr_a<kC, false>(pp, m0 / 8, 0), pb = addr_b<kGroup, true>(eg, 0, 0);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          if (kk > m0 / 16) break;
          uint32_t fa[2][4];
#pragma unroll
          for (int p = 0; p < 2; ++p) ldm4<false>(fa[p], pa + kk * 256 + p * kTile * 2);
          output_step<2, kGroup * kC>(y, fa, pb + kk * 512, fe + kk);
        }
      }
      const float fx = a.scale * gate[5 * kC + 3];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e);
        const float f = gate[row] * fx;
        float2 z[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          z[n] = make_float2(f * x[n][2 * e] + fy * y[n][2 * e], f * x[n][2 * e + 1] + fy * y[n][2 * e + 1]);
        set_row<T>(o + (long)row * a.Hv * a.dv + cw, a.dv - cw, vec, whole, row < rows, z);
      }
    }
    if (L::buffers == 1 && c0 + L::cols < a.dvp) {
      __syncthreads();
      output_load<T, DK>(slices, a, nv, c0 + L::cols);
    }
  }
}

template <typename T, int DK>
int run_prepare(const Problem& a, Range r, cudaStream_t stream) {
  constexpr int bytes = PrepareSmem<T, DK>::bytes;
  if (const int rc = with_smem(delta_prepare_kernel<T, DK>, bytes)) return rc;
  LaunchScope scope(kKindDeltaRule, stream);
  const long ctas = (long)a.B * a.Hk * r.n;
  // While SMs are left over, a value head of its own CTA costs only the products of
  // keys once more (a prompt of 77, 4 key and 8 value heads: 48.7 us from call to
  // result, 53.6 with both in turn); in a full grid that would be work for nothing.
  r.parts = ctas * a.rep <= 148 ? a.rep : 1;
  delta_prepare_kernel<T, DK><<<(unsigned)(ctas * r.parts), kThreads, bytes, stream>>>(a, r);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}
template <typename T, int DK>
int run_scan(const Problem& a, Range r, cudaStream_t stream) {
  constexpr int bytes = ScanSmem<Planes<T>::n, DK>::bytes;
  if (const int rc = with_smem(delta_scan_kernel<T, DK>, bytes)) return rc;
  LaunchScope scope(kKindDeltaRule, stream);
  const unsigned ctas = (unsigned)((long)a.B * a.Hv * (a.dvp / kSlice));
  if (r.n == a.nc) return launch_after(delta_scan_kernel<T, DK>, ctas, kThreads, bytes, stream, a, r);
  delta_scan_kernel<T, DK><<<ctas, kThreads, bytes, stream>>>(a, r);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}
template <typename T, int DK>
int run_output(const Problem& a, Range r, cudaStream_t stream) {
  constexpr int bytes = OutputSmem<T, DK>::bytes;
  if (const int rc = with_smem(delta_output_kernel<T, DK>, bytes)) return rc;
  LaunchScope scope(kKindDeltaRule, stream);
  const unsigned ctas = (unsigned)((long)a.B * a.Hv * r.n);
  if (r.n == a.nc) return launch_after(delta_output_kernel<T, DK>, ctas, kThreads, bytes, stream, a, r);
  delta_output_kernel<T, DK><<<ctas, kThreads, bytes, stream>>>(a, r);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

// A scan of few CTAs leaves most of every SM idle, so a long sequence is cut
// into ranges of chunks: while one is scanned, the next is prepared and the one
// before it gets its outputs on a side stream, joined before the call returns.
// Worth its launches where those two take long themselves, from 2048 chunks of
// heads on (about 0.1 ms of them at 128 x 128).
// The first range's preparation and the last one's outputs have no scan beside
// them, so those two are half as long (a prompt of 16384 900 us, in four equal
// ranges 934, two 958, eight 985).
constexpr int kEnds[] = {1, 3, 5, 6};  // of the ranges, in sixths of the chunks
constexpr int kRanges = sizeof(kEnds) / sizeof(int);
template <typename T, int DK>
int forward_typed(const Problem& a, cudaStream_t stream) {
  auto scan = [&](Range r) { return run_scan<T, DK>(a, r, stream); };
  int rc, device;
  Side* side = nullptr;
  if ((long)a.B * a.Hv * (a.dvp / kSlice) <= 148 && (long)a.B * a.Hv * a.nc >= 2048 && a.nc >= 16) {
    GRU_CUDA_TRY(cudaGetDevice(&device));
    if ((rc = side_stream(device, stream, &side))) return rc;
  }
  auto end = [&](int i) { return (int)((long)a.nc * kEnds[i] / kEnds[kRanges - 1]); };
  Range r{0, side ? end(0) : a.nc, 1}, before{0, 0, 1};
  if ((rc = run_prepare<T, DK>(a, r, stream))) return rc;
  if (side && (rc = stream_after(side->s, stream, side->fork))) return rc;
  if ((rc = scan(r))) return rc;
  for (int i = 1; side && i < kRanges; ++i) {
    before = r;
    r.first += r.n;
    r.n = end(i) - r.first;
    if ((rc = run_prepare<T, DK>(a, r, side->s))) return rc;
    GRU_CUDA_TRY(cudaEventRecord(side->fork, stream));  // the scan of the range before
    if ((rc = stream_after(stream, side->s, side->join))) return rc;
    if ((rc = scan(r))) return rc;
    GRU_CUDA_TRY(cudaStreamWaitEvent(side->s, side->fork, 0));
    if ((rc = run_output<T, DK>(a, before, side->s))) return rc;
  }
  if ((rc = run_output<T, DK>(a, r, stream))) return rc;
  return side ? stream_after(stream, side->s, side->join) : GRU_OK;
}

}  // namespace

int forward(const Problem& a, int dtype, cudaStream_t stream) {
  if (dtype == GRU_F32)
    return a.dk <= 64 ? forward_typed<float, 64>(a, stream) : forward_typed<float, 128>(a, stream);
  return a.dk <= 64 ? forward_typed<bf16, 64>(a, stream) : forward_typed<bf16, 128>(a, stream);
}

}  // namespace delta
}  // namespace gru
