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

// ---------------------------------------------------------------------------
// prepare: one CTA per (batch, key head, chunk), over the head's value heads.
// Latency-bound (a chain of small products between barriers), so it keeps its
// shared memory small enough for several CTAs on an SM.
// ---------------------------------------------------------------------------

constexpr int kLd = 68;  // row length of the FP32 64 x 64 tiles: a multiple of 4, not of 32
constexpr int kLx = 36;

template <typename T, int DK>
struct PrepareSmem {
  static constexpr int NP = Planes<T>::n;
  static constexpr int planes = 2 * NP * kC * DK * 2;
  static constexpr int tiles = (2 * kC * kLd + kC * kLx) * 4;  // N, W and X, over the planes once those are used up
  static constexpr int main = planes > tiles ? planes : tiles;
  static constexpr int bytes = main + kC * 8 + kGates * kC * 4 + kC * 4 + 64 * 4;
};

// acc[n] += A B_n of FP32 tiles in shared memory, A's columns times colscale[k]
// (SCALED): operands as three bf16 planes, which need no scale.  k0, k1: a range
// of k in multiples of 16; A at (m0, k), B at (k, n0).
template <int NT, bool SCALED>
__device__ __forceinline__ void mma_f32(float (&acc)[NT][4], const float* A, int lda, int m0, const float* B, int ldb,
                                        int n0, int k0, int k1, const float* colscale) {
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
  for (int k = k0; k < k1; k += 16) {
    uint32_t fa[3][4];
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
    for (int n = 0; n < NT; ++n) {
      uint32_t fb[2][3];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float* q = B + (k + c + 8 * j) * ldb + n0 + n * 8 + g;
        planes(q[0], q[ldb], fb[j]);
      }
      float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int i = 0; i <= s; ++i) mma_bf16(t, fa[i], fb[0][s - i], fb[1][s - i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] += t[e];
    }
  }
}

// One doubling of W's diagonal blocks, for 16 rows of it from m0 on by one
// warp: with the blocks W0 (rows o.. ) and W1 (rows s..) done, the block below
// W0 is X - W1 (B1 X), X = N10 - (N10 B0) W0.  First half: X into `x` and B1 X
// into shared memory; second half: the block into W.
template <int NT>
__device__ __forceinline__ void join_first(float (&x)[NT][4], const float* N, const float* W, float* X, int m0, int o,
                                           int s, const float* beta) {
  float t[NT][4];
  zero(t);
  mma_f32<NT, true>(t, N, kLd, m0, W, kLd, o, o, s, beta);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = frag_row(m0, e), c = frag_col(n * 8);
      const float2 f = *reinterpret_cast<const float2*>(N + r * kLd + o + c);
      x[n][2 * e] = f.x - t[n][2 * e];
      x[n][2 * e + 1] = f.y - t[n][2 * e + 1];
      *reinterpret_cast<float2*>(X + r * kLx + c) = make_float2(beta[r] * x[n][2 * e], beta[r] * x[n][2 * e + 1]);
    }
}
template <int NT>
__device__ __forceinline__ void join_second(const float (&x)[NT][4], float* W, const float* X, int m0, int o, int s) {
  float t[NT][4];
  zero(t);
  mma_f32<NT, false>(t, W, kLd, m0, X, kLx, 0, s, m0 + 16, nullptr);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float2*>(W + frag_row(m0, e) * kLd + o + frag_col(n * 8)) =
          make_float2(x[n][2 * e] - t[n][2 * e], x[n][2 * e + 1] - t[n][2 * e + 1]);
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
__global__ void __launch_bounds__(kThreads) delta_prepare_kernel(const Problem a, const bool fold_beta) {
  constexpr int NP = Planes<T>::n;
  constexpr int NQ = kC * DK / 4 / kThreads;
  extern __shared__ __align__(16) unsigned char smem[];
  using L = PrepareSmem<T, DK>;
  f16* ks = reinterpret_cast<f16*>(smem);
  f16* qs = ks + NP * kC * DK;
  float* N = reinterpret_cast<float*>(smem);  // over the planes
  float* W = N + kC * kLd;
  float* X = W + kC * kLd;
  double* G = reinterpret_cast<double*>(smem + L::main);
  float* gates = reinterpret_cast<float*>(G + kC);
  int* bad = reinterpret_cast<int*>(gates + kGates * kC);  // tokens whose key is not finite
  float* red = reinterpret_cast<float*>(bad + kC);         // [4][8] and scales

  const int chunk = blockIdx.x % a.nc, bh = blockIdx.x / a.nc;
  const int h = bh % a.Hk, b = bh / a.Hk;
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
    // a thread's four elements are half a row of a block: item j is elements
    // [4 j, 4 j + 4) of the tile as it lies in memory
    float4 kx[NQ], qx[NQ];
    float mk = 0.0f, mq = 0.0f;
    const bool whole = vq && vk && a.dk % 4 == 0;
    auto place = [&](int x, int& r, int& c) {
      const int j = threadIdx.x + x * kThreads, blk = j >> 4;
      r = (blk / (DK / 8)) * 8 + ((j >> 1) & 7), c = (blk % (DK / 8)) * 8 + (j & 1) * 4;
    };
    if (whole) {
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        int r, c;
        place(x, r, c);
        const bool in = r < rows && c < a.dk;
        kx[x] = load4(k + r * a.sk[1] + c, k, in);
        qx[x] = load4(q + r * a.sq[1] + c, q, in);
      }
    } else {
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        int r, c;
        place(x, r, c);
        const int left = r < rows ? a.dk - c : 0;
        kx[x] = load4_any(k + r * a.sk[1] + c, k, left);
        qx[x] = load4_any(q + r * a.sq[1] + c, q, left);
      }
    }
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      int r, c;
      place(x, r, c);
      float m = max_finite(max_finite(0.0f, kx[x].x), kx[x].y);
      mk = fmaxf(mk, max_finite(max_finite(m, kx[x].z), kx[x].w));
      m = max_finite(max_finite(0.0f, qx[x].x), qx[x].y);
      mq = fmaxf(mq, max_finite(max_finite(m, qx[x].z), qx[x].w));
      // A key that is not finite spoils its own token and the later ones (see
      // the gates); inside the products it would reach earlier ones too.
      if (!(fabsf(kx[x].x) + fabsf(kx[x].y) + fabsf(kx[x].z) + fabsf(kx[x].w) <= 3.4028235e38f)) {
        bool lost = false;
        float* f = &kx[x].x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(fabsf(f[i]) <= 3.4028235e38f)) f[i] = 0.0f, lost = true;
        if (lost) bad[r] = 1;
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
    f16* ko = a.kp + (long)blockIdx.x * NP * kC * DK;
    f16* qo = a.qp + (long)blockIdx.x * NP * kC * DK;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int at = (threadIdx.x + x * kThreads) * 4;
      uint32_t w0[NP], w1[NP];
      split2<NP>(kx[x].x, kx[x].y, ik, w0);
      split2<NP>(kx[x].z, kx[x].w, ik, w1);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        *reinterpret_cast<uint2*>(ks + p * kC * DK + at) = make_uint2(w0[p], w1[p]);
        *reinterpret_cast<uint2*>(ko + p * kC * DK + at) = make_uint2(w0[p], w1[p]);
      }
      split2<NP>(qx[x].x, qx[x].y, iq, w0);
      split2<NP>(qx[x].z, qx[x].w, iq, w1);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        *reinterpret_cast<uint2*>(qs + p * kC * DK + at) = make_uint2(w0[p], w1[p]);
        *reinterpret_cast<uint2*>(qo + p * kC * DK + at) = make_uint2(w0[p], w1[p]);
      }
    }
  }
  __syncthreads();

  // this warp's 16 x 32 of K K^T and Q K^T
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 32;
  float ak[4][4], aq[4][4];
  zero(ak);
  zero(aq);
  if (n0 <= m0) {  // the rest is above the diagonal
    const uint32_t pk = addr_a<DK, false>(ks, m0 / 8, 0), pq = addr_a<DK, false>(qs, m0 / 8, 0);
    const uint32_t pb = addr_b<DK, false>(ks, 0, n0 / 8);
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk) {
      uint32_t fk[NP][4], fq[NP][4], fb[NP][4][2];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        ldm4<false>(fk[p], pk + kk * 256 + p * kC * DK * 2);
        ldm4<false>(fq[p], pq + kk * 256 + p * kC * DK * 2);
      }
      load_b<NP, 4, false>(fb, pb + kk * 256, 32 * DK, kC * DK * 2);
      float t[4][4], u[4][4];
      zero(t);
      zero(u);
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

  for (int r = 0; r < a.rep; ++r) {
    const int hv = h * a.rep + r;
    const long nv = ((long)b * a.Hv + hv) * a.nc + chunk;
    if (warp == 0) {
      // sums of log decays in FP64: differences of neighbours stay exact to
      // FP32 where the sums are large
      double x[2];
      float be[2];
      unsigned lost[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        float gv = i < rows ? a.g[b * a.sg[0] + (t0 + i) * a.sg[1] + hv * a.sg[2]] : 0.0f;
        be[e] = i < rows ? a.beta[b * a.sb[0] + (t0 + i) * a.sb[1] + hv * a.sb[2]] : 0.0f;
        const bool off = bad[i] != 0 || !(gv <= 3.4028235e38f) || !(fabsf(be[e]) <= 3.4028235e38f);
        lost[e] = __ballot_sync(0xffffffffu, off);
        if (!(gv <= 3.4028235e38f)) gv = 0.0f;
        if (!(fabsf(be[e]) <= 3.4028235e38f)) be[e] = 0.0f;
        if (gv < kNoDecay) gv = kNoDecay;
        x[e] = gv;
      }
      // The first token with a key, decay or strength that is not finite: it
      // and those after it get NaN through e^G, those before it nothing.
      const int first = min(lost[0] ? 2 * (__ffs(lost[0]) - 1) : kC, lost[1] ? 2 * (__ffs(lost[1]) - 1) + 1 : kC);
      double s = x[0] + x[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
      }
      const double end = __shfl_sync(0xffffffffu, s, 31);
      const float nan = __uint_as_float(0x7fffffffu);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        const double gi = e ? s : s - x[1];
        G[i] = gi;
        gates[i] = i < first ? expf((float)gi) : nan;
        gates[kC + i] = expf((float)(end - gi));
        gates[2 * kC + i] = be[e];
        gates[3 * kC + i] = (float)gi;
        gates[4 * kC + i] = (float)(gi - (double)(float)gi);
      }
    }
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
          const float d = j + l <= i ? expf((float)(G[i] - G[j + l])) : 0.0f;
          nn[l] = j + l < i ? ak[n][2 * e + l] * d : 0.0f;
          const float p = j + l <= i ? aq[n][2 * e + l] * d * a.scale : 0.0f;
          pv[n][2 * e + l] = fold_beta ? p * gates[2 * kC + j + l] : p;
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
    {
      float x[2][4];
      if (warp == 2) join_first<2>(x, N, W, X, 16, 0, 16, beta);
      if (warp == 6) join_first<2>(x, N, W, X, 48, 32, 48, beta);
      __syncthreads();
      if (warp == 2) join_second<2>(x, W, X, 16, 0, 16);
      if (warp == 6) join_second<2>(x, W, X, 48, 32, 48);
      __syncthreads();
    }
    {
      float x[4][4];
      if (warp == 4) join_first<4>(x, N, W, X, 32, 0, 32, beta);
      if (warp == 6) join_first<4>(x, N, W, X, 48, 0, 32, beta);
      __syncthreads();
      if (warp == 4) join_second<4>(x, W, X, 32, 0, 32);
      if (warp == 6) join_second<4>(x, W, X, 48, 0, 32);
      __syncthreads();
    }
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
    if (threadIdx.x < 4) {
      const float v[4] = {plane_scale(iw), plane_scale(ip), red[32], red[33]};
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
// between three barriers a chunk, every warp's quarter with its own scale, so
// that no scale needs an exchange of its own.  K, W and the gates are loaded a
// chunk ahead; so are the warp's values of V, into registers.
//
// Bound by the chain of three dependent products a chunk.  (With a warp to 16
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
  copy_async(k, a.kp + nk * L::k, L::k * 2);
  copy_async(k + L::k, a.wp + nv * L::w, L::w * 2);
  copy_async(k + L::k + L::w, a.gates + nv * kGates * kC, kGates * kC * 4);
  cp_async_commit();
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads, 2) delta_scan_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n, MT = DK / 64;
  using L = ScanSmem<NP, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int slices = a.dvp / kSlice, groups = a.dvp / kGroup;
  const int bh = blockIdx.x / slices, hv = bh % a.Hv, b = bh / a.Hv;
  const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3, pair = threadIdx.x >> 7;
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
  const float* s0 = a.s0 ? a.s0 + (long)bh * a.dk * a.dv : nullptr;
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
  Columns<T> vt;
  auto load_v = [&](int chunk) {
    const int t = chunk * kC + quarter * 16;
    vt.start(v + t * a.sv[1], a.sv[1], a.T - t, a.dv - c0, vec);
  };
  auto state_out = [&](int chunk) {
    const long nv = nv0 + chunk;
    put_state<DK>(s, quarter, sp, ssc, chunk < a.nc ? a.states + (nv * 2 * groups + group) * kGroup * DK : nullptr,
                  (long)a.dvp * DK, a.sscale + (nv * groups + group) * 4);
  };
  scan_load<NP, DK>(smem, a, nk0, nv0);
  load_v(0);
  if (threadIdx.x < kSlice) first[threadIdx.x] = kC;
  state_out(0);
  for (int chunk = 0; chunk < a.nc; ++chunk) {
    const f16* kp = reinterpret_cast<const f16*>(smem + (chunk & 1) * L::stage);
    const f16* wp = kp + L::k;
    const float* gate = reinterpret_cast<const float*>(wp + L::w);
    const long nv = nv0 + chunk;
    cp_async_wait<0>();
    __syncthreads();
    if (chunk + 1 < a.nc) scan_load<NP, DK>(smem + ((chunk + 1) & 1) * L::stage, a, nk0 + chunk + 1, nv + 1);
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
      if (chunk + 1 < a.nc) load_v(chunk + 1);
      const float inv = plane_inv(warp_max(y));
      if (lane == 0) xsc[quarter] = plane_scale(inv);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // What is not finite is left out, since a zero of W times it would
          // reach earlier tokens, and put back below.
          const bool bad0 = !(fabsf(x[n][2 * e]) <= 3.4028235e38f) || !(fabsf(y[n][2 * e]) <= 3.4028235e38f);
          const bool bad1 = !(fabsf(x[n][2 * e + 1]) <= 3.4028235e38f) || !(fabsf(y[n][2 * e + 1]) <= 3.4028235e38f);
          off |= bad0 || bad1;
          uint32_t w[2];
          split2<2>(bad0 ? 0.0f : y[n][2 * e], bad1 ? 0.0f : y[n][2 * e + 1], inv, w);
          store_pair<2>(xp, 2 * kGroup * kC, quarter * 2 + e, n, w);
        }
    }
    off = __syncthreads_or(off);
    if (off) {  // rare, and the same for the whole CTA
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(fabsf(x[n][e]) <= 3.4028235e38f)) atomicMin(first + pair * kGroup + frag_col(n * 8) + (e & 1), row[e >> 1]);
      __syncthreads();
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
      const float inv = plane_inv(warp_max(x));
      // a scale below zero marks a quarter that holds something not finite
      bool lost = false;
      if (off) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) lost |= !(fabsf(x[n][e]) <= 3.4028235e38f);
        lost = __any_sync(0xffffffffu, lost);
      }
      if (lane == 0) a.escale[(nv * groups + group) * 4 + quarter] = lost ? -plane_scale(inv) : plane_scale(inv);
      f16* out = a.e + (nv * 2 * groups + group) * kGroup * kC;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t w[2];
          split2<2>(x[n][2 * e], x[n][2 * e + 1], inv, w);
          store_pair<2>(out, (long)a.dvp * kC, quarter * 2 + e, n, w);
        }
    }
    // S <- e^G S + K^T (e^(G_end - G) U)
    {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] *= gate[kC + row[e >> 1]] * gate[2 * kC + row[e >> 1]];
      const float inv = plane_inv(warp_max(x));
      if (lane == 0) ysc[quarter] = plane_scale(inv);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t w[2];
          split2<2>(x[n][2 * e], x[n][2 * e + 1], inv, w);
          store_pair<2>(yp, 2 * kGroup * kC, quarter * 2 + e, n, w);
        }
    }
    __syncthreads();
    if (off && threadIdx.x < kSlice) first[threadIdx.x] = kC;
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
// output: one CTA per (batch, value head, chunk); a warp takes 16 tokens x 16
// of a slice's 32 value columns, the next slice loads meanwhile.  bf16 outputs
// take the first plane only (2^-12 of the operands' size, against 2^-9 from
// rounding the output), which halves the reading: it is bound by memory.
// ---------------------------------------------------------------------------

template <typename T, int DK>
struct OutputSmem {
  static constexpr int NP = Planes<T>::n;  // planes used, of every operand
  static constexpr int q = NP * kC * DK, p = NP * kTile;
  static constexpr int s = NP * kSlice * DK, e = NP * kSlice * kC;
  static constexpr int bytes = (q + p + 2 * (s + e)) * 2 + kGates * kC * 4;
};

template <typename T, int DK>
__device__ __forceinline__ void output_load(f16* dst, const Problem& a, long nv, int c0) {
  using L = OutputSmem<T, DK>;
#pragma unroll
  for (int p = 0; p < L::NP; ++p) {
    copy_async(dst + p * kSlice * DK, a.states + (nv * 2 + p) * a.dvp * DK + (long)c0 * DK, kSlice * DK * 2);
    copy_async(dst + L::s + p * kSlice * kC, a.e + (nv * 2 + p) * a.dvp * kC + (long)c0 * kC, kSlice * kC * 2);
  }
  cp_async_commit();
}

// acc += A B over `steps` of 16, of which the first nk count; two at a time
// for four independent chains of products.  scale: one for `per` steps.
template <int NP, int STEPS, int PER>
__device__ __forceinline__ void output_product(float (&acc)[2][4], uint32_t pa, int plane_a, uint32_t pb, int plane_b,
                                               int nk, const float (&scale)[4]) {
#pragma unroll
  for (int kk = 0; kk < STEPS; kk += 2) {
    if (kk >= nk) break;
    float t[2][2][4];
    zero(t[0]);
    zero(t[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (kk + h >= nk) break;
      uint32_t fa[NP][4], fb[NP][2][2];
#pragma unroll
      for (int p = 0; p < NP; ++p) ldm4<false>(fa[p], pa + (kk + h) * 256 + p * plane_a);
      load_b<NP, 2, true>(fb, pb + (kk + h) * 512, 0, plane_b);
      mma_terms<NP, NP, 2>(t[h], fa, fb);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] += scale[kk / PER] * t[0][n][e] + scale[(kk + 1) / PER] * t[1][n][e];
  }
}

// y = P E where an error is not finite: element by element, because the zeros
// of P above its diagonal would spread it to earlier tokens.
template <int NP>
__device__ __noinline__ void output_by_element(float (&y)[2][4], const f16* pp, int m0, const f16* ep, float4 scale) {
  const float s[4] = {fabsf(scale.x), fabsf(scale.y), fabsf(scale.z), fabsf(scale.w)};
  for (int x = 0; x < 8; ++x) {
    const int n = x >> 2, e = x & 3;
    const int i = frag_row(m0, e >> 1), c = frag_col(n * 8) + (e & 1);
    float sum = 0.0f;
    for (int j = 0; j <= i; ++j) {
      const int ip = ((i >> 3) * 8 + (j >> 3)) * 64 + (i & 7) * 8 + (j & 7);
      const int ie = ((j >> 3) * 2 + (c >> 3)) * 64 + (j & 7) * 8 + (c & 7);
      float u = 0.0f, w = 0.0f;
      for (int p = 0; p < NP; ++p) {
        u += __half2float(pp[p * kTile + ip]);
        w += __half2float(ep[p * kSlice * kC + ie]);
      }
      sum += s[j >> 4] * (u * w);
    }
    y[n][e] = sum;
  }
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads) delta_output_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n;
  using L = OutputSmem<T, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  f16* qp = reinterpret_cast<f16*>(smem);
  f16* pp = qp + L::q;
  f16* slices = pp + L::p;
  float* gate = reinterpret_cast<float*>(slices + 2 * (L::s + L::e));

  const int chunk = blockIdx.x % a.nc, bh = blockIdx.x / a.nc;
  const int hv = bh % a.Hv, b = bh / a.Hv;
  const long nv = blockIdx.x, nk = ((long)b * a.Hk + hv / a.rep) * a.nc + chunk;
  copy_async(qp, a.qp + nk * L::q, L::q * 2);
  copy_async(pp, a.pp + nv * 2 * kTile, L::p * 2);
  copy_async(gate, a.gates + nv * kGates * kC, kGates * kC * 4);
  output_load<T, DK>(slices, a, nv, 0);
  const int warp = threadIdx.x >> 5;
  const int m0 = (warp >> 1) * 16, half = warp & 1;
  T* o = static_cast<T*>(a.o);
  const bool vec = a.dv % 2 == 0 && (reinterpret_cast<uintptr_t>(o) & (2 * sizeof(T) - 1)) == 0;
  for (int c0 = 0, buf = 0; c0 < a.dvp; c0 += kSlice, buf ^= 1) {
    cp_async_wait<0>();
    __syncthreads();
    if (c0 + kSlice < a.dvp) output_load<T, DK>(slices + (buf ^ 1) * (L::s + L::e), a, nv, c0 + kSlice);
    const f16* sp = slices + buf * (L::s + L::e);
    const f16* ep = sp + L::s;
    const long g = nv * (a.dvp / kGroup) + c0 / kGroup + half;
    const float4 fs = *reinterpret_cast<const float4*>(a.sscale + g * 4);
    const float4 fe = *reinterpret_cast<const float4*>(a.escale + g * 4);
    float x[2][4], y[2][4];
    zero(x);
    zero(y);
    output_product<NP, DK / 16, DK / 64>(x, addr_a<DK, false>(qp, m0 / 8, 0), kC * DK * 2,
                                         addr_b<kGroup, true>(sp + half * kGroup * DK, 0, 0), kSlice * DK * 2, DK / 16,
                                         {fs.x, fs.y, fs.z, fs.w});
    if (fminf(fminf(fe.x, fe.y), fminf(fe.z, fe.w)) < 0.0f) {
      output_by_element<NP>(y, pp, m0, ep + half * kGroup * kC, fe);
    } else {
      output_product<NP, 4, 1>(y, addr_a<kC, false>(pp, m0 / 8, 0), kTile * 2,
                             addr_b<kGroup, true>(ep + half * kGroup * kC, 0, 0), kSlice * kC * 2, m0 / 16 + 1,
                               {fe.x, fe.y, fe.z, fe.w});
    }
    const float fx = a.scale * gate[5 * kC + 3], fy = gate[5 * kC + 1];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e), c = c0 + frag_col(half * 16 + n * 8), t = chunk * kC + row;
        if (t < a.T) {
          const float f = gate[row] * fx;
          set2<T>(o + (((long)b * a.T + t) * a.Hv + hv) * a.dv + c, a.dv - c, vec, f * x[n][2 * e] + fy * y[n][2 * e],
                  f * x[n][2 * e + 1] + fy * y[n][2 * e + 1]);
        }
      }
  }
}

template <typename T, int DK>
int prepare_typed(const Problem& a, bool fold_beta, cudaStream_t stream) {
  using L = PrepareSmem<T, DK>;
  if (const int rc = with_smem(delta_prepare_kernel<T, DK>, L::bytes)) return rc;
  LaunchScope scope(kKindDeltaRule, stream);
  delta_prepare_kernel<T, DK><<<(unsigned)((long)a.B * a.Hk * a.nc), kThreads, L::bytes, stream>>>(a, fold_beta);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

template <typename T, int DK>
int forward_typed(const Problem& a, cudaStream_t stream) {
  if (const int rc = prepare_typed<T, DK>(a, true, stream)) return rc;
  using S = ScanSmem<Planes<T>::n, DK>;
  using O = OutputSmem<T, DK>;
  if (const int rc = with_smem(delta_scan_kernel<T, DK>, S::bytes)) return rc;
  if (const int rc = with_smem(delta_output_kernel<T, DK>, O::bytes)) return rc;
  LaunchScope scope(kKindDeltaRule, stream, 2);
  delta_scan_kernel<T, DK><<<(unsigned)((long)a.B * a.Hv * (a.dvp / kSlice)), kThreads, S::bytes, stream>>>(a);
  GRU_CUDA_TRY(cudaGetLastError());
  delta_output_kernel<T, DK><<<(unsigned)((long)a.B * a.Hv * a.nc), kThreads, O::bytes, stream>>>(a);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

}  // namespace

int prepare(const Problem& a, int dtype, bool fold_beta, cudaStream_t stream) {
  if (dtype == GRU_F32)
    return a.dk <= 64 ? prepare_typed<float, 64>(a, fold_beta, stream) : prepare_typed<float, 128>(a, fold_beta, stream);
  return a.dk <= 64 ? prepare_typed<bf16, 64>(a, fold_beta, stream) : prepare_typed<bf16, 128>(a, fold_beta, stream);
}

int forward(const Problem& a, int dtype, cudaStream_t stream) {
  if (dtype == GRU_F32)
    return a.dk <= 64 ? forward_typed<float, 64>(a, stream) : forward_typed<float, 128>(a, stream);
  return a.dk <= 64 ? forward_typed<bf16, 64>(a, stream) : forward_typed<bf16, 128>(a, stream);
}

}  // namespace delta
}  // namespace gru
