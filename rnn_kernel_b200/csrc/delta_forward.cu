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
// 128, two to a key head: 76 us).
// ---------------------------------------------------------------------------

constexpr int kLd = 68;  // row length of the FP32 64 x 64 tiles: a multiple of 4, not of 32
constexpr int kLx = 36;

// The gates that prepare makes, in shared memory: e^G, e^(G_end - G), beta, the
// exponents (integers) of e^G and of the keys, and the logarithms.
enum Local { kLocalLevel = 3, kLocalKey = 4, kLocalLog = 5, kLocal = 7 };

template <typename T, int DK>
struct PrepareSmem {
  static constexpr int NP = Planes<T>::n;
  static constexpr int planes = 2 * NP * kC * DK * 2;
  static constexpr int tiles = (2 * kC * kLd + kC * kLx) * 4;  // N, W and X, over the planes once those are used up
  static constexpr int main = planes > tiles ? planes : tiles;
  // gates of two value heads, tokens whose key is not finite, the largest
  // magnitudes of K's and Q's rows (then their scales), P's rows', W's exponents
  static constexpr int bytes = main + (2 * kLocal + 6) * kC * 4;
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
// not finite; `key`: scales of K's rows.
__device__ __forceinline__ void chunk_gates(const Problem& a, int b, int hv, int t0, int rows, const int* bad,
                                            const float* key, float* gates) {
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
  // what the planes of P leave out of a token's column: its key's size, in the
  // largest's, and its decay
  const int ke[2] = {exponent_of(key[2 * lane]), exponent_of(key[2 * lane + 1])};
  const int kmax = __reduce_max_sync(0xffffffffu, max(ke[0], ke[1]));
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    const double gi = e ? s : s - x[1];
    gates[i] = i < first ? expf((float)gi) : __uint_as_float(0x7fffffffu);
    gates[kC + i] = expf((float)(end - gi));
    gates[2 * kC + i] = be[e];
    const double g2 = gi * 1.4426950408889634;
    gates[kLocalLog * kC + i] = (float)g2;
    gates[(kLocalLog + 1) * kC + i] = (float)(g2 - (double)(float)g2);
    reinterpret_cast<int*>(gates)[kLocalLevel * kC + i] = (int)floor(g2);
    reinterpret_cast<int*>(gates)[kLocalKey * kC + i] = max(ke[e] - kmax, -60);
  }
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
  int* bad = reinterpret_cast<int*>(gates2 + 2 * kLocal * kC);  // tokens whose key is not finite
  float* ksc = reinterpret_cast<float*>(bad + kC);  // of K's rows and of Q's
  float* qsc = ksc + kC;
  float* prow = qsc + kC;                         // the largest of P's rows
  int* wrow = reinterpret_cast<int*>(prow + kC);  // exponents of the largest of W's rows, and of its columns
  int* wcol = wrow + kC;

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
  if (threadIdx.x < kC) bad[threadIdx.x] = 0, ksc[threadIdx.x] = 0.0f, qsc[threadIdx.x] = 0.0f;
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
    // The largest magnitudes of the rows: those of a thread's items, then of the
    // lanes that share them (bits 0 and 4), then of the warps.
    auto largest = [](const float4& f) { return max_mag(max_mag(max_mag(fabsf(f.x), f.y), f.z), f.w); };
    auto largest_finite = [](const float4& f) {
      return max_finite(max_finite(max_finite(max_finite(0.0f, f.x), f.y), f.z), f.w);
    };
    bool lost = false;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const float4 f = value(kr[x], x), g = value(qr[x], x);
      float mk = largest(f), mq = largest(g);
      int r, c;
      place(x, r, c);
      // A key that is not finite spoils its own token and the later ones (see the
      // gates); inside the products it would reach earlier ones too, so there it
      // counts as zero.
      if (!finite(mk)) {
        lost = true;
        bad[r] = 1;
        mk = largest_finite(f);
      }
      if (!finite(mq)) mq = largest_finite(g);
#pragma unroll
      for (int o = 1; o <= 16; o *= 16) {
        mk = fmaxf(mk, __shfl_xor_sync(0xffffffffu, mk, o));
        mq = fmaxf(mq, __shfl_xor_sync(0xffffffffu, mq, o));
      }
      if (!(lane & 17)) {  // magnitudes: integer order is theirs
        atomicMax(reinterpret_cast<int*>(ksc + r), __float_as_int(mk));
        atomicMax(reinterpret_cast<int*>(qsc + r), __float_as_int(mq));
      }
    }
    __syncthreads();
    if (threadIdx.x < kC) {
      ksc[threadIdx.x] = plane_scale(plane_inv(ksc[threadIdx.x]));
      qsc[threadIdx.x] = plane_scale(plane_inv(qsc[threadIdx.x]));
    }
    __syncthreads();
    f16* ko = a.kp + nk * NP * kC * DK;
    f16* qo = a.qp + nk * NP * kC * DK;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int at = (threadIdx.x + x * kThreads) * 4;
      int r, c;
      place(x, r, c);
      const float ik = plane_scale(ksc[r]), iq = plane_scale(qsc[r]);  // a power of two's inverse
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
  if (warp == 1) chunk_gates(a, b, h * a.rep + r0, t0, rows, bad, ksc, gates2 + (r0 & 1) * kLocal * kC);
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
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = frag_row(m0, e >> 1), j = frag_col(n0 + n * 8) + (e & 1);
      ak[n][e] = ak[n][e] * ksc[i] * ksc[j];
      aq[n][e] = aq[n][e] * qsc[i] * ksc[j];
    }
  __syncthreads();
  for (int x = threadIdx.x; x < kC * kLd; x += kThreads) W[x] = 0.0f;  // above its diagonal blocks it stays zero

  for (int r = r0; r < r1; ++r) {
    const int hv = h * a.rep + r;
    const long nv = ((long)b * a.Hv + hv) * a.nc + chunk;
    const float* gates = gates2 + (r & 1) * kLocal * kC;
    const int* level = reinterpret_cast<const int*>(gates + kLocalLevel * kC);
    const int* key = reinterpret_cast<const int*>(gates + kLocalKey * kC);
    float* out = a.gates + nv * kGates * kC;
    if (threadIdx.x < kC) prow[threadIdx.x] = 0.0f;
    __syncthreads();
    float pv[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = frag_row(m0, e), j = frag_col(n0 + n * 8);
        float nn[2];
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          // the decay, and what of it P's planes hold
          const float* log = gates + kLocalLog * kC;
          const float g = log_between(log, i, j + l), left = g + (float)(level[j + l] - level[i]);
          nn[l] = j + l < i ? ak[n][2 * e + l] * exp2f(g) : 0.0f;
          pv[n][2 * e + l] = j + l <= i ? aq[n][2 * e + l] * (exp2f(left) * a.scale) * power_of(127 - key[j + l]) : 0.0f;
        }
        *reinterpret_cast<float2*>(N + i * kLd + j) = make_float2(nn[0], nn[1]);
      }
    if (n0 <= m0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float m = 0.0f;
#pragma unroll
        for (int n = 0; n < 4; ++n) m = max_finite(max_finite(m, pv[n][2 * e]), pv[n][2 * e + 1]);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        if ((lane & 3) == 0) atomicMax(reinterpret_cast<int*>(prow + frag_row(m0, e)), __float_as_int(m));
      }
    }
    __syncthreads();
    f16* pp = a.pp + nv * 2 * kTile;
    const float ip[2] = {plane_inv(prow[frag_row(m0, 0)]), plane_inv(prow[frag_row(m0, 1)])};
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t w[2];
        split2<2>(pv[n][2 * e], pv[n][2 * e + 1], ip[e], w);
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
      chunk_gates(a, b, hv + 1, t0, rows, bad, ksc, gates2 + ((r + 1) & 1) * kLocal * kC);
    __syncthreads();
    if (warp < 4) join_second(jx, W, X, o1 + 16, o1, o1 + 16, n1);
    __syncthreads();
    // 32 -> 64: two row tiles, four column tiles
    const int m2 = 32 + (warp >> 2) * 16, n2 = (warp & 3) * 8;
    join_first(jx, N, W, X, m2, 0, 32, n2, beta);
    __syncthreads();
    join_second(jx, W, X, m2, 0, 32, n2);
    __syncthreads();
    // The exponents that W's columns leave out: the decays, and the largest of a
    // column in its rows' measure.  With keys of norm one that is about the key's
    // part; a larger key multiplies what later rows hold of earlier columns.
    constexpr int kNone = -(1 << 28);
    {
      const int row = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
      int m = kNone;
#pragma unroll
      for (int y = 0; y < 16; y += 4) {
        const float4 f = *reinterpret_cast<const float4*>(W + row * kLd + c + y);
        const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (v[z] != 0.0f) m = max(m, exponent_of(v[z]) + level[c + y + z]);
      }
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      if ((threadIdx.x & 3) == 0) wrow[row] = m == kNone ? 0 : m - level[row];
      if (threadIdx.x < kC) wcol[threadIdx.x] = kNone;
    }
    __syncthreads();
    {
      const int c = threadIdx.x & (kC - 1), r1 = threadIdx.x / kC * 16;
      int m = kNone;
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const float f = W[(r1 + y) * kLd + c];
        if (f != 0.0f) m = max(m, exponent_of(f) - level[r1 + y] - wrow[r1 + y]);
      }
      if (m != kNone) atomicMax(wcol + c, m + level[c]);
    }
    __syncthreads();
    auto size_w = [&](int c) { return max(wcol[c], -100); };  // none is above zero
    // W's planes: a thread takes two rows of eight elements of the tile's blocks.  A
    // row's largest quotient has the exponent of wrow: the column that gave it is none
    // larger in any row.
    f16* wp = a.wp + nv * 2 * kTile;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int j = threadIdx.x + x * kThreads, blk = j >> 3, row = (blk / 8) * 8 + (j & 7), c8 = blk % 8;
      const float* f = W + row * kLd + c8 * 8;
      const float inv = power_of(268 - max(wrow[row], 27));
      float v[8];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const int c = c8 * 8 + y;
        v[y] = f[y] * power_of(127 + level[c] - level[row] - size_w(c));
      }
      uint32_t w[4][2];
#pragma unroll
      for (int y = 0; y < 4; ++y) split2<2>(v[2 * y], v[2 * y + 1], inv, w[y]);
#pragma unroll
      for (int p = 0; p < 2; ++p)
        reinterpret_cast<uint4*>(wp + p * kTile)[j] = make_uint4(w[0][p], w[1][p], w[2][p], w[3][p]);
    }
    if (threadIdx.x < kC) {
      const int i = threadIdx.x;
      out[kDecay * kC + i] = gates[i];
      out[kRest * kC + i] = gates[kC + i];
      out[kBeta * kC + i] = gates[2 * kC + i];
      out[kScaleK * kC + i] = ksc[i];
      int* whole = reinterpret_cast<int*>(out);
      whole[kColumnW * kC + i] = size_w(i) - level[i];
      whole[kRowW * kC + i] = max(wrow[i], 27) - 14 - 127 + level[i];
      whole[kColumnP * kC + i] = key[i] - level[i];
      whole[kRowP * kC + i] = exponent_of(plane_scale(plane_inv(prow[i]))) - 127 + level[i];
      out[kScaleQ * kC + i] = qsc[i];
      out[kLog * kC + i] = gates[kLocalLog * kC + i];
      out[(kLog + 1) * kC + i] = gates[(kLocalLog + 1) * kC + i];
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
// with scales of a warp's own quarter or tokens, so that no scale needs an
// exchange of its own.  K, W and the gates are loaded a chunk ahead; so are the
// warp's values of V, into registers.
//
// Bound by the chain of three dependent products a chunk (3.2 us at 128 x 128, of
// which the tensor pipe is busy a quarter; 2.6 with a scale to 16 tokens and one
// plane of the states kept).  With a warp to 16 columns that keeps its whole state
// in registers and needs no barrier, the same work took 6.6 us where this took
// 2.6: one warp a scheduler hides none of its 3200 instructions' latencies.
// ---------------------------------------------------------------------------

template <int NP, int DK>
struct ScanSmem {
  static constexpr int k = NP * kC * DK, w = 2 * kTile;  // elements
  static constexpr int stage = (k + w) * 2 + kForward * kC * 4;
  static constexpr int s = 4 * kGroup * DK, x = 4 * kGroup * kC;  // two planes of two groups
  // scales of S and of U, weights of B R's tokens, a token for each column
  static constexpr int bytes = 2 * stage + (s + 2 * x) * 2 + 2 * 8 * 4 + 2 * (kC * 2 + 4 * 4) + kSlice * 4;
};

template <int NP, int DK>
__device__ __forceinline__ void scan_load(unsigned char* stage, const Problem& a, long nk, long nv) {
  using L = ScanSmem<NP, DK>;
  f16* k = reinterpret_cast<f16*>(stage);
  copy_async<L::k * 2, kThreads>(k, a.kp + nk * L::k);
  copy_async<L::w * 2, kThreads>(k + L::k, a.wp + nv * L::w);
  copy_async<kForward * kC * 4, kThreads>(k + L::k + L::w, a.gates + nv * kGates * kC);
  cp_async_commit();
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads, 2) delta_scan_kernel(const Problem a, const Range range) {
  constexpr int NP = Planes<T>::n, MT = DK / 64;
  using L = ScanSmem<NP, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int slices = a.dvp / kSlice, groups = a.dvp / kGroup;
  const int bh = blockIdx.x / slices, hv = bh % a.Hv, b = bh / a.Hv;
  const int pair = threadIdx.x >> 7, quarter = quarter_of(threadIdx.x);
  const int group = (blockIdx.x % slices) * 2 + pair, c0 = group * kGroup;
  const long nv0 = (long)bh * a.nc, nk0 = ((long)b * a.Hk + hv / a.rep) * a.nc;
  f16* base = reinterpret_cast<f16*>(smem + 2 * L::stage);
  f16* sp = base + pair * kGroup * DK;  // this group's first planes; the second are two groups on
  f16* xp = base + L::s + pair * kGroup * kC;
  f16* yp = xp + L::x;
  float* scales = reinterpret_cast<float*>(base + L::s + 2 * L::x);
  float* ssc = scales + pair * 4;
  float* ysc = scales + 8 + pair * 4;
  int* top = reinterpret_cast<int*>(scales + 16) + pair * 4;
  __half* factor = reinterpret_cast<__half*>(scales + 24) + pair * kC;
  int* first = reinterpret_cast<int*>(scales + 24 + kC);  // of each column, the first token that is not finite

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
    const int row[2] = {frag_row(quarter * 16, 0), frag_row(quarter * 16, 1)};  // this lane's tokens
    const float sk[2] = {gate[kScaleK * kC + row[0]], gate[kScaleK * kC + row[1]]};

    const int* whole = reinterpret_cast<const int*>(gate);
    int w[2];
    bool narrow;
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
          const float eg = gate[row[e]] * sk[e], be = gate[kBeta * kC + row[e]];
          const float2 vv = vt.get(n, e);
          x[n][2 * e] = vv.x - eg * x[n][2 * e];
          x[n][2 * e + 1] = vv.y - eg * x[n][2 * e + 1];
          y[n][2 * e] = be * x[n][2 * e];
          y[n][2 * e + 1] = be * x[n][2 * e + 1];
        }
      if (chunk + 1 < end) load_v(chunk + 1);
      // What is not finite is left out, since a zero of W times it would reach
      // earlier tokens, and put back below.
      float m = 0.0f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max_mag(m, y[n][e]);
      off = __any_sync(0xffffffffu, !finite(m));
      if (off) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[n][e] = finite(y[n][e]) && finite(x[n][e]) ? y[n][e] : 0.0f;
      }
      put_tokens<2>(y, quarter, xp, w, nullptr, nullptr);
      w[0] += whole[kColumnW * kC + row[0]];
      w[1] += whole[kColumnW * kC + row[1]];
      narrow = put_weights(w, quarter, factor, top);
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
    const int rw[2] = {whole[kRowW * kC + row[0]], whole[kRowW * kC + row[1]]};
    times_tokens<2, false, true>(x, wp, rw, quarter, xp, w, narrow, factor, top, -1.0f);
    if (off) {
      // a later token's error holds every earlier one's
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (row[e >> 1] > first[pair * kGroup + frag_col(n * 8) + (e & 1)]) x[n][e] = __uint_as_float(0x7fffffffu);
    }
    {
      put_tokens<2>(x, quarter, yp, w, a.e + (nv * groups + group) * 2 * kGroup * kC,
                    a.escale + (nv * groups + group) * kC);  // yp: on the way only
    }
    // S <- e^G S + K^T (e^(G_end - G) U)
    {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] *= gate[kRest * kC + row[e >> 1]] * gate[kBeta * kC + row[e >> 1]] * sk[e >> 1];
      __syncwarp();
      put_sum(x, quarter, yp, ysc);
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
    add_to_state<NP, DK>(s, kp, quarter, yp, ysc);
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
// by their last bit).  2048 chunks of heads of 128 x 128, bf16: 78 us, with one
// plane 46.  Bound by the latency of its loads; memory is a third busy.
// ---------------------------------------------------------------------------

template <typename T, int DK>
struct OutputSmem {
  static constexpr int cols = 64;
  static constexpr int q = Planes<T>::n * kC * DK, p = 2 * kTile;  // elements
  static constexpr int s = 2 * cols * DK, e = 2 * cols * kC;
  static constexpr int slice = s + e + 2 * (16 + 4 * kC);  // and the scales of S (four groups and quarters) and of E
  static constexpr int buffers = (q + p + 2 * slice) * 2 > 96 * 1024 ? 1 : 2;
  // P's exponents, and of four groups' tokens the weights' exponents, factors and tops
  static constexpr int bytes = (q + p + buffers * slice) * 2 + (kBackward + 1) * kC * 4 + 4 * (kC * 4 + kC * 2 + 2 * 4 * 4);
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
  if (threadIdx.x < 4 + 4 * 16) {
    const int t = threadIdx.x - 4, g = t < 0 ? threadIdx.x : t >> 4;
    if (c0 + g * kGroup < a.dvp)
      cp_async16(dst + L::s + L::e + threadIdx.x * 8, t < 0 ? a.sscale + (first + g) * 4 : a.escale + (first + g) * kC + (t & 15) * 4);
  }
  cp_async_commit();
}

// An element of P U, for a chunk with an error that is not finite: the zeros of P
// above its diagonal would spread it to earlier tokens.
__device__ __noinline__ float output_element(const f16* pp, int row, const int* column, const f16* ep, int plane,
                                             const float* scale, int i, int c) {
  float sum = 0.0f;
  for (int j = 0; j <= i; ++j) {
    const int ip = ((i >> 3) * 8 + (j >> 3)) * 64 + (i & 7) * 8 + (j & 7);
    const int ie = ((j >> 3) * 2 + (c >> 3)) * 64 + (j & 7) * 8 + (c & 7);
    float u = 0.0f, w = 0.0f;
    for (int p = 0; p < 2; ++p) {
      u += __half2float(pp[p * kTile + ip]);
      w += __half2float(ep[p * plane + ie]);
    }
    sum += power_of(row + column[j] + 127) * (fabsf(scale[j]) * (u * w));
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
  copy_async<kBackward * kC * 4, kThreads>(gate, a.gates + nv * kGates * kC);
  const int* gates = reinterpret_cast<const int*>(gate);
  int* column = reinterpret_cast<int*>(gate + kBackward * kC);  // P's, with the exponents of beta
  int* weight = column + kC;
  int* top = weight + 4 * kC;
  int* narrow = top + 4 * 4;
  __half* factor = reinterpret_cast<__half*>(narrow + 4 * 4);
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
      // P -> P B in place, eight columns at a time, but for powers of two that
      // leave |beta| in [1/2, 1]
      if (threadIdx.x < kC) {
        float& be = gate[kBeta * kC + threadIdx.x];
        const int up = exponent_of(be) + 1;  // of the least power above it, biased
        column[threadIdx.x] = gates[kColumnP * kC + threadIdx.x] + up - 127;
        be *= power_of(max(254 - up, 1));
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = threadIdx.x + i * kThreads;  // of 8 elements
        const float* be = gate + kBeta * kC + ((row >> 3) & 7) * 8;
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
          split2<2>(f.x * be[2 * j], f.y * be[2 * j + 1], 1.0f, w);
          r[0][j] = w[0], r[1][j] = w[1];
        }
#pragma unroll
        for (int p = 0; p < 2; ++p)
          reinterpret_cast<uint4*>(pp + p * kTile)[row] = make_uint4(r[p][0], r[p][1], r[p][2], r[p][3]);
      }
    }
    const f16* sp = slices + buf * L::slice;
    const f16* ep = sp + L::s;
    {
      // the weights of this slice's tokens: a thread has a group's token, half a warp
      // its 16 tokens
      const int w = exponent_of(reinterpret_cast<const float*>(ep + L::e)[16 + threadIdx.x]) + column[threadIdx.x & (kC - 1)];
      int m = w, least = w;
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      }
      weight[threadIdx.x] = w;
      factor[threadIdx.x] = __low2half(two_powers(w - m, 0));
      if ((threadIdx.x & 15) == 0) {
        top[threadIdx.x >> 4] = m;
        narrow[threadIdx.x >> 4] = m - least <= kNarrow;
      }
    }
    __syncthreads();
    if (L::buffers == 2 && c0 + L::cols < a.dvp) {
      buf ^= 1;
      output_load<T, DK>(slices + buf * L::slice, a, nv, c0 + L::cols);
    }
    const int cw = c0 + half * 32;  // this warp's columns; those it has are whole slices
    if (cw < a.dvp) {
      const float* fs = reinterpret_cast<const float*>(ep + L::e) + half * 8;
      const float* fe = reinterpret_cast<const float*>(ep + L::e) + 16 + half * 2 * kC;
      const f16* sg = sp + half * 4 * kGroup * DK;
      const f16* eg = ep + half * 4 * kGroup * kC;
      float x[4][4], y[4][4];
      zero(x);
      zero(y);
      {
        const uint32_t pa = addr_a<DK, false>(qp, m0 / 8, 0), pb = addr_b<kGroup, true>(sg, 0, 0);
        constexpr int per = DK / 64;  // steps to a scale
        float t[4][4];
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
          uint32_t fa[NP][4], fb[2][4][2];
#pragma unroll
          for (int p = 0; p < NP; ++p) ldm4<false>(fa[p], pa + kk * 256 + p * kC * DK * 2);
          load_b<2, 4, true>(fb, pb + kk * 512, 2 * kGroup * DK * 2, kGroup * DK * 2);
          // a bf16 output adds the steps of one scale up on the tensor core
          if (NP == 1 && kk % per != 0) {
#pragma unroll
            for (int p = 1; p >= 0; --p)
#pragma unroll
              for (int n = 0; n < 4; ++n) mma(t[n], fa[0], fb[p][n][0], fb[p][n][1]);
          } else {
            mma_terms<NP, 2, 4>(t, fa, fb);
          }
          if (NP == 1 && kk % per != per - 1) continue;
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[n][e] += fs[kk / per + (n >> 1) * 4] * t[n][e];
        }
      }
      bool lost = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) lost |= fe[i * 16] < 0.0f;
      const int row[2] = {frag_row(m0, 0), frag_row(m0, 1)};
      const int row_p[2] = {gates[kRowP * kC + row[0]], gates[kRowP * kC + row[1]]};
      if (lost) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            y[n][e] = output_element(pp, row_p[e >> 1], column, eg + (n >> 1) * 2 * kGroup * kC, kGroup * kC,
                                     fe + (n >> 1) * kC, row[e >> 1], frag_col((n & 1) * 8) + (e & 1));
      } else {
        const uint32_t pa = addr_a<kC, false>(pp, m0 / 8, 0), pb = addr_b<kGroup, true>(eg, 0, 0);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          if (kk > m0 / 16) break;
          uint32_t fp[2][4], fb[2][4][2];
#pragma unroll
          for (int p = 0; p < 2; ++p) ldm4<false>(fp[p], pa + kk * 256 + p * kTile * 2);
          load_b<2, 4, true>(fb, pb + kk * 512, 2 * kGroup * kC * 2, kGroup * kC * 2);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int group = half * 2 + g, *wg = weight + group * kC;
            Weights f;
            if (kk == m0 / 16 && !narrow[group * 4 + kk]) {
              const int own[2] = {wg[row[0]], wg[row[1]]};
              f = diagonal_weights<false, false>(own);
            } else {
              f = get_weights(kk, factor + group * kC, top + group * 4);
            }
            uint32_t fa[2][4], fg[2][2][2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
#pragma unroll
              for (int i = 0; i < 4; ++i) fa[p][i] = fp[p][i], fg[p][i >> 1][i & 1] = fb[p][2 * g + (i >> 1)][i & 1];
              weigh(fa[p], f);
            }
            float t[2][4];
            mma_terms<2, 2, 2>(t, fa, fg);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float r = power_of(f.top[e] + row_p[e]);
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                y[2 * g + n][2 * e] += r * t[n][2 * e];
                y[2 * g + n][2 * e + 1] += r * t[n][2 * e + 1];
              }
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f = gate[row[e]] * gate[kScaleQ * kC + row[e]] * a.scale;
        float2 z[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          z[n] = make_float2(f * x[n][2 * e] + y[n][2 * e], f * x[n][2 * e + 1] + y[n][2 * e + 1]);
        set_row<T>(o + (long)row[e] * a.Hv * a.dv + cw, a.dv - cw, vec, whole, row[e] < rows, z);
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
  // keys once more (a prompt of 77, 4 key and 8 value heads: 48 us from call to
  // result, 53 with both in turn); in a full grid that would be work for nothing.
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
// them, so those two are half as long (a prompt of 16384 1192 us, in four equal
// ranges 1232, two 1244, six 1262, not cut 1765).
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
