// The gated delta rule over chunks of 64 tokens: forward.
//
// With G_i the sum of the log decays of a chunk's tokens up to i, D_ij =
// e^(G_i - G_j), B = diag(beta), S0 the state before the chunk (kernels and
// comments use u_i = beta_i e_i, e_i the delta rule's prediction error):
//
//   N = strict_lower(K K^T o D)          W = (I + N B)^-1 N
//   R = V - diag(e^G) K S0               E = R - W (B R)       U = B E
//   O = scale (diag(e^G) Q S0 + lower(Q K^T o D) U)
//   S1 = e^G_end S0 + (diag(e^(G_end - G)) K)^T U
//
// W holds both inverses that forward and gradient need, without a division by
// beta: (I + N B)^-1 = I - W B and (I + B N)^-1 = I - B W.
//
// Three launches.  `prepare` (all chunks at once) computes W and the masked
// products of queries and keys.  `scan` is the only sequential part: a CTA
// owns 32 value columns of one head's state (columns do not interact), keeps
// them in registers as FP32 and walks the chunks; it writes the state before
// every chunk and E.  `output` (all chunks at once) computes O from them.

#include <algorithm>
#include <string>

#include "delta_common.cuh"

namespace gru {
namespace delta {
namespace {

// ---------------------------------------------------------------------------
// prepare: one CTA per (batch, key head, chunk).
// ---------------------------------------------------------------------------

constexpr int kLd = 68;          // row length of the FP32 64 x 64 tiles: a multiple of 4, not of 32

template <typename T, int DK>
struct PrepareSmem {
  static constexpr int NP = Planes<T>::n;
  static constexpr int planes = 2 * NP * kC * pitch(DK) * 2;
  static constexpr int tiles = 2 * kC * kLd * 4;  // N and W, over the planes once those are used up
  static constexpr int bytes = (planes > tiles ? planes : tiles) + 2 * kC * kLd * 4 + 32 * 36 * 4 + kC * 8 + kGates * kC * 4;
};

// q and k of one chunk as planes in shared memory and in the workspace.
template <typename T, int DK>
__device__ __forceinline__ void load_qk(const T* src, long stride, int rows, int dk, bool vec, bf16* dst, bf16* out) {
  constexpr int NP = Planes<T>::n;
  for (int i = threadIdx.x; i < kC * (DK / 4); i += kThreads) {
    const int r = i / (DK / 4), c = (i % (DK / 4)) * 4;
    const float4 f = get4<T>(src + r * stride + c, r < rows ? dk - c : 0, vec);
    uint32_t w0[NP], w1[NP];
    split2<NP>(f.x, f.y, w0);
    split2<NP>(f.z, f.w, w1);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint2 u = make_uint2(w0[p], w1[p]);
      *reinterpret_cast<uint2*>(dst + (p * kC + r) * pitch(DK) + c) = u;
      *reinterpret_cast<uint2*>(out + (p * kC + r) * DK + c) = u;
    }
  }
}

// One doubling of W's diagonal blocks: with the s x s blocks W0, W1 of a
// 2s x 2s block done, the block below is (I - W1 B1) N10 (I - B0 W0).
__device__ __forceinline__ void join_blocks(int s, const float* N, float* W, const float* beta, float* tmp) {
  const int total = (kC / (2 * s)) * s * s;
  for (int x = threadIdx.x; x < total; x += kThreads) {
    const int blk = x / (s * s), i = (x / s) % s, j = x % s, o = blk * 2 * s;
    const float* n = N + (o + s + i) * kLd + o;
    float a = n[j];
    for (int l = j + 1; l < s; ++l) a -= n[l] * beta[o + l] * W[(o + l) * kLd + o + j];
    tmp[(blk * s + i) * 36 + j] = a;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < total; x += kThreads) {
    const int blk = x / (s * s), i = (x / s) % s, j = x % s, o = blk * 2 * s;
    const float* w = W + (o + s + i) * kLd + o + s;
    float a = tmp[(blk * s + i) * 36 + j];
    for (int l = 0; l < i; ++l) a -= w[l] * beta[o + s + l] * tmp[(blk * s + l) * 36 + j];
    W[(o + s + i) * kLd + o + j] = a;
  }
  __syncthreads();
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads) delta_prepare_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n;
  extern __shared__ __align__(16) unsigned char smem[];
  using L = PrepareSmem<T, DK>;
  bf16* ks = reinterpret_cast<bf16*>(smem);
  bf16* qs = ks + NP * kC * pitch(DK);
  float* N = reinterpret_cast<float*>(smem);  // over the planes
  float* W = N + kC * kLd;
  float* kk = reinterpret_cast<float*>(smem + (L::planes > L::tiles ? L::planes : L::tiles));
  float* qk = kk + kC * kLd;
  float* tmp = qk + kC * kLd;
  double* G = reinterpret_cast<double*>(tmp + 32 * 36);
  float* gates = reinterpret_cast<float*>(G + kC);  // as Problem::gates

  const int chunk = blockIdx.x % a.nc, bh = blockIdx.x / a.nc;
  const int h = bh % a.Hk, b = bh / a.Hk;
  const int t0 = chunk * kC, rows = min(kC, a.T - t0);
  const T* q = static_cast<const T*>(a.q) + b * a.sq[0] + t0 * a.sq[1] + h * a.sq[2];
  const T* k = static_cast<const T*>(a.k) + b * a.sk[0] + t0 * a.sk[1] + h * a.sk[2];
  constexpr int am = 4 * sizeof(T) - 1;  // 4-element accesses
  const bool vq = ((reinterpret_cast<uintptr_t>(q) | (a.sq[1] * sizeof(T))) & am) == 0;
  const bool vk = ((reinterpret_cast<uintptr_t>(k) | (a.sk[1] * sizeof(T))) & am) == 0;
  load_qk<T, DK>(k, a.sk[1], rows, a.dk, vk, ks, a.kp + (long)blockIdx.x * NP * kC * DK);
  load_qk<T, DK>(q, a.sq[1], rows, a.dk, vq, qs, a.qp + (long)blockIdx.x * NP * kC * DK);
  __syncthreads();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 32;
  float ak[4][4], aq[4][4];
  zero(ak);
  zero(aq);
  if (n0 <= m0) {  // the rest is above the diagonal
    mma_tile<NP, NP, false, false, 4>(ak, ks, kC * pitch(DK), pitch(DK), m0, ks, kC * pitch(DK), pitch(DK), n0, 0, DK);
    mma_tile<NP, NP, false, false, 4>(aq, qs, kC * pitch(DK), pitch(DK), m0, ks, kC * pitch(DK), pitch(DK), n0, 0, DK);
  }
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = frag_row(m0, e) * kLd + frag_col(n0 + n * 8);
      *reinterpret_cast<float2*>(kk + at) = make_float2(ak[n][2 * e], ak[n][2 * e + 1]);
      *reinterpret_cast<float2*>(qk + at) = make_float2(aq[n][2 * e], aq[n][2 * e + 1]);
    }
  __syncthreads();

  for (int r = 0; r < a.rep; ++r) {
    const int hv = h * a.rep + r;
    const long nv = ((long)b * a.Hv + hv) * a.nc + chunk;
    if (warp == 0) {
      // sums of log decays in FP64: differences of neighbours stay exact to
      // FP32 where the sums are large
      double x[2];
      float be[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        float gv = i < rows ? a.g[b * a.sg[0] + (t0 + i) * a.sg[1] + hv * a.sg[2]] : 0.0f;
        if (gv < kNoDecay) gv = kNoDecay;
        x[e] = gv;
        be[e] = i < rows ? a.beta[b * a.sb[0] + (t0 + i) * a.sb[1] + hv * a.sb[2]] : 0.0f;
      }
      double s = x[0] + x[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
      }
      const double end = __shfl_sync(0xffffffffu, s, 31);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        const double gi = e ? s : s - x[1];
        G[i] = gi;
        gates[i] = expf((float)gi);
        gates[kC + i] = expf((float)(end - gi));
        gates[2 * kC + i] = be[e];
        gates[3 * kC + i] = (float)gi;
        gates[4 * kC + i] = (float)(gi - (double)(float)gi);
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < kGates * kC; x += kThreads) a.gates[nv * kGates * kC + x] = gates[x];
    bf16* pp = a.pp + nv * 3 * kC * kC;
    for (int x = threadIdx.x; x < kC * kC / 2; x += kThreads) {
      const int i = x / (kC / 2), j = (x % (kC / 2)) * 2;
      const float d0 = j <= i ? expf((float)(G[i] - G[j])) : 0.0f;
      const float d1 = j + 1 <= i ? expf((float)(G[i] - G[j + 1])) : 0.0f;
      const float2 kv = *reinterpret_cast<const float2*>(kk + i * kLd + j);
      const float2 qv = *reinterpret_cast<const float2*>(qk + i * kLd + j);
      *reinterpret_cast<float2*>(N + i * kLd + j) =
          make_float2(j < i ? kv.x * d0 : 0.0f, j + 1 < i ? kv.y * d1 : 0.0f);
      *reinterpret_cast<float2*>(W + i * kLd + j) = make_float2(0.0f, 0.0f);
      put2<3>(pp, kC * kC, kC, i, j, j <= i ? qv.x * d0 * a.scale : 0.0f, j + 1 <= i ? qv.y * d1 * a.scale : 0.0f);
    }
    __syncthreads();
    // W's 16 x 16 diagonal blocks, a thread per column, row by row:
    // W_ic = N_ic - sum_j N_ij beta_j W_jc
    if (threadIdx.x < kC) {
      const int o = threadIdx.x & ~15, c = threadIdx.x & 15;
      float w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = N[(o + i) * kLd + o + c];
#pragma unroll
        for (int j = 0; j < i; ++j) s -= N[(o + i) * kLd + o + j] * w[j];
        W[(o + i) * kLd + o + c] = s;
        w[i] = s * gates[2 * kC + o + i];
      }
    }
    __syncthreads();
    join_blocks(16, N, W, gates + 2 * kC, tmp);
    join_blocks(32, N, W, gates + 2 * kC, tmp);
    bf16* wp = a.wp + nv * 3 * kC * kC;
    for (int x = threadIdx.x; x < kC * kC / 2; x += kThreads) {
      const int i = x / (kC / 2), j = (x % (kC / 2)) * 2;
      const float2 f = *reinterpret_cast<const float2*>(W + i * kLd + j);
      put2<3>(wp, kC * kC, kC, i, j, f.x, f.y);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// scan: one CTA per (batch, value head, 32 value columns), chunk after chunk.
// ---------------------------------------------------------------------------

template <int NP, int DK>
struct ScanSmem {
  static constexpr int k = NP * kC * pitch(DK);      // elements
  static constexpr int w = 3 * kC * pitch(kC);
  static constexpr int stage = (k + w) * 2 + 3 * kC * 4;  // bytes
  static constexpr int s = 3 * DK * pitch(kSlice);
  static constexpr int x = 3 * kC * pitch(kSlice);
  static constexpr int bytes = 2 * stage + (s + 2 * x) * 2;
};

template <int NP, int DK>
__device__ __forceinline__ void scan_load(unsigned char* stage, const Problem& a, long nk, long nv) {
  using L = ScanSmem<NP, DK>;
  bf16* k = reinterpret_cast<bf16*>(stage);
  copy_rows<DK>(k, a.kp + nk * NP * kC * DK, NP * kC);
  copy_rows<kC>(k + L::k, a.wp + nv * 3 * kC * kC, 3 * kC);
  float* sc = reinterpret_cast<float*>(k + L::k + L::w);
  if (threadIdx.x < 3 * kC / 4) cp_async16(sc + threadIdx.x * 4, a.gates + nv * kGates * kC + threadIdx.x * 4);
  cp_async_commit();
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads) delta_scan_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n;
  constexpr int NT = DK / 32;  // 8-column tiles of the state per warp: 16 x 32 (DK 128) or 16 x 16 (DK 64)
  using L = ScanSmem<NP, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  bf16* sp = reinterpret_cast<bf16*>(smem + 2 * L::stage);
  bf16* xp = sp + L::s;
  bf16* yp = xp + L::x;
  constexpr int ldx = pitch(kSlice), plx = kC * ldx, pls = DK * ldx;

  const int slices = a.dvp / kSlice;
  const int slice = blockIdx.x % slices, bh = blockIdx.x / slices;
  const int hv = bh % a.Hv, b = bh / a.Hv;
  const int c0 = slice * kSlice;
  const int warp = threadIdx.x >> 5;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 16;         // of the 64 x 32 tiles
  const int ms = DK == 128 ? warp * 16 : m0, ns = DK == 128 ? 0 : n0;  // of the state
  const long nv0 = (long)bh * a.nc, nk0 = ((long)b * a.Hk + hv / a.rep) * a.nc;

  float s[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = frag_row(ms, e >> 1), c = c0 + frag_col(ns + n * 8) + (e & 1);
      s[n][e] = (a.s0 && r < a.dk && c < a.dv) ? a.s0[((long)bh * a.dk + r) * a.dv + c] : 0.0f;
    }

  const T* v = static_cast<const T*>(a.v) + b * a.sv[0] + hv * a.sv[2] + c0;
  float vr[2][4];
  auto load_v = [&](int chunk) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = chunk * kC + frag_row(m0, e), c = frag_col(n0 + n * 8);
        const T* p = v + t * a.sv[1] + c;
        const bool in = t < a.T;
        vr[n][2 * e] = in && c0 + c < a.dv ? as_float(p[0]) : 0.0f;
        vr[n][2 * e + 1] = in && c0 + c + 1 < a.dv ? as_float(p[1]) : 0.0f;
      }
  };
  auto put_state = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        put2<3>(sp, pls, ldx, frag_row(ms, e), frag_col(ns + n * 8), s[n][2 * e], s[n][2 * e + 1]);
  };

  scan_load<NP, DK>(smem, a, nk0, nv0);
  load_v(0);
  put_state();
  for (int chunk = 0; chunk < a.nc; ++chunk) {
    unsigned char* stage = smem + (chunk & 1) * L::stage;
    const bf16* kp = reinterpret_cast<const bf16*>(stage);
    const bf16* wp = kp + L::k;
    const float* gate = reinterpret_cast<const float*>(wp + L::w);
    const long nv = nv0 + chunk;
    cp_async_wait<0>();
    __syncthreads();
    if (chunk + 1 < a.nc) scan_load<NP, DK>(smem + ((chunk + 1) & 1) * L::stage, a, nk0 + chunk + 1, nv + 1);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(a.states + (nv * DK + frag_row(ms, e)) * a.dvp + c0 + frag_col(ns + n * 8)) =
            make_float2(s[n][2 * e], s[n][2 * e + 1]);

    float acc[2][4], r[2][4];
    zero(acc);
    mma_tile<NP, 3, false, true, 2>(acc, kp, kC * pitch(DK), pitch(DK), m0, sp, pls, ldx, n0, 0, DK);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e);
        const float eg = gate[row], be = gate[2 * kC + row];
        r[n][2 * e] = vr[n][2 * e] - eg * acc[n][2 * e];
        r[n][2 * e + 1] = vr[n][2 * e + 1] - eg * acc[n][2 * e + 1];
        put2<3>(xp, plx, ldx, row, frag_col(n0 + n * 8), be * r[n][2 * e], be * r[n][2 * e + 1]);
      }
    if (chunk + 1 < a.nc) load_v(chunk + 1);
    __syncthreads();
    zero(acc);
    mma_tile<3, 3, false, true, 2>(acc, wp, kC * pitch(kC), pitch(kC), m0, xp, plx, ldx, n0, 0, m0 + 16);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e), col = frag_col(n0 + n * 8);
        const float e0 = r[n][2 * e] - acc[n][2 * e], e1 = r[n][2 * e + 1] - acc[n][2 * e + 1];
        *reinterpret_cast<float2*>(a.e + (nv * kC + row) * a.dvp + c0 + col) = make_float2(e0, e1);
        const float f = gate[kC + row] * gate[2 * kC + row];
        put2<3>(yp, plx, ldx, row, col, f * e0, f * e1);
      }
    __syncthreads();
    float ds[NT][4];
    zero(ds);
    mma_tile<NP, 3, true, true, NT>(ds, kp, kC * pitch(DK), pitch(DK), ms, yp, plx, ldx, ns, 0, kC);
    const float decay = gate[kC - 1];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = decay * s[n][e] + ds[n][e];
    put_state();
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = frag_row(ms, e >> 1), c = c0 + frag_col(ns + n * 8) + (e & 1);
      if (r < a.dk && c < a.dv) a.s_out[((long)bh * a.dk + r) * a.dv + c] = s[n][e];
    }
}

// ---------------------------------------------------------------------------
// output: one CTA per (batch, value head, chunk).
// ---------------------------------------------------------------------------

// Planes of the state and of U: bf16 outputs need no more than two (2^-18 of
// the operands' size, against 2^-9 from rounding the output).
template <typename T>
struct OutPlanes {
  static constexpr int n = Planes<T>::n == 1 ? 2 : 3;
};

template <typename T, int DK>
struct OutputSmem {
  static constexpr int NP = Planes<T>::n, NO = OutPlanes<T>::n;
  static constexpr int q = NP * kC * pitch(DK), p = NO * kC * pitch(kC);
  static constexpr int s = NO * DK * pitch(kSlice), u = NO * kC * pitch(kSlice);
  static constexpr int bytes = (q + p + s + u) * 2 + 3 * kC * 4;
};

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads) delta_output_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n, NO = OutPlanes<T>::n;
  using L = OutputSmem<T, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  bf16* qp = reinterpret_cast<bf16*>(smem);
  bf16* pp = qp + L::q;
  bf16* sp = pp + L::p;
  bf16* up = sp + L::s;
  float* gate = reinterpret_cast<float*>(up + L::u);
  constexpr int ldx = pitch(kSlice), plx = kC * ldx, pls = DK * ldx;

  const int chunk = blockIdx.x % a.nc, bh = blockIdx.x / a.nc;
  const int hv = bh % a.Hv, b = bh / a.Hv;
  const long nv = blockIdx.x, nk = ((long)b * a.Hk + hv / a.rep) * a.nc + chunk;
  copy_rows<DK>(qp, a.qp + nk * NP * kC * DK, NP * kC);
  copy_rows<kC>(pp, a.pp + nv * 3 * kC * kC, NO * kC);
  if (threadIdx.x < 3 * kC / 4) cp_async16(gate + threadIdx.x * 4, a.gates + nv * kGates * kC + threadIdx.x * 4);
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 16;
  T* o = static_cast<T*>(a.o);
  const bool vec = a.dv % 2 == 0 && (reinterpret_cast<uintptr_t>(o) & (2 * sizeof(T) - 1)) == 0;
  for (int c0 = 0; c0 < a.dvp; c0 += kSlice) {
    load_slice<NO>(sp, pls, a.states + nv * DK * a.dvp + c0, a.dvp, DK);
    for (int i = threadIdx.x; i < kC * (kSlice / 4); i += kThreads) {
      const int r = i / (kSlice / 4), c = (i % (kSlice / 4)) * 4;
      const float4 f = *reinterpret_cast<const float4*>(a.e + (nv * kC + r) * a.dvp + c0 + c);
      const float be = gate[2 * kC + r];
      put2<NO>(up, plx, ldx, r, c, be * f.x, be * f.y);
      put2<NO>(up, plx, ldx, r, c + 2, be * f.z, be * f.w);
    }
    __syncthreads();
    float x[2][4], y[2][4];
    zero(x);
    zero(y);
    mma_tile<NP, NO, false, true, 2>(x, qp, kC * pitch(DK), pitch(DK), m0, sp, pls, ldx, n0, 0, DK);
    mma_tile<NO, NO, false, true, 2>(y, pp, kC * pitch(kC), pitch(kC), m0, up, plx, ldx, n0, 0, m0 + 16);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e), c = c0 + frag_col(n0 + n * 8), t = chunk * kC + row;
        if (t < a.T) {
          const float f = a.scale * gate[row];
          set2<T>(o + (((long)b * a.T + t) * a.Hv + hv) * a.dv + c, a.dv - c, vec, f * x[n][2 * e] + y[n][2 * e],
                  f * x[n][2 * e + 1] + y[n][2 * e + 1]);
        }
      }
    __syncthreads();
  }
}

template <typename T, int DK>
int prepare_typed(const Problem& a, cudaStream_t stream) {
  using L = PrepareSmem<T, DK>;
  if (const int rc = with_smem(delta_prepare_kernel<T, DK>, L::bytes)) return rc;
  LaunchScope scope(kKindDeltaRule, stream);
  delta_prepare_kernel<T, DK><<<(unsigned)((long)a.B * a.Hk * a.nc), kThreads, L::bytes, stream>>>(a);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

template <typename T, int DK>
int forward_typed(const Problem& a, cudaStream_t stream) {
  if (const int rc = prepare_typed<T, DK>(a, stream)) return rc;
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

int prepare(const Problem& a, int dtype, cudaStream_t stream) {
  if (dtype == GRU_F32)
    return a.dk <= 64 ? prepare_typed<float, 64>(a, stream) : prepare_typed<float, 128>(a, stream);
  return a.dk <= 64 ? prepare_typed<bf16, 64>(a, stream) : prepare_typed<bf16, 128>(a, stream);
}

int forward(const Problem& a, int dtype, cudaStream_t stream) {
  if (dtype == GRU_F32)
    return a.dk <= 64 ? forward_typed<float, 64>(a, stream) : forward_typed<float, 128>(a, stream);
  return a.dk <= 64 ? forward_typed<bf16, 64>(a, stream) : forward_typed<bf16, 128>(a, stream);
}

}  // namespace delta
}  // namespace gru
