// The gated delta rule over chunks of 64 tokens: gradient.
//
// In the notation of the forward, with dS1 the gradient of the state after a
// chunk and P = scale lower(Q K^T o D):
//
//   dU = P^T dO + diag(e^(G_end - G)) K dS1        Z = dU - W^T (B dU)
//   dV = B Z            dbeta_i = Z_i . E_i
//   dS0 = scale Q^T diag(e^G) dO + e^G_end dS1 - K^T diag(e^G) B Z
//   dP' = scale lower(dO U^T) o D                  M = -B strict_lower(Z U^T) o D
//   dQ     = scale diag(e^G) dO S0^T + dP' K
//   dK_row = -diag(e^G) B Z S0^T + M K             (k_i where it carries e^+G_i)
//   dK_col = diag(e^(G_end - G)) U dS1^T + dP'^T Q + M^T K     (where e^-G_i)
//   dg_t = sum_{i >= t} x_i + sum_{i >= t > j} y_ij + sum_{j < t} z_j + e^G_end <S0, dS1>
//
// where x_i = q_i . dq_i + k_i . dk_row_i and z_j = k_j . dk_col_j of the terms
// with the states only, and y_ij = dP'_ij q_i . k_j + M_ij k_i . k_j: what the
// decay of token t multiplies, and nothing besides (running sums of q . dq -
// k . dk would do, but cancel most of their digits).
//
// The chunks' products of queries, keys and W are computed again (`prepare`)
// rather than kept from the forward.  `dout` (all chunks) computes P^T dO;
// `scan` walks the chunks backwards as the forward's scan does, a CTA per head
// and 32 value columns, and leaves dS1 and Z; `grads` (all chunks) does the
// rest, a CTA per key head, over its value heads in a fixed order.

#include "delta_common.cuh"

namespace gru {
namespace delta {
namespace {

template <typename T>
__device__ __forceinline__ bool vec4_ok(const T* p, long stride) {
  return ((reinterpret_cast<uintptr_t>(p) | (stride * sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
}

// A chunk's rows of the output gradient, kSlice columns from c0, as planes.
template <typename T>
__device__ __forceinline__ void load_dout(bf16* dst, const T* p, long stride, int rows, int cols, bool vec) {
  constexpr int NP = Planes<T>::n;
  for (int i = threadIdx.x; i < kC * (kSlice / 4); i += kThreads) {
    const int r = i / (kSlice / 4), c = (i % (kSlice / 4)) * 4;
    const float4 f = get4<T>(p + r * stride + c, r < rows ? cols - c : 0, vec);
    put2<NP>(dst, kC * pitch(kSlice), pitch(kSlice), r, c, f.x, f.y);
    put2<NP>(dst, kC * pitch(kSlice), pitch(kSlice), r, c + 2, f.z, f.w);
  }
}

// ---------------------------------------------------------------------------
// dout: P^T dO, one CTA per (batch, value head, chunk).
// ---------------------------------------------------------------------------

template <typename T>
struct DoutSmem {
  static constexpr int p = 3 * kC * pitch(kC), d = Planes<T>::n * kC * pitch(kSlice);
  static constexpr int bytes = (p + d) * 2;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) delta_dout_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n;
  using L = DoutSmem<T>;
  extern __shared__ __align__(16) unsigned char smem[];
  bf16* pp = reinterpret_cast<bf16*>(smem);
  bf16* op = pp + L::p;
  constexpr int ldx = pitch(kSlice), plx = kC * ldx;
  const int chunk = blockIdx.x % a.nc, bh = blockIdx.x / a.nc;
  const int hv = bh % a.Hv, b = bh / a.Hv;
  const int t0 = chunk * kC, rows = min(kC, a.T - t0);
  const long nv = blockIdx.x, stride = (long)a.Hv * a.dv;
  const T* dout = static_cast<const T*>(a.dout) + ((long)b * a.T + t0) * stride + (long)hv * a.dv;
  const bool vec = vec4_ok(dout, a.dv);
  copy_rows<kC>(pp, a.pp + nv * 3 * kC * kC, 3 * kC);
  cp_async_commit();
  cp_async_wait<0>();
  const int warp = threadIdx.x >> 5;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 16;
  for (int c0 = 0; c0 < a.dvp; c0 += kSlice) {
    load_dout<T>(op, dout + c0, stride, rows, a.dv - c0, vec);
    __syncthreads();
    float acc[2][4];
    zero(acc);
    mma_tile<3, NP, true, true, 2>(acc, pp, kC * pitch(kC), pitch(kC), m0, op, plx, ldx, n0, m0, kC);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(a.du0 + (nv * kC + frag_row(m0, e)) * a.dvp + c0 + frag_col(n0 + n * 8)) =
            make_float2(acc[n][2 * e], acc[n][2 * e + 1]);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// scan: one CTA per (batch, value head, 32 value columns), last chunk first.
// ---------------------------------------------------------------------------

template <int NP, int DK>
struct BackSmem {
  static constexpr int k = NP * kC * pitch(DK);
  static constexpr int w = 3 * kC * pitch(kC);
  static constexpr int stage = (2 * k + w) * 2 + 3 * kC * 4;
  static constexpr int stages = NP == 3 && DK == 128 ? 1 : 2;  // two do not fit there
  static constexpr int s = 3 * DK * pitch(kSlice);
  static constexpr int x = 3 * kC * pitch(kSlice);
  static constexpr int bytes = stages * stage + (s + 3 * x) * 2;
};

template <int NP, int DK>
__device__ __forceinline__ void back_load(unsigned char* stage, const Problem& a, long nk, long nv) {
  using L = BackSmem<NP, DK>;
  bf16* k = reinterpret_cast<bf16*>(stage);
  copy_rows<DK>(k, a.kp + nk * NP * kC * DK, NP * kC);
  copy_rows<DK>(k + L::k, a.qp + nk * NP * kC * DK, NP * kC);
  copy_rows<kC>(k + 2 * L::k, a.wp + nv * 3 * kC * kC, 3 * kC);
  float* sc = reinterpret_cast<float*>(k + 2 * L::k + L::w);
  if (threadIdx.x < 3 * kC / 4) cp_async16(sc + threadIdx.x * 4, a.gates + nv * kGates * kC + threadIdx.x * 4);
  cp_async_commit();
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads) delta_back_scan_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n;
  constexpr int NT = DK / 32;
  using L = BackSmem<NP, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  bf16* sp = reinterpret_cast<bf16*>(smem + L::stages * L::stage);
  bf16* xp = sp + L::s;
  bf16* yp = xp + L::x;
  bf16* op = yp + L::x;
  constexpr int ldx = pitch(kSlice), plx = kC * ldx, pls = DK * ldx;

  const int slices = a.dvp / kSlice;
  const int slice = blockIdx.x % slices, bh = blockIdx.x / slices;
  const int hv = bh % a.Hv, b = bh / a.Hv;
  const int c0 = slice * kSlice;
  const int warp = threadIdx.x >> 5;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 16;
  const int ms = DK == 128 ? warp * 16 : m0, ns = DK == 128 ? 0 : n0;
  const long nv0 = (long)bh * a.nc, nk0 = ((long)b * a.Hk + hv / a.rep) * a.nc;

  float d[NT][4];  // the gradient of the state after the chunk
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = frag_row(ms, e >> 1), c = c0 + frag_col(ns + n * 8) + (e & 1);
      d[n][e] = (a.ds_out && r < a.dk && c < a.dv) ? a.ds_out[((long)bh * a.dk + r) * a.dv + c] : 0.0f;
    }
  const long stride = (long)a.Hv * a.dv;
  const long at = (long)b * a.T * stride + (long)hv * a.dv + c0;
  const T* dout = a.dout ? static_cast<const T*>(a.dout) + at : nullptr;
  T* dv = static_cast<T*>(a.dv_) + at;
  const bool vec = a.dv % 2 == 0;
  float dr[2][4], ur[2][4];
  auto load_rows = [&](int chunk) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e), t = chunk * kC + row, c = frag_col(n0 + n * 8);
        const bool in = dout && t < a.T;
        dr[n][2 * e] = in && c0 + c < a.dv ? as_float(dout[t * stride + c]) : 0.0f;
        dr[n][2 * e + 1] = in && c0 + c + 1 < a.dv ? as_float(dout[t * stride + c + 1]) : 0.0f;
        const float2 u = dout ? *reinterpret_cast<const float2*>(a.du0 + ((nv0 + chunk) * kC + row) * a.dvp + c0 + c)
                              : make_float2(0.0f, 0.0f);
        ur[n][2 * e] = u.x;
        ur[n][2 * e + 1] = u.y;
      }
  };
  auto put_state = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        put2<3>(sp, pls, ldx, frag_row(ms, e), frag_col(ns + n * 8), d[n][2 * e], d[n][2 * e + 1]);
  };

  int buf = 0;
  back_load<NP, DK>(smem, a, nk0 + a.nc - 1, nv0 + a.nc - 1);
  load_rows(a.nc - 1);
  put_state();
  for (int chunk = a.nc - 1; chunk >= 0; --chunk) {
    unsigned char* stage = smem + buf * L::stage;
    const bf16* kp = reinterpret_cast<const bf16*>(stage);
    const bf16* qp = kp + L::k;
    const bf16* wp = qp + L::k;
    const float* gate = reinterpret_cast<const float*>(wp + L::w);
    const long nv = nv0 + chunk;
    cp_async_wait<0>();
    __syncthreads();
    if (L::stages == 2 && chunk > 0) {
      buf ^= 1;
      back_load<NP, DK>(smem + buf * L::stage, a, nk0 + chunk - 1, nv - 1);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(a.dstates + (nv * DK + frag_row(ms, e)) * a.dvp + c0 + frag_col(ns + n * 8)) =
            make_float2(d[n][2 * e], d[n][2 * e + 1]);

    float acc[2][4], du[2][4];
    zero(acc);
    mma_tile<NP, 3, false, true, 2>(acc, kp, kC * pitch(DK), pitch(DK), m0, sp, pls, ldx, n0, 0, DK);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e), col = frag_col(n0 + n * 8);
        const float er = gate[kC + row], be = gate[2 * kC + row], f = gate[row] * a.scale;
        du[n][2 * e] = ur[n][2 * e] + er * acc[n][2 * e];
        du[n][2 * e + 1] = ur[n][2 * e + 1] + er * acc[n][2 * e + 1];
        put2<3>(xp, plx, ldx, row, col, be * du[n][2 * e], be * du[n][2 * e + 1]);
        put2<3>(op, plx, ldx, row, col, f * dr[n][2 * e], f * dr[n][2 * e + 1]);
      }
    if (chunk > 0) load_rows(chunk - 1);
    __syncthreads();
    zero(acc);
    mma_tile<3, 3, true, true, 2>(acc, wp, kC * pitch(kC), pitch(kC), m0, xp, plx, ldx, n0, m0, kC);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e), col = frag_col(n0 + n * 8), t = chunk * kC + row;
        const float z0 = du[n][2 * e] - acc[n][2 * e], z1 = du[n][2 * e + 1] - acc[n][2 * e + 1];
        const float be = gate[2 * kC + row], f = -gate[row] * be;
        *reinterpret_cast<float2*>(a.z + (nv * kC + row) * a.dvp + c0 + col) = make_float2(z0, z1);
        put2<3>(yp, plx, ldx, row, col, f * z0, f * z1);
        if (t < a.T) set2<T>(dv + t * stride + col, a.dv - c0 - col, vec, be * z0, be * z1);
      }
    __syncthreads();
    float x[NT][4];
    zero(x);
    mma_tile<NP, 3, true, true, NT>(x, qp, kC * pitch(DK), pitch(DK), ms, op, plx, ldx, ns, 0, kC);
    mma_tile<NP, 3, true, true, NT>(x, kp, kC * pitch(DK), pitch(DK), ms, yp, plx, ldx, ns, 0, kC);
    const float decay = gate[kC - 1];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[n][e] = decay * d[n][e] + x[n][e];
    put_state();
    if (L::stages == 1 && chunk > 0) {
      __syncthreads();
      back_load<NP, DK>(smem, a, nk0 + chunk - 1, nv - 1);
    }
  }
  if (a.ds0) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = frag_row(ms, e >> 1), c = c0 + frag_col(ns + n * 8) + (e & 1);
        if (r < a.dk && c < a.dv) a.ds0[((long)bh * a.dk + r) * a.dv + c] = d[n][e];
      }
  }
}

// ---------------------------------------------------------------------------
// grads: one CTA per (batch, key head, chunk).
// ---------------------------------------------------------------------------

template <int NP, int DK>
struct GradSmem {
  static constexpr int qk = NP * kC * pitch(DK);
  static constexpr int s = 3 * DK * pitch(kSlice), x = 3 * kC * pitch(kSlice), o = NP * kC * pitch(kSlice);
  static constexpr int slices = 2 * s + 2 * x + o;   // while walking the value columns
  static constexpr int tiles = 2 * 3 * kC * pitch(kC) + 2 * kC * (kC + 1);  // afterwards; y in FP32
  static constexpr int bytes = (2 * qk + (slices > tiles ? slices : tiles)) * 2 + kGates * kC * 4 + (5 * kC + 16) * 4;
};

// The value at (row, col) and (row, col + 1) of a tile held as planes.
template <int NP>
__device__ __forceinline__ float2 take2(const bf16* p, int plane, int ld, int row, int col) {
  float2 f = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = NP - 1; i >= 0; --i) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p + i * plane + row * ld + col);
    f.x += __uint_as_float(w << 16);
    f.y += __uint_as_float(w & 0xffff0000u);
  }
  return f;
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads) delta_grads_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n;
  constexpr int NT = DK / 16;  // a warp's half of the key columns, in 8-column tiles
  using L = GradSmem<NP, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  bf16* qp = reinterpret_cast<bf16*>(smem);
  bf16* kp = qp + L::qk;
  bf16* s0p = kp + L::qk;
  bf16* dsp = s0p + L::s;
  bf16* up = dsp + L::s;
  bf16* zp = up + L::x;
  bf16* op = zp + L::x;
  bf16* dpp = s0p;  // over the slices
  bf16* mp = dpp + 3 * kC * pitch(kC);
  float* gate = reinterpret_cast<float*>(s0p + (L::slices > L::tiles ? L::slices : L::tiles));
  float* y = reinterpret_cast<float*>(mp + 3 * kC * pitch(kC));  // [64][65]
  float* red = gate + kGates * kC;  // x and z of the two column halves, F; then one value per warp
  float* wred = red + 5 * kC;
  constexpr int ldx = pitch(kSlice), plx = kC * ldx, pls = DK * ldx;
  constexpr int ldq = pitch(DK), plq = kC * ldq, ldc = pitch(kC), plc = kC * ldc;

  const int chunk = blockIdx.x % a.nc, bh = blockIdx.x / a.nc;
  const int hk = bh % a.Hk, b = bh / a.Hk;
  const int t0 = chunk * kC, rows = min(kC, a.T - t0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = (warp >> 1) * 16, half = warp & 1;
  const long stride = (long)a.Hv * a.dv;

  copy_rows<DK>(qp, a.qp + (long)blockIdx.x * NP * kC * DK, NP * kC);
  copy_rows<DK>(kp, a.kp + (long)blockIdx.x * NP * kC * DK, NP * kC);
  cp_async_commit();
  cp_async_wait<0>();

  for (int r = 0; r < a.rep; ++r) {
    const int hv = hk * a.rep + r;
    const long nv = ((long)b * a.Hv + hv) * a.nc + chunk;
    const T* dout = a.dout ? static_cast<const T*>(a.dout) + ((long)b * a.T + t0) * stride + (long)hv * a.dv : nullptr;
    const bool vec = vec4_ok(dout, a.dv);
    __syncthreads();
    for (int i = threadIdx.x; i < kGates * kC; i += kThreads) gate[i] = a.gates[nv * kGates * kC + i];
    float dp[4][4], da[4][4], dq[NT][4], dkr[NT][4], dkc[NT][4];
    zero(dp);
    zero(da);
    zero(dq);
    zero(dkr);
    zero(dkc);
    float sdot = 0.0f, bdot[2] = {0.0f, 0.0f};
    __syncthreads();
    for (int c0 = 0; c0 < a.dvp; c0 += kSlice) {
      for (int i = threadIdx.x; i < DK * (kSlice / 4); i += kThreads) {
        const int x = i / (kSlice / 4), c = (i % (kSlice / 4)) * 4;
        const float4 f = *reinterpret_cast<const float4*>(a.states + (nv * DK + x) * a.dvp + c0 + c);
        const float4 g = *reinterpret_cast<const float4*>(a.dstates + (nv * DK + x) * a.dvp + c0 + c);
        put2<3>(s0p, pls, ldx, x, c, f.x, f.y);
        put2<3>(s0p, pls, ldx, x, c + 2, f.z, f.w);
        put2<3>(dsp, pls, ldx, x, c, g.x, g.y);
        put2<3>(dsp, pls, ldx, x, c + 2, g.z, g.w);
        sdot += (f.x * g.x + f.y * g.y) + (f.z * g.z + f.w * g.w);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = threadIdx.x + j * kThreads;
        const int x = i / (kSlice / 4), c = (i % (kSlice / 4)) * 4;
        const float4 f = *reinterpret_cast<const float4*>(a.e + (nv * kC + x) * a.dvp + c0 + c);
        const float4 g = *reinterpret_cast<const float4*>(a.z + (nv * kC + x) * a.dvp + c0 + c);
        const float be = gate[2 * kC + x];
        put2<3>(up, plx, ldx, x, c, be * f.x, be * f.y);
        put2<3>(up, plx, ldx, x, c + 2, be * f.z, be * f.w);
        put2<3>(zp, plx, ldx, x, c, g.x, g.y);
        put2<3>(zp, plx, ldx, x, c + 2, g.z, g.w);
        bdot[j] += (f.x * g.x + f.y * g.y) + (f.z * g.z + f.w * g.w);
      }
      load_dout<T>(op, dout + c0, stride, dout ? rows : 0, a.dv - c0, vec);
      __syncthreads();
      if (half * 32 <= m0) {
        mma_tile<NP, 3, false, false, 4>(dp, op, plx, ldx, m0, up, plx, ldx, half * 32, 0, kSlice);
        mma_tile<3, 3, false, false, 4>(da, zp, plx, ldx, m0, up, plx, ldx, half * 32, 0, kSlice);
      }
      mma_tile<NP, 3, false, false, NT>(dq, op, plx, ldx, m0, s0p, pls, ldx, half * (DK / 2), 0, kSlice);
      mma_tile<3, 3, false, false, NT>(dkr, zp, plx, ldx, m0, s0p, pls, ldx, half * (DK / 2), 0, kSlice);
      mma_tile<3, 3, false, false, NT>(dkc, up, plx, ldx, m0, dsp, pls, ldx, half * (DK / 2), 0, kSlice);
      __syncthreads();
    }
    // the masked 64 x 64 products, over the slices' memory
    {
      float qk[4][4], kk[4][4];
      zero(qk);
      zero(kk);
      if (half * 32 <= m0) {
        mma_tile<NP, NP, false, false, 4>(qk, qp, plq, ldq, m0, kp, plq, ldq, half * 32, 0, DK);
        mma_tile<NP, NP, false, false, 4>(kk, kp, plq, ldq, m0, kp, plq, ldq, half * 32, 0, DK);
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = frag_row(m0, e), j = frag_col(half * 32 + n * 8);
          float u[2], w[2];
#pragma unroll
          for (int l = 0; l < 2; ++l) {
            const float dec = j + l <= i ? expf((gate[3 * kC + i] - gate[3 * kC + j + l]) +
                                                (gate[4 * kC + i] - gate[4 * kC + j + l])) : 0.0f;
            u[l] = j + l <= i ? a.scale * dec * dp[n][2 * e + l] : 0.0f;
            w[l] = j + l < i ? -gate[2 * kC + i] * dec * da[n][2 * e + l] : 0.0f;
            y[i * (kC + 1) + j + l] = j + l < i ? u[l] * qk[n][2 * e + l] + w[l] * kk[n][2 * e + l] : 0.0f;
          }
          put2<3>(dpp, plc, ldc, i, j, u[0], u[1]);
          put2<3>(mp, plc, ldc, i, j, w[0], w[1]);
        }
    }
    float xs[2] = {0.0f, 0.0f}, zs[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e), col = frag_col(half * (DK / 2) + n * 8);
        const float eg = gate[row], er = gate[kC + row], be = gate[2 * kC + row];
        const float2 kv = take2<NP>(kp, plq, ldq, row, col), qv = take2<NP>(qp, plq, ldq, row, col);
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          dq[n][2 * e + l] *= a.scale * eg;
          dkr[n][2 * e + l] *= -eg * be;
          dkc[n][2 * e + l] *= er;
        }
        xs[e] += (qv.x * dq[n][2 * e] + qv.y * dq[n][2 * e + 1]) + (kv.x * dkr[n][2 * e] + kv.y * dkr[n][2 * e + 1]);
        zs[e] += kv.x * dkc[n][2 * e] + kv.y * dkc[n][2 * e + 1];
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        xs[e] += __shfl_xor_sync(0xffffffffu, xs[e], o);
        zs[e] += __shfl_xor_sync(0xffffffffu, zs[e], o);
      }
      if ((lane & 3) == 0) {
        red[half * kC + frag_row(m0, e)] = xs[e];
        red[(2 + half) * kC + frag_row(m0, e)] = zs[e];
      }
    }
    __syncthreads();
    const int nb = half * (DK / 2);
    mma_tile<3, NP, false, true, NT>(dq, dpp, plc, ldc, m0, kp, plq, ldq, nb, 0, m0 + 16);
    mma_tile<3, NP, false, true, NT>(dkr, mp, plc, ldc, m0, kp, plq, ldq, nb, 0, m0 + 16);
    mma_tile<3, NP, true, true, NT>(dkc, dpp, plc, ldc, m0, qp, plq, ldq, nb, m0, kC);
    mma_tile<3, NP, true, true, NT>(dkc, mp, plc, ldc, m0, kp, plq, ldq, nb, m0, kC);
    if (threadIdx.x < kC) {
      // y_ij -> sum over the columns before j
      float* row = y + threadIdx.x * (kC + 1);
      float run = 0.0f;
      for (int j = 0; j < kC; ++j) {
        const float t = row[j];
        row[j] = run;
        run += t;
      }
    }
    __syncthreads();
    {
      const int t = threadIdx.x >> 2;
      float f = 0.0f;
      for (int i = t + (threadIdx.x & 3); i < kC; i += 4) f += y[i * (kC + 1) + t];
      f += __shfl_xor_sync(0xffffffffu, f, 1);
      f += __shfl_xor_sync(0xffffffffu, f, 2);
      if ((threadIdx.x & 3) == 0) red[4 * kC + t] = f;
    }
    float end = gate[kC - 1] * sdot;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) end += __shfl_xor_sync(0xffffffffu, end, o);
    if (lane == 0) wred[warp] = end;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      bdot[j] += __shfl_xor_sync(0xffffffffu, bdot[j], 1);
      bdot[j] += __shfl_xor_sync(0xffffffffu, bdot[j], 2);
      bdot[j] += __shfl_xor_sync(0xffffffffu, bdot[j], 4);
      const int x = (threadIdx.x + j * kThreads) / (kSlice / 4);
      if ((lane & 7) == 0 && x < rows) a.dbeta[((long)b * a.T + t0 + x) * a.Hv + hv] = bdot[j];
    }
    __syncthreads();
    if (warp == 0) {
      // two tokens a lane: x summed from the end, z from the start
      double x[2], z[2], last = 0.0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        x[e] = (double)red[i] + red[kC + i];
        z[e] = (double)red[2 * kC + i] + red[3 * kC + i];
      }
      double sx = x[0] + x[1], sz = z[0] + z[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_down_sync(0xffffffffu, sx, o), w = __shfl_up_sync(0xffffffffu, sz, o);
        if (lane + o < 32) sx += u;
        if (lane >= o) sz += w;
      }
      for (int w = 0; w < kThreads / 32; ++w) last += wred[w];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        if (i < rows) {
          const float gv = a.g[b * a.sg[0] + (t0 + i) * a.sg[1] + hv * a.sg[2]];
          const double from = e ? sx - x[0] : sx, before = e ? sz - z[1] : sz - z[0] - z[1];
          // a decay of zero passes no gradient
          a.dg[((long)b * a.T + t0 + i) * a.Hv + hv] =
              gv < kNoDecay ? 0.0f : (float)(from + before + red[4 * kC + i] + last);
        }
      }
    }
    // dq and dk of a key head are the sums over its value heads
    float* accq = a.dqk + (long)blockIdx.x * 2 * kC * DK;
    float* acck = accq + kC * DK;
    const bool pair = a.dk % 2 == 0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e), col = frag_col(nb + n * 8);
        float2 x = make_float2(dq[n][2 * e], dq[n][2 * e + 1]);
        float2 y = make_float2(dkr[n][2 * e] + dkc[n][2 * e], dkr[n][2 * e + 1] + dkc[n][2 * e + 1]);
        float2* px = reinterpret_cast<float2*>(accq + row * DK + col);
        float2* py = reinterpret_cast<float2*>(acck + row * DK + col);
        if (r > 0) {
          x.x += px->x, x.y += px->y;
          y.x += py->x, y.y += py->y;
        }
        if (r + 1 < a.rep) {
          *px = x;
          *py = y;
        } else if (row < rows) {
          const long o = (((long)b * a.T + t0 + row) * a.Hk + hk) * a.dk + col;
          set2<T>(static_cast<T*>(a.dq) + o, a.dk - col, pair, x.x, x.y);
          set2<T>(static_cast<T*>(a.dk_) + o, a.dk - col, pair, y.x, y.y);
        }
      }
  }
}

template <typename T, int DK>
int backward_typed(const Problem& a, cudaStream_t stream) {
  using D = DoutSmem<T>;
  using S = BackSmem<Planes<T>::n, DK>;
  using G = GradSmem<Planes<T>::n, DK>;
  if (const int rc = with_smem(delta_dout_kernel<T>, D::bytes)) return rc;
  if (const int rc = with_smem(delta_back_scan_kernel<T, DK>, S::bytes)) return rc;
  if (const int rc = with_smem(delta_grads_kernel<T, DK>, G::bytes)) return rc;
  LaunchScope scope(kKindDeltaRule, stream, a.dout ? 3 : 2);
  if (a.dout) {
    delta_dout_kernel<T><<<(unsigned)((long)a.B * a.Hv * a.nc), kThreads, D::bytes, stream>>>(a);
    GRU_CUDA_TRY(cudaGetLastError());
  }
  delta_back_scan_kernel<T, DK><<<(unsigned)((long)a.B * a.Hv * (a.dvp / kSlice)), kThreads, S::bytes, stream>>>(a);
  GRU_CUDA_TRY(cudaGetLastError());
  delta_grads_kernel<T, DK><<<(unsigned)((long)a.B * a.Hk * a.nc), kThreads, G::bytes, stream>>>(a);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

}  // namespace

int backward(const Problem& a, int dtype, cudaStream_t stream) {
  if (const int rc = prepare(a, dtype, stream)) return rc;
  if (dtype == GRU_F32)
    return a.dk <= 64 ? backward_typed<float, 64>(a, stream) : backward_typed<float, 128>(a, stream);
  return a.dk <= 64 ? backward_typed<bf16, 64>(a, stream) : backward_typed<bf16, 128>(a, stream);
}

}  // namespace delta
}  // namespace gru
