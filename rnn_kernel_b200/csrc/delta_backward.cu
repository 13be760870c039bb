// The gated delta rule over chunks of 64 tokens: gradient.
//
// In the notation of the forward, with dS1 the gradient of the state after a
// chunk:
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
// K, Q, W and P come as the forward left them.  `scan` walks the chunks backwards as the forward's scan does and leaves dS1,
// Z and dO as planes; `grads` (all chunks at once) does the rest, a CTA per key
// head, over its value heads in a fixed order.

#include "delta_scan.cuh"

namespace gru {
namespace delta {
namespace {

// ---------------------------------------------------------------------------
// scan: one CTA per (batch, value head, 32 value columns), last chunk first, in
// the forward scan's division of work: eight warps, four quarters of the rows x
// two groups of 16 columns, dS in registers, planes through shared memory
// between three barriers a chunk (2048 chunks of heads of 128 x 128, bf16: 260 us;
// bound by the chain of four dependent products a chunk).
// ---------------------------------------------------------------------------

template <int NP, int DK, int STAGES>
struct BackSmem {
  static constexpr int k = NP * kC * DK, w = 2 * kTile;  // elements; K, Q, W, P
  static constexpr int stage = 2 * (k + w) * 2 + kBackward * kC * 4;
  // two planes of two groups (of dO, NP): dS, B dU, e^G B Z, e^G dO; dO
  static constexpr int s = 4 * kGroup * DK, x = 4 * kGroup * kC, o = NP * 2 * kGroup * kC;
  // scales of dS, e^G B Z and e^G dO, weights of B dU's and dO's tokens
  static constexpr int bytes = STAGES * stage + (s + 3 * x + o) * 2 + 3 * 8 * 4 + 4 * (kC * 2 + 4 * 4);
};

template <int NP, int DK>
__device__ __forceinline__ void back_load(unsigned char* stage, const Problem& a, long nk, long nv) {
  using L = BackSmem<NP, DK, 1>;
  f16* p = reinterpret_cast<f16*>(stage);
  copy_async<L::k * 2, kThreads>(p, a.kp + nk * L::k);
  copy_async<L::k * 2, kThreads>(p + L::k, a.qp + nk * L::k);
  copy_async<L::w * 2, kThreads>(p + 2 * L::k, a.wp + nv * L::w);
  copy_async<L::w * 2, kThreads>(p + 2 * L::k + L::w, a.pp + nv * L::w);
  copy_async<kBackward * kC * 4, kThreads>(p + 2 * (L::k + L::w), a.gates + nv * kGates * kC);
  cp_async_commit();
}

// STAGES: with two the next chunk's tiles load during this one; with one they
// load between chunks, and two CTAs fit on an SM.
template <typename T, int DK, int STAGES>
__global__ void __launch_bounds__(kThreads, 2) delta_back_scan_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n, MT = DK / 64;
  using L = BackSmem<NP, DK, STAGES>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int slices = a.dvp / kSlice, groups = a.dvp / kGroup;
  const int bh = blockIdx.x / slices, hv = bh % a.Hv, b = bh / a.Hv;
  const int pair = threadIdx.x >> 7, quarter = quarter_of(threadIdx.x);
  const int group = (blockIdx.x % slices) * 2 + pair, c0 = group * kGroup;
  const long nv0 = (long)bh * a.nc, nk0 = ((long)b * a.Hk + hv / a.rep) * a.nc;
  let_next_start();
  f16* base = reinterpret_cast<f16*>(smem + STAGES * L::stage);
  f16* sp = base + pair * kGroup * DK;
  f16* up = base + L::s + pair * kGroup * kC;  // B dU
  f16* zp = up + L::x;                         // -e^G B Z
  f16* qop = zp + L::x;                        // scale e^G dO
  f16* op = base + L::s + 3 * L::x + pair * kGroup * kC;
  float* scales = reinterpret_cast<float*>(base + L::s + 3 * L::x + L::o) + pair * 4;
  float *ssc = scales, *zsc = scales + 8, *qosc = scales + 16;
  int* utop = reinterpret_cast<int*>(scales - pair * 4 + 24) + pair * 4;
  int* otop = utop + 8;
  __half* ufactor = reinterpret_cast<__half*>(scales - pair * 4 + 40) + pair * kC;
  __half* ofactor = ufactor + 2 * kC;
  const int row[2] = {frag_row(quarter * 16, 0), frag_row(quarter * 16, 1)};  // this lane's tokens
  int ow[2];    // exponents of their dO's scales and of P's rows
  int next[2];  // those, of the chunk whose dO is loaded
  bool onarrow;

  float d[MT][2][4];  // the gradient of the state after the chunk
  const float* ds = a.ds_out ? a.ds_out + (long)bh * a.dk * a.dv : nullptr;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = frag_row((quarter * MT + m) * 16, e >> 1), c = c0 + frag_col(n * 8) + (e & 1);
        d[m][n][e] = ds && r < a.dk && c < a.dv ? ds[(long)r * a.dv + c] : 0.0f;
      }
  const long stride = (long)a.Hv * a.dv;
  const long at = (long)b * a.T * stride + (long)hv * a.dv + c0;
  const T* dout = a.dout ? static_cast<const T*>(a.dout) + at : nullptr;
  T* dv = static_cast<T*>(a.dv_) + at;
  const int cols = a.dv - c0;
  const bool vec = pairs_ok<T>(a.dout, 0, 0, 0, a.dv);
  Columns<T, 2> od;
  auto load_dout = [&](int chunk) {
    const int t = chunk * kC + quarter * 16;
    od.start(dout + (dout ? t * stride : 0), stride, dout ? a.T - t : 0, cols, vec);
#pragma unroll
    for (int e = 0; e < 2; ++e) next[e] = reinterpret_cast<const int*>(a.gates)[((nv0 + chunk) * kGates + kRowP) * kC + row[e]];
  };
  auto dout_tile = [&](float (&x)[2][4]) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = od.get(n, e);
        x[n][2 * e] = f.x;
        x[n][2 * e + 1] = f.y;
      }
  };
  auto put_dout = [&](int chunk) {
    float x[2][4];
    dout_tile(x);
    const long nv = nv0 + chunk;
    put_tokens<NP>(x, quarter, op, ow, a.dop + (nv * groups + group) * NP * kGroup * kC,
                   a.doscale + (nv * groups + group) * kC);
#pragma unroll
    for (int e = 0; e < 2; ++e) ow[e] += next[e];
    onarrow = put_weights(ow, quarter, ofactor, otop);
  };
  auto state_out = [&](int chunk) {
    const long nv = nv0 + chunk;
    put_state<DK>(d, quarter, sp, ssc, chunk >= 0 ? a.dstates + (nv * groups + group) * 2 * kGroup * DK : nullptr,
                     a.dsscale + (nv * groups + group) * 4);
  };
  back_load<NP, DK>(smem, a, nk0 + a.nc - 1, nv0 + a.nc - 1);
  load_dout(a.nc - 1);
  state_out(a.nc - 1);
  put_dout(a.nc - 1);
  int buf = 0;
  for (int chunk = a.nc - 1; chunk >= 0; --chunk) {
    const f16* kp = reinterpret_cast<const f16*>(smem + buf * L::stage);
    const f16* qp = kp + L::k;
    const f16* wp = qp + L::k;
    const f16* pp = wp + L::w;
    const float* gate = reinterpret_cast<const float*>(pp + L::w);
    const long nv = nv0 + chunk;
    cp_async_wait<0>();
    __syncthreads();
    if (STAGES == 2 && chunk > 0) {
      buf ^= 1;
      back_load<NP, DK>(smem + buf * L::stage, a, nk0 + chunk - 1, nv - 1);
    }
    const int* whole = reinterpret_cast<const int*>(gate);
    const float sk[2] = {gate[kScaleK * kC + row[0]], gate[kScaleK * kC + row[1]]};
    float x[2][4], y[2][4];
    // scale e^G dO, for Q^T
    dout_tile(x);
    if (chunk > 0) load_dout(chunk - 1);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] *= a.scale * gate[row[e >> 1]] * gate[kScaleQ * kC + row[e >> 1]];
    put_sum(x, quarter, qop, qosc);
    // dU
    times_state<NP, DK>(x, kp, quarter * 2, sp, ssc);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] *= sk[e >> 1] * gate[kRest * kC + row[e >> 1]];
    {
      const int left[2] = {whole[kColumnP * kC + row[0]], whole[kColumnP * kC + row[1]]};
      times_tokens<NP, true, false>(x, pp, left, quarter, op, ow, onarrow, ofactor, otop, 1.0f);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[n][e] = x[n][e] * gate[kBeta * kC + row[e >> 1]];
    int w[2];
    bool narrow;
    {
      put_tokens<2>(y, quarter, up, w, nullptr, nullptr);
#pragma unroll
      for (int e = 0; e < 2; ++e) w[e] += whole[kRowW * kC + row[e]];
      narrow = put_weights(w, quarter, ufactor, utop);
    }
    group_sync(pair);
    // Z and dV
    {
      const int left[2] = {whole[kColumnW * kC + row[0]], whole[kColumnW * kC + row[1]]};
      times_tokens<2, true, true>(x, wp, left, quarter, up, w, narrow, ufactor, utop, -1.0f);
      put_tokens<2>(x, quarter, zp, w, a.z + (nv * groups + group) * 2 * kGroup * kC,
                    a.zscale + (nv * groups + group) * kC);  // zp: on the way only
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = chunk * kC + row[e], c = frag_col(n * 8);
        const float be = gate[kBeta * kC + row[e]], eg = gate[row[e]] * sk[e];
        x[n][2 * e] *= be;
        x[n][2 * e + 1] *= be;
        if (t < a.T) set2<T>(dv + t * stride + c, cols - c, a.dv % 2 == 0, x[n][2 * e], x[n][2 * e + 1]);
        y[n][2 * e] = -eg * x[n][2 * e];
        y[n][2 * e + 1] = -eg * x[n][2 * e + 1];
      }
    __syncwarp();
    put_sum(y, quarter, zp, zsc);
    group_sync(pair);
    const float decay = gate[kC - 1];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[m][n][e] *= decay;
    add_to_state<NP, DK>(d, qp, quarter, qop, qosc);
    add_to_state<NP, DK>(d, kp, quarter, zp, zsc);
    state_out(chunk - 1);
    if (chunk > 0) put_dout(chunk - 1);
    if (STAGES == 1 && chunk > 0) {
      __syncthreads();
      back_load<NP, DK>(smem, a, nk0 + chunk - 1, nv - 1);
    }
  }
  if (!a.ds0) return;
  float* out = a.ds0 + (long)bh * a.dk * a.dv;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = frag_row((quarter * MT + m) * 16, e >> 1), c = c0 + frag_col(n * 8) + (e & 1);
        if (r < a.dk && c < a.dv) out[(long)r * a.dv + c] = d[m][n][e];
      }
}

// ---------------------------------------------------------------------------
// grads: one CTA per (batch, key head, chunk).  It walks the value columns in
// steps of 16 (one step of the products' inner dimension), the next stage of one
// or two steps loading meanwhile.  A warp keeps 16 tokens x 32 key columns of
// dQ, dK_row and dK_col, and of 16 or 32 tokens of dO U^T and Z U^T, in
// registers: sixteen warps for 128 key columns, eight for 64, where two CTAs
// then share an SM (2048 chunks of heads of 64, FP32: 190 us, sixteen warps of half
// the tile took a fifth more; of 128, bf16: 326 us).  Bound by the latency of products
// and barriers; the tensor pipe is a third busy, the most of any of these kernels.
//
// dP' and M are summed over along both sides, so they are held twice: with the other
// factor's scales in them and a scale a row, and the same a column.  One tile with one
// scale would give a token the digits that the largest of 64 leaves it.
// ---------------------------------------------------------------------------

// A lower 64 x 64 matrix as its ten 16 x 16 tiles on and below the diagonal.
constexpr int kLower = 10 * 256;
__device__ __forceinline__ int lower_tile(int r16, int c16) { return r16 * (r16 + 1) / 2 + c16; }
// A (16 rows m, 16 of k) of one: stored [m][k], or [k][m] (TRANS).
template <bool TRANS>
__device__ __forceinline__ uint32_t addr_lower(const f16* p, int m16, int k16) {
  const int i = (threadIdx.x >> 3) & 3;
  const int tile = TRANS ? lower_tile(k16, m16) : lower_tile(m16, k16);
  return smem_addr(p) + (tile * 256 + (TRANS ? i : (i & 1) * 2 + (i >> 1)) * 64 + (threadIdx.x & 7) * 8) * 2;
}

template <int NP, int DK>
struct GradSmem {
  static constexpr int split = DK / 32;           // warps that share 16 tokens' columns
  static constexpr int threads = 128 * split;
  static constexpr int steps = split / 2;         // of 16 value columns to a stage
  static constexpr int qk = NP * kC * DK;  // elements
  static constexpr int s = 2 * kGroup * DK, x = 2 * kGroup * kC, o = NP * kGroup * kC;
  // a stage: S, dS, E, Z, dO, each [step][plane], and their scales
  static constexpr int planes = steps * (2 * s + 2 * x + o);
  static constexpr int stage = planes + steps * 2 * (2 * 4 + 3 * kC);
  // bytes: dP' and M twice, scaled by rows and by columns; y in FP32; over the stages
  static constexpr int tiles = 4 * 2 * kLower * 2 + kC * (kC + 1) * 4;
  static constexpr int main = 2 * stage * 2 > tiles ? 2 * stage * 2 : tiles;
  static constexpr int least = 2 * qk * 2 + (main + 15) / 16 * 16 + kGates * kC * 4 + ((2 * split + 1 + 4) * kC + 4 * split) * 4;
  // dq and dk of the value heads so far, every thread's own, where that fits
  // (not for FP32 inputs of 128 key columns: in global memory there)
  static constexpr int sums = 2 * kC * DK * 4;
  static constexpr bool sums_fit = least + sums <= 227 * 1024;
  static constexpr int bytes = least + (sums_fit ? sums : 0);
};

// A stage from the g-th group on (of all chunks' groups).
template <int NP, int DK>
__device__ __forceinline__ void grad_load(f16* dst, const Problem& a, long g) {
  using L = GradSmem<NP, DK>;
  constexpr int n = L::steps, threads = L::threads;
  copy_async<n * L::s * 2, threads>(dst, a.states + g * L::s);
  copy_async<n * L::s * 2, threads>(dst + n * L::s, a.dstates + g * L::s);
  copy_async<n * L::x * 2, threads>(dst + 2 * n * L::s, a.e + g * L::x);
  copy_async<n * L::x * 2, threads>(dst + n * (2 * L::s + L::x), a.z + g * L::x);
  copy_async<n * L::o * 2, threads>(dst + n * (2 * L::s + 2 * L::x), a.dop + g * L::o);
  // scales: of S and of dS, then of the tokens of E, Z and dO
  if (threadIdx.x < n * (2 + 3 * 16)) {
    const int t = threadIdx.x - 2 * n, what = t / (16 * n);
    const float* from = t < 0 ? (threadIdx.x < n ? a.sscale + (g + threadIdx.x) * 4 : a.dsscale + (g + threadIdx.x - n) * 4)
                              : (what == 0 ? a.escale : what == 1 ? a.zscale : a.doscale) + g * kC + t % (16 * n) * 4;
    cp_async16(dst + L::planes + threadIdx.x * 8, from);
  }
  cp_async_commit();
}

// The value pair `word` of a tile held as planes, without its scale.
template <int NP>
__device__ __forceinline__ float2 take2(const f16* p, int plane, int word) {
  float2 f = __half22float2(reinterpret_cast<const __half2*>(p)[word]);
  if (NP == 2) {
    const float2 l = __half22float2(reinterpret_cast<const __half2*>(p + plane)[word]);
    f.x += l.x;
    f.y += l.y;
  }
  return f;
}

// acc += A B, one step of 16, times the scales of the rows and a lane's columns.
template <int NA, int NB, int NT>
__device__ __forceinline__ void step_add(float (&acc)[NT][4], const float (&row)[2], const float (&column)[NT][2],
                                         const uint32_t (&fa)[NA][4], const uint32_t (&fb)[NB][NT][2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float t[NT / 2][4];
    uint32_t g[NB][NT / 2][2];
#pragma unroll
    for (int p = 0; p < NB; ++p)
#pragma unroll
      for (int i = 0; i < NT / 2; ++i) g[p][i][0] = fb[p][h * NT / 2 + i][0], g[p][i][1] = fb[p][h * NT / 2 + i][1];
    mma_terms<NA, NB, NT / 2>(t, fa, g);
#pragma unroll
    for (int i = 0; i < NT / 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[h * NT / 2 + i][e] += row[e >> 1] * column[h * NT / 2 + i][e & 1] * t[i][e];
  }
}
// The same with one scale for the first half of the tiles' columns, and for the second.
template <int NA, int NB, int NT>
__device__ __forceinline__ void step_add(float (&acc)[NT][4], const float (&row)[2], float f0, float f1,
                                         const uint32_t (&fa)[NA][4], const uint32_t (&fb)[NB][NT][2]) {
  float column[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) column[i][0] = column[i][1] = i < NT / 2 ? f0 : f1;
  step_add<NA, NB, NT>(acc, row, column, fa, fb);
}

// acc += A B over steps [k0, k1) of the tokens, times the scales of A's rows: A a
// lower 64 x 64 tile (rows m, or transposed), B a [64 x DK] tile from column block
// n8, without its scales.
template <int NP, int DK, bool TA, int NT>
__device__ __forceinline__ void token_product(float (&acc)[NT][4], const float (&row)[2], const f16* A, int m16, const f16* B,
                                              int n8, int k0, int k1) {
  for (int kk = k0; kk < k1; ++kk) {
    uint32_t fa[2][4], fb[NP][NT][2];
    const uint32_t pa = addr_lower<TA>(A, m16, kk);
#pragma unroll
    for (int p = 0; p < 2; ++p) ldm4<TA>(fa[p], pa + p * kLower * 2);
    load_b<NP, NT, true>(fb, addr_b<DK, true>(B, 2 * kk, n8), 256, kC * DK * 2);
    step_add<2, NP, NT>(acc, row, 1.0f, 1.0f, fa, fb);
  }
}

template <typename T, int DK>
__global__ void __launch_bounds__(GradSmem<Planes<T>::n, DK>::threads, DK == 64 ? 2 : 1)
    delta_grads_kernel(const Problem a) {
  constexpr int NP = Planes<T>::n;
  using L = GradSmem<NP, DK>;
  constexpr int split = L::split, threads = L::threads;
  constexpr int NT = 4;          // a warp's 32 key columns, in 8-column tiles
  constexpr int NC = 8 / split;  // its columns of the 64 x 64 products
  extern __shared__ __align__(16) unsigned char smem[];
  f16* qp = reinterpret_cast<f16*>(smem);
  f16* kp = qp + L::qk;
  f16* main = kp + L::qk;
  // over the stages: dP' with K's scales and a scale a row, M likewise; dP' with
  // Q's scales and a scale a column, M with K's
  f16* dpr = main;
  f16* mr = dpr + 2 * kLower;
  f16* dpc = mr + 2 * kLower;
  f16* mc = dpc + 2 * kLower;
  float* y = reinterpret_cast<float*>(mc + 2 * kLower);  // [64][65]
  float* gate = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(main) + (L::main + 15) / 16 * 16);
  float* red = gate + kGates * kC;  // x and z of the warps that share tokens, F
  float* largest = red + (2 * split + 1) * kC;  // magnitudes of dP' and M, rows' and columns': [4][64]
  float* wred = largest + 4 * kC;  // values per warp

  const int chunk = blockIdx.x % a.nc, bh = blockIdx.x / a.nc;
  const int hk = bh % a.Hk, b = bh / a.Hk;
  const int t0 = chunk * kC, rows = min(kC, a.T - t0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rw[2] = {frag_row(warp / split * 16, 0), frag_row(warp / split * 16, 1)};  // this lane's tokens
  // This warp's tokens; its part of the columns, and whether that holds any of the
  // 64 x 64 products' lower half.  The parts turn from row to row: were they the
  // warp's remainder, one of the SM's quarters would have twice the others' products.
  const int m0 = warp / split * 16, col = (warp - warp / split * split / 4) & (split - 1);
  const bool below = col * NC * 8 <= m0;
  const int groups = a.dvp / kGroup;

  copy_async<L::qk * 2, threads>(qp, a.qp + (long)blockIdx.x * L::qk);
  copy_async<L::qk * 2, threads>(kp, a.kp + (long)blockIdx.x * L::qk);
  wait_for_before();

  for (int r = 0; r < a.rep; ++r) {
    const int hv = hk * a.rep + r;
    const long nv = ((long)b * a.Hv + hv) * a.nc + chunk;
    __syncthreads();
    copy_async<kGates * kC * 4, threads>(gate, a.gates + nv * kGates * kC);
    grad_load<NP, DK>(main, a, nv * groups);
    if (threadIdx.x < kC) {
#pragma unroll
      for (int i = 0; i < 4; ++i) largest[i * kC + threadIdx.x] = 0.0f;
    }
    float dp[NC][4], da[NC][4], dq[NT][4], dkr[NT][4], dkc[NT][4];
    zero(dp);
    zero(da);
    zero(dq);
    zero(dkr);
    zero(dkc);
    float sdot = 0.0f, bdot[2] = {0.0f, 0.0f};
    for (int g = 0; g < groups; ++g) {
      constexpr int n = L::steps;
      const int i = g % n, at = g / n & 1;
      const f16* stage = main + at * L::stage;
      if (i == 0) {
        cp_async_wait<0>();
        __syncthreads();
        if (g + n < groups) grad_load<NP, DK>(main + (at ^ 1) * L::stage, a, nv * groups + g + n);
      }
      const f16* sp = stage + i * L::s;
      const f16* dsp = sp + n * L::s;
      const f16* ep = stage + 2 * n * L::s + i * L::x;
      const f16* zp = ep + n * L::x;
      const f16* op = stage + n * (2 * L::s + 2 * L::x) + i * L::o;
      // scales: of the quarters of the key columns (S, dS) and of the tokens
      const float* ss = reinterpret_cast<const float*>(stage + L::planes) + i * 4;
      const float *sds = ss + 4 * n, *se = ss - i * 4 + 8 * n + i * kC, *sz = se + n * kC, *so = sz + n * kC;
      const int kq = col * 4 / split;         // quarter of this warp's first key column
      constexpr int k2 = split == 4 ? 0 : 1;  // and of its last
      // a scale below zero only marks tokens
      const float fE[2] = {fabsf(se[rw[0]]), fabsf(se[rw[1]])}, fZ[2] = {fabsf(sz[rw[0]]), fabsf(sz[rw[1]])};
      const float fO[2] = {fabsf(so[rw[0]]), fabsf(so[rw[1]])};
      auto state_dot = [&] {
#pragma unroll
        for (int j = 0; j < kGroup * DK / 2 / threads; ++j) {
          // block warp + 4 split j is of the rows 8 (warp / 2 + 2 split j) ..., in quarter q
          const int word = threadIdx.x + j * threads, q = (warp / 2 + 2 * split * j) * 8 / (DK / 4);
          const float2 u = take2<2>(sp, kGroup * DK, word), v = take2<2>(dsp, kGroup * DK, word);
          sdot += (ss[q] * sds[q]) * (u.x * v.x + u.y * v.y);
        }
      };
      // of eight warps, half begin with what takes shared memory and no tensor core
      // (training 64 x 512 505 us, 510 where all end with it; sixteen are spread by
      // themselves)
      const bool early = split == 2 && (m0 & 16);
      if (early) state_dot();
      uint32_t fz[2][4], fe[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        ldm4<false>(fz[p], addr_a<kGroup, false>(zp, m0 / 8, 0) + p * kGroup * kC * 2);
        ldm4<false>(fe[p], addr_a<kGroup, false>(ep, m0 / 8, 0) + p * kGroup * kC * 2);
      }
      if (col == 0) {
        // Z . E of this lane's two tokens
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 u = pair(fz[0][j], fz[1][j]), w = pair(fe[0][j], fe[1][j]);
          bdot[j & 1] += fZ[j & 1] * fE[j & 1] * (u.x * w.x + u.y * w.y);
        }
      }
      {
        uint32_t fb[2][NT][2];
        load_b<2, NT, false>(fb, addr_b<kGroup, false>(dsp, 0, col * NT), 512, kGroup * DK * 2);
        step_add<2, 2, NT>(dkc, fE, sds[kq], sds[kq + k2], fe, fb);
      }
      uint32_t fo[NP][4];
#pragma unroll
      for (int p = 0; p < NP; ++p) ldm4<false>(fo[p], addr_a<kGroup, false>(op, m0 / 8, 0) + p * kGroup * kC * 2);
      {
        uint32_t fb[2][NT][2];
        load_b<2, NT, false>(fb, addr_b<kGroup, false>(sp, 0, col * NT), 512, kGroup * DK * 2);
        step_add<NP, 2, NT>(dq, fO, ss[kq], ss[kq + k2], fo, fb);
        step_add<2, 2, NT>(dkr, fZ, ss[kq], ss[kq + k2], fz, fb);
      }
      if (below) {
        uint32_t fb[2][NC][2];
        load_b<2, NC, false>(fb, addr_b<kGroup, false>(ep, 0, col * NC), 512, kGroup * kC * 2);
        float f[NC][2];
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int l = 0; l < 2; ++l) f[n][l] = fabsf(se[frag_col((col * NC + n) * 8) + l]);
        step_add<NP, 2, NC>(dp, fO, f, fo, fb);
        step_add<2, 2, NC>(da, fZ, f, fz, fb);
      }
      if (!early) state_dot();
    }
    __syncthreads();
    // the masked 64 x 64 products, over the stages' memory
    const float sk[2] = {gate[kScaleK * kC + rw[0]], gate[kScaleK * kC + rw[1]]};
    const float sq[2] = {gate[kScaleQ * kC + rw[0]], gate[kScaleQ * kC + rw[1]]};
    float sc[NC][2];  // K's scales of this lane's columns
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int l = 0; l < 2; ++l) sc[n][l] = gate[kScaleK * kC + frag_col((col * NC + n) * 8) + l];
    {
      float qk[NC][4], kk[NC][4];
      zero(qk);
      zero(kk);
      if (below) {
#pragma unroll
        for (int k = 0; k < DK / 16; ++k) {
          uint32_t fa[NP][4], fb[NP][NC][2];
          load_b<NP, NC, false>(fb, addr_b<DK, false>(kp, 2 * k, col * NC), 32 * DK, kC * DK * 2);
#pragma unroll
          for (int p = 0; p < NP; ++p) ldm4<false>(fa[p], addr_a<DK, false>(qp, m0 / 8, 2 * k) + p * kC * DK * 2);
          step_add<NP, NP, NC>(qk, sq, sc, fa, fb);
#pragma unroll
          for (int p = 0; p < NP; ++p) ldm4<false>(fa[p], addr_a<DK, false>(kp, m0 / 8, 2 * k) + p * kC * DK * 2);
          step_add<NP, NP, NC>(kk, sk, sc, fa, fb);
        }
      }
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = frag_row(m0, e), j = frag_col((col * NC + n) * 8);
#pragma unroll
          for (int l = 0; l < 2; ++l) {
            const float dec = j + l <= i ? decay_between(gate + kLog * kC, i, j + l) * gate[kBeta * kC + j + l]
                                         : 0.0f;
            float& u = dp[n][2 * e + l];
            float& w = da[n][2 * e + l];
            u = j + l <= i ? a.scale * dec * u : 0.0f;
            w = j + l < i ? -gate[kBeta * kC + i] * dec * w : 0.0f;
            y[i * (kC + 1) + j + l] = j + l < i ? u * qk[n][2 * e + l] + w * kk[n][2 * e + l] : 0.0f;
          }
        }
    }
    // the largest of dP' and M of every row, with K's scales, and of every column,
    // with Q's and K's
    if (below) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mu = 0.0f, mw = 0.0f;
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int l = 0; l < 2; ++l) {
            mu = max_finite(mu, dp[n][2 * e + l] * sc[n][l]);
            mw = max_finite(mw, da[n][2 * e + l] * sc[n][l]);
          }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, o));
          mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, o));
        }
        if ((lane & 3) == 0) {
          atomicMax(reinterpret_cast<int*>(largest + rw[e]), __float_as_int(mu));
          atomicMax(reinterpret_cast<int*>(largest + kC + rw[e]), __float_as_int(mw));
        }
      }
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          float mu = max_finite(max_finite(0.0f, dp[n][l] * sq[0]), dp[n][2 + l] * sq[1]);
          float mw = max_finite(max_finite(0.0f, da[n][l] * sk[0]), da[n][2 + l] * sk[1]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, o));
            mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, o));
          }
          if (lane < 4) {
            const int j = frag_col((col * NC + n) * 8) + l;
            atomicMax(reinterpret_cast<int*>(largest + 2 * kC + j), __float_as_int(mu));
            atomicMax(reinterpret_cast<int*>(largest + 3 * kC + j), __float_as_int(mw));
          }
        }
    }
    float xs[2] = {0.0f, 0.0f}, zs[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = frag_row(m0, e);
        const int word = ((m0 / 8 + e) * (DK / 8) + col * NT + n) * 32 + lane;
        const float eg = gate[row], er = gate[kRest * kC + row], be = gate[kBeta * kC + row];
        const float2 kv = take2<NP>(kp, kC * DK, word), qv = take2<NP>(qp, kC * DK, word);
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          dq[n][2 * e + l] *= a.scale * eg;
          dkr[n][2 * e + l] *= -eg * be;
          dkc[n][2 * e + l] *= er * be;
        }
        xs[e] += sq[e] * (qv.x * dq[n][2 * e] + qv.y * dq[n][2 * e + 1]) +
                 sk[e] * (kv.x * dkr[n][2 * e] + kv.y * dkr[n][2 * e + 1]);
        zs[e] += sk[e] * (kv.x * dkc[n][2 * e] + kv.y * dkc[n][2 * e + 1]);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        xs[e] += __shfl_xor_sync(0xffffffffu, xs[e], o);
        zs[e] += __shfl_xor_sync(0xffffffffu, zs[e], o);
        bdot[e] += __shfl_xor_sync(0xffffffffu, bdot[e], o);
      }
      const int row = frag_row(m0, e);
      if ((lane & 3) == 0) {
        red[col * kC + row] = xs[e];
        red[(split + col) * kC + row] = zs[e];
        if (col == 0 && row < rows) a.dbeta[((long)b * a.T + t0 + row) * a.Hv + hv] = bdot[e];
      }
    }
    float end = gate[kC - 1] * sdot;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) end += __shfl_xor_sync(0xffffffffu, end, o);
    if (lane == 0) wred[warp] = end;
    __syncthreads();
    // scales of the products' rows: of this lane's tokens as rows, and as columns
    // of what is transposed
    float scale[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) scale[i][e] = plane_scale(plane_inv(largest[i * kC + rw[e]]));
    const float iu[2] = {plane_inv(largest[rw[0]]), plane_inv(largest[rw[1]])};
    const float iw[2] = {plane_inv(largest[kC + rw[0]]), plane_inv(largest[kC + rw[1]])};
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int c8 = col * NC + n;
      if (c8 / 2 > m0 / 16) continue;
      const int j = frag_col(c8 * 8);
      const float ju[2] = {plane_inv(largest[2 * kC + j]), plane_inv(largest[2 * kC + j + 1])};
      const float jw[2] = {plane_inv(largest[3 * kC + j]), plane_inv(largest[3 * kC + j + 1])};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int word = lower_tile(m0 / 16, c8 / 2) * 128 + (e * 2 + (c8 & 1)) * 32 + lane;
        uint32_t u[2], w[2], x[2], z[2];
        split2<2>(dp[n][2 * e] * sc[n][0], dp[n][2 * e + 1] * sc[n][1], iu[e], u);
        split2<2>(da[n][2 * e] * sc[n][0], da[n][2 * e + 1] * sc[n][1], iw[e], w);
        split2<2>(dp[n][2 * e] * ju[0], dp[n][2 * e + 1] * ju[1], sq[e], x);
        split2<2>(da[n][2 * e] * jw[0], da[n][2 * e + 1] * jw[1], sk[e], z);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          reinterpret_cast<uint32_t*>(dpr + p * kLower)[word] = u[p];
          reinterpret_cast<uint32_t*>(mr + p * kLower)[word] = w[p];
          reinterpret_cast<uint32_t*>(dpc + p * kLower)[word] = x[p];
          reinterpret_cast<uint32_t*>(mc + p * kLower)[word] = z[p];
        }
      }
    }
    {
      // y_ij -> sum over the columns before j, `per` threads to a row
      constexpr int per = threads / kC, n = kC / per;
      float* part = y + (threadIdx.x / per) * (kC + 1) + (threadIdx.x % per) * n;
      float v[n], sum = 0.0f;
#pragma unroll
      for (int j = 0; j < n; ++j) {
        v[j] = part[j];
        sum += v[j];
      }
      float run = 0.0f;  // of the parts before
#pragma unroll
      for (int k = 0; k < per - 1; ++k) {
        const float f = __shfl_sync(0xffffffffu, sum, k, per);
        if (threadIdx.x % per > k) run += f;
      }
#pragma unroll
      for (int j = 0; j < n; ++j) {
        part[j] = run;
        run += v[j];
      }
    }
    __syncthreads();
    token_product<NP, DK, false, NT>(dq, scale[0], dpr, m0 / 16, kp, col * NT, 0, m0 / 16 + 1);
    token_product<NP, DK, false, NT>(dkr, scale[1], mr, m0 / 16, kp, col * NT, 0, m0 / 16 + 1);
    token_product<NP, DK, true, NT>(dkc, scale[2], dpc, m0 / 16, qp, col * NT, m0 / 16, kC / 16);
    token_product<NP, DK, true, NT>(dkc, scale[3], mc, m0 / 16, kp, col * NT, m0 / 16, kC / 16);
    float log_decay[2];  // of the two tokens that a lane of warp 0 ends with
#pragma unroll
    for (int e = 0; e < 2; ++e)
      log_decay[e] = warp == 0 && 2 * lane + e < rows
                         ? a.g[b * a.sg[0] + (t0 + 2 * lane + e) * a.sg[1] + hv * a.sg[2]] : 0.0f;
    {
      constexpr int per = threads / kC;
      const int t = threadIdx.x / per;
      float f = 0.0f;
      for (int i = t + threadIdx.x % per; i < kC; i += per) f += y[i * (kC + 1) + t];
#pragma unroll
      for (int o = 1; o < per; o <<= 1) f += __shfl_xor_sync(0xffffffffu, f, o);
      if (threadIdx.x % per == 0) red[2 * split * kC + t] = f;
    }
    __syncthreads();
    if (warp == 0) {
      // two tokens a lane: x summed from the end, z from the start
      double x[2], z[2], last = lane < 4 * split ? wred[lane] : 0.0f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        x[e] = z[e] = 0.0;
#pragma unroll
        for (int c = 0; c < split; ++c) {
          x[e] += red[c * kC + i];
          z[e] += red[(split + c) * kC + i];
        }
      }
      double sx = x[0] + x[1], sz = z[0] + z[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_down_sync(0xffffffffu, sx, o), w = __shfl_up_sync(0xffffffffu, sz, o);
        if (lane + o < 32) sx += u;
        if (lane >= o) sz += w;
        last += __shfl_xor_sync(0xffffffffu, last, o);
      }
      // of the lanes after this one, and of those before: nothing is taken off again
      sx = __shfl_down_sync(0xffffffffu, sx, 1);
      sz = __shfl_up_sync(0xffffffffu, sz, 1);
      if (lane == 31) sx = 0.0;
      if (lane == 0) sz = 0.0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * lane + e;
        if (i < rows) {
          const double from = e ? sx + x[1] : sx + x[0] + x[1], before = e ? sz + z[0] : sz;
          // a decay of zero passes no gradient
          a.dg[((long)b * a.T + t0 + i) * a.Hv + hv] =
              log_decay[e] < kNoDecay ? 0.0f : (float)(from + before + red[2 * split * kC + i] + last);
        }
      }
    }
    // dq and dk of a key head are the sums over its value heads: a thread's
    // pair i is sum[i * threads]
    float2* sum = reinterpret_cast<float2*>(L::sums_fit ? reinterpret_cast<float*>(smem + L::least)
                                                        : a.dqk + (long)blockIdx.x * 2 * kC * DK) + threadIdx.x;
    const bool even = a.dk % 2 == 0;
    const bool whole = a.dk % 8 == 0 && ((reinterpret_cast<uintptr_t>(a.dq) | reinterpret_cast<uintptr_t>(a.dk_)) & 15) == 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float2 x[NT], z[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        x[n] = make_float2(dq[n][2 * e], dq[n][2 * e + 1]);
        z[n] = make_float2(dkr[n][2 * e] + dkc[n][2 * e], dkr[n][2 * e + 1] + dkc[n][2 * e + 1]);
        float2* px = sum + (n * 4 + e * 2) * threads;
        float2* pz = px + threads;
        if (r > 0) {
          x[n].x += px->x, x[n].y += px->y;
          z[n].x += pz->x, z[n].y += pz->y;
        }
        if (r + 1 < a.rep) {
          *px = x[n];
          *pz = z[n];
        }
      }
      if (r + 1 == a.rep) {
        const int row = frag_row(m0, e), c = col * NT * 8;
        const long o = (((long)b * a.T + t0 + row) * a.Hk + hk) * a.dk + c;
        set_row<T>(static_cast<T*>(a.dq) + o, a.dk - c, even, whole, row < rows, x);
        set_row<T>(static_cast<T*>(a.dk_) + o, a.dk - c, even, whole, row < rows, z);
      }
    }
  }
}

template <typename T, int DK, int STAGES>
int launch_scan(const Problem& a, cudaStream_t stream) {
  constexpr int bytes = BackSmem<Planes<T>::n, DK, STAGES>::bytes;
  if (const int rc = with_smem(delta_back_scan_kernel<T, DK, STAGES>, bytes)) return rc;
  delta_back_scan_kernel<T, DK, STAGES>
      <<<(unsigned)((long)a.B * a.Hv * (a.dvp / kSlice)), kThreads, bytes, stream>>>(a);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

template <typename T, int DK>
int backward_typed(const Problem& a, cudaStream_t stream) {
  using G = GradSmem<Planes<T>::n, DK>;
  const int grad_bytes = a.rep > 1 ? G::bytes : G::least;  // one value head has nothing to add up
  if (const int rc = with_smem(delta_grads_kernel<T, DK>, grad_bytes)) return rc;
  LaunchScope scope(kKindDeltaRule, stream, 2);
  // one stage where two CTAs then share an SM and there are that many, or
  // where two stages do not fit (FP32 inputs of 128 key columns)
  constexpr int kMost = 227 * 1024;
  constexpr bool fits = BackSmem<Planes<T>::n, DK, 2>::bytes <= kMost;
  constexpr bool share = 2 * (BackSmem<Planes<T>::n, DK, 1>::bytes + 1024) <= 228 * 1024;
  const bool many = (long)a.B * a.Hv * (a.dvp / kSlice) > 148;
  if constexpr (fits) {
    if (const int rc = many && share ? launch_scan<T, DK, 1>(a, stream) : launch_scan<T, DK, 2>(a, stream)) return rc;
  } else {
    if (const int rc = launch_scan<T, DK, 1>(a, stream)) return rc;
  }
  return launch_after(delta_grads_kernel<T, DK>, (unsigned)((long)a.B * a.Hk * a.nc), G::threads, grad_bytes, stream, a);
}

}  // namespace

int backward(const Problem& a, int dtype, cudaStream_t stream) {
  if (dtype == GRU_F32)
    return a.dk <= 64 ? backward_typed<float, 64>(a, stream) : backward_typed<float, 128>(a, stream);
  return a.dk <= 64 ? backward_typed<bf16, 64>(a, stream) : backward_typed<bf16, 128>(a, stream);
}

}  // namespace delta
}  // namespace gru
