// Shared device code of the gated delta rule's kernels (sm_100a).
//
// The chunked kernels need FP32-grade products (states, gates' gradients and
// FP32 tensors are FP32) from tensor cores that multiply 16-bit numbers.  FP32
// numbers are held as two FP16 planes with a power of two that some of them
// share, x = s (h + l), h = fp16(x / s), l = fp16(x / s - h): s puts the largest
// magnitude in [2^14, 2^15), so a value keeps 22 bits down to 2^-17 of the
// largest, and 2^-39 of the largest below.  A product of two such tiles is three
// plane products (l h', h l', h h'; l l' is below 2^-22 of the result), half the
// work of three bf16 planes.  bf16 inputs are one plane: exact down to 2^-31 of
// the largest, and 2^-39 of it below.
//
// What shares a scale.  Of K, Q, the errors and the gradients of outputs: a
// token's head, or 16 value columns of it.  Of W and P: a token's row, without the
// other tokens' own sizes and the decays between (Weights, below).  So no token's
// digits depend on another's magnitude, but where a state holds both.  Of a state
// and its gradient: a quarter of the key columns x 16 value columns; of what a chunk
// adds to one: 16 tokens x 16 value columns.
//
// Tiles in memory are made of 8 x 8 blocks of 128 consecutive bytes, the unit
// that ldmatrix reads (transposed or not, without bank conflicts) and that a
// warp's accumulators write as 32 x 4 bytes.
#pragma once

#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "../../include/rnn_kernel_b200.h"

namespace gru {
namespace delta {

constexpr int kC = 64;      // tokens per chunk
constexpr int kGroup = 16;  // value columns to a tile of states, errors and their gradients
constexpr int kSlice = 32;  // value columns of a scan's CTA; they are padded to a multiple of this
constexpr int kThreads = 256;
constexpr int kTile = kC * kC;  // elements of a token x token tile

// Rows of Problem::gates, 64 numbers each, one to a token.  A scan loads those
// up to its last.
enum Gate {
  kDecay = 0,    // e^G_i
  kRest = 1,     // e^(G_end - G_i)
  kBeta = 2,
  kScaleK = 3,   // of the planes of K
  kColumnW = 4,  // exponents (integers) of what the planes of W leave out, see Weights
  kRowW = 5,
  kForward = 6,  // rows that the forward scan needs
  kScaleQ = 6,
  kColumnP = 7,
  kRowP = 8,
  kBackward = 9,
  kLog = 9,      // G_i / log 2 as two floats
  kGates = 11
};

// Log decays below this count as this: e^-1000 is zero in FP32, and sums of 64
// of them (in FP64) still tell neighbouring tokens apart, which -inf would not.
constexpr float kNoDecay = -1000.0f;

typedef __nv_bfloat16 bf16;
typedef __half f16;

template <typename T>
struct Planes;  // planes of an input tensor
template <>
struct Planes<float> {
  static constexpr int n = 2;
};
template <>
struct Planes<bf16> {
  static constexpr int n = 1;
};

// One gated-delta problem; strides in elements.
struct Problem {
  const void *q, *k, *v;
  const float *g, *beta, *s0;
  void* o;
  float* s_out;
  long sq[3], sk[3], sv[3], sg[3], sb[3];  // batch, token, head
  int B, T, Hk, Hv, dk, dv;
  int rep;   // value heads per key head
  int nc;    // chunks
  int dvp;   // dv rounded up to a multiple of kSlice
  float scale;
  // workspace; n = (b * H + h) * nc + chunk, tiles of 8 x 8 blocks
  f16* kp;       // [n over Hk][NP][64 x DK]
  f16* qp;       // [n over Hk][NP][64 x DK]
  f16* wp;       // [n over Hv][2][64 x 64]
  f16* pp;       // [n over Hv][2][64 x 64]
  float* gates;  // [n over Hv][kGates][64]
  // Tiles of 16 value columns each, [n over Hv][group][2][rows x 16], rows the
  // key columns of a state or the tokens.  Scales: of a state's quarters, [n
  // over Hv][group][4], of tokens, [n over Hv][group][64].
  f16* states;   // the state before the chunk
  float* sscale;
  f16* e;        // v - S'^T k, so that u = beta e
  float* escale;
  // gradient
  const void* dout;
  const float* ds_out;
  void *dq, *dk_, *dv_;
  float *dg, *dbeta, *ds0;
  f16* z;
  float* zscale;
  f16* dstates;  // the gradient of the state after the chunk
  float* dsscale;
  f16* dop;      // the output's gradient, one plane if it is bf16
  float* doscale;
  float* dqk;    // [n over Hk][2][64][DK]: dq and dk summed over a key head's value heads
};

int forward(const Problem& a, int dtype, cudaStream_t stream);
int backward(const Problem& a, int dtype, cudaStream_t stream);

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N));
}
// BYTES (a multiple of 16) from global to shared memory by THREADS threads:
// one address each, the rest constant offsets.
template <int BYTES, int THREADS>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  constexpr int n = BYTES / 16, full = n / THREADS, rest = n % THREADS;
  char* d = static_cast<char*>(dst) + threadIdx.x * 16;
  const char* s = static_cast<const char*>(src) + threadIdx.x * 16;
#pragma unroll
  for (int i = 0; i < full; ++i) cp_async16(d + i * THREADS * 16, s + i * THREADS * 16);
  if (rest > 0 && threadIdx.x < rest) cp_async16(d + full * THREADS * 16, s + full * THREADS * 16);
}

template <bool TRANS>
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// d = A B + d, and d = A B.
__device__ __forceinline__ void mma_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------------------
// Operands in shared memory, COLS elements to a row of blocks.  Each function
// gives this lane's address for the first block; moving by whole blocks adds
// 128 bytes a column of blocks, 16 * COLS a row of blocks.
// ---------------------------------------------------------------------------

template <int COLS>
__device__ __forceinline__ uint32_t block_addr(const f16* p, int r8, int c8) {
  return smem_addr(p) + ((r8 * (COLS / 8) + c8) * 64 + (threadIdx.x & 7) * 8) * 2;
}
// A (16 rows m, 16 of k): stored [m][k], or [k][m] (TRANS).
template <int COLS, bool TRANS>
__device__ __forceinline__ uint32_t addr_a(const f16* p, int m8, int k8) {
  const int i = (threadIdx.x >> 3) & 3;
  return TRANS ? block_addr<COLS>(p, k8 + (i >> 1), m8 + (i & 1)) : block_addr<COLS>(p, m8 + (i & 1), k8 + (i >> 1));
}
// B (16 of k, two 8-column tiles n): stored [k][n] (TRANS), or [n][k].
template <int COLS, bool TRANS>
__device__ __forceinline__ uint32_t addr_b(const f16* p, int k8, int n8) {
  const int i = (threadIdx.x >> 3) & 3;
  return TRANS ? block_addr<COLS>(p, k8 + (i & 1), n8 + (i >> 1)) : block_addr<COLS>(p, n8 + (i >> 1), k8 + (i & 1));
}

// t[n] = A B_n over one step of 16 in k, smallest plane products first.  The
// tensor core truncates when it adds into its accumulator, so every step has
// fresh ones and callers add those up in FP32 (rounded to nearest).
template <int NA, int NB, int NT>
__device__ __forceinline__ void mma_terms(float (&t)[NT][4], const uint32_t (&fa)[NA][4], const uint32_t (&fb)[NB][NT][2]) {
  constexpr int kTop = (NA > NB ? NA : NB) - 1;
  bool first = true;
#pragma unroll
  for (int s = kTop; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i)
      if (i < NA && s - i < NB) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (first) mma_zero(t[n], fa[i], fb[s - i][n][0], fb[s - i][n][1]);
          else mma(t[n], fa[i], fb[s - i][n][0], fb[s - i][n][1]);
        }
        first = false;
      }
}

// B fragments of NT (even) tiles: `next` bytes from one pair of tiles to the
// next, `plane` bytes from plane to plane.
template <int NB, int NT, bool TRANS>
__device__ __forceinline__ void load_b(uint32_t (&fb)[NB][NT][2], uint32_t addr, int next, int plane) {
#pragma unroll
  for (int p = 0; p < NB; ++p)
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t r[4];
      ldm4<TRANS>(r, addr + p * plane + (n / 2) * next);
      fb[p][n][0] = r[0], fb[p][n][1] = r[1], fb[p][n + 1][0] = r[2], fb[p][n + 1][1] = r[3];
    }
}

// The logarithm of e^(G_i - G_j), from its two rows, and that.
__device__ __forceinline__ float log_between(const float* log, int i, int j) {
  return (log[i] - log[j]) + (log[kC + i] - log[kC + j]);
}
__device__ __forceinline__ float decay_between(const float* log, int i, int j) { return exp2f(log_between(log, i, j)); }

template <int NT>
__device__ __forceinline__ void zero(float (&acc)[NT][4]) {
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
}

// Row and first column of accumulator pair h (0: rows 0-7, 1: rows 8-15) of an
// 8-column tile at (m0, n0).
__device__ __forceinline__ int frag_row(int m0, int h) { return m0 + ((threadIdx.x & 31) >> 2) + 8 * h; }
__device__ __forceinline__ int frag_col(int n0) { return n0 + (threadIdx.x & 3) * 2; }

// ---------------------------------------------------------------------------
// Planes.
// ---------------------------------------------------------------------------

// 1 / s for a tile whose largest magnitude is m (a finite number).  Tiles
// below 2^-100 share the scale of 2^-100.
__device__ __forceinline__ float plane_inv(float m) {
  const int eb = max((int)(__float_as_uint(m) >> 23), 27);
  return __uint_as_float((unsigned)(268 - eb) << 23);
}
__device__ __forceinline__ float plane_scale(float inv) { return __uint_as_float((254u << 23) - __float_as_uint(inv)); }

// A power of two's exponent, biased, and back: zero below FP32's normal numbers (a
// decay of that size forgets), the largest above.
__device__ __forceinline__ int exponent_of(float x) { return (int)((__float_as_uint(x) >> 23) & 0xffu); }
__device__ __forceinline__ float power_of(int biased) { return __uint_as_float((unsigned)min(max(biased, 0), 254) << 23); }

// Two values (times inv) as planes, packed {low half: a, high half: b}.
template <int NP>
__device__ __forceinline__ void split2(float a, float b, float inv, uint32_t (&w)[NP]) {
  a *= inv;
  b *= inv;
  const __half2 h = __floats2half2_rn(a, b);
  w[0] = *reinterpret_cast<const uint32_t*>(&h);
  if (NP == 2) {
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    w[NP - 1] = *reinterpret_cast<const uint32_t*>(&l);
  }
}

// The numbers that two packed planes stand for.
__device__ __forceinline__ float2 pair(uint32_t h, uint32_t l) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&l));
  return make_float2(x.x + y.x, x.y + y.y);
}

// The larger of m and |x|; a NaN wins.
__device__ __forceinline__ float max_mag(float m, float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(m), "f"(fabsf(x)));
  return y;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028235e38f; }
// The larger of m and |x| if that is finite: what is not must not take the
// other values' scale.
__device__ __forceinline__ float max_finite(float m, float x) { return fmaxf(m, finite(x) ? fabsf(x) : 0.0f); }
// The largest of non-negative numbers over the warp; a NaN wins.
__device__ __forceinline__ float warp_largest(float m) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
}
// The largest finite magnitude of a warp's tile, and whether all are finite.
template <int NT>
__device__ __forceinline__ float warp_max(const float (&x)[NT][4], bool& all_finite) {
  float m = 0.0f;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max_mag(m, x[n][e]);
  m = warp_largest(m);
  all_finite = finite(m);
  if (!all_finite) {
    m = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = max_finite(m, x[n][e]);
    m = warp_largest(m);
  }
  return m;
}
template <int NT>
__device__ __forceinline__ float warp_max(const float (&x)[NT][4]) {
  bool all_finite;
  return warp_max<NT>(x, all_finite);
}

// The largest finite magnitudes of the two rows of a lane in a warp's 16 x 16
// tile, and whether all of the tile is finite.
__device__ __forceinline__ void row_max(const float (&x)[2][4], float (&m)[2], bool& all_finite) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    m[e] = max_mag(max_mag(max_mag(fabsf(x[0][2 * e]), x[0][2 * e + 1]), x[1][2 * e]), x[1][2 * e + 1]);
    m[e] = max_mag(m[e], __shfl_xor_sync(0xffffffffu, m[e], 1));
    m[e] = max_mag(m[e], __shfl_xor_sync(0xffffffffu, m[e], 2));
  }
  all_finite = !__any_sync(0xffffffffu, !finite(m[0]) || !finite(m[1]));
  if (!all_finite) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[e] = 0.0f;
#pragma unroll
      for (int n = 0; n < 2; ++n) m[e] = max_finite(max_finite(m[e], x[n][2 * e]), x[n][2 * e + 1]);
      m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 1));
      m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 2));
    }
  }
}

// Writes 16 rows (from row block r8) x 16 columns of accumulators, times their
// row's inv, as NP planes of a tile of 16 columns in shared memory (`plane` elements apart),
// and into `out`, if given, 16 bytes a lane.  Four blocks of 128 consecutive
// bytes, which is what stmatrix writes at once.
template <int NP>
__device__ __forceinline__ void store_rows(f16* tile, int plane, int r8, const float (&x)[2][4], const float (&inv)[2],
                                           f16* out, int out_plane) {
  uint32_t w[2][2][NP];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) split2<NP>(x[n][2 * e], x[n][2 * e + 1], inv[e], w[e][n]);
  const int at = r8 * 128 + (threadIdx.x & 31) * 8;
#pragma unroll
  for (int p = 0; p < NP; ++p)
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(smem_addr(tile + p * plane + at)),
                 "r"(w[0][0][p]), "r"(w[0][1][p]), "r"(w[1][0][p]), "r"(w[1][1][p])
                 : "memory");
  if (out) {
    __syncwarp();
#pragma unroll
    for (int p = 0; p < NP; ++p)
      *reinterpret_cast<uint4*>(out + p * out_plane + at) = *reinterpret_cast<const uint4*>(tile + p * plane + at);
  }
}

// ---------------------------------------------------------------------------
// Products over tokens: sum_j A_ij x_j, A a token x token matrix (W or P), x_j
// tokens whose planes have a scale s_j each.
//
// The planes of A leave out what its rows and columns differ by,
//
//   A_ij = 2^Row_i A'_ij 2^Column_j:
//
// 2^Column_j is about |k_j| e^-G_j (in W, where keys of any size multiply one another,
// the largest that the column has in its rows' measure, for |k_j|), 2^Row_i what is
// left, so that a row's largest A' has an FP16 number's size; the decays' exponents,
// as large as they may be, are integers and only their differences are ever taken.  So
// |A'_ij| spans little, and a 16 x 16 tile of it is multiplied as A'_ij 2^(w_j - w),
// w_j the exponent of s_j 2^Column_j (of s_j 2^Row_j, for sums over A's rows), w the
// largest of those that a row adds up: in the tile on the diagonal only the tokens up
// to i (from i on), without i itself in W, whose diagonal is zero.  What falls below
// FP16's range there is below 2^-24 of a term of the largest size.
// ---------------------------------------------------------------------------

// A lane's factors for an A fragment, {rows 0-7, 8-15} x {k = 0-7, 8-15}, and the
// exponents w of its two rows.
struct Weights {
  __half2 f[2][2];
  int top[2];
};

__device__ __forceinline__ __half2 two_powers(int a, int b) {
  const float x = __uint_as_float((unsigned)(min(max(a, -60), 0) + 127) << 23);
  const float y = __uint_as_float((unsigned)(min(max(b, -60), 0) + 127) << 23);
  return __floats2half2_rn(x, y);
}

// 16 tokens whose exponents are this close serve the tile on the diagonal as they
// serve the others: A' in both planes times 2^-16 is still exact in FP16 (training 4 x
// 2048 885 us, with every diagonal on its own 900).
constexpr int kNarrow = 16;

// What a warp's 16 tokens bring to the tiles: factors and the exponent, in shared
// memory; whether they are narrow.  own: the exponents of the lane's rows, lane / 4 and
// lane / 4 + 8.
__device__ __forceinline__ bool put_weights(const int (&own)[2], int quarter, __half* factor, int* top) {
  const int lane = threadIdx.x & 31, m = __reduce_max_sync(0xffffffffu, max(own[0], own[1]));
  const int least = __reduce_min_sync(0xffffffffu, min(own[0], own[1]));
  if ((lane & 3) == 0) {
    const __half2 f = two_powers(own[0] - m, own[1] - m);
    factor[quarter * 16 + (lane >> 2)] = __low2half(f);
    factor[quarter * 16 + (lane >> 2) + 8] = __high2half(f);
  }
  if (lane == 0) top[quarter] = m;
  return m - least <= kNarrow;
}
__device__ __forceinline__ Weights get_weights(int kk, const __half* factor, const int* top) {
  Weights r;
  const int c = kk * 16 + (threadIdx.x & 3) * 2;
#pragma unroll
  for (int k = 0; k < 2; ++k) r.f[0][k] = r.f[1][k] = *reinterpret_cast<const __half2*>(factor + c + 8 * k);
  r.top[0] = r.top[1] = top[kk];
  return r;
}

// For the tile on the diagonal, whose tokens are the warp's own, where they are not
// narrow: the largest up to a row, or from it on (DOWN), without it (STRICT).
template <bool DOWN, bool STRICT>
__device__ __forceinline__ Weights diagonal_weights(const int (&own)[2]) {
  Weights r;
  const int lane = threadIdx.x & 31, from = (lane & 3) * 8;
  // of tokens 2c, 2c + 1, 2c + 8, 2c + 9, c = lane & 3
  const int w[4] = {__shfl_sync(0xffffffffu, own[0], from), __shfl_sync(0xffffffffu, own[0], from + 4),
                    __shfl_sync(0xffffffffu, own[1], from), __shfl_sync(0xffffffffu, own[1], from + 4)};
  int a = own[DOWN ? 1 : 0], b = own[DOWN ? 0 : 1];  // the rows that count first, and the others
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    const int x = DOWN ? __shfl_down_sync(0xffffffffu, a, o) : __shfl_up_sync(0xffffffffu, a, o);
    const int y = DOWN ? __shfl_down_sync(0xffffffffu, b, o) : __shfl_up_sync(0xffffffffu, b, o);
    if (DOWN ? lane + o < 32 : lane >= o) {
      a = max(a, x);
      b = max(b, y);
    }
  }
  const int all = __shfl_sync(0xffffffffu, a, DOWN ? 0 : 31);
  b = max(b, all);
  if (STRICT) {
    const int x = DOWN ? __shfl_down_sync(0xffffffffu, a, 4) : __shfl_up_sync(0xffffffffu, a, 4);
    const int y = DOWN ? __shfl_down_sync(0xffffffffu, b, 4) : __shfl_up_sync(0xffffffffu, b, 4);
    const bool edge = DOWN ? lane >= 28 : lane < 4;
    a = edge ? -(1 << 28) : x;  // nothing there
    b = edge ? all : y;
  }
  r.top[0] = DOWN ? b : a;
  r.top[1] = DOWN ? a : b;
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int k = 0; k < 2; ++k) r.f[e][k] = two_powers(w[2 * k] - r.top[e], w[2 * k + 1] - r.top[e]);
  return r;
}

__device__ __forceinline__ void weigh(uint32_t (&fa)[4], const Weights& w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&fa[i]), w.f[i & 1][i >> 1]);
    fa[i] = *reinterpret_cast<const uint32_t*>(&x);
  }
}

// ---------------------------------------------------------------------------
// Elements of either input type.
// ---------------------------------------------------------------------------

// Four consecutive elements as they lie in memory, and as numbers.
template <typename T>
struct Quad;
template <>
struct Quad<float> {
  typedef float4 type;
  static __device__ __forceinline__ float4 get(const float4& r) { return r; }
  static __device__ __forceinline__ float4 make(float x, float y, float z, float w) { return make_float4(x, y, z, w); }
};
template <>
struct Quad<bf16> {
  typedef uint2 type;
  static __device__ __forceinline__ float4 get(const uint2& r) {
    return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                       __uint_as_float(r.y & 0xffff0000u));
  }
  static __device__ __forceinline__ uint2 make(bf16 x, bf16 y, bf16 z, bf16 w) {
    return make_uint2(__bfloat16_as_ushort(x) | (uint32_t)__bfloat16_as_ushort(y) << 16,
                      __bfloat16_as_ushort(z) | (uint32_t)__bfloat16_as_ushort(w) << 16);
  }
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(bf16 x) { return __bfloat162float(x); }
// Four elements one by one, of which `left` are there: the others are read
// from `safe`, so that there is no branch and all loads are in flight together,
// and count as zero.
template <typename T>
__device__ __forceinline__ float4 load4_any(const T* p, const T* safe, int left) {
  const float x = as_float(*(left > 0 ? p : safe)), y = as_float(*(left > 1 ? p + 1 : safe));
  const float z = as_float(*(left > 2 ? p + 2 : safe)), w = as_float(*(left > 3 ? p + 3 : safe));
  return make_float4(left > 0 ? x : 0.0f, left > 1 ? y : 0.0f, left > 2 ? z : 0.0f, left > 3 ? w : 0.0f);
}

template <typename T>
__device__ __forceinline__ T as_type(float x);
template <>
__device__ __forceinline__ float as_type<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 as_type<bf16>(float x) { return __float2bfloat16_rn(x); }

// Two consecutive values, stored where they exist.
template <typename T>
__device__ __forceinline__ void set2(T* p, int left, bool vec, float a, float b);
template <>
__device__ __forceinline__ void set2<float>(float* p, int left, bool vec, float a, float b) {
  if (vec && left >= 2) {
    *reinterpret_cast<float2*>(p) = make_float2(a, b);
  } else {
    if (left > 0) p[0] = a;
    if (left > 1) p[1] = b;
  }
}
template <>
__device__ __forceinline__ void set2<bf16>(bf16* p, int left, bool vec, float a, float b) {
  if (vec && left >= 2) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
  } else {
    if (left > 0) p[0] = __float2bfloat16_rn(a);
    if (left > 1) p[1] = __float2bfloat16_rn(b);
  }
}

// A row of four accumulator tiles, 32 columns over four lanes, stored at p where
// `in` and they exist (`left` of them do).  `pairs`: p allows two-element accesses;
// `whole`: 16-byte ones too, and `left` is a multiple of 8.  Then bf16 goes between
// the lanes first, so that each stores 16 bytes once instead of 4 four times.
template <typename T>
__device__ __forceinline__ void set_row(T* p, int left, bool pairs, bool whole, bool in, const float2 (&x)[4]) {
  const int lane = threadIdx.x & 3;
  if (sizeof(T) == 2 && whole) {
    uint32_t w[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x[n].x, x[n].y);
      w[n] = *reinterpret_cast<const uint32_t*>(&v);
    }
    // lane i's word j becomes lane j's word i
#pragma unroll
    for (int o = 1; o < 4; o <<= 1)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (!(n & o)) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & o ? w[n] : w[n + o], o);
          if (lane & o) w[n] = got; else w[n + o] = got;
        }
    if (in && lane * 8 < left) *reinterpret_cast<uint4*>(p + lane * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if (in) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int c = n * 8 + lane * 2;
      set2<T>(p + c, left - c, pairs, x[n].x, x[n].y);
    }
  }
}

// A warp's 16 tokens x 8 or 16 value columns of a [token][column] tensor, as
// accumulator tiles.  `start` issues the loads and `get` gives a value pair,
// zero where the tensor has none: nothing between the two waits for memory.
template <typename T>
struct PairOf;
template <>
struct PairOf<float> {
  typedef float2 type;
  static __device__ __forceinline__ float2 make(float x, float y) { return make_float2(x, y); }
  static __device__ __forceinline__ float2 get(float2 r) { return r; }
};
template <>
struct PairOf<bf16> {
  typedef uint32_t type;
  static __device__ __forceinline__ uint32_t make(bf16 x, bf16 y) {
    return __bfloat16_as_ushort(x) | (uint32_t)__bfloat16_as_ushort(y) << 16;
  }
  static __device__ __forceinline__ float2 get(uint32_t r) {
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
  }
};
// NT column tiles of 8.
template <typename T, int NT>
struct Columns {
  typename PairOf<T>::type raw[NT][2];
  int tokens, cols;  // that there are from the tile's first on
  bool whole;        // all of the tile is there, the same for the warp
  // vec: columns and strides are even and p is aligned to two elements
  __device__ __forceinline__ void start(const T* p, long stride, int tokens_, int cols_, bool vec) {
    tokens = tokens_;
    cols = cols_;
    whole = tokens >= 16 && cols >= NT * 8;
    if (whole && vec) {
      const T* q = p + frag_row(0, 0) * stride + frag_col(0);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          raw[n][e] = *reinterpret_cast<const typename PairOf<T>::type*>(q + e * 8 * stride + n * 8);
      return;
    }
    if (tokens <= 0 || cols <= 0) return;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = frag_col(n * 8);
        const T* q = p + min(frag_row(0, e), tokens - 1) * stride;
        raw[n][e] = PairOf<T>::make(q[min(c, cols - 1)], q[min(c + 1, cols - 1)]);
      }
  }
  __device__ __forceinline__ float2 get(int n, int e) const {
    float2 f = PairOf<T>::get(raw[n][e]);
    if (whole) return f;
    const int c = frag_col(n * 8);
    const bool in = frag_row(0, e) < tokens;
    f.x = in && c < cols ? f.x : 0.0f;
    f.y = in && c + 1 < cols ? f.y : 0.0f;
    return f;
  }
};
template <typename T>
__device__ __forceinline__ bool pairs_ok(const void* p, long s0, long s1, long s2, int cols) {
  return (reinterpret_cast<uintptr_t>(p) & (2 * sizeof(T) - 1)) == 0 && ((s0 | s1 | s2 | cols) & 1) == 0;
}

template <typename K>
inline int with_smem(K kernel, int bytes) {
  GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return GRU_OK;
}

// The kernels of a call follow one another, and each starts as soon as the last
// CTAs of the one before have: it reads what was there before the call, then
// waits for all that the one before writes (a prompt of 77: 48 us from call to
// result, 53 in turn; training 4 x 2048 885 us either way).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P>
inline int launch_after(void (*kernel)(P...), unsigned ctas, unsigned threads, int bytes, cudaStream_t stream, P... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = ctas;
  config.blockDim = threads;
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  GRU_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, args...));
  return GRU_OK;
}

}  // namespace delta
}  // namespace gru
