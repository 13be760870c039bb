// Shared device code of the gated delta rule's kernels (sm_100a).
//
// The chunked kernels need FP32-grade products (the states, the gates' and the
// FP32 inputs' gradients are FP32), on tensor cores that multiply bf16: an FP32
// operand is held as three bf16 planes x = x0 + x1 + x2 (x0 = bf16(x), x1 =
// bf16(x - x0), x2 = bf16(x - x0 - x1): the residue is below 2^-26 |x|), and a
// product of two such operands is the six plane products whose weight is above
// 2^-24, a product with a bf16 operand (which is one plane, exactly) three.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "../../include/rnn_kernel_b200.h"

namespace gru {
namespace delta {

constexpr int kC = 64;         // tokens per chunk
constexpr int kSlice = 32;     // value columns that one CTA of a scan (one pass of a loop) works on
constexpr int kThreads = 256;  // 8 warps: 4 tiles of 16 rows x 2 halves of the columns

constexpr int kGates = 5;      // rows of Problem::gates
// Log decays below this count as this: e^-1000 is zero in FP32, and sums of 64
// of them (in FP64) still tell neighbouring tokens apart, which -inf would not.
constexpr float kNoDecay = -1000.0f;

typedef __nv_bfloat16 bf16;

// Rows of 16-bit elements in shared memory are padded by 16 bytes: the eight
// 16-byte rows of an ldmatrix then fall into eight different bank groups for
// every row length used here (32, 64, 128).
__host__ __device__ constexpr int pitch(int cols) { return cols + 8; }

template <typename T>
struct Planes;  // planes that hold a value of the input type exactly
template <>
struct Planes<float> {
  static constexpr int n = 3;
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
  int dvp;   // dv rounded up to whole slices
  float scale;
  // workspace; n = (b * H + h) * nc + chunk
  bf16* kp;      // [n over Hk][NP][64][DK]
  bf16* qp;      // [n over Hk][NP][64][DK]
  bf16* wp;      // [n over Hv][3][64][64]
  bf16* pp;      // [n over Hv][3][64][64]
  float* gates;  // [n over Hv][kGates][64]: e^G_i, e^(G_end - G_i), beta_i, G_i as two floats
  float* states; // [n over Hv][DK][dvp]: the state before the chunk
  float* e;      // [n over Hv][64][dvp]: v - S'^T k, so that u = beta e
  // gradient
  const void* dout;
  const float* ds_out;
  void *dq, *dk_, *dv_;
  float *dg, *dbeta, *ds0;
  float* du0;    // [n over Hv][64][dvp]: P^T dO
  float* z;      // [n over Hv][64][dvp]
  float* dstates;// [n over Hv][DK][dvp]: the gradient of the state after the chunk
  float* dqk;    // [n over Hk][2][64][DK]: dq and dk summed over a key head's value heads
};

int prepare(const Problem& a, int dtype, cudaStream_t stream);
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

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two values as planes, packed {low half: a, high half: b}.
template <int NP>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&w)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
    if (i + 1 < NP) {
      a -= __uint_as_float(w[i] << 16);
      b -= __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// A tile in shared memory, as planes: `stride` elements from plane to plane.
template <int NP, int PITCH>
struct Tile {
  bf16* p;
  static constexpr int np = NP;
  static constexpr int ld = PITCH;
  template <int ROWS>
  __device__ static constexpr int elems() { return NP * ROWS * PITCH; }
};

// acc[NT][4] += A (16 rows from m0) x B (NT * 8 columns from n0) over k in
// [k0, k1) (multiples of 16).  A's planes hold [m][k] (TA false) or [k][m];
// B's hold [k][n] (TB true) or [n][k].  sa / sb: elements between planes.
//
// The tensor core truncates when it adds into its accumulator.  So every 32 of
// k go into fresh accumulators, smallest plane products first, and those are
// added to acc in FP32 (rounded to nearest).
template <int NA, int NB, bool TA, bool TB, int NT>
__device__ __forceinline__ void mma_tile(float (&acc)[NT][4], const bf16* a, int sa, int lda, int m0, const bf16* b,
                                         int sb, int ldb, int n0, int k0, int k1) {
  static_assert(NT % 2 == 0, "pairs of 8-column tiles");
  const int lane = threadIdx.x & 31;
  const uint32_t pa = smem_addr(a) + 2 * (TA ? ((lane & 7) + (lane >> 4) * 8) * lda + m0 + ((lane >> 3) & 1) * 8
                                             : (m0 + (lane & 15)) * lda + (lane >> 4) * 8);
  const uint32_t pb = smem_addr(b) + 2 * (TB ? (lane & 15) * ldb + n0 + (lane >> 4) * 8
                                             : (n0 + (lane & 7) + (lane >> 4) * 8) * ldb + ((lane >> 3) & 1) * 8);
  constexpr int kTop = (NA > NB ? NA : NB) - 1;  // planes i, j with i + j <= kTop
  for (int kb = k0; kb < k1; kb += 32) {
    float t[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) t[i][j] = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = kb + 16 * h;
      if (k < k1) {
        uint32_t fa[NA][4];
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          const uint32_t at = pa + 2 * (i * sa + (TA ? k * lda : k));
          if (TA) ldm4t(fa[i], at); else ldm4(fa[i], at);
        }
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t fb[NB][4];
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const uint32_t at = pb + 2 * (i * sb + (TB ? k * ldb + n * 8 : n * 8 * ldb + k));
            if (TB) ldm4t(fb[i], at); else ldm4(fb[i], at);
          }
#pragma unroll
          for (int s = kTop; s >= 0; --s)
#pragma unroll
            for (int i = 0; i <= s; ++i) {
              const int j = s - i;
              if (i < NA && j < NB) {
                mma(t[n], fa[i], fb[j][0], fb[j][1]);
                mma(t[n + 1], fa[i], fb[j][2], fb[j][3]);
              }
            }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += t[i][j];
  }
}

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

// Stores (a, b) at [row][col], [row][col + 1] of each plane.
template <int NP>
__device__ __forceinline__ void put2(bf16* p, int plane, int ld, int row, int col, float a, float b) {
  uint32_t w[NP];
  split2<NP>(a, b, w);
#pragma unroll
  for (int i = 0; i < NP; ++i) *reinterpret_cast<uint32_t*>(p + i * plane + row * ld + col) = w[i];
}

// Four consecutive values, zero past `left`.
template <typename T>
__device__ __forceinline__ float4 get4(const T* p, int left, bool vec);
template <>
__device__ __forceinline__ float4 get4<float>(const float* p, int left, bool vec) {
  if (vec && left >= 4) return *reinterpret_cast<const float4*>(p);
  return make_float4(left > 0 ? p[0] : 0.f, left > 1 ? p[1] : 0.f, left > 2 ? p[2] : 0.f, left > 3 ? p[3] : 0.f);
}
template <>
__device__ __forceinline__ float4 get4<bf16>(const bf16* p, int left, bool vec) {
  if (vec && left >= 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
  }
  return make_float4(left > 0 ? __bfloat162float(p[0]) : 0.f, left > 1 ? __bfloat162float(p[1]) : 0.f,
                     left > 2 ? __bfloat162float(p[2]) : 0.f, left > 3 ? __bfloat162float(p[3]) : 0.f);
}

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(bf16 x) { return __bfloat162float(x); }
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

template <typename K>
inline int with_smem(K kernel, int bytes) {
  GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return GRU_OK;
}

// Rows of `cols` 16-bit elements from a dense array into padded shared rows.
template <int COLS>
__device__ __forceinline__ void copy_rows(bf16* dst, const bf16* src, int rows) {
  constexpr int per = COLS / 8;
  for (int i = threadIdx.x; i < rows * per; i += kThreads) {
    const int r = i / per, c = i % per;
    cp_async16(dst + r * pitch(COLS) + c * 8, src + (long)r * COLS + c * 8);
  }
}

// rows x kSlice FP32 values (row stride ld) as planes in padded shared rows.
template <int NP>
__device__ __forceinline__ void load_slice(bf16* dst, int plane, const float* src, long ld, int rows) {
  for (int i = threadIdx.x; i < rows * (kSlice / 4); i += kThreads) {
    const int r = i / (kSlice / 4), c = (i % (kSlice / 4)) * 4;
    const float4 f = *reinterpret_cast<const float4*>(src + r * ld + c);
    put2<NP>(dst, plane, pitch(kSlice), r, c, f.x, f.y);
    put2<NP>(dst, plane, pitch(kSlice), r, c + 2, f.z, f.w);
  }
}

}  // namespace delta
}  // namespace gru
