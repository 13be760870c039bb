// What the selective scan, the causal convolution and the layer norm share:
// loads and stores of FP32 or bf16 rows as FP32, the sigmoid, and the sum of
// partial results in a fixed order.
#pragma once

#include <cuda_bf16.h>

#include <string>

#include "common.cuh"
#include "../../include/rnn_kernel_b200.h"

namespace gru {

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements, aligned to min(16, N * sizeof(T)) bytes.
template <int N>
__device__ __forceinline__ void load_row(const float* p, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 r = *reinterpret_cast<const float4*>(p + i);
      v[i] = r.x, v[i + 1] = r.y, v[i + 2] = r.z, v[i + 3] = r.w;
    }
  } else if constexpr (N == 2) {
    const float2 r = *reinterpret_cast<const float2*>(p);
    v[0] = r.x, v[1] = r.y;
  } else {
    static_assert(N == 1, "1, 2 or a multiple of 4");
    v[0] = *p;
  }
}
template <int N>
__device__ __forceinline__ void load_row(const bf16* p, float (&v)[N]) {
  auto two = [&](int i, unsigned r) {
    v[i] = __uint_as_float(r << 16);
    v[i + 1] = __uint_as_float(r & 0xffff0000u);
  };
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const uint4 r = *reinterpret_cast<const uint4*>(p + i);
      two(i, r.x), two(i + 2, r.y), two(i + 4, r.z), two(i + 6, r.w);
    }
  } else if constexpr (N == 4) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    two(0, r.x), two(2, r.y);
  } else if constexpr (N == 2) {
    two(0, *reinterpret_cast<const unsigned*>(p));
  } else {
    static_assert(N == 1, "1, 2, 4 or a multiple of 8");
    v[0] = __bfloat162float(*p);
  }
}
template <int N>
__device__ __forceinline__ void store_row(float* p, const float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else if constexpr (N == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else {
    static_assert(N == 1, "1, 2 or a multiple of 4");
    *p = v[0];
  }
}
template <int N>
__device__ __forceinline__ void store_row(bf16* p, const float (&v)[N]) {
  auto two = [&](int i) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(v[i], v[i + 1]);
    return *reinterpret_cast<const unsigned*>(&r);
  };
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
      *reinterpret_cast<uint4*>(p + i) = make_uint4(two(i), two(i + 2), two(i + 4), two(i + 6));
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(two(0), two(2));
  } else if constexpr (N == 2) {
    *reinterpret_cast<unsigned*>(p) = two(0);
  } else {
    static_assert(N == 1, "1, 2, 4 or a multiple of 8");
    *p = __float2bfloat16_rn(v[0]);
  }
}

// The numbers that T would hold.
template <typename T, int N>
__device__ __forceinline__ void round_row(float (&v)[N]) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (N % 2 == 0) {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(v[i], v[i + 1]);
        const unsigned w = *reinterpret_cast<const unsigned*>(&r);
        v[i] = __uint_as_float(w << 16), v[i + 1] = __uint_as_float(w & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = to_f32(from_f32<T>(v[i]));
    }
  }
}

// The hardware's 2^x and 1 / x.  Numbers below 2^-126 count as zero, which spares the
// steps that scale them.
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_of(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + e^-x), 0 below -87.3.  Off by at most |x| 2^-23.7 + 2^-21.2 of itself where x is
// negative: the exponent's product rounded (2^-24 of it) with a constant that is (1.4e-8), the
// exponential 2^-22, the sum 2^-24, the reciprocal 2^-23.  That is 2^-19.2 at -16, 2^-17.1 at -87.
__device__ __forceinline__ float sigmoid_of(float x) { return rcp_of(1.0f + exp2_of(x * -1.4426950408889634f)); }

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// N consecutive elements as they are stored, so that a load can be under way
// while the numbers before it are worked on.
template <typename T, int N>
struct Raw {
  static constexpr int kBytes = N * (int)sizeof(T), kWords = kBytes / 4;
  static_assert(N == 1 || kBytes == 4 || kBytes == 8 || kBytes % 16 == 0, "one element, or whole accesses");
  unsigned v[kWords > 0 ? kWords : 1];
  T one;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (N == 1) {
      one = *p;
    } else if constexpr (kBytes == 4) {
      v[0] = *reinterpret_cast<const unsigned*>(p);
    } else if constexpr (kBytes == 8) {
      const uint2 r = *reinterpret_cast<const uint2*>(p);
      v[0] = r.x, v[1] = r.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 r = reinterpret_cast<const uint4*>(p)[i / 4];
        v[i] = r.x, v[i + 1] = r.y, v[i + 2] = r.z, v[i + 3] = r.w;
      }
    }
  }
  __device__ __forceinline__ void get(float (&f)[N]) const {
    if constexpr (N == 1) {
      f[0] = to_f32(one);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = __uint_as_float(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
};

// store(c, sum over p of part[p * stride + c]) for c < cols: FP64 sums in a
// fixed order, so results do not change from run to run.  ROWS threads share a
// column.
template <typename Store, int ROWS>
__global__ void __launch_bounds__(32 * ROWS) sum_parts_kernel(const float* __restrict__ part, int parts, long stride,
                                                              long cols, Store store) {
  __shared__ double s[ROWS][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long c = blockIdx.x * 32L + tx;
  double acc = 0.0;
  if (c < cols)
#pragma unroll 8
    for (int p = ty; p < parts; p += ROWS) acc += (double)part[p * stride + c];
  s[ty][tx] = acc;
  __syncthreads();
#pragma unroll
  for (int n = ROWS / 2; n > 0; n /= 2) {
    if (ty < n) s[ty][tx] += s[ty + n][tx];
    __syncthreads();
  }
  if (ty == 0 && c < cols) store(c, (float)s[0][tx]);
}
template <typename Store>
int sum_parts(const float* part, int parts, long stride, long cols, Store store, cudaStream_t stream) {
  const unsigned ctas = (unsigned)((cols + 31) / 32);
  if (parts > 32) sum_parts_kernel<Store, 32><<<ctas, 1024, 0, stream>>>(part, parts, stride, cols, store);
  else sum_parts_kernel<Store, 4><<<ctas, 128, 0, stream>>>(part, parts, stride, cols, store);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

// Writes x to FP32 or bf16 memory.
__device__ __forceinline__ void put(void* p, long i, int dtype, float x) {
  if (dtype == GRU_F32) static_cast<float*>(p)[i] = x;
  else static_cast<bf16*>(p)[i] = __float2bfloat16_rn(x);
}

// N elements of a parameter from i on as FP32.  whole: they lie on a boundary of
// min(16, N elements) bytes.  One branch on the type around all loads: a branch
// around each would wait for each (16 of them took 10 us at a kernel's start).
template <int N>
__device__ __forceinline__ void get_row(const void* p, long i, int dtype, bool whole, float (&v)[N]) {
  if (dtype == GRU_F32) {
    const float* f = static_cast<const float*>(p) + i;
    if (whole) {
      load_row<N>(f, v);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = f[e];
    }
  } else {
    const bf16* f = static_cast<const bf16*>(p) + i;
    if (whole) {
      load_row<N>(f, v);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = __bfloat162float(f[e]);
    }
  }
}

inline int refuse(const char* what, const char* msg, int code = GRU_ERR_INVALID) {
  set_error(std::string(what) + ": " + msg);
  return code;
}
inline uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }
inline uintptr_t elem_size(int dtype) { return dtype == GRU_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == GRU_F32 || dtype == GRU_BF16; }

// Hands out 256-byte aligned pieces of a buffer; with a null base it only
// counts.
struct Pieces {
  char* base;
  size_t used = 0;
  float* floats(size_t n) {
    float* p = base ? reinterpret_cast<float*>(base + used) : nullptr;
    used += align_up(n * sizeof(float), 256);
    return p;
  }
};

// The SMs of the current device (148 where they cannot be read).
inline int sms_here() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  const int n = sm_count(dev);
  return n > 0 ? n : 148;
}

}  // namespace gru
