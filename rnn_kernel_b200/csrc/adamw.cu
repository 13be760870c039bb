// AdamW over many tensors in one launch, with moments held in 32 or in 8 bits.
//
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2
//   p <- (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in FP32 whatever the weights' type (FP32 or bf16, rounded once when stored).
// All tensors' moments live in one buffer each, in which every tensor starts at
// a multiple of 256 elements (one quantisation block); a CTA updates 2048
// consecutive elements of one tensor, a warp one block, a lane 2 x 4 elements,
// so every access is a coalesced 16-byte one (8 for bf16, 4 for codes).  The
// tensor table travels in the kernel's parameters: no copy, no device table.
//
// 8-bit moments.  A block's 256 values share an FP32 scale, absmax / 1.875;
// the code of r = |x| / scale holds r's exponent and 3 mantissa bits:
//   first moment   sign, 4 exponent bits: 2^-15 .. 1.875 (and zero)
//   second moment  5 exponent bits:       2^-31 .. 1.875 (and zero)
// A logarithmic code, because v spans many decades inside a block and a linear
// one would round most of it to zero, and v divides: a nonzero v is never
// coded as zero.  Rounding is stochastic, from a hash of (seed, step,
// position): an update moves v by 0.1 % where codes are 6 - 12 % apart, so
// rounding to nearest would stop the average altogether, while here its
// expectation is exact (above the least code).  The arithmetic up to the codes
// is IEEE-rounded operation by operation (the __f*_rn calls, no contraction),
// so codes do not depend on the compiler.
//
// HBM-bound: FP32 weights with 32-bit moments move 28 bytes an element, with
// 8-bit moments 16.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "../../include/rnn_kernel_b200.h"

namespace gru {
namespace {

constexpr int kBlock = 256;         // elements per quantisation block = per warp
constexpr int kThreads = 256;
constexpr int kChunk = kBlock * (kThreads / 32);  // elements per CTA
constexpr float kInvTop = (float)(1.0 / 1.875);  // the largest code stands for 1.875 scales

struct Entry {
  void* p;
  const void* g;
  long n;
  long off;        // of the tensor's moments, a multiple of kBlock
  float decay;     // 1 - lr * weight_decay
  float step;      // lr / (1 - b1^t), or lr with device scalars
  float inv_bc2;   // 1 / sqrt(1 - b2^t)
  int chunk;       // first CTA of this tensor
  int vec;         // p and g allow 4-element accesses
  int pad;
};

template <int N>
struct Table {
  Entry e[N];
};

struct Common {
  void* m;
  void* v;
  float* sm;
  float* sv;
  const float* scal;  // device scalars (1 / (1 - b1^t), 1 / sqrt(1 - b2^t), key) or null
  float b1, omb1, b2, omb2, eps, gscale;
  unsigned key;
  int count;
};

__device__ __forceinline__ float code_value(unsigned low, int ebits) {
  return low ? __uint_as_float((low << 20) + ((128u - (1u << ebits)) << 23)) : 0.0f;
}

__device__ __forceinline__ float decode_m(unsigned c, float scale) {
  const float x = code_value(c & 0x7fu, 4);
  return __fmul_rn((c & 0x80u) ? -x : x, scale);
}

__device__ __forceinline__ float decode_v(unsigned c, float scale) { return __fmul_rn(code_value(c, 5), scale); }

// 32 random bits of a position: 16 for each moment.
__device__ __forceinline__ unsigned noise_bits(long i, unsigned key) {
  unsigned h = (unsigned)i * 0x9E3779B1u + key + (unsigned)((unsigned long long)i >> 32) * 0xC2B2AE3Du;
  h = (h ^ (h >> 15)) * 0xB5297A4Du;
  h = (h ^ (h >> 13)) * 0x68E31DA5u;
  return h ^ (h >> 16);
}

// The code whose value is r rounded up or down at random (16 random bits
// below the 3 mantissa bits; the 4 bits below those are truncated).
__device__ __forceinline__ int round_code(float r, unsigned n16, int ebits) {
  const int c = (int)((__float_as_uint(r) + (n16 << 4)) >> 20) - (int)((128u - (1u << ebits)) << 3);
  return min(c, (1 << (ebits + 3)) - 1);
}

__device__ __forceinline__ unsigned encode_m(float m, float inv, unsigned n16) {
  constexpr float least = 1.125f / 32768.0f;
  const float r = __fmul_rn(fabsf(m), inv);
  int c = round_code(r, n16, 4);
  if (r < least) c = r > __fmul_rn((float)n16, least / 65536.0f) ? 1 : 0;
  return (unsigned)c | (m < 0.0f ? 0x80u : 0u);
}

__device__ __forceinline__ unsigned encode_v(float v, float inv, unsigned n16) {
  const float r = __fmul_rn(v, inv);
  const int c = max(round_code(r, n16, 5), 1);
  return r > 0.0f ? (unsigned)c : 0u;
}

// A block's scale from the warp's largest magnitude (as bits: for
// non-negative floats integer order is value order, and a NaN is above all).
// Below 2^-100 the reciprocal would overflow: the block counts as zero.
__device__ __forceinline__ float block_scale(unsigned amax_bits) {
  const float s = __fmul_rn(__uint_as_float(__reduce_max_sync(0xffffffffu, amax_bits)), kInvTop);
  return s < 0x1p-100f ? 0.0f : s;
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, long left, int vec, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, long left, int vec, float (&x)[4]) {
  if (vec && left >= 4) {
    const float4 f = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = i < left ? p[i] : 0.0f;
  }
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, long left, int vec, float (&x)[4]) {
  if (vec && left >= 4) {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
    x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xffff0000u);
    x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = i < left ? __bfloat162float(p[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, long left, int vec, const float (&x)[4]);
template <>
__device__ __forceinline__ void store4<float>(float* p, long left, int vec, const float (&x)[4]) {
  if (vec && left >= 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = x[i];
  }
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, long left, int vec, const float (&x)[4]) {
  if (vec && left >= 4) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    uint2 u;
    u.x = *reinterpret_cast<const unsigned*>(&a);
    u.y = *reinterpret_cast<const unsigned*>(&b);
    __stcs(reinterpret_cast<uint2*>(p), u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = __float2bfloat16_rn(x[i]);
  }
}

// kBits: 32 or 8.
template <typename T, int kBits, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<N> tab,
                                                         const __grid_constant__ Common c) {
  // the last tensor whose first CTA is not after this one
  int lo = 0, hi = c.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.e[mid].chunk <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const Entry& e = tab.e[lo];
  const int lane = threadIdx.x & 31;
  // first element of this warp's block, in the tensor and in the moments
  const long at = (long)(blockIdx.x - e.chunk) * kChunk + (threadIdx.x >> 5) * kBlock;
  if (at >= e.n) return;
  const long so = e.off + at;

  float p[2][4], g[2][4], m[2][4], v[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long i = at + h * 128 + lane * 4;
    load4<T>(static_cast<const T*>(e.g) + i, e.n - i, e.vec, g[h]);
    load4<T>(static_cast<const T*>(e.p) + i, e.n - i, e.vec, p[h]);
    if (kBits == 32) {
      load4<float>(static_cast<const float*>(c.m) + so + h * 128 + lane * 4, 4, 1, m[h]);
      load4<float>(static_cast<const float*>(c.v) + so + h * 128 + lane * 4, 4, 1, v[h]);
    }
  }
  if (kBits == 8) {
    unsigned cm[2], cv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      cm[h] = reinterpret_cast<const unsigned*>(static_cast<const unsigned char*>(c.m) + so)[h * 32 + lane];
      cv[h] = reinterpret_cast<const unsigned*>(static_cast<const unsigned char*>(c.v) + so)[h * 32 + lane];
    }
    const float sm = c.sm[so / kBlock], sv = c.sv[so / kBlock];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[h][i] = decode_m((cm[h] >> (8 * i)) & 0xffu, sm);
        v[h][i] = decode_v((cv[h] >> (8 * i)) & 0xffu, sv);
      }
  }
  float step = e.step, inv_bc2 = e.inv_bc2;
  unsigned key = c.key;
  if (c.scal) {
    step = __fmul_rn(step, c.scal[0]);
    inv_bc2 = c.scal[1];
    key = __float_as_uint(c.scal[2]);
  }
  unsigned am = 0, av = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gg = __fmul_rn(g[h][i], c.gscale);
      m[h][i] = __fadd_rn(__fmul_rn(m[h][i], c.b1), __fmul_rn(gg, c.omb1));
      v[h][i] = __fadd_rn(__fmul_rn(v[h][i], c.b2), __fmul_rn(__fmul_rn(gg, gg), c.omb2));
      const float den = __fadd_rn(__fmul_rn(__fsqrt_rn(v[h][i]), inv_bc2), c.eps);
      p[h][i] = __fsub_rn(__fmul_rn(p[h][i], e.decay), __fdiv_rn(__fmul_rn(m[h][i], step), den));
      am = max(am, __float_as_uint(m[h][i]) & 0x7fffffffu);
      av = max(av, __float_as_uint(v[h][i]) & 0x7fffffffu);
    }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long i = at + h * 128 + lane * 4;
    store4<T>(static_cast<T*>(e.p) + i, e.n - i, e.vec, p[h]);
    if (kBits == 32) {
      // the elements between the tensor's end and its block's are zero: g is
      store4<float>(static_cast<float*>(c.m) + so + h * 128 + lane * 4, 4, 1, m[h]);
      store4<float>(static_cast<float*>(c.v) + so + h * 128 + lane * 4, 4, 1, v[h]);
    }
  }
  if (kBits == 8) {
    const float sm = block_scale(am), sv = block_scale(av);
    const float im = sm == 0.0f ? 0.0f : __frcp_rn(sm), iv = sv == 0.0f ? 0.0f : __frcp_rn(sv);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned cm = 0, cv = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned r = noise_bits(so + h * 128 + lane * 4 + i, key);
        cm |= encode_m(m[h][i], im, r >> 16) << (8 * i);
        cv |= encode_v(v[h][i], iv, r & 0xffffu) << (8 * i);
      }
      reinterpret_cast<unsigned*>(static_cast<unsigned char*>(c.m) + so)[h * 32 + lane] = cm;
      reinterpret_cast<unsigned*>(static_cast<unsigned char*>(c.v) + so)[h * 32 + lane] = cv;
    }
    if (lane == 0) {
      c.sm[so / kBlock] = sm;
      c.sv[so / kBlock] = sv;
    }
  }
}

// One thread: counts the step and leaves its bias corrections and rounding
// key in device memory, for steps replayed from a CUDA graph.
__global__ void adamw_scalars_kernel(long long* step, double b1, double b2, unsigned seed, float* scal) {
  const long long t = ++*step;
  scal[0] = (float)(1.0 / (1.0 - pow(b1, (double)t)));
  scal[1] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  scal[2] = __uint_as_float(seed * 0x8DA6B343u + (unsigned)t * 0xD8163841u);
}

// 8-bit moments as the FP32 values that they stand for; a thread takes 4
// codes of each moment.  HBM-bound: 10 bytes an element.
__global__ void __launch_bounds__(256) adamw_decode_kernel(const unsigned* __restrict__ m, const unsigned* __restrict__ v,
                                                           const float* __restrict__ sm, const float* __restrict__ sv,
                                                           long n4, float4* __restrict__ om, float4* __restrict__ ov) {
  const long stride = (long)gridDim.x * blockDim.x;
  for (long i = blockIdx.x * (long)blockDim.x + threadIdx.x; i < n4; i += stride) {
    const unsigned a = __ldcs(m + i), b = __ldcs(v + i);
    const float s = sm[i / (kBlock / 4)], t = sv[i / (kBlock / 4)];
    __stcs(om + i, make_float4(decode_m(a & 0xffu, s), decode_m((a >> 8) & 0xffu, s), decode_m((a >> 16) & 0xffu, s),
                               decode_m(a >> 24, s)));
    __stcs(ov + i, make_float4(decode_v(b & 0xffu, t), decode_v((b >> 8) & 0xffu, t), decode_v((b >> 16) & 0xffu, t),
                               decode_v(b >> 24, t)));
  }
}

inline bool aligned(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <typename T, int kBits, int N>
int launch(const Table<N>& t, const Common& c, int ctas, cudaStream_t stream) {
  LaunchScope scope(kKindOptimizer, stream);
  adamw_kernel<T, kBits, N><<<ctas, kThreads, 0, stream>>>(t, c);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

// Fills tables of at most N tensors (and 2^30 CTAs) and launches each.
template <typename T, int kBits, int N>
int run(const gru_adamw_tensor* ts, int count, Common c, cudaStream_t stream) {
  const unsigned va = 4 * sizeof(T);
  Table<N> t;
  int k = 0;
  long ctas = 0;
  for (int i = 0; i < count; ++i) {
    if (ts[i].n == 0) continue;
    const long need = (ts[i].n + kChunk - 1) / kChunk;
    if (k == N || ctas + need > (1L << 30)) {
      c.count = k;
      if (const int rc = launch<T, kBits, N>(t, c, (int)ctas, stream)) return rc;
      k = 0;
      ctas = 0;
    }
    t.e[k++] = Entry{ts[i].param, ts[i].grad, ts[i].n, ts[i].state_offset, ts[i].decay, ts[i].step_size,
                     ts[i].inv_sqrt_bc2, (int)ctas, aligned(ts[i].param, va) && aligned(ts[i].grad, va), 0};
    ctas += need;
  }
  if (k == 0) return GRU_OK;
  c.count = k;
  return launch<T, kBits, N>(t, c, (int)ctas, stream);
}

// Tables of 32 tensors (1.8 KB of kernel parameters) or of 512 (28 KB, of
// the 32 KB a launch may carry): a launch's parameters are copied whole.
template <typename T, int kBits>
int run_sized(const gru_adamw_tensor* ts, int count, const Common& c, cudaStream_t stream) {
  if (count <= 32) return run<T, kBits, 32>(ts, count, c, stream);
  return run<T, kBits, 512>(ts, count, c, stream);
}

}  // namespace
}  // namespace gru

using namespace gru;

extern "C" int gru_adamw_step(const gru_adamw_tensor* tensors, int count, int dtype, int state_bits, void* exp_avg,
                              void* exp_avg_sq, float* scale_avg, float* scale_sq, long state_elems, double beta1,
                              double beta2, double eps, double grad_scale, unsigned seed, long long step,
                              long long* device_step, float* device_scalars, void* stream_) {
  clear_error();
  if (count < 0 || (count > 0 && !tensors)) {
    set_error("gru_adamw_step: need count >= 0 and a tensor table");
    return GRU_ERR_INVALID;
  }
  if ((dtype != GRU_F32 && dtype != GRU_BF16) || (state_bits != 32 && state_bits != 8)) {
    set_error("gru_adamw_step: dtype must be GRU_F32 or GRU_BF16 and state_bits 32 or 8");
    return GRU_ERR_UNSUPPORTED;
  }
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0)) {
    set_error("gru_adamw_step: need 0 <= beta1, beta2 < 1 and eps >= 0");
    return GRU_ERR_INVALID;
  }
  if (device_step && !device_scalars) {
    set_error("gru_adamw_step: device_step needs device_scalars");
    return GRU_ERR_INVALID;
  }
  bool any = false;
  for (int i = 0; i < count; ++i) {
    const gru_adamw_tensor& t = tensors[i];
    if (t.n < 0 || (t.n > 0 && (!t.param || !t.grad))) {
      set_error("gru_adamw_step: a tensor has a negative size or a null pointer");
      return GRU_ERR_INVALID;
    }
    const unsigned es = dtype == GRU_F32 ? 4 : 2;
    if (!aligned(t.param, es) || !aligned(t.grad, es)) {
      set_error("gru_adamw_step: a tensor is not aligned to its element size");
      return GRU_ERR_INVALID;
    }
    if (t.state_offset < 0 || t.state_offset % kBlock != 0 || t.state_offset > state_elems ||
        t.n > state_elems - t.state_offset || t.n > (1L << 40)) {
      set_error("gru_adamw_step: a tensor's moments must start at a multiple of 256 and end inside the buffers");
      return GRU_ERR_INVALID;
    }
    any = any || t.n > 0;
  }
  if (any && (!exp_avg || !exp_avg_sq || (state_bits == 8 && (!scale_avg || !scale_sq)) || state_elems % kBlock != 0 ||
              !aligned(exp_avg, 16) || !aligned(exp_avg_sq, 16))) {
    set_error("gru_adamw_step: moments (and 8-bit scales) must be non-null, 16-byte aligned, a multiple of 256 long");
    return GRU_ERR_INVALID;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (device_step) {
    LaunchScope scope(kKindOptimizer, stream);
    adamw_scalars_kernel<<<1, 1, 0, stream>>>(device_step, beta1, beta2, seed, device_scalars);
    GRU_CUDA_TRY(cudaGetLastError());
  }
  if (!any) return GRU_OK;
  const Common c{exp_avg, exp_avg_sq, scale_avg, scale_sq, device_scalars, (float)beta1, (float)(1.0 - beta1),
                 (float)beta2, (float)(1.0 - beta2), (float)eps, (float)grad_scale,
                 seed * 0x8DA6B343u + (unsigned)step * 0xD8163841u, 0};
  if (dtype == GRU_F32)
    return state_bits == 32 ? run_sized<float, 32>(tensors, count, c, stream)
                            : run_sized<float, 8>(tensors, count, c, stream);
  return state_bits == 32 ? run_sized<__nv_bfloat16, 32>(tensors, count, c, stream)
                          : run_sized<__nv_bfloat16, 8>(tensors, count, c, stream);
}

extern "C" int gru_adamw_decode(const void* exp_avg, const void* exp_avg_sq, const float* scale_avg,
                                const float* scale_sq, long state_elems, float* out_avg, float* out_avg_sq,
                                void* stream_) {
  clear_error();
  if (state_elems < 0 || state_elems % kBlock != 0) {
    set_error("gru_adamw_decode: state_elems must be a multiple of 256");
    return GRU_ERR_INVALID;
  }
  if (state_elems == 0) return GRU_OK;
  if (!exp_avg || !exp_avg_sq || !scale_avg || !scale_sq || !out_avg || !out_avg_sq || !aligned(exp_avg, 16) ||
      !aligned(exp_avg_sq, 16) || !aligned(out_avg, 16) || !aligned(out_avg_sq, 16)) {
    set_error("gru_adamw_decode: pointers must be non-null and 16-byte aligned");
    return GRU_ERR_INVALID;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const long n4 = state_elems / 4;
  LaunchScope scope(kKindOptimizer, stream);
  adamw_decode_kernel<<<(int)std::min<long>((n4 + 255) / 256, 148L * 16), 256, 0, stream>>>(
      static_cast<const unsigned*>(exp_avg), static_cast<const unsigned*>(exp_avg_sq), scale_avg, scale_sq, n4,
      reinterpret_cast<float4*>(out_avg), reinterpret_cast<float4*>(out_avg_sq));
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}
