// AdamW over many tensors in one launch, with moments held in 32 or in 8 bits.
//
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2
//   p <- (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in FP32 whatever the weights' type (FP32 or bf16, rounded once when stored).
// All tensors' moments live in one buffer each, in which every tensor starts at
// a multiple of 256 elements (one quantisation block); a CTA updates 2048
// (with 8-bit moments up to 16384) consecutive elements of one tensor, a warp a block at a time, a lane 2 x 4 elements,
// so every access is a coalesced 16-byte one (8 for bf16, 4 for codes).  The
// tensor table travels in the kernel's parameters: no copy, no device table.
//
// 8-bit moments.  A block's 256 values share an FP32 scale, absmax / 1.875;
// the code of r = |x| / scale holds r's exponent and 3 mantissa bits:
//   first moment   sign, 4 exponent bits: 2^-15 .. 1.875 (and zero)
//   second moment  5 exponent bits:       2^-31 .. 1.875 (and zero)
// A logarithmic code, because v spans many decades inside a block and a linear
// one would round most of it to zero, and v divides: a nonzero v is never
// coded as zero, unless its quotient by the scale is below FP32's range, and
// beside a v coded as zero (a gradient whose square vanishes) no m is rounded
// up to the least code: eps alone would divide it.  Rounding is stochastic, from a hash of (seed, step,
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
constexpr int kRow = kBlock * (kThreads / 32);  // elements that a CTA's warps take at a time
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
  int rows;  // kRow elements that a CTA takes, one after the other
};

__device__ __forceinline__ float code_value(unsigned low, int ebits) {
  return low ? __uint_as_float((low << 20) + ((128u - (1u << ebits)) << 23)) : 0.0f;
}

__device__ __forceinline__ float value_m(unsigned c) {
  const float x = code_value(c & 0x7fu, 4);
  return (c & 0x80u) ? -x : x;
}
__device__ __forceinline__ float value_v(unsigned c) { return code_value(c, 5); }
__device__ __forceinline__ float decode_m(unsigned c, float scale) { return __fmul_rn(value_m(c), scale); }
__device__ __forceinline__ float decode_v(unsigned c, float scale) { return __fmul_rn(value_v(c), scale); }

// The larger of two magnitudes; a NaN wins.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// 32 random bits of a position, 16 for each moment.  noise_base is linear in
// the position (inside a block, whose elements share their upper 32 bits).
__device__ __forceinline__ unsigned noise_base(long i, unsigned key) {
  return (unsigned)i * 0x9E3779B1u + key + (unsigned)((unsigned long long)i >> 32) * 0xC2B2AE3Du;
}
__device__ __forceinline__ unsigned noise_bits(unsigned h) {
  h = (h ^ (h >> 15)) * 0xB5297A4Du;
  h = (h ^ (h >> 13)) * 0x68E31DA5u;
  return h ^ (h >> 16);
}

// The code whose value is r rounded up or down at random, from 16 random bits
// (shifted to `noise`) below the 3 mantissa bits; the 4 bits below those are
// truncated.  Below 1 where r is below the least code.
__device__ __forceinline__ int round_code(float r, unsigned noise, int ebits) {
  const unsigned base = (128u - (1u << ebits)) << 23;
  return min((int)(__float_as_uint(r) + noise - base) >> 20, (1 << (ebits + 3)) - 1);
}

constexpr float kLeast = 1.125f / 32768.0f;  // the least first moment that a code stands for

// A first moment below that: the least code or zero, at random.
__device__ __forceinline__ int round_least(float r, unsigned n16) {
  // n16 / 65536, exactly, without the slow integer conversion
  const float u = __uint_as_float(0x3f800000u | (n16 << 7)) - 1.0f;
  return r > __fmul_rn(u, kLeast) ? 1 : 0;
}

// A block's scale from the warp's largest magnitude (as bits: for
// non-negative floats integer order is value order, and a NaN is above all).
// Below 2^-100 the reciprocal would overflow: the block counts as zero.
__device__ __forceinline__ float block_scale(unsigned amax_bits) {
  const float s = __fmul_rn(__uint_as_float(__reduce_max_sync(0xffffffffu, amax_bits)), kInvTop);
  return s < 0x1p-100f ? 0.0f : s;
}

// Four consecutive elements: `vec` where all four exist and one access can
// take them, else those of them that exist (zeros for the others).
template <typename T>
__device__ __forceinline__ void load4(const T* p, int left, bool vec, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, int left, bool vec, float (&x)[4]) {
  if (vec) {
    const float4 f = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = i < left ? p[i] : 0.0f;
  }
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, int left, bool vec, float (&x)[4]) {
  if (vec) {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
    x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xffff0000u);
    x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = i < left ? __bfloat162float(p[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, int left, bool vec, const float (&x)[4]);
template <>
__device__ __forceinline__ void store4<float>(float* p, int left, bool vec, const float (&x)[4]) {
  if (vec) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = x[i];
  }
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, int left, bool vec, const float (&x)[4]) {
  if (vec) {
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

// The step's square root and quotient.  With 8-bit moments the kernel is near
// its instruction limit (86 slots an element at copy bandwidth), so it takes
// the hardware's approximations, good to 2 ulp of a step that the moments
// themselves know to 4 bits; codes and scales do not depend on them.
template <int kBits>
__device__ __forceinline__ float root(float x) {
  if (kBits == 32) return __fsqrt_rn(x);
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int kBits>
__device__ __forceinline__ float ratio(float x, float y) {
  if (kBits == 32) return __fdiv_rn(x, y);
  float z;  // y is a normal number, or zero where v and eps are
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(z) : "f"(y));
  return __fmul_rn(x, z);
}

// kBits: 32 or 8.
//
// What bounds it: memory with 32-bit moments; with 8-bit ones the integer pipe
// (two instructions a cycle and SM) comes close: the codes' values come from
// a table in shared memory instead of integer arithmetic, codes are packed by
// multiply-adds (another pipe), and a first moment below the least code is the
// rare case of a branch over a lane's eight elements.
template <typename T, int kBits, int N>
__global__ void __launch_bounds__(kThreads, kBits == 8 ? 5 : 4) adamw_kernel(const __grid_constant__ Table<N> tab,
                                                         const __grid_constant__ Common c) {
  __shared__ float lut[kBits == 8 ? 512 : 1];
  if (kBits == 8) {
    lut[threadIdx.x] = value_m(threadIdx.x);
    lut[256 + threadIdx.x] = value_v(threadIdx.x);
    __syncthreads();
  }
  // the last tensor whose first CTA is not after this one
  int lo = 0, hi = c.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.e[mid].chunk <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const Entry& e = tab.e[lo];
  const int lane = threadIdx.x & 31;
  float step = e.step, inv_bc2 = e.inv_bc2;
  unsigned key = c.key;
  if (c.scal) {
    step = __fmul_rn(step, c.scal[0]);
    inv_bc2 = c.scal[1];
    key = __float_as_uint(c.scal[2]);
  }
#pragma unroll 1
  for (int w = 0; w < c.rows; ++w) {
    // first element of this warp's block, in the tensor and in the moments
    const long at = ((long)(blockIdx.x - e.chunk) * c.rows + w) * kRow + (threadIdx.x >> 5) * kBlock;
    if (at >= e.n) return;
    const long so = e.off + at;

    float p[2][4], g[2][4], m[2][4], v[2][4];
    const int there = (int)min((long)kBlock, e.n - at);
    const bool vec = e.vec && there == kBlock;  // the same for the whole warp
    T* bp = static_cast<T*>(e.p) + at + lane * 4;
    const T* bg = static_cast<const T*>(e.g) + at + lane * 4;
    float* fm = static_cast<float*>(c.m) + so + lane * 4;
    float* fv = static_cast<float*>(c.v) + so + lane * 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      load4<T>(bg + h * 128, there - h * 128 - lane * 4, vec, g[h]);
      load4<T>(bp + h * 128, there - h * 128 - lane * 4, vec, p[h]);
      if (kBits == 32) {
        load4<float>(fm + h * 128, 4, true, m[h]);
        load4<float>(fv + h * 128, 4, true, v[h]);
      }
    }
    unsigned* bm = reinterpret_cast<unsigned*>(static_cast<unsigned char*>(c.m) + so) + lane;
    unsigned* bv = reinterpret_cast<unsigned*>(static_cast<unsigned char*>(c.v) + so) + lane;
    if (kBits == 8) {
      unsigned cm[2], cv[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        cm[h] = bm[h * 32];
        cv[h] = bv[h * 32];
      }
      const float sm = c.sm[so / kBlock], sv = c.sv[so / kBlock];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m[h][i] = __fmul_rn(lut[(cm[h] >> (8 * i)) & 0xffu], sm);
          v[h][i] = __fmul_rn(lut[256 + ((cv[h] >> (8 * i)) & 0xffu)], sv);
        }
    }
    float am = 0.0f, av = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float gg = __fmul_rn(g[h][i], c.gscale);
        m[h][i] = __fadd_rn(__fmul_rn(m[h][i], c.b1), __fmul_rn(gg, c.omb1));
        v[h][i] = __fadd_rn(__fmul_rn(v[h][i], c.b2), __fmul_rn(__fmul_rn(gg, gg), c.omb2));
        const float den = __fadd_rn(__fmul_rn(root<kBits>(v[h][i]), inv_bc2), c.eps);
        p[h][i] = __fsub_rn(__fmul_rn(p[h][i], e.decay), ratio<kBits>(__fmul_rn(m[h][i], step), den));
        if (kBits == 8) {
          am = max_nan(am, fabsf(m[h][i]));
          av = max_nan(av, v[h][i]);
        }
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      store4<T>(bp + h * 128, there - h * 128 - lane * 4, vec, p[h]);
      if (kBits == 32) {
        // the elements between the tensor's end and its block's are zero: g is
        store4<float>(fm + h * 128, 4, true, m[h]);
        store4<float>(fv + h * 128, 4, true, v[h]);
      }
    }
    if (kBits == 8) {
      const float sm = block_scale(__float_as_uint(am)), sv = block_scale(__float_as_uint(av));
      const float im = sm == 0.0f ? 0.0f : __frcp_rn(sm), iv = sv == 0.0f ? 0.0f : __frcp_rn(sv);
      int km[2][4];
      unsigned rnd[2][4], cv[2] = {0, 0};
      bool low = false;
      const unsigned base = noise_base(so + lane * 4, key);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 3; i >= 0; --i) {
          rnd[h][i] = noise_bits(base + (unsigned)(h * 128 + i) * 0x9E3779B1u);
          const float r = __fmul_rn(fabsf(m[h][i]), im), q = __fmul_rn(v[h][i], iv);
          km[h][i] = round_code(r, (rnd[h][i] >> 12) & 0xffff0u, 4);
          low |= r < kLeast;
          // a nonzero second moment is never coded as zero: it divides
          const int k = max(round_code(q, (rnd[h][i] << 4) & 0xffff0u, 5), (int)min(__float_as_uint(q), 1u));
          cv[h] = cv[h] * 256u + (unsigned)k;
        }
        bv[h * 32] = cv[h];
      }
      if (low) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float r = __fmul_rn(fabsf(m[h][i]), im);
            if (r < kLeast) km[h][i] = (cv[h] >> (8 * i)) & 0xffu ? round_least(r, rnd[h][i] >> 16) : 0;
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        unsigned cm = 0;
#pragma unroll
        for (int i = 3; i >= 0; --i)
          cm = cm * 256u + ((unsigned)km[h][i] | ((__float_as_uint(m[h][i]) >> 24) & 0x80u));
        bm[h * 32] = cm;
      }
      if (lane == 0) {
        c.sm[so / kBlock] = sm;
        c.sv[so / kBlock] = sv;
      }
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
    const long chunk = (long)kRow * c.rows, need = (ts[i].n + chunk - 1) / chunk;
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

// Tables of 32 tensors (1.8 KB of kernel parameters) or of 256 (14 KB): a
// launch's parameters are copied whole, so a few tensors get the small one.
template <typename T, int kBits>
int run_sized(const gru_adamw_tensor* ts, int count, const Common& c, cudaStream_t stream) {
  if (count <= 32) return run<T, kBits, 32>(ts, count, c, stream);
  return run<T, kBits, 256>(ts, count, c, stream);
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
  // a block of second moments below 2^-100 counts as zero: eps must not be
  // smaller than their roots, or their step would be divided by next to nothing
  if (state_bits == 8 && !(eps >= 0x1p-50)) {
    set_error("gru_adamw_step: need eps >= 2^-50 with 8-bit moments");
    return GRU_ERR_INVALID;
  }
  if (device_step && !device_scalars) {
    set_error("gru_adamw_step: device_step needs device_scalars");
    return GRU_ERR_INVALID;
  }
  long total = 0;
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
    total += t.n;
  }
  if (total > 0 && (!exp_avg || !exp_avg_sq || (state_bits == 8 && (!scale_avg || !scale_sq)) || state_elems % kBlock != 0 ||
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
  if (total == 0) return GRU_OK;
  // With 8-bit moments a CTA first builds its decoding table, so a large step
  // lets it take up to eight rows while two waves of CTAs remain (201 M
  // weights: 1027 us with eight rows, 1074 with one); a small one, and 32-bit
  // moments, spread over as many CTAs as there are.
  const long all = total / (kRow * 2L * 5 * 148);
  const int rows = state_bits == 8 ? (int)std::min(std::max(all, 1L), 8L) : 1;
  const Common c{exp_avg, exp_avg_sq, scale_avg, scale_sq, device_scalars, (float)beta1, (float)(1.0 - beta1),
                 (float)beta2, (float)(1.0 - beta2), eps > 0.0 ? std::max((float)eps, 1.17549435e-38f) : 0.0f,
                 (float)grad_scale,
                 seed * 0x8DA6B343u + (unsigned)step * 0xD8163841u, 0, rows};
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
