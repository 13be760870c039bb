// Layer normalisation of rows, with the sum of a residual stream in front, and
// its gradient (contract in include/rnn_kernel_b200.h).
//
//   s = x + residual (in the residual's type);  n = (s - mean) rstd;  y = n w + b
//   ds += rstd (g - mean(g) - n mean(g n)) with g = dy w;  dw = sum dy n;  db = sum dy
//
// A row is read and written once and held between: a warp holds rows
// of up to 1024 bf16 or 512 FP32 elements, a CTA longer ones, 16 bytes a thread
// and load; the next row's loads are under way meanwhile.  One load a thread stays
// in registers, and two of FP32; the other forms spill, the warps' most, as all are compiled
// for CTAs of 1024 threads (gradient: 512).  A first sum gives a mean
// that rounding leaves a little off where a row has a large offset; the distances
// from it, which are exact there, give the rest of the mean (`shift`) and the
// variance, so an offset costs no digits.  y is the norm of s as it is stored: the
// gradient, which reads s again, sees the same numbers.  CTAs go over the rows with
// the weights (and the sums of dw and db) in registers; the CTAs' sums are added in
// a fixed order by a second launch.
//
// Bound by memory: 8192 rows of 2048 with a residual, bf16, forward 26 us (134 MB, 79 %
// of the copy rate), gradient 36 (134 MB, 57 %: two CTAs an SM by their registers, and
// a barrier a row); 32768 rows of 256, FP32, forward 12 us (67 MB, 85 %), gradient 17
// (101 MB, 89 %).  By local memory where registers are spilled: 8192 rows with a residual,
// timed with the launches, of 768 bf16 78 and 56 us (50 MB each, 8 us; gradient 178
// with an FP32 residual), of 4096 61 and 114 (268 MB, 41 us).

#include <algorithm>

#include "row_ops.cuh"

namespace gru {
namespace {

constexpr int kMaxWidth = 16384;
constexpr int kNormCtas = 148 * 4;  // most CTAs of the gradient, whose sums the workspace holds

struct Norm {
  const void *x, *res, *w, *b;
  void *y, *s;
  float* stats;  // [3][rows]: the first mean, what it lacks, 1 / deviation
  // gradient: s is read; x, y, res and b are unused
  const void *dy, *ds;
  void *dx, *dres;
  float* part;  // [CTA][2][D]
  long R, xs, rs, dys, dss;  // rows, and elements between them
  int D, wtype, wvec;  // wvec: the weights lie on boundaries of a load
  float eps;
};

// Sums K numbers over the threads of a row.
template <int K, bool CTA>
__device__ __forceinline__ void row_sum(float (&v)[K], float* smem) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if constexpr (CTA) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) smem[k * 32 + warp] = v[k];
    __syncthreads();
    if (warps <= 8) {  // eight lanes hold the warps' sums, four times over
#pragma unroll
      for (int k = 0; k < K; ++k) {
        v[k] = (lane & 7) < warps ? smem[k * 32 + (lane & 7)] : 0.0f;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = warp_sum(lane < warps ? smem[k * 32 + lane] : 0.0f);
    }
  }
}

// Elementwise on V neighbours, two in an operation: V is 1 or even.
template <int V>
__device__ __forceinline__ void add_to(float (&v)[V], float c) {
  if constexpr (V == 1) v[0] += c;
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 r = __fadd2_rn(make_float2(v[e], v[e + 1]), make_float2(c, c));
      v[e] = r.x, v[e + 1] = r.y;
    }
}
template <int V>
__device__ __forceinline__ void scale(float (&v)[V], float c) {
  if constexpr (V == 1) v[0] *= c;
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 r = __fmul2_rn(make_float2(v[e], v[e + 1]), make_float2(c, c));
      v[e] = r.x, v[e + 1] = r.y;
    }
}
template <int V>
__device__ __forceinline__ void add_row(float (&v)[V], const float (&w)[V]) {
  if constexpr (V == 1) v[0] += w[0];
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 r = __fadd2_rn(make_float2(v[e], v[e + 1]), make_float2(w[e], w[e + 1]));
      v[e] = r.x, v[e + 1] = r.y;
    }
}
// v = a b + c
template <int V>
__device__ __forceinline__ void fma_row(float (&v)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V == 1) v[0] = fmaf(a[0], b[0], c[0]);
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 r = __ffma2_rn(make_float2(a[e], a[e + 1]), make_float2(b[e], b[e + 1]), make_float2(c[e], c[e + 1]));
      v[e] = r.x, v[e + 1] = r.y;
    }
}
// acc += a, and acc += a b, as two sums (of odd and even places).
template <int V>
__device__ __forceinline__ void sum_into(float2& acc, const float (&a)[V]) {
  if constexpr (V == 1) acc.x += a[0];
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) acc = __fadd2_rn(acc, make_float2(a[e], a[e + 1]));
}
template <int V>
__device__ __forceinline__ void dot_into(float2& acc, const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) acc.x = fmaf(a[0], b[0], acc.x);
  else
#pragma unroll
    for (int e = 0; e < V; e += 2) acc = __ffma2_rn(make_float2(a[e], a[e + 1]), make_float2(b[e], b[e + 1]), acc);
}

// V elements a load, NV loads a thread; RES: there is a residual (type TR).
template <typename TX, typename TR, bool RES, int V, int NV, bool CTA>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const Norm a) {
  __shared__ float smem[2][64];
  const int per = CTA ? blockDim.x : 32;
  const int tid = CTA ? threadIdx.x : threadIdx.x & 31;
  const long first = CTA ? blockIdx.x : (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long step = CTA ? gridDim.x : (long)gridDim.x * (blockDim.x >> 5);
  const float inv = 1.0f / (float)a.D;
  float w[NV][V], b[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = min((i * per + tid) * V, a.D - V);  // threads past the row read its last
    get_row<V>(a.w, c, a.wtype, a.wvec, w[i]);
    get_row<V>(a.b ? a.b : a.w, c, a.wtype, a.wvec, b[i]);
    if (!a.b)
#pragma unroll
      for (int e = 0; e < V; ++e) b[i][e] = 0.0f;
  }
  Raw<TX, V> xn[NV];
  Raw<TR, V> tn[NV];
  auto load = [&](long r) {
    const TX* x = static_cast<const TX*>(a.x) + r * a.xs;
    const TR* res = static_cast<const TR*>(a.res) + r * a.rs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * per + tid) * V;
      if (c < a.D) {
        xn[i].load(x + c);
        if (RES) tn[i].load(res + c);
      }
    }
  };
  if (first < a.R) load(first);
  for (long r = first; r < a.R; r += step) {
    float v[NV][V], t[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * per + tid) * V < a.D) {
        xn[i].get(v[i]);
        if (RES) tn[i].get(t[i]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = t[i][e] = 0.0f;
      }
    }
    if (r + step < a.R) load(r + step);
    float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * per + tid) * V;
      if (RES) {
        add_row<V>(v[i], t[i]);
        if (c < a.D) store_row<V>(static_cast<TR*>(a.s) + r * a.D + c, v[i]);
        round_row<TR, V>(v[i]);
      }
      sum_into<V>(acc, v[i]);
    }
    float sum[1] = {acc.x + acc.y};
    row_sum<1, CTA>(sum, smem[0]);
    const float mean = sum[0] * inv;
    float2 first_sum = make_float2(0.0f, 0.0f), square = first_sum;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * per + tid) * V < a.D) {
        add_to<V>(v[i], -mean);
        sum_into<V>(first_sum, v[i]);
        dot_into<V>(square, v[i], v[i]);
      }
    float sums[2] = {first_sum.x + first_sum.y, square.x + square.y};
    row_sum<2, CTA>(sums, smem[1]);
    const float shift = sums[0] * inv;
    const float var = sums[1] * inv - shift * shift;  // shift is small beside the deviation, or all but 0
    const float rstd = rsqrtf((var < 0.0f ? 0.0f : var) + a.eps);
    if (tid == 0 && a.stats) {
      a.stats[r] = mean;
      a.stats[a.R + r] = shift;
      a.stats[2 * a.R + r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * per + tid) * V;
      if (c >= a.D) continue;
      add_to<V>(v[i], -shift);
      scale<V>(v[i], rstd);
      fma_row<V>(v[i], v[i], w[i], b[i]);
      store_row<V>(static_cast<TX*>(a.y) + r * a.D + c, v[i]);
    }
  }
}

// TS: the type of s and ds (the residual's, or x's without one).
template <typename TX, typename TS, int V, int NV, bool CTA>
__global__ void __launch_bounds__(512) norm_backward_kernel(const Norm a) {
  extern __shared__ float dyn[];
  __shared__ float smem[2][64];
  const int per = CTA ? blockDim.x : 32;
  const int tid = CTA ? threadIdx.x : threadIdx.x & 31;
  const long first = CTA ? blockIdx.x : (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long step = CTA ? gridDim.x : (long)gridDim.x * (blockDim.x >> 5);
  const float inv = 1.0f / (float)a.D;
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    get_row<V>(a.w, min((i * per + tid) * V, a.D - V), a.wtype, a.wvec, w[i]);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = db[i][e] = 0.0f;
  }
  Raw<TS, V> sn[NV], dn[NV];
  Raw<TX, V> gn[NV];
  float stats[3];
  auto load = [&](long r) {
    const TS* s = static_cast<const TS*>(a.s) + r * a.xs;
    const TX* dy = static_cast<const TX*>(a.dy) + r * a.dys;
    const TS* ds = static_cast<const TS*>(a.ds) + r * a.dss;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * per + tid) * V;
      if (c < a.D) {
        sn[i].load(s + c);
        gn[i].load(dy + c);
        if (a.ds) dn[i].load(ds + c);
      }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) stats[k] = a.stats[k * a.R + r];
  };
  if (first < a.R) load(first);
  int turn = 0;
  for (long r = first; r < a.R; r += step, turn ^= 1) {
    float n[NV][V], g[NV][V], ds[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      sn[i].get(n[i]);
      gn[i].get(g[i]);
      if (a.ds) dn[i].get(ds[i]);
    }
    const float mean = stats[0], shift = stats[1], rstd = stats[2];
    if (r + step < a.R) load(r + step);
    float2 gs = make_float2(0.0f, 0.0f), gn_ = gs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * per + tid) * V >= a.D) continue;
      add_to<V>(n[i], -mean);
      add_to<V>(n[i], -shift);
      scale<V>(n[i], rstd);
      add_row<V>(db[i], g[i]);
      fma_row<V>(dw[i], g[i], n[i], dw[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) g[i][e] *= w[i][e];
      sum_into<V>(gs, g[i]);
      dot_into<V>(gn_, g[i], n[i]);
    }
    float sums[2] = {gs.x + gs.y, gn_.x + gn_.y};
    row_sum<2, CTA>(sums, smem[turn]);
    const float m0 = -sums[0] * inv * rstd, m1 = -sums[1] * inv * rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * per + tid) * V;
      if (c >= a.D) continue;
      // rstd g - rstd mean(g) - n rstd mean(g n) (+ ds)
      scale<V>(g[i], rstd);
      add_to<V>(g[i], m0);
      scale<V>(n[i], m1);
      add_row<V>(g[i], n[i]);
      if (a.ds) add_row<V>(g[i], ds[i]);
      if (a.dx) store_row<V>(static_cast<TX*>(a.dx) + r * a.D + c, g[i]);
      if (a.dres) store_row<V>(static_cast<TS*>(a.dres) + r * a.D + c, g[i]);
    }
  }
  float* part = a.part + (long)blockIdx.x * 2 * a.D;
  if (CTA) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = (i * per + tid) * V + e;
        if (c < a.D) part[c] = dw[i][e], part[a.D + c] = db[i][e];
      }
  } else {  // the warps' sums, in their order
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
    float* mine = dyn + warp * 2 * a.D;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = (i * per + tid) * V + e;
        if (c < a.D) mine[c] = dw[i][e], mine[a.D + c] = db[i][e];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.D; c += blockDim.x) {
      float t = dyn[c];
      for (int k = 1; k < warps; ++k) t += dyn[k * 2 * a.D + c];
      part[c] = t;
    }
  }
}

struct StoreNorm {
  void *dw, *db;
  int D, dtype;
  __device__ __forceinline__ void operator()(long c, float x) const {
    if (c < D) put(dw, c, dtype, x);
    else if (db) put(db, c - D, dtype, x);
  }
};

// How a row is dealt out.
struct Shape {
  int nv, threads, rows;  // loads a thread, threads a CTA, rows a CTA at a time
  bool cta;
};
// v elements a load: warps hold rows of up to 4 loads a lane, where there are rows
// enough for four of them on every SM; CTAs hold the others in as many loads a thread
// as `most` threads need, eight elements a thread where that takes no more than 256 of them.
Shape shape_of(int D, int v, int most, long rows) {
  const int loads = ceil_div(D, v);
  const int warp_loads = v == 1 ? 8 : 4;
  Shape s;
  s.cta = loads > 32 * warp_loads || (v > 1 && loads > 32 && rows < 4 * 148);
  if (!s.cta) {
    s.nv = 1;
    while (s.nv * 32 < loads) s.nv *= 2;
    s.threads = 128, s.rows = 4;
    return s;
  }
  s.nv = v == 1 ? 8 : 1;
  while (s.nv * 32 < loads && s.nv * v < 8 && rows >= 148) s.nv *= 2;
  if (s.nv * 256 < loads) s.nv *= 2;
  while (s.nv * most < loads) s.nv *= 2;
  s.threads = (ceil_div(loads, s.nv) + 31) / 32 * 32, s.rows = 1;
  return s;
}

template <typename TX, typename TR, bool RES, int V>
int launch_forward(const Norm& a, cudaStream_t stream) {
  const Shape s = shape_of(a.D, V, 1024, a.R);
  const long need = (a.R + s.rows - 1) / s.rows;
  const unsigned ctas = (unsigned)std::min<long>(need, (long)sms_here() * std::max(1, 2048 / s.threads));
  LaunchScope scope(kKindLayerNorm, stream);
#define GRU_NORM(NV, CTA)                                                                    \
  if (s.nv == NV && s.cta == CTA) {                                                          \
    norm_forward_kernel<TX, TR, RES, V, NV, CTA><<<ctas, s.threads, 0, stream>>>(a);         \
    GRU_CUDA_TRY(cudaGetLastError());                                                        \
    return GRU_OK;                                                                           \
  }
  GRU_NORM(1, false)
  GRU_NORM(2, false)
  GRU_NORM(4, false)
  if constexpr (V == 1) {
    GRU_NORM(8, false)
    GRU_NORM(8, true)
    GRU_NORM(16, true)
  } else {
    GRU_NORM(1, true)
    GRU_NORM(2, true)
    if constexpr (V == 4) {  // two loads of eight hold the longest row
      GRU_NORM(4, true)
    }
  }
#undef GRU_NORM
  return refuse("gru_layer_norm_forward", "no kernel for this width", GRU_ERR_UNSUPPORTED);
}

template <typename TX, typename TS, int V>
int launch_backward(const Norm& a, const StoreNorm& store, cudaStream_t stream) {
  const Shape s = shape_of(a.D, V, 512, a.R);
  const long need = (a.R + s.rows - 1) / s.rows;
  const long fit = std::min<long>(kNormCtas, (long)sms_here() * std::max(1, 1024 / s.threads));
  const unsigned ctas = (unsigned)std::min(need, fit);
  const size_t smem = s.cta ? 0 : sizeof(float) * 4 * 2 * a.D;
  LaunchScope scope(kKindLayerNorm, stream, 2);
#define GRU_NORM(NV, CTA)                                                                    \
  if (s.nv == NV && s.cta == CTA) {                                                          \
    norm_backward_kernel<TX, TS, V, NV, CTA><<<ctas, s.threads, smem, stream>>>(a);          \
    GRU_CUDA_TRY(cudaGetLastError());                                                        \
    return sum_parts(a.part, (int)ctas, 2L * a.D, 2L * a.D, store, stream);                  \
  }
  GRU_NORM(1, false)
  GRU_NORM(2, false)
  GRU_NORM(4, false)
  if constexpr (V == 1) {
    GRU_NORM(8, false)
    GRU_NORM(8, true)
    GRU_NORM(16, true)
    GRU_NORM(32, true)
  } else {
    GRU_NORM(1, true)
    GRU_NORM(2, true)
    GRU_NORM(4, true)
    if constexpr (V == 4) {
      GRU_NORM(8, true)
    }
  }
#undef GRU_NORM
  return refuse("gru_layer_norm_backward", "no kernel for this width", GRU_ERR_UNSUPPORTED);
}

int check(const char* me, const gru_norm_args* p) {
  if (!p) return refuse(me, "null arguments");
  if (!known(p->dtype) || !known(p->residual_dtype) || !known(p->weight_dtype))
    return refuse(me, "types must be GRU_F32 or GRU_BF16", GRU_ERR_UNSUPPORTED);
  if ((p->residual_dtype != p->dtype && p->residual_dtype != GRU_F32) ||
      (p->weight_dtype != p->dtype && p->weight_dtype != GRU_F32))
    return refuse(me, "the residual and the weights must be FP32 or of x's type", GRU_ERR_UNSUPPORTED);
  if (p->rows < 0 || p->width < 1) return refuse(me, "need rows >= 0 and width >= 1");
  if (p->width > kMaxWidth) return refuse(me, "the width must be in [1, 16384]", GRU_ERR_UNSUPPORTED);
  if (!(p->eps >= 0.0f)) return refuse(me, "eps must not be negative");
  return GRU_OK;
}

bool misaligned(const void* p, int dtype) { return bits(p) & (elem_size(dtype) - 1); }

}  // namespace
}  // namespace gru

using namespace gru;

extern "C" size_t gru_layer_norm_workspace_bytes(const gru_norm_args* p) {
  if (check("gru_layer_norm_workspace_bytes", p)) return 0;
  return align_up(sizeof(float) * 2 * (size_t)p->width * (size_t)std::min<long>(kNormCtas, std::max(1L, p->rows)), 256);
}

extern "C" int gru_layer_norm_forward(const gru_norm_args* p, const void* x, const void* residual, const void* weight,
                                      const void* bias, void* out, void* sum, float* stats, void* stream_) {
  clear_error();
  const char* me = "gru_layer_norm_forward";
  if (const int rc = check(me, p)) return rc;
  if (p->rows == 0) return GRU_OK;
  if (!x || !weight || !out || (residual != nullptr) != (sum != nullptr))
    return refuse(me, "null tensor, or a sum without a residual");
  if (misaligned(x, p->dtype) || misaligned(out, p->dtype) || misaligned(residual, p->residual_dtype) ||
      misaligned(sum, p->residual_dtype) || misaligned(weight, p->weight_dtype) || misaligned(bias, p->weight_dtype) ||
      (bits(stats) & 3))
    return refuse(me, "a tensor is not aligned to its element size");
  Norm a{};
  a.x = x, a.res = residual, a.w = weight, a.b = bias, a.y = out, a.s = sum, a.stats = stats;
  a.R = p->rows, a.xs = p->row_stride, a.rs = p->residual_row_stride;
  a.D = p->width, a.wtype = p->weight_dtype, a.eps = p->eps;
  const int v = p->dtype == GRU_F32 ? 4 : 8;
  const bool vec = a.D % v == 0 && a.xs % v == 0 && (!residual || a.rs % v == 0) &&
                   ((bits(x) | bits(residual) | bits(out) | bits(sum)) & 15) == 0;
  a.wvec = vec && ((bits(weight) | bits(bias)) & 15) == 0;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (p->dtype == GRU_F32) {
    if (residual) return vec ? launch_forward<float, float, true, 4>(a, stream) : launch_forward<float, float, true, 1>(a, stream);
    return vec ? launch_forward<float, float, false, 4>(a, stream) : launch_forward<float, float, false, 1>(a, stream);
  }
  if (!residual) return vec ? launch_forward<bf16, bf16, false, 8>(a, stream) : launch_forward<bf16, bf16, false, 1>(a, stream);
  if (p->residual_dtype == GRU_F32)
    return vec ? launch_forward<bf16, float, true, 8>(a, stream) : launch_forward<bf16, float, true, 1>(a, stream);
  return vec ? launch_forward<bf16, bf16, true, 8>(a, stream) : launch_forward<bf16, bf16, true, 1>(a, stream);
}

extern "C" int gru_layer_norm_backward(const gru_norm_args* p, const void* sum, const void* weight, const float* stats,
                                       const void* dout, const void* dsum, void* dx, void* dresidual,
                                       void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream_) {
  clear_error();
  const char* me = "gru_layer_norm_backward";
  if (const int rc = check(me, p)) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!dweight || misaligned(dweight, p->weight_dtype) || misaligned(dbias, p->weight_dtype))
    return refuse(me, "null or misaligned gradient of the weight");
  if (p->rows == 0) {
    const size_t n = elem_size(p->weight_dtype) * p->width;
    GRU_CUDA_TRY(cudaMemsetAsync(dweight, 0, n, stream));
    if (dbias) GRU_CUDA_TRY(cudaMemsetAsync(dbias, 0, n, stream));
    return GRU_OK;
  }
  const int st = p->residual_dtype;  // s's type; x's without a residual
  if (!sum || !weight || !stats || !dout) return refuse(me, "null tensor");
  if (misaligned(sum, st) || misaligned(dsum, st) || misaligned(dresidual, st) || misaligned(dout, p->dtype) ||
      misaligned(dx, p->dtype) || misaligned(weight, p->weight_dtype) || (bits(stats) & 3))
    return refuse(me, "a tensor is not aligned to its element size");
  if (!workspace || (bits(workspace) & 15) || workspace_bytes < gru_layer_norm_workspace_bytes(p))
    return refuse(me, "workspace too small or not 16-byte aligned");
  Norm a{};
  a.s = const_cast<void*>(sum), a.w = weight, a.stats = const_cast<float*>(stats);
  a.dy = dout, a.ds = dsum, a.dx = dx, a.dres = dresidual, a.part = static_cast<float*>(workspace);
  a.R = p->rows, a.xs = p->row_stride, a.dys = a.dss = p->width;
  a.D = p->width, a.wtype = p->weight_dtype, a.eps = p->eps;
  const int v = p->dtype == GRU_F32 ? 4 : 8;
  const bool vec = a.D % v == 0 && a.xs % v == 0 &&
                   ((bits(sum) | bits(dout) | bits(dsum) | bits(dx) | bits(dresidual)) & 15) == 0;
  a.wvec = vec && (bits(weight) & 15) == 0;
  const StoreNorm store{dweight, dbias, a.D, p->weight_dtype};
  if (p->dtype == GRU_F32)
    return vec ? launch_backward<float, float, 4>(a, store, stream) : launch_backward<float, float, 1>(a, store, stream);
  if (st == GRU_F32)
    return vec ? launch_backward<bf16, float, 8>(a, store, stream) : launch_backward<bf16, float, 1>(a, store, stream);
  return vec ? launch_backward<bf16, bf16, 8>(a, store, stream) : launch_backward<bf16, bf16, 1>(a, store, stream);
}
