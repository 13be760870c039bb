// Gradient of the selective scan.
//
// With gy the gradient of y (dout silu(z) where there is a gate) and r_t what
// the tokens behind t hand back to h_t:
//
//   dh_t = C_t gy_t + r_t;   r_{t-1} = a_t dh_t
//   dC_t = sum over channels of gy_t h_t;   dB_t = sum over channels of dt_t x_t dh_t
//   dx_t = skip gy_t + dt_t sum_n B_t dh_t
//   ddt_t = x_t sum_n B_t dh_t + sum_n A w_t,   w_t = dh_t a_t h_{t-1};   dA = sum_t dt_t w_t
//
// The forward's shape, backwards: a CTA owns 32 channels of one sequence, a lane
// each, and goes over blocks of 64 tokens from the last to the first, 8 tokens a
// warp.  The forward kept the state before each block.  For four states at a time a
// warp computes its tokens' decays once and from them its tokens' effect on the
// state (P h + S) and on what is handed back (P r + R); both meet the other
// warps' in shared memory, and the warp goes over its tokens forwards for h and
// backwards for the gradients.  Sums over channels are butterflies over the
// lanes in which each round halves the values, so that 64 values take 62
// exchanges; the tiles' sums of dB and dC are added by a second launch, in a
// fixed order, as are those over sequences of dA, dskip and dbias.
// Bound by instructions.

#include <algorithm>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {
namespace {

constexpr int kTok = 8;  // tokens of a warp
constexpr int kWarps = kMark / kTok;

// Shared memory in floats.
struct Lay {
  int bs, cs, ex, carry, rate, da, sums, total;
};
__host__ __device__ inline Lay layout(int ng) {
  Lay l;
  int n = 0;
  l.bs = n, n += kMark * ng * 4;
  l.cs = n, n += kMark * ng * 4;
  l.ex = n, n += 2 * kWarps * 3 * kLanes * 4;
  l.carry = n, n += 2 * ng * kLanes * 4;
  l.rate = n, n += ng * kLanes * 4;
  l.da = n, n += kWarps * ng * kLanes * 4;
  l.sums = n, n += 2 * kWarps * kLanes;
  l.total = n;
  return l;
}

// One round of the butterfly: lanes with `bit` keep the upper half of 2 M values
// and hand over the lower, the others the other way around.
template <int M>
__device__ __forceinline__ void halve(float* v, int bit, bool upper) {
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const float send = upper ? v[i] : v[i + M], keep = upper ? v[i + M] : v[i];
    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps, 1) scan_backward_kernel(const Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lay l = layout(p.ng);
  const int tile = blockIdx.x % p.tiles, b = blockIdx.x / p.tiles;
  const int group = tile / p.per_group, local = (tile - group * p.per_group) * kLanes + lane;
  const bool live = local < p.R;
  const int d = group * p.R + (live ? local : 0);
  const int np = p.ng * 4;
  float* bs = sm + l.bs + w * kTok * np;
  float* cs = sm + l.cs + w * kTok * np;
  float4* ex = reinterpret_cast<float4*>(sm + l.ex);
  float4* carry = reinterpret_cast<float4*>(sm + l.carry);
  float4* rate = reinterpret_cast<float4*>(sm + l.rate);
  float4* das = reinterpret_cast<float4*>(sm + l.da) + w * p.ng * kLanes + lane;

  const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
  const int blocks = ceil_div(p.T, kMark);
  for (int g = w; g < p.ng; g += kWarps) {
    float r[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = 4 * g + j;
      r[j] = live && n < p.N ? decay_rate(p.a[(long)d * p.N + n]) : 0.0f;
      s[j] = live && n < p.N && p.dlast ? p.dlast[((long)b * p.D + d) * p.N + n] : 0.0f;
    }
    rate[g * kLanes + lane] = make_float4(r[0], r[1], r[2], r[3]);
    carry[g * kLanes + lane] = make_float4(s[0], s[1], s[2], s[3]);
  }
  for (int g = 0; g < p.ng; ++g) das[g * kLanes] = make_float4(0.f, 0.f, 0.f, 0.f);
  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + d;
  const T* dt = static_cast<const T*>(p.dt) + b * p.dts[0] + d;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.zs[0] + d : nullptr;
  const T* bm = static_cast<const T*>(p.b) + b * p.bs[0] + group * p.bs[2];
  const T* cm = static_cast<const T*>(p.c) + b * p.cs[0] + group * p.cs[2];
  const long dense = (long)b * p.T * p.D + d;
  const T* dout = p.dout ? static_cast<const T*>(p.dout) + dense : nullptr;
  float dskip = 0.0f, dbias = 0.0f;
  __syncthreads();

  int turn = 0;
  for (int i = blocks - 1; i >= 0; --i) {
    const int t0 = i * kMark + w * kTok, here = min(max(p.T - t0, 0), kTok);
    float step[kTok], xv[kTok], gy[kTok], sdt = 0.0f;
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      const bool in = live && t < here;
      xv[t] = in ? to_f32(x[(t0 + t) * p.xs[1]]) : 0.0f;
      step[t] = in ? to_f32(dt[(t0 + t) * p.dts[1]]) : 0.0f;
      gy[t] = in && dout ? to_f32(dout[(long)(t0 + t) * p.D]) : 0.0f;
    }
    if (z)
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        const float v = live && t < here ? to_f32(z[(t0 + t) * p.zs[1]]) : 0.0f;
        gy[t] *= v * sigmoid_of(v);
      }
    for (int k = lane; k < kTok * np; k += 32) {
      const int t = k / np, n = k - t * np;
      const bool in = t < here && n < p.N;
      bs[k] = in ? to_f32(bm[(t0 + t) * p.bs[1] + n]) : 0.0f;
      cs[k] = in ? to_f32(cm[(t0 + t) * p.cs[1] + n]) : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      step[t] = live && t < here ? step_of(p, step[t], bias) : 0.0f;
      sdt += step[t];
    }
    float y[kTok], sb[kTok], sa[kTok];
#pragma unroll
    for (int t = 0; t < kTok; ++t) y[t] = sb[t] = sa[t] = 0.0f;
    __syncwarp();
    for (int g = 0; g < p.ng; ++g, turn ^= 1) {
      const float4 rt4 = rate[g * kLanes + lane];
      const float rt[4] = {rt4.x, rt4.y, rt4.z, rt4.w};
      float a[kTok][4], s[4], r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = r[j] = 0.0f;
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        const float4 b4 = *reinterpret_cast<const float4*>(bs + t * np + 4 * g);
        const float bv[4] = {b4.x, b4.y, b4.z, b4.w}, du = step[t] * xv[t];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[t][j] = exp2_of(step[t] * rt[j]);
          s[j] = fmaf(a[t][j], s[j], du * bv[j]);
        }
      }
#pragma unroll
      for (int t = kTok - 1; t >= 0; --t) {
        const float4 c4 = *reinterpret_cast<const float4*>(cs + t * np + 4 * g);
        const float cv[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = a[t][j] * fmaf(cv[j], gy[t], r[j]);
      }
      float4* e = ex + turn * kWarps * 3 * kLanes;
      e[(w * 3 + 0) * kLanes + lane] =
          make_float4(exp2_of(sdt * rt[0]), exp2_of(sdt * rt[1]), exp2_of(sdt * rt[2]), exp2_of(sdt * rt[3]));
      e[(w * 3 + 1) * kLanes + lane] = make_float4(s[0], s[1], s[2], s[3]);
      e[(w * 3 + 2) * kLanes + lane] = make_float4(r[0], r[1], r[2], r[3]);
      float4 h4 = reinterpret_cast<const float4*>(
          p.marks)[((((long)b * p.tiles + tile) * p.nmarks + i) * p.ng + g) * kLanes + lane];
      __syncthreads();
      float4 r4 = carry[(((blocks - 1 - i) & 1) * p.ng + g) * kLanes + lane];
      for (int k = 0; k < w; ++k) {
        const float4 q = e[(k * 3 + 0) * kLanes + lane], v = e[(k * 3 + 1) * kLanes + lane];
        h4.x = fmaf(q.x, h4.x, v.x), h4.y = fmaf(q.y, h4.y, v.y), h4.z = fmaf(q.z, h4.z, v.z), h4.w = fmaf(q.w, h4.w, v.w);
      }
      for (int k = kWarps - 1; k > w; --k) {
        const float4 q = e[(k * 3 + 0) * kLanes + lane], v = e[(k * 3 + 2) * kLanes + lane];
        r4.x = fmaf(q.x, r4.x, v.x), r4.y = fmaf(q.y, r4.y, v.y), r4.z = fmaf(q.z, r4.z, v.z), r4.w = fmaf(q.w, r4.w, v.w);
      }
      const float h0[4] = {h4.x, h4.y, h4.z, h4.w};
      float h[kTok][4];
      r[0] = r4.x, r[1] = r4.y, r[2] = r4.z, r[3] = r4.w;
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        const float4 b4 = *reinterpret_cast<const float4*>(bs + t * np + 4 * g);
        const float bv[4] = {b4.x, b4.y, b4.z, b4.w}, du = step[t] * xv[t];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[t][j] = fmaf(a[t][j], t ? h[t - 1][j] : h0[j], du * bv[j]);
      }
      float4 da = das[g * kLanes];
      float da4[4] = {da.x, da.y, da.z, da.w};
      float sums[kTok];
#pragma unroll
      for (int t = kTok - 1; t >= 0; --t) {
        const float4 b4 = *reinterpret_cast<const float4*>(bs + t * np + 4 * g);
        const float4 c4 = *reinterpret_cast<const float4*>(cs + t * np + 4 * g);
        const float bv[4] = {b4.x, b4.y, b4.z, b4.w}, cv[4] = {c4.x, c4.y, c4.z, c4.w};
        const float du = step[t] * xv[t];
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float dh = fmaf(cv[j], gy[t], r[j]);
          y[t] = fmaf(cv[j], h[t][j], y[t]);
          sb[t] = fmaf(bv[j], dh, sb[t]);
          v[j] = dh * du;
          v[4 + j] = gy[t] * h[t][j];
          r[j] = a[t][j] * dh;
          const float wt = r[j] * (t ? h[t - 1][j] : h0[j]);
          sa[t] = fmaf(rt[j], wt, sa[t]);
          da4[j] = fmaf(step[t], wt, da4[j]);
        }
        halve<4>(v, 16, lane & 16);
        halve<2>(v, 8, lane & 8);
        halve<1>(v, 4, lane & 4);
        sums[t] = v[0];
      }
      das[g * kLanes] = make_float4(da4[0], da4[1], da4[2], da4[3]);
      // a lane now holds dB (lane < 16) or dC of state (lane >> 2) & 3, for all
      // tokens, over a quarter of the lanes each
      halve<4>(sums, 2, lane & 2);
      halve<2>(sums, 1, lane & 1);
      {
        const int t = (lane & 2 ? 4 : 0) + (lane & 1 ? 2 : 0);
        float* part = p.part_bc + ((((long)b * p.tiles + tile) * p.T + t0 + t) * 2 + (lane >> 4)) * np + 4 * g + ((lane >> 2) & 3);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (t + k < here) part[(long)k * 2 * np] = sums[k];
      }
      if (w == 0) {
        carry[(((blocks - i) & 1) * p.ng + g) * kLanes + lane] = make_float4(r[0], r[1], r[2], r[3]);
        if (i == 0 && live && p.ds0) {
          float* ds0 = p.ds0 + ((long)b * p.D + d) * p.N + 4 * g;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * g + j < p.N) ds0[j] = r[j];
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      if (!live || t >= here) continue;
      const long at = dense + (long)(t0 + t) * p.D;
      const float g = p.skip ? skip * gy[t] : 0.0f;
      static_cast<T*>(p.dx)[at] = from_f32<T>(fmaf(step[t], sb[t], g));
      float raw = fmaf(xv[t], sb[t], sa[t] * 0.6931471805599453f);  // rt is A / ln 2
      if (p.softplus) {
        const float v = to_f32(dt[(t0 + t) * p.dts[1]]) + bias;
        raw *= v > 20.0f ? 1.0f : 1.0f / (1.0f + expf(-v));
      }
      static_cast<T*>(p.ddt)[at] = from_f32<T>(raw);
      dbias += raw;
      dskip = fmaf(gy[t], xv[t], dskip);
      if (z) {
        const float v = to_f32(z[(t0 + t) * p.zs[1]]), s = sigmoid_of(v);
        const float full = p.skip ? fmaf(skip, xv[t], y[t]) : y[t];
        const float go = dout ? to_f32(dout[(long)(t0 + t) * p.D]) : 0.0f;
        static_cast<T*>(p.dz)[at] = from_f32<T>(go * full * s * fmaf(v, 1.0f - s, 1.0f));
      }
    }
    __syncwarp();
  }
  float* sums = sm + l.sums;
  sums[w * kLanes + lane] = dskip;
  sums[(kWarps + w) * kLanes + lane] = dbias;
  __syncthreads();
  if (!live) return;
  if (w < 2) {
    float s = 0.0f;
    for (int k = 0; k < kWarps; ++k) s += sums[(w * kWarps + k) * kLanes + lane];
    p.part_ch[((long)b * 2 + w) * p.D + d] = s;
  }
  const float4* all = reinterpret_cast<const float4*>(sm + l.da) + lane;
  for (int g = w; g < p.ng; g += kWarps) {
    float4 s = all[g * kLanes];
    for (int k = 1; k < kWarps; ++k) {
      const float4 v = all[(k * p.ng + g) * kLanes];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * g + j < p.N) p.part_a[((long)b * p.D + d) * p.N + 4 * g + j] = v[j];
  }
}

// dB and dC: the sums over a group's tiles of 32 channels, in their order.
template <typename T>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const Problem p) {
  const int np = p.ng * 4;
  const long i = blockIdx.x * 256L + threadIdx.x;  // (b, t, group, which, state)
  const long total = (long)p.B * p.T * p.G * 2 * np;
  if (i >= total) return;
  const int n = (int)(i % np);
  long rest = i / np;
  const int which = (int)(rest % 2);
  rest /= 2;
  const int group = (int)(rest % p.G);
  rest /= p.G;
  const long t = rest % p.T, b = rest / p.T;
  if (n >= p.N) return;
  const long row = 2L * np;
  const float* part = p.part_bc + ((b * p.tiles + (long)group * p.per_group) * p.T + t) * row + which * np + n;
  double s = 0.0;
#pragma unroll 4
  for (int k = 0; k < p.per_group; ++k) s += (double)part[k * p.T * row];
  static_cast<T*>(which ? p.dc : p.db)[((b * p.T + t) * p.G + group) * p.N + n] = from_f32<T>((float)s);
}

struct StoreF32 {
  float* out;
  __device__ __forceinline__ void operator()(long c, float x) const { out[c] = x; }
};
struct StoreChannels {
  float *dskip, *dbias;
  int D;
  __device__ __forceinline__ void operator()(long c, float x) const {
    if (c < D) {
      if (dskip) dskip[c] = x;
    } else if (dbias) {
      dbias[c - D] = x;
    }
  }
};

template <typename T>
int launch_backward(const Problem& p, cudaStream_t stream) {
  const size_t smem = layout(p.ng).total * sizeof(float);
  GRU_CUDA_TRY(cudaFuncSetAttribute(scan_backward_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  LaunchScope scope(kKindSelectiveScan, stream, 4);
  scan_backward_kernel<T><<<(unsigned)((long)p.B * p.tiles), 32 * kWarps, smem, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  const long sums = (long)p.B * p.T * p.G * 2 * p.ng * 4;
  sum_tiles_kernel<T><<<(unsigned)((sums + 255) / 256), 256, 0, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  const long an = (long)p.D * p.N;
  if (const int rc = sum_parts(p.part_a, p.B, an, an, StoreF32{p.da}, stream)) return rc;
  return sum_parts(p.part_ch, p.B, 2L * p.D, 2L * p.D, StoreChannels{p.dskip, p.dbias, p.D}, stream);
}

}  // namespace

int backward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? launch_backward<float>(p, stream) : launch_backward<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
