// Forward of the selective scan over all tokens.
//
//   h[n] = e^{dt A[n]} h[n] + dt x B[n];   y = sum_n C[n] h[n] + skip x;   out = y silu(z)
//
// A CTA owns 32 channels of one sequence, a lane each, and goes over the time in
// blocks; every warp has 16 tokens of a block.  For four states at a time a warp
// computes its tokens' decays once (kept in registers), and from them what its
// tokens make of a state: h -> P h + S with P = e^{A sum dt}.  The warps' P and S
// meet in shared memory; each warp then has the state before its first token
// from those ahead of it, and goes over its tokens again with that.  B and C are
// broadcast reads of shared memory; the sum over n is the lane's own.
// One exponential per token, channel and state (16 a cycle and SM) is what
// bounds it.

#include <algorithm>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {
namespace {

constexpr int kTok = 16;  // tokens of a warp

// Shared memory in floats.
struct Lay {
  int dts, dus, bs, cs, ex, carry, rate, total;
};
__host__ __device__ inline Lay layout(int warps, int ng) {
  Lay l;
  int n = 0;
  l.dts = n, n += warps * kTok * kLanes;
  l.dus = n, n += warps * kTok * kLanes;
  l.bs = n, n += warps * kTok * ng * 4;
  l.cs = n, n += warps * kTok * ng * 4;
  l.ex = n, n += 2 * warps * 2 * kLanes * 4;
  l.carry = n, n += 2 * ng * kLanes * 4;
  l.rate = n, n += ng * kLanes * 4;
  l.total = n;
  return l;
}

template <typename T>
__global__ void __launch_bounds__(256, 2) scan_forward_kernel(const Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int warps = blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lay l = layout(warps, p.ng);
  const int tile = blockIdx.x % p.tiles, b = blockIdx.x / p.tiles;
  const int group = tile / p.per_group, local = (tile - group * p.per_group) * kLanes + lane;
  const bool live = local < p.R;
  const int d = group * p.R + (live ? local : 0);
  const int np = p.ng * 4;
  float* dts = sm + l.dts + w * kTok * kLanes + lane;
  float* dus = sm + l.dus + w * kTok * kLanes + lane;
  float* bs = sm + l.bs + w * kTok * np;
  float* cs = sm + l.cs + w * kTok * np;
  float4* ex = reinterpret_cast<float4*>(sm + l.ex);
  float4* carry = reinterpret_cast<float4*>(sm + l.carry);
  float4* rate = reinterpret_cast<float4*>(sm + l.rate);

  const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
  for (int g = w; g < p.ng; g += warps) {
    float r[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = 4 * g + j;
      r[j] = live && n < p.N ? decay_rate(p.a[(long)d * p.N + n]) : 0.0f;
      s[j] = live && n < p.N && p.s0 ? p.s0[((long)b * p.D + d) * p.N + n] : 0.0f;
    }
    rate[g * kLanes + lane] = make_float4(r[0], r[1], r[2], r[3]);
    carry[g * kLanes + lane] = make_float4(s[0], s[1], s[2], s[3]);
  }
  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + d;
  const T* dt = static_cast<const T*>(p.dt) + b * p.dts[0] + d;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.zs[0] + d : nullptr;
  const T* bm = static_cast<const T*>(p.b) + b * p.bs[0] + group * p.bs[2];
  const T* cm = static_cast<const T*>(p.c) + b * p.cs[0] + group * p.cs[2];
  T* out = static_cast<T*>(p.out) + (long)b * p.T * p.D + d;
  __syncthreads();

  int turn = 0;
  const int block = warps * kTok, blocks = ceil_div(p.T, block);
  for (int i = 0; i < blocks; ++i) {
    const int t0 = i * block + w * kTok, here = min(max(p.T - t0, 0), kTok);
    float y[kTok], sdt = 0.0f;
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      const bool in = live && t < here;
      y[t] = in ? to_f32(x[(t0 + t) * p.xs[1]]) : 0.0f;
      dts[t * kLanes] = in ? to_f32(dt[(t0 + t) * p.dts[1]]) : 0.0f;
    }
    for (int k = lane; k < kTok * np; k += 32) {
      const int t = k / np, n = k - t * np;
      const bool in = t < here && n < p.N;
      bs[k] = in ? to_f32(bm[(t0 + t) * p.bs[1] + n]) : 0.0f;
      cs[k] = in ? to_f32(cm[(t0 + t) * p.cs[1] + n]) : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      const float step = live && t < here ? step_of(p, dts[t * kLanes], bias) : 0.0f;
      dts[t * kLanes] = step;
      dus[t * kLanes] = step * y[t];
      sdt += step;
      y[t] *= skip;
    }
    if (!p.skip)
#pragma unroll
      for (int t = 0; t < kTok; ++t) y[t] = 0.0f;
    __syncwarp();
    for (int g = 0; g < p.ng; ++g, turn ^= 1) {
      const float4 rt = rate[g * kLanes + lane];
      float a[kTok][4];
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        const float step = dts[t * kLanes], du = dus[t * kLanes];
        const float4 bv = *reinterpret_cast<const float4*>(bs + t * np + 4 * g);
        a[t][0] = exp2_of(step * rt.x), a[t][1] = exp2_of(step * rt.y);
        a[t][2] = exp2_of(step * rt.z), a[t][3] = exp2_of(step * rt.w);
        s.x = fmaf(a[t][0], s.x, du * bv.x), s.y = fmaf(a[t][1], s.y, du * bv.y);
        s.z = fmaf(a[t][2], s.z, du * bv.z), s.w = fmaf(a[t][3], s.w, du * bv.w);
      }
      float4* e = ex + turn * warps * 2 * kLanes;
      e[(w * 2 + 0) * kLanes + lane] =
          make_float4(exp2_of(sdt * rt.x), exp2_of(sdt * rt.y), exp2_of(sdt * rt.z), exp2_of(sdt * rt.w));
      e[(w * 2 + 1) * kLanes + lane] = s;
      __syncthreads();
      float4 h = carry[((i & 1) * p.ng + g) * kLanes + lane];
      for (int k = 0; k < w; ++k) {
        const float4 q = e[(k * 2 + 0) * kLanes + lane], v = e[(k * 2 + 1) * kLanes + lane];
        h.x = fmaf(q.x, h.x, v.x), h.y = fmaf(q.y, h.y, v.y), h.z = fmaf(q.z, h.z, v.z), h.w = fmaf(q.w, h.w, v.w);
      }
      if (p.marks && t0 % kMark == 0 && here > 0)
        reinterpret_cast<float4*>(p.marks)[((((long)b * p.tiles + tile) * p.nmarks + t0 / kMark) * p.ng + g) * kLanes + lane] = h;
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        const float du = dus[t * kLanes];
        const float4 bv = *reinterpret_cast<const float4*>(bs + t * np + 4 * g);
        const float4 cv = *reinterpret_cast<const float4*>(cs + t * np + 4 * g);
        h.x = fmaf(a[t][0], h.x, du * bv.x), h.y = fmaf(a[t][1], h.y, du * bv.y);
        h.z = fmaf(a[t][2], h.z, du * bv.z), h.w = fmaf(a[t][3], h.w, du * bv.w);
        y[t] = fmaf(cv.x, h.x, y[t]), y[t] = fmaf(cv.y, h.y, y[t]);
        y[t] = fmaf(cv.z, h.z, y[t]), y[t] = fmaf(cv.w, h.w, y[t]);
      }
      if (w == warps - 1) {
        carry[(((i + 1) & 1) * p.ng + g) * kLanes + lane] = h;
        if (i == blocks - 1 && live) {
          float* last = p.last + ((long)b * p.D + d) * p.N + 4 * g;
          const float v[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * g + j < p.N) last[j] = v[j];
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      if (!live || t >= here) continue;
      float v = y[t];
      if (z) {
        const float gate = to_f32(z[(t0 + t) * p.zs[1]]);
        v *= gate * sigmoid_of(gate);
      }
      out[(long)(t0 + t) * p.D] = from_f32<T>(v);
    }
    __syncwarp();
  }
}

}  // namespace

template <typename T>
int launch_forward(const Problem& p, cudaStream_t stream) {
  int warps = std::min(8, ceil_div(p.T, kTok));
  const size_t most = 227 * 1024;
  while (warps > 1 && layout(warps, p.ng).total * sizeof(float) > most) warps /= 2;
  const size_t smem = layout(warps, p.ng).total * sizeof(float);
  GRU_CUDA_TRY(cudaFuncSetAttribute(scan_forward_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  LaunchScope scope(kKindSelectiveScan, stream);
  scan_forward_kernel<T><<<(unsigned)((long)p.B * p.tiles), warps * 32, smem, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

int forward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? launch_forward<float>(p, stream) : launch_forward<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
