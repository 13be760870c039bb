// Forward of the selective scan over all tokens.
//
//   h[n] = e^{dt A[n]} h[n] + dt x B[n];   y = sum_n C[n] h[n] + skip x;   out = y silu(z)
//
// A CTA owns 32 channels of one sequence, a lane each; every warp has two (four
// above 32) of the states and goes through all tokens with them in registers, so
// that each decay is computed once and nothing is exchanged along the time.  What
// a token has per channel (the step by softplus, dt x, the gate) is worked out by
// one warp for all, two tokens at a time, and passes through shared memory, as do
// B and C (by state: one broadcast read serves four tokens of 32 channels) and the
// warps' shares of y.  Blocks of 16 tokens, one barrier each: the next block's
// inputs are prepared and the last block's outputs finished beside a block's scan.
// Neighbouring tokens share a packed FP32 operation in all but the recurrence.
//
// Sequences too few to fill the GPU are cut into segments: a first launch finds
// what each makes of a state (h -> e^{A sum dt} h + S), then all segments run side
// by side, each putting the segments ahead of it together first.
// One exponential per token, channel and state (16 a cycle and SM) is the bound.

#include <algorithm>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {
namespace {

// Shared memory in floats.
struct Lay {
  int step, du, bs, cs, part, total;
};
__host__ __device__ inline Lay layout(int warps, int np) {
  Lay l;
  int n = 0;
  l.step = n, n += 2 * kBlock * kLanes;
  l.du = n, n += 2 * kBlock * kLanes;
  l.bs = n, n += 2 * np * kRow;
  l.cs = n, n += 2 * np * kRow;
  l.part = n, n += 2 * warps * kBlock * kLanes;
  l.total = n;
  return l;
}

// SG: states of a warp.  SUM: only what the segments make of a state.  MOST: threads
// at most.  ONE: there are eight warps at least, so that each has one pair of a
// block's tokens to prepare and finish, or none.  W: the warps, where they are known
// (8, for the usual 16 states: their sums' addresses are constants then), or 0.
// K: elements of B and C a thread moves at most.
template <typename T, int SG, bool SUM, int MOST, bool ONE, int W, int K>
__global__ void __launch_bounds__(MOST, MOST == 256 ? 3 : 1) scan_forward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int warps = W ? W : blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lay l = layout(warps, p.np);
  const Place q = place(p);
  if (SUM && q.seg == p.segs - 1) return;
  const T* x = static_cast<const T*>(p.x) + q.b * p.xb + q.d;
  const T* dt = static_cast<const T*>(p.dt) + q.b * p.dtb + q.d;
  const T* z = p.z ? static_cast<const T*>(p.z) + q.b * p.zb + q.d : nullptr;
  const T* bm = static_cast<const T*>(p.b) + q.b * p.bb + q.group * p.bg;
  const T* cm = static_cast<const T*>(p.c) + q.b * p.cb + q.group * p.cg;
  T* out = static_cast<T*>(p.out) + (long)q.b * p.T * p.D + q.d;
  const float bias = p.bias ? p.bias[q.d] : 0.0f, skip = p.skip ? p.skip[q.d] : 0.0f;

  float rt[SG], h[SG];
#pragma unroll
  for (int j = 0; j < SG; ++j) {
    const int n = SG * w + j;
    const bool in = q.live && n < p.N;
    rt[j] = in ? decay_rate(p.a[(long)q.d * p.N + n]) : 0.0f;
    h[j] = !SUM && in && p.s0 ? p.s0[((long)q.b * p.D + q.d) * p.N + n] : 0.0f;
  }
  if (!SUM)
    for (int s = 0; s < q.seg; ++s) {
      const long at = (long)q.unit * p.segs + s;
      const float steps = p.seg_steps[at * kLanes + lane];
#pragma unroll
      for (int j = 0; j < SG; ++j)
        h[j] = fmaf(exp2_of(rt[j] * steps), h[j], p.seg_sums[(at * p.np + SG * w + j) * kLanes + lane]);
    }

  // Of the block after the next: a pair of tokens and some of B and C.  (Where
  // warps are fewer than pairs, the others are loaded when they are needed.)
  const int lastt = q.end - 1;
  const bool first_pair = !ONE || w < kBlock / 2;
  Pair<T> nx, nd, nz;
  Few<T, K> few;
  few.init(p, bm, cm);
  auto prefetch = [&](int t0) {
    if (first_pair) {
      const int t = t0 + 2 * w;
      nx.load(x, p.xst, t, lastt);
      nd.load(dt, p.dtst, t, lastt);
      if (!SUM && z) nz.load(z, p.zst, t, lastt);
    }
    few.load(p, t0, lastt);
  };
  Pair<T> cx, cz, ox, oz;  // of the next block, and of the one that is finished
  auto prepare_pair = [&](const Pair<T>& px, const Pair<T>& pd, int t, int at, int buf) {
    const float s0 = t <= lastt ? step_of(p.softplus, to_f32(pd.x), bias) : 0.0f;
    const float s1 = t < lastt ? step_of(p.softplus, to_f32(pd.y), bias) : 0.0f;
    const float u0 = t <= lastt ? s0 * to_f32(px.x) : 0.0f, u1 = t < lastt ? s1 * to_f32(px.y) : 0.0f;
    pair_in(sm + l.step + buf * kBlock * kLanes, at) = make_float2(s0, s1);
    pair_in(sm + l.du + buf * kBlock * kLanes, at) = make_float2(u0, u1);
  };
  auto prepare = [&](int t0, int buf) {
    if (first_pair) prepare_pair(nx, nd, t0 + 2 * w, pair_at(2 * w, lane), buf);
    if (!ONE)
      for (int u = w + warps; u < kBlock / 2; u += warps) {
        Pair<T> px, pd;
        px.load(x, p.xst, t0 + 2 * u, lastt), pd.load(dt, p.dtst, t0 + 2 * u, lastt);
        prepare_pair(px, pd, t0 + 2 * u, pair_at(2 * u, lane), buf);
      }
    few.store(sm + l.bs + buf * p.np * kRow, sm + l.cs + buf * p.np * kRow, t0, lastt);
    ox = cx, oz = cz, cx = nx, cz = nz;
  };
  // part: [quad][warp][lane]
  auto finish_pair = [&](const Pair<T>& px, const Pair<T>& pz, int u, int t, int buf) {
    const float* part = sm + l.part + buf * warps * kBlock * kLanes + ((u >> 1) * warps * kLanes + lane) * 4 + 2 * (u & 1);
    float2 y = twice(0.0f);
    if (p.skip) y = make_float2(skip * to_f32(px.x), skip * to_f32(px.y));
#pragma unroll (W ? W : 4)
    for (int k = 0; k < warps; ++k) y = __fadd2_rn(y, *reinterpret_cast<const float2*>(part + k * 4 * kLanes));
    if (z) {
      const float z0 = to_f32(pz.x), z1 = to_f32(pz.y);
      y.x *= z0 * gate_of(z0), y.y *= z1 * gate_of(z1);
    }
    if (q.live) {
      T* to = row_at(out, t, p.ost);
      to[0] = from_f32<T>(y.x);
      if (t < lastt) to[p.D] = from_f32<T>(y.y);
    }
  };
  auto finish = [&](int t0, int buf) {
    if (first_pair && t0 + 2 * w <= lastt) finish_pair(ox, oz, w, t0 + 2 * w, buf);
    if (!ONE)
      for (int u = w + warps; u < kBlock / 2 && t0 + 2 * u <= lastt; u += warps) {
        Pair<T> px, pz;
        px.load(x, p.xst, t0 + 2 * u, lastt);
        if (z) pz.load(z, p.zst, t0 + 2 * u, lastt);
        finish_pair(px, pz, u, t0 + 2 * u, buf);
      }
  };

  prefetch(q.first);
  prepare(q.first, 0);
  prefetch(q.first + kBlock);
  __syncthreads();
  float total = 0.0f;
  float* mark = p.marks + (((long)q.unit * p.nmarks + q.first / kBlock) * p.np + SG * w) * kLanes + lane;
  int buf = 0;
  for (int t0 = q.first; t0 < q.end; t0 += kBlock, buf ^= 1) {
    if (t0 + kBlock < q.end) {
      prepare(t0 + kBlock, buf ^ 1);
      prefetch(t0 + 2 * kBlock);
    } else {
      ox = cx, oz = cz;
    }
    if (!SUM && p.marks) {
#pragma unroll
      for (int j = 0; j < SG; ++j)
        if (SG * w + j < p.N) mark[j * kLanes] = h[j];
      mark += p.np * kLanes;
    }
    const float4* step = reinterpret_cast<const float4*>(sm + l.step + buf * kBlock * kLanes) + lane;
    const float4* du = reinterpret_cast<const float4*>(sm + l.du + buf * kBlock * kLanes) + lane;
    const float* bs = sm + l.bs + (buf * p.np + SG * w) * kRow;
    const float* cs = sm + l.cs + (buf * p.np + SG * w) * kRow;
    float4* part = reinterpret_cast<float4*>(sm + l.part + buf * warps * kBlock * kLanes) + w * kLanes + lane;
#pragma unroll
    for (int t = 0; t < kBlock / 4; ++t) {
      const float4 s = step[t * kLanes], u = du[t * kLanes];
      float2 y0 = twice(0.0f), y1 = twice(0.0f);
      if (SUM) total += (s.x + s.y) + (s.z + s.w);
#pragma unroll
      for (int j = 0; j < SG; ++j) {
        const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
        const float2 e0 = __fmul2_rn(make_float2(s.x, s.y), twice(rt[j])), e1 = __fmul2_rn(make_float2(s.z, s.w), twice(rt[j]));
        const float2 v0 = __fmul2_rn(make_float2(u.x, u.y), make_float2(bv.x, bv.y));
        const float2 v1 = __fmul2_rn(make_float2(u.z, u.w), make_float2(bv.z, bv.w));
        float2 h0, h1;
        h0.x = fmaf(exp2_of(e0.x), h[j], v0.x);
        h0.y = fmaf(exp2_of(e0.y), h0.x, v0.y);
        h1.x = fmaf(exp2_of(e1.x), h0.y, v1.x);
        h1.y = fmaf(exp2_of(e1.y), h1.x, v1.y);
        h[j] = h1.y;
        if (!SUM) {
          const float4 cv = *reinterpret_cast<const float4*>(cs + j * kRow + 4 * t);
          y0 = __ffma2_rn(make_float2(cv.x, cv.y), h0, y0);
          y1 = __ffma2_rn(make_float2(cv.z, cv.w), h1, y1);
        }
      }
      if (!SUM) part[t * warps * kLanes] = make_float4(y0.x, y0.y, y1.x, y1.y);
    }
    __syncthreads();
    if (!SUM) finish(t0, buf);
  }
  if (SUM) {
    const long at = (long)q.unit * p.segs + q.seg;
#pragma unroll
    for (int j = 0; j < SG; ++j)
      if (SG * w + j < p.np) p.seg_sums[(at * p.np + SG * w + j) * kLanes + lane] = h[j];
    if (w == 0) p.seg_steps[at * kLanes + lane] = total;
  } else if (q.seg == p.segs - 1 && q.live) {
    float* last = p.last + ((long)q.b * p.D + q.d) * p.N + SG * w;
#pragma unroll
    for (int j = 0; j < SG; ++j)
      if (SG * w + j < p.N) last[j] = h[j];
  }
}

template <typename T, int SG, int MOST, bool ONE, int W, int K>
int launch_forward(const Problem& p, cudaStream_t stream) {
  const int warps = (p.N + SG - 1) / SG;
  const size_t smem = layout(warps, p.np).total * sizeof(float);
  const unsigned ctas = (unsigned)((long)p.B * p.tiles * p.segs);
  LaunchScope scope(kKindSelectiveScan, stream, p.segs > 1 ? 2 : 1);
  if (p.segs > 1) {
    GRU_CUDA_TRY(cudaFuncSetAttribute(scan_forward_kernel<T, SG, true, MOST, ONE, W, K>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    scan_forward_kernel<T, SG, true, MOST, ONE, W, K><<<ctas, 32 * warps, smem, stream>>>(p);
    GRU_CUDA_TRY(cudaGetLastError());
  }
  GRU_CUDA_TRY(cudaFuncSetAttribute(scan_forward_kernel<T, SG, false, MOST, ONE, W, K>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  scan_forward_kernel<T, SG, false, MOST, ONE, W, K><<<ctas, 32 * warps, smem, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

template <typename T>
int forward_of(const Problem& p, cudaStream_t stream) {
  if (p.N <= 14) return launch_forward<T, 2, 256, false, 0, 2>(p, stream);
  if (p.N <= 16) return launch_forward<T, 2, 256, true, 8, 1>(p, stream);
  return p.N <= 32 ? launch_forward<T, 2, 512, true, 0, 2>(p, stream) : launch_forward<T, 4, 512, true, 0, 4>(p, stream);
}

}  // namespace

int forward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? forward_of<float>(p, stream) : forward_of<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
