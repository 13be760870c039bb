// Forward of the selective scan over all tokens.
//
//   h[n] = e^{dt A[n]} h[n] + dt x B[n];   y = sum_n C[n] h[n] + skip x;   out = y silu(z)
//
// A CTA owns 32 channels of one sequence, a lane each; every warp has four of the
// states and goes through all tokens with them in registers, so that each decay is
// computed once and nothing is exchanged along the time.  What a token has per
// channel (the step by softplus, dt x, the gate) is worked out by one warp for
// all, four tokens at a time, and passes through shared memory, as do B and C (by
// state: one broadcast read serves four tokens of 32 channels) and the warps'
// shares of y.  Blocks of 16 tokens: the next one's inputs are copied in beside a
// block's scan; between two barriers its outputs are finished and they are prepared.
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

// Shared memory in floats; elem: bytes of an element.
struct Lay {
  int step, du, bs, cs, part, in, few, total;
};
__host__ __device__ inline Lay layout(int warps, int N, int elem) {
  const int np = warps * kStates;
  Lay l;
  int n = 0;
  l.step = n, n += kBlock * kLanes;
  l.du = n, n += kBlock * kLanes;
  l.bs = n, n += np * kRow;
  l.cs = n, n += np * kRow;
  l.part = n, n += warps * kBlock * kLanes;  // [quad][warp][lane] float4
  l.in = n, n += 3 * kBlock * kLanes * elem / 4;
  l.few = n, n += 2 * kBlock * N * elem / 4;
  l.total = n;
  return l;
}

// SUM: only what the segments make of a state.  MOST: threads at most.  W: the
// warps, where they are known (4, for the usual 16 states: addresses are constants
// then, and each warp has one quad of tokens to prepare and finish), or 0.
template <typename T, bool SUM, int MOST, int W>
__global__ void __launch_bounds__(MOST, MOST == 128 ? 6 : 1) scan_forward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int warps = W ? W : blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31, np = warps * kStates;
  const Lay l = layout(warps, p.N, sizeof(T));
  const Place q = place(p);
  if (SUM && q.seg == p.segs - 1) return;
  const T* x = static_cast<const T*>(p.x) + q.b * p.xb + q.d0;
  const T* dt = static_cast<const T*>(p.dt) + q.b * p.dtb + q.d0;
  const T* z = p.z && !SUM ? static_cast<const T*>(p.z) + q.b * p.zb + q.d0 : nullptr;
  const T* bm = static_cast<const T*>(p.b) + q.b * p.bb + q.group * p.bg;
  const T* cm = static_cast<const T*>(p.c) + q.b * p.cb + q.group * p.cg;
  T* out = static_cast<T*>(p.out) + (long)q.b * p.T * p.D + q.d;
  const float bias = p.bias ? p.bias[q.d] : 0.0f, skip = p.skip ? p.skip[q.d] : 0.0f;
  const int lastt = q.end - 1, n0 = kStates * w;
  T* in = reinterpret_cast<T*>(sm + l.in);
  T* few = reinterpret_cast<T*>(sm + l.few);
  constexpr int kTile = kBlock * kLanes;
  auto fetch = [&](int t0) {
    fetch_rows(in, x, p.xst, t0, lastt, q.width, p.wide_rows);
    fetch_rows(in + kTile, dt, p.dtst, t0, lastt, q.width, p.wide_rows);
    if (z) fetch_rows(in + 2 * kTile, z, p.zst, t0, lastt, q.width, p.wide_rows);
    fetch_few(few, bm, p.bst, t0, lastt, p.N, p.wide_few);
    fetch_few(few + kBlock * p.N, cm, p.cst, t0, lastt, p.N, p.wide_few);
  };
  fetch(q.first);

  float rt[kStates], h[kStates];
#pragma unroll
  for (int j = 0; j < kStates; ++j) {
    const bool in = q.live && n0 + j < p.N;
    rt[j] = in ? decay_rate(p.a[(long)q.d * p.N + n0 + j]) : 0.0f;
    h[j] = !SUM && in && p.s0 ? p.s0[((long)q.b * p.D + q.d) * p.N + n0 + j] : 0.0f;
  }
  if (!SUM)
    for (int s = 0; s < q.seg; ++s) {
      const long at = (long)q.unit * p.segs + s;
      const float steps = p.seg_steps[at * kLanes + lane];
#pragma unroll
      for (int j = 0; j < kStates; ++j)
        h[j] = fmaf(exp2_of(rt[j] * steps), h[j], p.seg_sums[(at * p.np + n0 + j) * kLanes + lane]);
    }

  float4* step = reinterpret_cast<float4*>(sm + l.step) + lane;
  float4* du = reinterpret_cast<float4*>(sm + l.du) + lane;
  float4* part = reinterpret_cast<float4*>(sm + l.part) + lane;
  const float* bs = sm + l.bs + n0 * kRow;
  const float* cs = sm + l.cs + n0 * kRow;
  // What finish() needs of the warp's first quad; the inputs are overwritten before.
  float own[4], gate[4];
  auto outer = [&](int u, float (&o)[4], float (&g)[4]) {
    quad_of(in, u, lane, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = p.skip ? o[i] * skip : 0.0f;
    if (z) {
      quad_of(in + 2 * kTile, u, lane, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] *= gate_of(g[i]);
    }
  };
  auto prepare = [&](int t0) {
    for (int u = w; u < kQuads; u += warps) {
      float s[4], v[4];
      quad_of(in + kTile, u, lane, s);
      quad_of(in, u, lane, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = step_of(p.softplus, s[i], bias);
        v[i] *= s[i];
      }
      if (!q.live || t0 + 4 * u + 3 > lastt)  // lanes without a channel keep states of zero
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!q.live || t0 + 4 * u + i > lastt) s[i] = v[i] = 0.0f;
      step[u * kLanes] = as4(s), du[u * kLanes] = as4(v);
      if (!SUM && u == w) outer(u, own, gate);
      if (W) break;
    }
    turn_few(p, few, few + kBlock * p.N, sm + l.bs, sm + l.cs, np, q.end - t0);
  };
  auto finish = [&](int t0) {
    for (int u = w; u < kQuads; u += warps) {
      const int t = t0 + 4 * u;
      float4 sum = part[u * warps * kLanes];
#pragma unroll (W ? W : 4)
      for (int k = 1; k < warps; ++k) sum = add4(sum, part[(u * warps + k) * kLanes]);
      float y[4] = {sum.x, sum.y, sum.z, sum.w}, o[4], g[4];
      if (u == w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = own[i], g[i] = gate[i];
      } else {  // fewer warps than quads: from memory once more
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = min(t + i, lastt);
          o[i] = p.skip ? skip * to_f32(*row_at(x + q.d - q.d0, at, p.xst)) : 0.0f;
          g[i] = z ? to_f32(*row_at(z + q.d - q.d0, at, p.zst)) : 0.0f;
          g[i] *= gate_of(g[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] += o[i];
        if (z) y[i] *= g[i];
      }
      if (q.live) {
        T* to = row_at(out, t, p.ost);
        if (t + 3 <= lastt) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *row_at(to, i, p.ost) = from_f32<T>(y[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t + i <= lastt) *row_at(to, i, p.ost) = from_f32<T>(y[i]);
        }
      }
      if (W) break;
    }
  };

  copies_done();
  __syncthreads();
  prepare(q.first);
  __syncthreads();
  float total = 0.0f;
  float* mark = p.marks + (((long)q.unit * p.nmarks + q.first / kBlock) * p.np + n0) * kLanes + lane;
  for (int t0 = q.first; t0 <= lastt; t0 += kBlock) {
    const bool more = t0 + kBlock <= lastt;
    if (more) fetch(t0 + kBlock);
    if (!SUM && p.marks) {
#pragma unroll
      for (int j = 0; j < kStates; ++j) mark[j * kLanes] = h[j];
      mark += p.np * kLanes;
    }
#pragma unroll
    for (int t = 0; t < kQuads; ++t) {
      const float4 s = step[t * kLanes], u = du[t * kLanes];
      float2 y0 = twice(0.0f), y1 = twice(0.0f);
      if (SUM) total += (s.x + s.y) + (s.z + s.w);
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
        const float2 e0 = __fmul2_rn(lo(s), twice(rt[j])), e1 = __fmul2_rn(hi(s), twice(rt[j]));
        const float2 v0 = __fmul2_rn(lo(u), lo(bv)), v1 = __fmul2_rn(hi(u), hi(bv));
        float2 h0, h1;
        h0.x = fmaf(exp2_of(e0.x), h[j], v0.x);
        h0.y = fmaf(exp2_of(e0.y), h0.x, v0.y);
        h1.x = fmaf(exp2_of(e1.x), h0.y, v1.x);
        h1.y = fmaf(exp2_of(e1.y), h1.x, v1.y);
        h[j] = h1.y;
        if (!SUM) {
          const float4 cv = *reinterpret_cast<const float4*>(cs + j * kRow + 4 * t);
          y0 = __ffma2_rn(lo(cv), h0, y0);
          y1 = __ffma2_rn(hi(cv), h1, y1);
        }
      }
      if (!SUM) part[(t * warps + w) * kLanes] = make_float4(y0.x, y0.y, y1.x, y1.y);
    }
    copies_done();
    __syncthreads();
    if (!SUM) finish(t0);
    if (more) prepare(t0 + kBlock);
    __syncthreads();
  }
  if (SUM) {
    const long at = (long)q.unit * p.segs + q.seg;
#pragma unroll
    for (int j = 0; j < kStates; ++j) p.seg_sums[(at * p.np + n0 + j) * kLanes + lane] = h[j];
    if (w == 0) p.seg_steps[at * kLanes + lane] = total;
  } else if (q.seg == p.segs - 1 && q.live) {
    float* last = p.last + ((long)q.b * p.D + q.d) * p.N + n0;
#pragma unroll
    for (int j = 0; j < kStates; ++j)
      if (n0 + j < p.N) last[j] = h[j];
  }
}

template <typename T, int MOST, int W>
int launch_forward(const Problem& p, cudaStream_t stream) {
  const int warps = p.np / kStates;
  const size_t smem = layout(warps, p.N, sizeof(T)).total * sizeof(float);
  const unsigned ctas = (unsigned)((long)p.B * p.tiles * p.segs);
  LaunchScope scope(kKindSelectiveScan, stream, p.segs > 1 ? 2 : 1);
  if (p.segs > 1) {
    auto kernel = scan_forward_kernel<T, true, MOST, W>;
    GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<ctas, 32 * warps, smem, stream>>>(p);
    GRU_CUDA_TRY(cudaGetLastError());
  }
  auto kernel = scan_forward_kernel<T, false, MOST, W>;
  GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<ctas, 32 * warps, smem, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

template <typename T>
int forward_of(const Problem& p, cudaStream_t stream) {
  if (p.np == 16) return launch_forward<T, 128, 4>(p, stream);
  return p.np < 16 ? launch_forward<T, 128, 0>(p, stream) : launch_forward<T, 512, 0>(p, stream);
}

}  // namespace

int forward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? forward_of<float>(p, stream) : forward_of<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
