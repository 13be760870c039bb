// Forward of the selective scan over all tokens.
//
//   h[n] = e^{dt A[n]} h[n] + dt x B[n];   y = sum_n C[n] h[n] + skip x;   out = y silu(z)
//
// A CTA owns 64 channels of one sequence, two neighbours a lane, which share every
// packed FP32 operation; every warp has four (two, below 12) of the states and goes
// through all tokens with them in registers, so that each decay is computed once
// and nothing is exchanged along the time.  What a token has per channel (the step
// by softplus, dt x, the gate) is worked out by one warp for all, two tokens at a
// time, and passes through shared memory, as do B and C (each number twice: one
// broadcast read serves two tokens of 64 channels) and the warps' shares of y.
// Blocks of 16 tokens: the next one's inputs are copied in beside a block's scan;
// between two barriers its outputs are finished and they are prepared.
//
// The hardware's exponential is off by up to 2^-22, to one side for neighbouring
// arguments, and a state that remembers a thousand tokens would gather that a
// thousand times (3e-6 of it).  So a block's start is carried over the block by
// e^{A sum dt} and not by the product of its decays: the difference of the two, of
// the start, is put in at the block's end (4e-7).
//
// Sequences too few to fill the GPU are cut into segments: a first launch finds
// what each makes of a state (h -> e^{A sum dt} h + S), then all segments run side
// by side, each putting the segments ahead of it together first.
//
// The floor is one exponential per token, channel and state (16 a cycle and SM).  64
// sequences of 512 tokens, 512 channels, 16 states, FP32: 173 us, of which the
// exponentials would take 58 and memory 41.  No unit is full (issue slots 52 %,
// exponentials 46 %, shared memory 54 %): the latencies of a token's chain, with 12.7
// warps an SM on average (registers allow 16; the 512 CTAs are 13.8).  16384 tokens of 2048 channels in 32 segments,
// bf16: 195 us the first pass (exponentials 71 % busy), 283 the second.  Left out in
// turn, exponentials, copies, preparation and B and C took 20 to 30 us each of 185,
// finish() and the blocks' carrying 12 to 14.

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
__host__ __device__ inline Lay layout(int warps, int np, int N, int elem) {
  Lay l;
  int n = 0;
  l.step = n, n += kBlock * kTile;
  l.du = n, n += kBlock * kTile;
  l.bs = n, n += np * kRow;
  l.cs = n, n += np * kRow;
  l.part = n, n += warps * kBlock * kTile;  // [pair of tokens][warp][lane] float4
  l.in = n, n += 3 * kBlock * kTile * elem / 4;
  l.few = n, n += 2 * kBlock * N * elem / 4;
  l.total = n;
  return l;
}

// SG: states of a warp.  SUM: only what the segments make of a state.  PADS: some of
// them are not there (an infinite dt x times their B of 0 makes NaN of them, and in
// the gradient an infinite gradient of y times their C: that is kept out of the sums over
// states, which took 2 % where all are there and were asked for).  MOST: threads
// at most.  OCC: CTAs of an SM.  W: the warps, where they are known (addresses are
// constants then, and what finish() needs stays in registers), or 0.
template <typename T, int SG, bool SUM, bool PADS, int MOST, int OCC, int W>
__global__ void __launch_bounds__(MOST, OCC) scan_forward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int threads = W ? 32 * W : blockDim.x, warps = W ? W : threads >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lay l = layout(warps, p.np, p.N, sizeof(T));
  const Place q = place(p, SUM ? p.segs - 1 : p.segs, 0);
  const T* x = static_cast<const T*>(p.x) + q.b * p.xb + q.d0;
  const T* dt = static_cast<const T*>(p.dt) + q.b * p.dtb + q.d0;
  const T* z = p.z && !SUM ? static_cast<const T*>(p.z) + q.b * p.zb + q.d0 : nullptr;
  const T* bm = static_cast<const T*>(p.b) + q.b * p.bb + q.group * p.bg;
  const T* cm = static_cast<const T*>(p.c) + q.b * p.cb + q.group * p.cg;
  T* out = static_cast<T*>(p.out) + (long)q.b * p.T * p.D + q.d;
  const float2 bias = two_of(p.bias, q), skip = two_of(p.skip, q);
  const int lastt = q.end - 1, n0 = SG * w;
  T* in = reinterpret_cast<T*>(sm + l.in);
  T* few = reinterpret_cast<T*>(sm + l.few);
  constexpr int kRows = kBlock * kTile;
  Feed<T> feed;
  feed.init(p, bm, cm);
  auto fetch = [&](int t0) {
    feed.row(in, x, p.xst, t0, lastt, q.width, p.row_piece);
    feed.row(in + kRows, dt, p.dtst, t0, lastt, q.width, p.row_piece);
    if (z) feed.row(in + 2 * kRows, z, p.zst, t0, lastt, q.width, p.row_piece);
    feed.bc(p, few, bm, cm, t0, lastt);
  };
  fetch(q.first);

  float2 rt[SG], h[SG];
#pragma unroll
  for (int j = 0; j < SG; ++j) {
    const float2 a = two_of(p.a, q, n0 + j, p.N);
    rt[j] = make_float2(decay_rate(a.x), decay_rate(a.y));
    h[j] = SUM ? twice(0.0f) : two_of(p.s0 ? p.s0 + (long)q.b * p.D * p.N : nullptr, q, n0 + j, p.N);
  }
  if (!SUM)
#pragma unroll 4
    for (int s = 0; s < q.seg; ++s) {
      const long at = (long)q.unit * p.segs + s;
      const float2 steps = both(p.seg_steps + at * kTile, 0, lane);
#pragma unroll
      for (int j = 0; j < SG; ++j)
        h[j] = behind_segment(h[j], passed(rt[j], steps), both(p.seg_sums + (at * p.np + n0 + j) * kTile, 0, lane));
    }

  float4* step = reinterpret_cast<float4*>(sm + l.step) + lane;  // [pair of tokens][lane]
  float4* du = reinterpret_cast<float4*>(sm + l.du) + lane;
  float4* part = reinterpret_cast<float4*>(sm + l.part) + lane;
  const float* bs = sm + l.bs + n0 * kRow;
  const float* cs = sm + l.cs + n0 * kRow;
  // What finish() needs of the warp's first pairs; the inputs are overwritten before.
  constexpr int kOwn = W ? (kPairs + W - 1) / W : 1;
  float own[kOwn][4], gate[kOwn][4];
  auto prepare = [&](int t0) {
#pragma unroll
    for (int k = 0; k < (W ? kOwn : kPairs); ++k) {
      const int u = w + k * warps;
      if (u >= kPairs) break;
      float s[4], v[4];
      four(in + kRows, u, lane, s);
      four(in, u, lane, v);
      if (!SUM && k < kOwn) {
        constexpr int kLast = kOwn - 1;
        float(&o)[4] = own[k < kOwn ? k : kLast];
        float(&g)[4] = gate[k < kOwn ? k : kLast];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = p.skip ? (i & 1 ? skip.y : skip.x) * v[i] : 0.0f;
        if (z) {
          four(in + 2 * kRows, u, lane, g);
#pragma unroll
          for (int i = 0; i < 4; ++i) g[i] *= sigmoid_of(g[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = step_of(p.softplus, s[i], i & 1 ? bias.y : bias.x);
        v[i] *= s[i];
      }
      // tokens that are not there, and lanes without a channel, whose states stay zero
      if (!q.second || t0 + 2 * u + 1 > lastt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(i & 1 ? q.second : q.live) || t0 + 2 * u + i / 2 > lastt) s[i] = v[i] = 0.0f;
      step[u * kLanes] = as4(s), du[u * kLanes] = as4(v);
    }
    turn_few(p, few, sm + l.bs, sm + l.cs, p.np, q.end - t0);
  };
  auto finish = [&](int t0) {
#pragma unroll
    for (int k = 0; k < (W ? kOwn : kPairs); ++k) {
      const int u = w + k * warps, t = t0 + 2 * u;
      if (u >= kPairs || t > lastt) break;
      float4 sum = part[u * warps * kLanes];
#pragma unroll (W ? W : 4)
      for (int i = 1; i < warps; ++i) sum = add4(sum, part[(u * warps + i) * kLanes]);
      float y[4] = {sum.x, sum.y, sum.z, sum.w}, g[4];
      if (k < kOwn) {
        constexpr int kLast = kOwn - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] += own[k < kOwn ? k : kLast][i], g[i] = gate[k < kOwn ? k : kLast][i];
      } else if (q.live) {  // fewer warps than pairs: from memory once more
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = min(t + i / 2, lastt), c = q.d - q.d0 + (i & 1 ? q.second : 0);
          if (p.skip) y[i] = fmaf(i & 1 ? skip.y : skip.x, to_f32(*row_at(x + c, at, p.xst)), y[i]);
          if (z) {
            g[i] = to_f32(*row_at(z + c, at, p.zst));
            g[i] *= sigmoid_of(g[i]);
          }
        }
      }
      if (p.sums) {
        float* kept = p.sums + ((long)q.b * p.T + t) * p.D + q.d;
        put_both(kept, y[0], y[1], q, p.even_sums);
        if (t < lastt) put_both(kept + p.D, y[2], y[3], q, p.even_sums);
      }
      if (z)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] *= g[i];
      T* to = row_at(out, t, p.ost);
      put_both(to, y[0], y[1], q, p.even_out);
      if (t < lastt) put_both(to + p.D, y[2], y[3], q, p.even_out);
    }
  };

  copies_done();
  __syncthreads();
  prepare(q.first);
  __syncthreads();
  float2 total = twice(0.0f);
  float* mark = p.marks + (((long)q.unit * p.nmarks + q.first / kBlock) * p.np + n0) * kTile + 2 * lane;
  for (int t0 = q.first; t0 <= lastt; t0 += kBlock) {
    const bool more = t0 + kBlock <= lastt;
    if (more) fetch(t0 + kBlock);
    if (!SUM && p.marks) {
#pragma unroll
      for (int j = 0; j < SG; ++j) *reinterpret_cast<float2*>(mark + j * kTile) = h[j];
      mark += p.np * kTile;
    }
    float2 before[SG], all[SG], steps = twice(0.0f);  // the start, the product of decays, the sum of steps
#pragma unroll
    for (int j = 0; j < SG; ++j) before[j] = h[j], all[j] = twice(1.0f);
#pragma unroll
    for (int t = 0; t < kPairs; ++t) {
      const float4 s = step[t * kLanes], u = du[t * kLanes];
      float2 y0 = twice(0.0f), y1 = twice(0.0f);
      steps = __fadd2_rn(steps, __fadd2_rn(lo(s), hi(s)));
#pragma unroll
      for (int j = 0; j < SG; ++j) {
        const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
        const float2 a0 = exp2_of(__fmul2_rn(lo(s), rt[j])), a1 = exp2_of(__fmul2_rn(hi(s), rt[j]));
        const float2 h0 = __ffma2_rn(a0, h[j], __fmul2_rn(lo(u), lo(bv)));
        const float2 h1 = __ffma2_rn(a1, h0, __fmul2_rn(hi(u), hi(bv)));
        h[j] = h1;
        all[j] = __fmul2_rn(all[j], __fmul2_rn(a0, a1));
        if (!SUM && (!PADS || n0 + j < p.N)) {
          const float4 cv = *reinterpret_cast<const float4*>(cs + j * kRow + 4 * t);
          y0 = __ffma2_rn(lo(cv), h0, y0);
          y1 = __ffma2_rn(hi(cv), h1, y1);
        }
      }
      if (!SUM) part[(t * warps + w) * kLanes] = as4(y0, y1);
    }
#pragma unroll
    for (int j = 0; j < SG; ++j) h[j] = carried(h[j], before[j], passed(rt[j], steps), all[j]);
    if (SUM) total = __fadd2_rn(total, steps);
    copies_done();
    __syncthreads();
    if (!SUM) finish(t0);
    if (more) prepare(t0 + kBlock);
    __syncthreads();
  }
  if (SUM) {
    const long at = (long)q.unit * p.segs + q.seg;
#pragma unroll
    for (int j = 0; j < SG; ++j)
      *reinterpret_cast<float2*>(p.seg_sums + (at * p.np + n0 + j) * kTile + 2 * lane) = h[j];
    if (w == 0) *reinterpret_cast<float2*>(p.seg_steps + at * kTile + 2 * lane) = total;
  } else if (q.seg == p.segs - 1) {
#pragma unroll
    for (int j = 0; j < SG; ++j) put_two(p.last + (long)q.b * p.D * p.N, q, n0 + j, p.N, h[j]);
  }
}

template <typename T, int SG, int MOST, int OCC, int W>
int launch_forward(const Problem& p, cudaStream_t stream) {
  const int warps = p.np / SG;
  const size_t smem = layout(warps, p.np, p.N, sizeof(T)).total * sizeof(float);
  const long units = (long)p.B * p.tiles;
  LaunchScope scope(kKindSelectiveScan, stream, p.segs > 1 ? 2 : 1);
  if (p.segs > 1) {
    auto kernel = scan_forward_kernel<T, SG, true, false, MOST, OCC, W>;
    GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<(unsigned)(units * (p.segs - 1)), 32 * warps, smem, stream>>>(p);
    GRU_CUDA_TRY(cudaGetLastError());
  }
  auto kernel = p.N == p.np ? scan_forward_kernel<T, SG, false, false, MOST, OCC, W> : scan_forward_kernel<T, SG, false, true, MOST, OCC, W>;
  GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<(unsigned)(units * p.segs), 32 * warps, smem, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

// States of a warp: four, which share a token's loads and its share of y; two below 12
// states, for threads to copy and prepare with.  (64 sequences of 512 tokens, 512
// channels, four and two states a warp: 8 states 156 and 115 us, 12 states 162 and
// 205, 16 states 187 and 210, 32 states 337 and 390.)  As many CTAs an SM as leave a
// thread some 110 to 128 registers, of which 8 to 44 bytes are spilled: 80 for one or two
// CTAs more took 199 us instead of 172 at 16 states, 358 instead of 299 at 32.  (17 to 28
// states have three CTAs and 80 registers all the same, and spill 124 bytes; two were not
// measured there.)  Known warps where the states are usual
// (8 states 135 us with any number of warps, 115 with four).
template <typename T>
int forward_of(const Problem& p, cudaStream_t stream) {
  if (p.np == 4) return launch_forward<T, 2, 64, 7, 2>(p, stream);
  if (p.np == 8) return launch_forward<T, 2, 128, 4, 4>(p, stream);
  if (p.np == 12) return launch_forward<T, 4, 96, 5, 3>(p, stream);
  if (p.np == 16) return launch_forward<T, 4, 128, 4, 4>(p, stream);
  if (p.np < 32) return launch_forward<T, 4, 224, 3, 0>(p, stream);
  if (p.np == 32) return launch_forward<T, 4, 256, 2, 8>(p, stream);
  if (p.np == 64) return launch_forward<T, 4, 512, 1, 16>(p, stream);
  return launch_forward<T, 4, 512, 1, 0>(p, stream);
}

}  // namespace

// Warps of a CTA, and CTAs of an SM, as above.
Fit forward_fit(int np) {
  return {np < 12 ? np / 2 : np / 4, np == 4 ? 7 : np == 8 ? 4 : np == 12 ? 5 : np == 16 ? 4 : np < 32 ? 3 : np == 32 ? 2 : 1};
}

int forward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? forward_of<float>(p, stream) : forward_of<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
