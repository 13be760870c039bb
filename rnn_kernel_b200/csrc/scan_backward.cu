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
// each, a warp two states at a time (twice two above 32 states), and goes over
// blocks of 16 tokens from the last to the first.  The forward kept the state
// before each block; from it a warp computes its states at the block's tokens,
// with the decays, in registers, and then goes over the tokens backwards.  The
// warps' shares of y, sum_n B dh and sum_n A w meet in shared memory, where two
// tokens a warp are finished.  Sums over channels are butterflies over the lanes in
// which each round halves the values: 64 values (16 tokens, 2 states, dB and dC)
// take 62 exchanges and leave a lane two sums.  The tiles' sums of dB and dC are
// added by a second launch, in a fixed order, as are those over sequences of dA,
// dskip and dbias.  Segments as in the forward.  Bound by instructions: some 26
// per token, channel and state, of them 8 for the sums over channels.

#include <algorithm>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {

namespace {

// Shared memory in floats.
struct Lay {
  int step, du, gy, bs, cs, part, sums, total;
};
__host__ __device__ inline Lay layout(int warps, int np) {
  Lay l;
  int n = 0;
  l.step = n, n += kBlock * kLanes;
  l.du = n, n += kBlock * kLanes;
  l.gy = n, n += kBlock * kLanes;
  l.bs = n, n += np * kRow;
  l.cs = n, n += np * kRow;
  l.part = n, n += warps * 3 * kBlock * kLanes;  // y, sum B dh, sum A w
  l.sums = n, n += 2 * warps * kLanes;
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

// GW: pairs of states of a warp.  SUM: only what the segments hand back.  MOST, ONE,
// W and K as in the forward.
template <typename T, int GW, bool SUM, int MOST, bool ONE, int W, int K>
__global__ void __launch_bounds__(MOST, MOST == 256 ? 2 : 1) scan_backward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int warps = W ? W : blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lay l = layout(warps, p.np);
  const Place q = place(p);
  if (SUM && q.seg == 0) return;
  const T* x = static_cast<const T*>(p.x) + q.b * p.xb + q.d;
  const T* dt = static_cast<const T*>(p.dt) + q.b * p.dtb + q.d;
  const T* z = p.z ? static_cast<const T*>(p.z) + q.b * p.zb + q.d : nullptr;
  const T* bm = static_cast<const T*>(p.b) + q.b * p.bb + q.group * p.bg;
  const T* cm = static_cast<const T*>(p.c) + q.b * p.cb + q.group * p.cg;
  const long dense = (long)q.b * p.T * p.D + q.d;
  const T* dout = p.dout ? static_cast<const T*>(p.dout) + dense : nullptr;
  const float bias = p.bias ? p.bias[q.d] : 0.0f, skip = p.skip ? p.skip[q.d] : 0.0f;

  // states 2 (g warps + w) and the next
  float rt[GW][2], back[GW][2];
  float2 da[GW][2];
#pragma unroll
  for (int g = 0; g < GW; ++g)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = 2 * (g * warps + w) + j;
      const bool in = q.live && n < p.N;
      rt[g][j] = in ? decay_rate(p.a[(long)q.d * p.N + n]) : 0.0f;
      back[g][j] = !SUM && in && p.dlast ? p.dlast[((long)q.b * p.D + q.d) * p.N + n] : 0.0f;
      da[g][j] = twice(0.0f);
    }
  if (!SUM)
    for (int s = p.segs - 1; s > q.seg; --s) {
      const long at = (long)q.unit * p.segs + s;
      const float steps = p.seg_steps[at * kLanes + lane];
#pragma unroll
      for (int g = 0; g < GW; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int n = 2 * (g * warps + w) + j;
          if (n < p.np)
            back[g][j] = fmaf(exp2_of(rt[g][j] * steps), back[g][j], p.seg_sums[(at * p.np + n) * kLanes + lane]);
        }
    }

  Pair<T> nx, nd, nz, ng;  // a pair of the next block's tokens; of this one's below
  Pair<T> cx, cd, cz, cg;
  Few<T, K> few;
  few.init(p, bm, cm);
  const int lastt = q.end - 1;
  auto load = [&](int t, Pair<T>& px, Pair<T>& pd, Pair<T>& pz, Pair<T>& pg) {
    px.load(x, p.xst, t, lastt);
    pd.load(dt, p.dtst, t, lastt);
    if (z) pz.load(z, p.zst, t, lastt);
    if (dout) pg.load(dout, p.ost, t, lastt);
  };
  const bool first_pair = !ONE || w < kBlock / 2;
  auto prefetch = [&](int t0) {
    if (first_pair) load(t0 + 2 * w, nx, nd, nz, ng);
    few.load(p, t0, lastt);
  };
  auto prepare_pair = [&](const Pair<T>& px, const Pair<T>& pd, const Pair<T>& pz, const Pair<T>& pg, int t, int at) {
    const bool a = q.live && t <= lastt, b = q.live && t < lastt;
    const float s0 = a ? step_of(p.softplus, to_f32(pd.x), bias) : 0.0f;
    const float s1 = b ? step_of(p.softplus, to_f32(pd.y), bias) : 0.0f;
    float g0 = a && dout ? to_f32(pg.x) : 0.0f, g1 = b && dout ? to_f32(pg.y) : 0.0f;
    if (z) {
      const float z0 = to_f32(pz.x), z1 = to_f32(pz.y);
      g0 = a ? g0 * (z0 * gate_of(z0)) : 0.0f, g1 = b ? g1 * (z1 * gate_of(z1)) : 0.0f;
    }
    pair_in(sm + l.step, at) = make_float2(s0, s1);
    pair_in(sm + l.du, at) = make_float2(a ? s0 * to_f32(px.x) : 0.0f, b ? s1 * to_f32(px.y) : 0.0f);
    pair_in(sm + l.gy, at) = make_float2(g0, g1);
  };
  auto prepare = [&](int t0) {
    if (first_pair) prepare_pair(nx, nd, nz, ng, t0 + 2 * w, pair_at(2 * w, lane));
    if (!ONE)
      for (int u = w + warps; u < kBlock / 2; u += warps) {
        Pair<T> px, pd, pz, pg;
        load(t0 + 2 * u, px, pd, pz, pg);
        prepare_pair(px, pd, pz, pg, t0 + 2 * u, pair_at(2 * u, lane));
      }
    few.store(sm + l.bs, sm + l.cs, t0, lastt);
    cx = nx, cd = nd, cz = nz, cg = ng;
  };
  float dskip = 0.0f, dbias = 0.0f;
  // A token's sums over the states, and what follows from them.
  auto finish_token = [&](T px, T pd, T pz, T pg, float y, float sb, float sa, float gy, float step, int t) {
    const float xv = to_f32(px);
    const float gx = fmaf(step, sb, p.skip ? skip * gy : 0.0f);
    float raw = fmaf(xv, sb, sa * 0.6931471805599453f);  // rt is A / ln 2
    if (p.softplus) raw *= gate_of(to_f32(pd) + bias);
    const long at = dense + (long)t * p.D;
    static_cast<T*>(p.dx)[at] = from_f32<T>(gx), static_cast<T*>(p.ddt)[at] = from_f32<T>(raw);
    if (z) {
      const float v = to_f32(pz), s = gate_of(v), full = p.skip ? fmaf(skip, xv, y) : y, go = dout ? to_f32(pg) : 0.0f;
      static_cast<T*>(p.dz)[at] = from_f32<T>(go * full * (s * fmaf(v, 1.0f - s, 1.0f)));
    }
    dbias += raw, dskip = fmaf(gy, xv, dskip);
  };
  // part: [quad][y, sum B dh, sum A w][warp][lane]
  auto finish_pair = [&](const Pair<T>& px, const Pair<T>& pd, const Pair<T>& pz, const Pair<T>& pg, int u, int t) {
    float2 sum[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      sum[i] = twice(0.0f);
      if (i == 0 && !z) continue;
      const float* part = sm + l.part + (((u >> 1) * 3 + i) * warps * kLanes + lane) * 4 + 2 * (u & 1);
#pragma unroll (W ? W : 4)
      for (int k = 0; k < warps; ++k) sum[i] = __fadd2_rn(sum[i], *reinterpret_cast<const float2*>(part + k * 4 * kLanes));
    }
    if (!q.live) return;
    const int at = pair_at(2 * u, lane);
    const float2 gy = pair_in(sm + l.gy, at), step = pair_in(sm + l.step, at);
    finish_token(px.x, pd.x, pz.x, pg.x, sum[0].x, sum[1].x, sum[2].x, gy.x, step.x, t);
    if (t < lastt) finish_token(px.y, pd.y, pz.y, pg.y, sum[0].y, sum[1].y, sum[2].y, gy.y, step.y, t + 1);
  };
  auto finish = [&](int t0) {
    if (first_pair && t0 + 2 * w <= lastt) finish_pair(cx, cd, cz, cg, w, t0 + 2 * w);
    if (!ONE)
      for (int u = w + warps; u < kBlock / 2 && t0 + 2 * u <= lastt; u += warps) {
        Pair<T> px, pd, pz, pg;
        load(t0 + 2 * u, px, pd, pz, pg);
        finish_pair(px, pd, pz, pg, u, t0 + 2 * u);
      }
  };

  const float4* step = reinterpret_cast<const float4*>(sm + l.step) + lane;
  const float4* du = reinterpret_cast<const float4*>(sm + l.du) + lane;
  const float4* gy = reinterpret_cast<const float4*>(sm + l.gy) + lane;
  float total = 0.0f;
  const int start = q.first + (q.end - 1 - q.first) / kBlock * kBlock;  // the last block
  // the marks of this warp's first state; its lanes' rows of partial sums
  const float* mark = p.marks + (((long)q.unit * p.nmarks + start / kBlock) * p.np + 2 * w) * kLanes + lane;
  float* bc = p.part_bc + (((long)q.unit * p.np + 2 * w + ((lane >> 3) & 1)) * 2 + (lane >> 4)) * p.T;
  const int mine = (lane & 4 ? 8 : 0) + (lane & 2 ? 4 : 0) + (lane & 1 ? 2 : 0);
  prefetch(start);
  prepare(start);
  if (start > q.first) prefetch(start - kBlock);
  __syncthreads();
  for (int t0 = start; t0 >= q.first; t0 -= kBlock) {
#pragma unroll
    for (int g = 0; g < GW; ++g) {
      const int n0 = 2 * (g * warps + w);
      const float* bs = sm + l.bs + n0 * kRow;
      const float* cs = sm + l.cs + n0 * kRow;
      if (GW > 1 && n0 >= p.np) {  // no such states: nothing to add
        continue;
      }
      float a[2][kBlock], h[2][kBlock], h0[2] = {0.0f, 0.0f};
      if (!SUM) {
#pragma unroll
        for (int j = 0; j < 2; ++j) h0[j] = n0 + j < p.N ? mark[(g * 2 * warps + j) * kLanes] : 0.0f;
      }
#pragma unroll
      for (int t = 0; t < kBlock / 4; ++t) {
        const float4 s = step[t * kLanes], u = du[t * kLanes];
        if (SUM) total += (s.x + s.y) + (s.z + s.w);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 e0 = __fmul2_rn(make_float2(s.x, s.y), twice(rt[g][j]));
          const float2 e1 = __fmul2_rn(make_float2(s.z, s.w), twice(rt[g][j]));
          a[j][4 * t] = exp2_of(e0.x), a[j][4 * t + 1] = exp2_of(e0.y);
          a[j][4 * t + 2] = exp2_of(e1.x), a[j][4 * t + 3] = exp2_of(e1.y);
          if (!SUM) {
            const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
            const float2 v0 = __fmul2_rn(make_float2(u.x, u.y), make_float2(bv.x, bv.y));
            const float2 v1 = __fmul2_rn(make_float2(u.z, u.w), make_float2(bv.z, bv.w));
            h[j][4 * t] = fmaf(a[j][4 * t], t ? h[j][t ? 4 * t - 1 : 0] : h0[j], v0.x);
            h[j][4 * t + 1] = fmaf(a[j][4 * t + 1], h[j][4 * t], v0.y);
            h[j][4 * t + 2] = fmaf(a[j][4 * t + 2], h[j][4 * t + 1], v1.x);
            h[j][4 * t + 3] = fmaf(a[j][4 * t + 3], h[j][4 * t + 2], v1.y);
          }
        }
      }
      float sums[kBlock];
      float2 da2[2] = {twice(0.0f), twice(0.0f)};  // of the block: short sums first
      float4* part = reinterpret_cast<float4*>(sm + l.part) + w * kLanes + lane;
      const int next = warps * kLanes;
#pragma unroll
      for (int t = kBlock / 4 - 1; t >= 0; --t) {
        const float4 s = step[t * kLanes], u = du[t * kLanes], gv = gy[t * kLanes];
        float2 y0 = twice(0.0f), y1 = y0, b0 = y0, b1 = y0, w0 = y0, w1 = y0;
        if (!SUM && g > 0) {
          const float4 py = part[3 * t * next], pb = part[(3 * t + 1) * next], pw = part[(3 * t + 2) * next];
          y0 = make_float2(py.x, py.y), y1 = make_float2(py.z, py.w), b0 = make_float2(pb.x, pb.y), b1 = make_float2(pb.z, pb.w);
          w0 = make_float2(pw.x, pw.y), w1 = make_float2(pw.z, pw.w);
        }
        float v[16];  // [dB, dC][state][token]
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 cv = *reinterpret_cast<const float4*>(cs + j * kRow + 4 * t);
          const float2 c0 = make_float2(cv.x, cv.y), c1 = make_float2(cv.z, cv.w);
          const float2 g0 = make_float2(gv.x, gv.y), g1 = make_float2(gv.z, gv.w);
          const float2 cg0 = __fmul2_rn(c0, g0), cg1 = __fmul2_rn(c1, g1);
          float2 d0, d1, r0, r1;
          d1.y = cg1.y + back[g][j];
          r1.y = a[j][4 * t + 3] * d1.y;
          d1.x = cg1.x + r1.y;
          r1.x = a[j][4 * t + 2] * d1.x;
          d0.y = cg0.y + r1.x;
          r0.y = a[j][4 * t + 1] * d0.y;
          d0.x = cg0.x + r0.y;
          r0.x = back[g][j] = a[j][4 * t] * d0.x;
          if (SUM) continue;
          const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
          const float2 h01 = make_float2(h[j][4 * t], h[j][4 * t + 1]), h23 = make_float2(h[j][4 * t + 2], h[j][4 * t + 3]);
          r0.x *= t ? h[j][t ? 4 * t - 1 : 0] : h0[j];  // w
          r0.y *= h01.x, r1.x *= h01.y, r1.y *= h23.x;
          y0 = __ffma2_rn(c0, h01, y0), y1 = __ffma2_rn(c1, h23, y1);
          b0 = __ffma2_rn(make_float2(bv.x, bv.y), d0, b0), b1 = __ffma2_rn(make_float2(bv.z, bv.w), d1, b1);
          w0 = __ffma2_rn(twice(rt[g][j]), r0, w0), w1 = __ffma2_rn(twice(rt[g][j]), r1, w1);
          da2[j] = __ffma2_rn(make_float2(s.x, s.y), r0, da2[j]);
          da2[j] = __ffma2_rn(make_float2(s.z, s.w), r1, da2[j]);
          const float2 vb0 = __fmul2_rn(d0, make_float2(u.x, u.y)), vb1 = __fmul2_rn(d1, make_float2(u.z, u.w));
          const float2 vc0 = __fmul2_rn(g0, h01), vc1 = __fmul2_rn(g1, h23);
          v[4 * j] = vb0.x, v[4 * j + 1] = vb0.y, v[4 * j + 2] = vb1.x, v[4 * j + 3] = vb1.y;
          v[8 + 4 * j] = vc0.x, v[9 + 4 * j] = vc0.y, v[10 + 4 * j] = vc1.x, v[11 + 4 * j] = vc1.y;
        }
        if (SUM) continue;
        part[3 * t * next] = make_float4(y0.x, y0.y, y1.x, y1.y);
        part[(3 * t + 1) * next] = make_float4(b0.x, b0.y, b1.x, b1.y);
        part[(3 * t + 2) * next] = make_float4(w0.x, w0.y, w1.x, w1.y);
        halve<8>(v, 16, lane & 16);
        halve<4>(v, 8, lane & 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[4 * t + e] = v[e];
      }
      if (SUM) continue;
      da[g][0] = __fadd2_rn(da[g][0], da2[0]), da[g][1] = __fadd2_rn(da[g][1], da2[1]);
      // a lane holds dB (lane < 16) or dC of state (lane >> 3) & 1, for all tokens,
      // over an eighth of the lanes each
      halve<8>(sums, 4, lane & 4);
      halve<4>(sums, 2, lane & 2);
      halve<2>(sums, 1, lane & 1);
      const int t = t0 + mine;
      float* to = bc + (long)g * 4 * warps * p.T + t;
      if (t <= lastt) to[0] = sums[0];
      if (t < lastt) to[1] = sums[1];
    }
    mark -= p.np * kLanes;
    __syncthreads();
    if (!SUM) finish(t0);
    if (t0 > q.first) {
      // finish() reads this block's steps and gradients of its own pairs, which
      // are the pairs that prepare() overwrites
      prepare(t0 - kBlock);
      if (t0 - kBlock > q.first) prefetch(t0 - 2 * kBlock);
    }
    __syncthreads();
  }
  if (SUM) {
    const long at = (long)q.unit * p.segs + q.seg;
#pragma unroll
    for (int g = 0; g < GW; ++g)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = 2 * (g * warps + w) + j;
        if (n < p.np) p.seg_sums[(at * p.np + n) * kLanes + lane] = back[g][j];
      }
    if (w == 0) p.seg_steps[at * kLanes + lane] = total / GW;
    return;
  }
  float* sums = sm + l.sums;
  sums[w * kLanes + lane] = dskip;
  sums[(warps + w) * kLanes + lane] = dbias;
  __syncthreads();
  if (!q.live) return;
  const long at = (long)q.b * p.segs + q.seg;
  for (int k = w; k < 2; k += warps) {
    float s = 0.0f;
    for (int o = 0; o < warps; ++o) s += sums[(k * warps + o) * kLanes + lane];
    p.part_ch[(at * 2 + k) * p.D + q.d] = s;
  }
#pragma unroll
  for (int g = 0; g < GW; ++g)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = 2 * (g * warps + w) + j;
      if (n >= p.N) continue;
      p.part_a[(at * p.D + q.d) * p.N + n] = da[g][j].x + da[g][j].y;
      if (q.seg == 0 && p.ds0) p.ds0[((long)q.b * p.D + q.d) * p.N + n] = back[g][j];
    }
}

// dB and dC: the sums over a group's tiles of 32 channels, in their order.  A
// thread has a token, so that the partial sums are read along the time.
template <typename T>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const Problem p) {
  const long i = blockIdx.x * 256L + threadIdx.x;  // (b, group, state, which, t)
  const long t = i % p.T;
  long rest = i / p.T;
  const int which = (int)(rest % 2);
  rest /= 2;
  const int n = (int)(rest % p.N);
  rest /= p.N;
  const int group = (int)(rest % p.G);
  const long b = rest / p.G;
  if (b >= p.B) return;
  const long tile = (long)p.np * 2 * p.T;
  const float* part = p.part_bc + (b * p.tiles + (long)group * p.per_group) * tile + ((long)n * 2 + which) * p.T + t;
  double s = 0.0;
#pragma unroll 8
  for (int k = 0; k < p.per_group; ++k) s += (double)part[k * tile];
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

template <typename T, int GW, int MOST, bool ONE, int W, int K>
int launch_backward(const Problem& p, cudaStream_t stream) {
  const int warps = ceil_div(p.N, 2 * GW);
  const size_t smem = layout(warps, p.np).total * sizeof(float);
  const unsigned ctas = (unsigned)((long)p.B * p.tiles * p.segs);
  LaunchScope scope(kKindSelectiveScan, stream, p.segs > 1 ? 5 : 4);
  if (p.segs > 1) {
    GRU_CUDA_TRY(cudaFuncSetAttribute(scan_backward_kernel<T, GW, true, MOST, ONE, W, K>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    scan_backward_kernel<T, GW, true, MOST, ONE, W, K><<<ctas, 32 * warps, smem, stream>>>(p);
    GRU_CUDA_TRY(cudaGetLastError());
  }
  GRU_CUDA_TRY(cudaFuncSetAttribute(scan_backward_kernel<T, GW, false, MOST, ONE, W, K>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  scan_backward_kernel<T, GW, false, MOST, ONE, W, K><<<ctas, 32 * warps, smem, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  const long sums = (long)p.B * p.T * p.G * 2 * p.N;
  sum_tiles_kernel<T><<<(unsigned)((sums + 255) / 256), 256, 0, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  const long an = (long)p.D * p.N;
  if (const int rc = sum_parts(p.part_a, p.B * p.segs, an, an, StoreF32{p.da}, stream)) return rc;
  return sum_parts(p.part_ch, p.B * p.segs, 2L * p.D, 2L * p.D, StoreChannels{p.dskip, p.dbias, p.D}, stream);
}

template <typename T>
int backward_of(const Problem& p, cudaStream_t stream) {
  if (p.N <= 14) return launch_backward<T, 1, 256, false, 0, 2>(p, stream);
  if (p.N <= 16) return launch_backward<T, 1, 256, true, 8, 1>(p, stream);
  return p.N <= 32 ? launch_backward<T, 1, 512, true, 0, 2>(p, stream) : launch_backward<T, 2, 512, true, 0, 4>(p, stream);
}

}  // namespace

int backward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? backward_of<float>(p, stream) : backward_of<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
