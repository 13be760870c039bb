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
// The forward's shape, backwards: a CTA owns 64 channels of one sequence, two a
// lane, a warp two states (twice two above 16), and goes over blocks of 16 tokens
// from the last to the first.  The forward kept the state before each block; from
// it a warp computes its states at eight tokens, with the decays, in registers, and
// then goes over the tokens backwards, first for the later eight (for them it passes
// the earlier ones once more: half an exponential, where twice as many kept states
// would cost as much in memory traffic), and what the gate multiplied, for dz.  The
// warps' shares of sum_n B dh and sum_n A w meet in shared memory, where each warp
// finishes a token.  Sums over
// channels: the lane's two, then butterflies over the lanes in which each round
// halves the values: 32 values (8 tokens, 2 states, dB and dC) take 31 exchanges and
// leave a lane one sum.  The tiles' sums of dB and dC are added by a second launch,
// in a fixed order, as are those over sequences of dA, dskip and dbias.  Segments as
// in the forward.
//
// 64 sequences of 512 tokens, 512 channels, 16 states, FP32: 500 us; its exponentials
// would take 87, its memory 82.  Bound by instructions and their latencies (issue slots
// 50 % with the 16 warps an SM that 128 registers a thread allow; shared memory's
// wavefronts 60 %).  It took 551 when it made what the gate multiplied once more, instead
// of reading it; left out in turn, the finishing of tokens then took 92 us, the
// preparation 60, copies 42, the earlier tokens' second pass 28, the butterflies 28.

#include <algorithm>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {

namespace {

constexpr int kHalf = kBlock / 2;

// Shared memory in floats; elem: bytes of an element.
struct Lay {
  int step, du, gy, xs, sg, bs, cs, part, marks, in, kept, few, sums, total;
};
__host__ __device__ inline Lay layout(int warps, int np, int N, int elem) {
  Lay l;
  int n = 0;
  l.step = n, n += kBlock * kTile;
  l.du = n, n += kBlock * kTile;  // dt x
  l.gy = n, n += kBlock * kTile;  // gradient of y
  l.xs = n, n += kBlock * kTile;
  l.sg = n, n += kBlock * kTile;  // softplus'
  l.bs = n, n += np * kRow;
  l.cs = n, n += np * kRow;
  l.part = n, n += warps * 2 * kHalf * kTile;  // [token][sum B dh, sum A w][warp][lane] float2
  l.marks = n, n += 2 * np * kTile;  // of this block and the next
  l.in = n, n += 4 * kBlock * kTile * elem / 4;
  l.kept = n, n += kBlock * kTile;
  l.few = n, n += 2 * kBlock * N * elem / 4;
  l.sums = n, n += 2 * warps * kTile;
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

// GW: pairs of states of a warp.  SUM: only what the segments hand back.  PADS, MOST, OCC
// and W as in the forward.
template <typename T, int GW, bool SUM, bool PADS, int MOST, int OCC, int W>
__global__ void __launch_bounds__(MOST, OCC) scan_backward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int threads = W ? 32 * W : blockDim.x, warps = W ? W : threads >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lay l = layout(warps, p.np, p.N, sizeof(T));
  const Place q = place(p, SUM ? p.segs - 1 : p.segs, SUM ? 1 : 0);
  const T* x = static_cast<const T*>(p.x) + q.b * p.xb + q.d0;
  const T* dt = static_cast<const T*>(p.dt) + q.b * p.dtb + q.d0;
  const T* z = p.z ? static_cast<const T*>(p.z) + q.b * p.zb + q.d0 : nullptr;
  const T* bm = static_cast<const T*>(p.b) + q.b * p.bb + q.group * p.bg;
  const T* cm = static_cast<const T*>(p.c) + q.b * p.cb + q.group * p.cg;
  const T* dout = p.dout ? static_cast<const T*>(p.dout) + (long)q.b * p.T * p.D + q.d0 : nullptr;
  const long dense = (long)q.b * p.T * p.D + q.d;
  const float* kept = z && !SUM ? p.sums + (long)q.b * p.T * p.D + q.d0 : nullptr;
  const float2 bias = two_of(p.bias, q), skip = two_of(p.skip, q);
  const int lastt = q.end - 1;
  T* in = reinterpret_cast<T*>(sm + l.in);
  T* few = reinterpret_cast<T*>(sm + l.few);
  constexpr int kRows = kBlock * kTile;
  Feed<T> feed;
  feed.init(p, bm, cm);
  Feed<float> feed_kept;
  auto fetch = [&](int t0) {
    feed.row(in, x, p.xst, t0, lastt, q.width, p.row_piece);
    feed.row(in + kRows, dt, p.dtst, t0, lastt, q.width, p.row_piece);
    if (z) feed.row(in + 2 * kRows, z, p.zst, t0, lastt, q.width, p.row_piece);
    if (dout) feed.row(in + 3 * kRows, dout, p.ost, t0, lastt, q.width, p.dout_piece);
    if (kept) feed_kept.row(sm + l.kept, kept, p.D * 4, t0, lastt, q.width, p.sums_piece);
    feed.bc(p, few, bm, cm, t0, lastt);
  };
  auto fetch_marks = [&](int t0, int buf) {
    const float4* from = reinterpret_cast<const float4*>(p.marks + ((long)q.unit * p.nmarks + t0 / kBlock) * p.np * kTile);
    for (int e = threadIdx.x; e < p.np * kTile / 4; e += threads) copy<16>(reinterpret_cast<float4*>(sm + l.marks + buf * p.np * kTile) + e, from + e);
  };
  const int start = q.first + (lastt - q.first) / kBlock * kBlock;  // the last block
  fetch(start);
  if (!SUM) fetch_marks(start, 0);

  // states 2 (g warps + w) and the next
  float2 rt[GW][2], back[GW][2], da[GW][2];
#pragma unroll
  for (int g = 0; g < GW; ++g)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = 2 * (g * warps + w) + j;
      const float2 a = two_of(p.a, q, n, p.N);
      rt[g][j] = make_float2(decay_rate(a.x), decay_rate(a.y));
      back[g][j] = SUM ? twice(0.0f) : two_of(p.dlast ? p.dlast + (long)q.b * p.D * p.N : nullptr, q, n, p.N);
      da[g][j] = twice(0.0f);
    }
  if (!SUM)
#pragma unroll 4
    for (int s = p.segs - 1; s > q.seg; --s) {
      const long at = (long)q.unit * p.segs + s;
      const float2 steps = both(p.seg_steps + at * kTile, 0, lane);
#pragma unroll
      for (int g = 0; g < GW; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int n = 2 * (g * warps + w) + j;
          back[g][j] = behind_segment(back[g][j], passed(rt[g][j], steps),
                                      both(p.seg_sums + (at * p.np + n) * kTile, 0, lane));
        }
    }

  float4* rows = reinterpret_cast<float4*>(sm) + lane;  // [array][pair of tokens][lane]
  const int a_step = l.step / 4, a_du = l.du / 4, a_gy = l.gy / 4;
  float2* shares = reinterpret_cast<float2*>(sm + l.part) + lane;
  float2* ends = reinterpret_cast<float2*>(sm) + lane;  // [array][token][lane], of what finish() alone reads
  // What two tokens have per channel.
  auto prepare = [&](int t0) {
    for (int u = w; u < kPairs; u += warps) {
      const int t = t0 + 2 * u;
      float s[4], v[4], g[4] = {0.0f, 0.0f, 0.0f, 0.0f}, xv[4], sg[4];
      four(in, u, lane, xv);
      four(in + kRows, u, lane, s);
      if (dout) four(in + 3 * kRows, u, lane, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float bi = i & 1 ? bias.y : bias.x;
        sg[i] = p.softplus ? sigmoid_of(s[i] + bi) : 1.0f;
        s[i] = step_of(p.softplus, s[i], bi);
        v[i] = s[i] * xv[i];
      }
      if (z) {
        float zv[4], y[4];
        four(in + 2 * kRows, u, lane, zv);
        if (!SUM) four(sm + l.kept, u, lane, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float c = sigmoid_of(zv[i]);
          if (!SUM) y[i] *= g[i] * (c * fmaf(zv[i], 1.0f - c, 1.0f));
          g[i] *= zv[i] * c;
        }
        if (!SUM && t <= lastt) {
          T* dz = row_at(static_cast<T*>(p.dz) + dense, t, p.ost);
          put_both(dz, y[0], y[1], q, p.even_out);
          if (t < lastt) put_both(dz + p.D, y[2], y[3], q, p.even_out);
        }
      }
      if (!q.second || t + 1 > lastt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(i & 1 ? q.second : q.live) || t + i / 2 > lastt) s[i] = v[i] = g[i] = 0.0f;
      float4* to = rows + u * kLanes;
      to[a_step] = as4(s), to[a_du] = as4(v), to[a_gy] = as4(g);
      if (!SUM)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float2* at = ends + (2 * u + i) * kLanes;
          at[l.xs / 2] = make_float2(xv[2 * i], xv[2 * i + 1]);
          at[l.sg / 2] = make_float2(sg[2 * i], sg[2 * i + 1]);
        }
      if (W >= kPairs) break;
    }
    turn_few(p, few, sm + l.bs, sm + l.cs, p.np, q.end - t0);
  };
  float2 dskip = twice(0.0f), dbias = twice(0.0f);
  // A half's tokens' sums over the states, and what follows from them; a token a warp.
  auto finish = [&](int t0, int half) {
    for (int e = w; e < kHalf; e += warps) {
      const int t = t0 + half * kHalf + e;
      if (t > lastt) break;
      float2 sum[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2* part = shares + (e * 2 + i) * warps * kLanes;
        sum[i] = part[0];
#pragma unroll (W ? W : 4)
        for (int k = 1; k < warps; ++k) sum[i] = __fadd2_rn(sum[i], part[k * kLanes]);
      }
      auto of = [&](int a) {
        return reinterpret_cast<const float2*>(rows + a + (half * (kHalf / 2) + e / 2) * kLanes)[e & 1];
      };
      const float2* end = ends + (half * kHalf + e) * kLanes;
      const float2 s = of(a_step), g = of(a_gy), xv = end[l.xs / 2], sg = end[l.sg / 2];
      const float2 sb = sum[0], sa = sum[1];
      const float2 raw = __fmul2_rn(__ffma2_rn(xv, sb, __fmul2_rn(sa, twice(0.6931471805599453f))), sg);  // rt is A / ln 2
      const float2 gx = __ffma2_rn(s, sb, p.skip ? __fmul2_rn(skip, g) : twice(0.0f));
      put_both(row_at(static_cast<T*>(p.dx) + dense, t, p.ost), gx.x, gx.y, q, p.even_out);
      put_both(row_at(static_cast<T*>(p.ddt) + dense, t, p.ost), raw.x, raw.y, q, p.even_out);
      dbias = __fadd2_rn(dbias, raw), dskip = __ffma2_rn(g, xv, dskip);
    }
  };

  float2 total = twice(0.0f);
  // the lanes' rows of partial sums, and their token of a half
  float* bc = p.part_bc + (((long)q.unit * p.np + 2 * w + ((lane >> 3) & 1)) * 2 + (lane >> 4)) * p.T;
  copies_done();
  __syncthreads();
  prepare(start);
  __syncthreads();
  int buf = 0;
  for (int t0 = start; t0 >= q.first; t0 -= kBlock, buf ^= 1) {
    const bool more = t0 > q.first;
    if (more) {
      fetch(t0 - kBlock);
      if (!SUM) fetch_marks(t0 - kBlock, buf ^ 1);
    }
#pragma unroll 1
    for (int half = 1; half >= 0; --half) {
#pragma unroll
      for (int g = 0; g < GW; ++g) {
        // one pair's work behind the other's: mixed by the compiler, its registers went to
        // memory (32 states 1164 us instead of 954)
        if (g > 0) __syncwarp();
        const int n0 = 2 * (g * warps + w);
        const float* bs = sm + l.bs + n0 * kRow;
        const float* cs = sm + l.cs + n0 * kRow;
        const float4* step = rows + a_step + half * (kHalf / 2) * kLanes;
        if (SUM) {
          const float4* gy = rows + a_gy + half * (kHalf / 2) * kLanes;
          float2 behind[2] = {back[g][0], back[g][1]}, all[2] = {twice(1.0f), twice(1.0f)}, steps = twice(0.0f);
#pragma unroll
          for (int t = kHalf / 2 - 1; t >= 0; --t) {
            const float4 s = step[t * kLanes], gv = gy[t * kLanes];
            steps = __fadd2_rn(steps, __fadd2_rn(lo(s), hi(s)));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float4 cv = *reinterpret_cast<const float4*>(cs + j * kRow + 4 * (half * (kHalf / 2) + t));
              float2& r = back[g][j];
              const float2 a0 = exp2_of(__fmul2_rn(lo(s), rt[g][j])), a1 = exp2_of(__fmul2_rn(hi(s), rt[g][j]));
              r = __fmul2_rn(a1, __ffma2_rn(hi(cv), hi(gv), r));
              r = __fmul2_rn(a0, __ffma2_rn(lo(cv), lo(gv), r));
              all[j] = __fmul2_rn(all[j], __fmul2_rn(a0, a1));
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
            back[g][j] = carried(back[g][j], behind[j], passed(rt[g][j], steps), all[j]);
          if (g == 0) total = __fadd2_rn(total, steps);
          continue;
        }
        float2 a[2][kHalf], h[2][kHalf], before[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) before[j] = both(sm + l.marks + (buf * p.np + n0 + j) * kTile, 0, lane);
        if (half) {  // pass the earlier eight
#pragma unroll
          for (int t = 0; t < kHalf / 2; ++t) {
            const float4 s = rows[a_step + t * kLanes], u = rows[a_du + t * kLanes];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
              before[j] = __ffma2_rn(exp2_of(__fmul2_rn(lo(s), rt[g][j])), before[j], __fmul2_rn(lo(u), lo(bv)));
              before[j] = __ffma2_rn(exp2_of(__fmul2_rn(hi(s), rt[g][j])), before[j], __fmul2_rn(hi(u), hi(bv)));
            }
          }
        }
        bs += 4 * half * (kHalf / 2), cs += 4 * half * (kHalf / 2);
        const float4* du = rows + a_du + half * (kHalf / 2) * kLanes;
        const float4* gy = rows + a_gy + half * (kHalf / 2) * kLanes;
        // what is handed back is carried over the tokens as the forward carries a state
        float2 behind[2] = {back[g][0], back[g][1]}, all[2] = {twice(1.0f), twice(1.0f)}, steps = twice(0.0f);
#pragma unroll
        for (int t = 0; t < kHalf / 2; ++t) {
          const float4 s = step[t * kLanes], u = du[t * kLanes];
          steps = __fadd2_rn(steps, __fadd2_rn(lo(s), hi(s)));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
            a[j][2 * t] = exp2_of(__fmul2_rn(lo(s), rt[g][j]));
            a[j][2 * t + 1] = exp2_of(__fmul2_rn(hi(s), rt[g][j]));
            h[j][2 * t] = __ffma2_rn(a[j][2 * t], t ? h[j][t ? 2 * t - 1 : 0] : before[j], __fmul2_rn(lo(u), lo(bv)));
            h[j][2 * t + 1] = __ffma2_rn(a[j][2 * t + 1], h[j][2 * t], __fmul2_rn(hi(u), hi(bv)));
            all[j] = __fmul2_rn(all[j], __fmul2_rn(a[j][2 * t], a[j][2 * t + 1]));
          }
          __syncwarp();  // a pair of tokens after another, for the registers' sake (516 -> 509 us)
        }
        float sums[kHalf];
        float2 da2[2] = {twice(0.0f), twice(0.0f)};  // of the half: short sums first
#pragma unroll
        for (int t = kHalf / 2 - 1; t >= 0; --t) {
          const float4 s = step[t * kLanes], u = du[t * kLanes], gv = gy[t * kLanes];
          float2* share0 = shares + (2 * t * 2 * warps + w) * kLanes;  // of the tokens 2 t and 2 t + 1
          float2* share1 = share0 + 2 * warps * kLanes;
          float2 b0 = twice(0.0f), b1 = b0, w0 = b0, w1 = b0;
          if (g > 0) {
            b0 = share0[0], w0 = share0[warps * kLanes];
            b1 = share1[0], w1 = share1[warps * kLanes];
          }
          float v[8];  // [dB, dC][state][token]
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float4 cv = *reinterpret_cast<const float4*>(cs + j * kRow + 4 * t);
            const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
            const float2 h0 = h[j][2 * t], h1 = h[j][2 * t + 1], hb = t ? h[j][t ? 2 * t - 1 : 0] : before[j];
            const bool there = !PADS || n0 + j < p.N;  // assignments below: as selects 22 states took 944 us, not 840
            float2 d1 = __ffma2_rn(hi(cv), hi(gv), back[g][j]);
            if (!there) d1 = twice(0.0f);
            const float2 r1 = __fmul2_rn(a[j][2 * t + 1], d1);
            float2 d0 = __ffma2_rn(lo(cv), lo(gv), r1);
            if (!there) d0 = twice(0.0f);
            back[g][j] = __fmul2_rn(a[j][2 * t], d0);
            const float2 q1 = __fmul2_rn(r1, h0), q0 = __fmul2_rn(back[g][j], hb);  // w
            b0 = __ffma2_rn(lo(bv), d0, b0), b1 = __ffma2_rn(hi(bv), d1, b1);
            if (there) w0 = __ffma2_rn(rt[g][j], q0, w0), w1 = __ffma2_rn(rt[g][j], q1, w1);
            da2[j] = __ffma2_rn(lo(s), q0, da2[j]), da2[j] = __ffma2_rn(hi(s), q1, da2[j]);
            v[2 * j] = fmaf(d0.y, u.y, d0.x * u.x), v[2 * j + 1] = fmaf(d1.y, u.w, d1.x * u.z);
            v[4 + 2 * j] = fmaf(h0.y, gv.y, h0.x * gv.x), v[5 + 2 * j] = fmaf(h1.y, gv.w, h1.x * gv.z);
          }
          share0[0] = b0, share0[warps * kLanes] = w0;
          share1[0] = b1, share1[warps * kLanes] = w1;
          halve<4>(v, 16, lane & 16);
          halve<2>(v, 8, lane & 8);
          sums[2 * t] = v[0], sums[2 * t + 1] = v[1];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          da[g][j] = __fadd2_rn(da[g][j], da2[j]);
          back[g][j] = carried(back[g][j], behind[j], passed(rt[g][j], steps), all[j]);
        }
        // a lane holds dB (lane < 16) or dC of state (lane >> 3) & 1, for all eight
        // tokens, over an eighth of the lanes each
        halve<4>(sums, 4, lane & 4);
        halve<2>(sums, 2, lane & 2);
        halve<1>(sums, 1, lane & 1);
        const int t = t0 + half * kHalf + (lane & 7);
        if (t <= lastt) bc[(long)g * 4 * warps * p.T + t] = sums[0];
      }
      if (SUM) continue;
      if (half == 0) copies_done();
      __syncthreads();
      finish(t0, half);
      if (half) __syncthreads();
    }
    if (SUM) copies_done();
    __syncthreads();  // finish() reads rows that prepare() overwrites
    if (more) prepare(t0 - kBlock);
    __syncthreads();
  }
  if (SUM) {
    const long at = (long)q.unit * p.segs + q.seg;
#pragma unroll
    for (int g = 0; g < GW; ++g)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = 2 * (g * warps + w) + j;
        *reinterpret_cast<float2*>(p.seg_sums + (at * p.np + n) * kTile + 2 * lane) = back[g][j];
      }
    if (w == 0) *reinterpret_cast<float2*>(p.seg_steps + at * kTile + 2 * lane) = total;
    return;
  }
  float2* sums = reinterpret_cast<float2*>(sm + l.sums) + lane;
  sums[w * kLanes] = dskip;
  sums[(warps + w) * kLanes] = dbias;
  __syncthreads();
  const long at = (long)q.b * p.segs + q.seg;
  for (int k = w; k < 2; k += warps) {
    float2 s = twice(0.0f);
    for (int o = 0; o < warps; ++o) s = __fadd2_rn(s, sums[(k * warps + o) * kLanes]);
    put_two(p.part + at * p.D * (p.N + 2) + (long)p.D * (p.N + k), q, 0, 1, s);
  }
#pragma unroll
  for (int g = 0; g < GW; ++g)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = 2 * (g * warps + w) + j;
      put_two(p.part + at * p.D * (p.N + 2), q, n, p.N, da[g][j]);
      if (q.seg == 0 && p.ds0) put_two(p.ds0 + (long)q.b * p.D * p.N, q, n, p.N, back[g][j]);
    }
}

// dB and dC: the sums over a group's tiles of 64 channels, in their order.  A warp
// has 128 tokens of a row (b, group, state, dB or dC), four a lane, so that the partial
// sums are read along the time.  Eight tiles are added in FP32, by pairs, and their sums
// in FP64.  (A thread a token, and every tile in FP64: 27 us instead of 9 for 32 tiles of 4 x
// 2048 tokens, by the divisions of its index and the conversions.)
constexpr int kSumTokens = 128;
template <typename T>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const Problem p, long rows) {
  const int blocks = (p.T + kSumTokens - 1) / kSumTokens;
  const long item = blockIdx.x * 8L + (threadIdx.x >> 5);
  const long row = item / blocks;
  if (row >= rows) return;
  const int t0 = (int)(item - row * blocks) * kSumTokens + (threadIdx.x & 31);
  const int which = (int)(row & 1);
  const long state = row >> 1, bg = state / p.N, b = bg / p.G;
  const int n = (int)(state - bg * p.N), group = (int)(bg - b * p.G);
  const long tile = (long)p.np * 2 * p.T;
  const float* part = p.part_bc + (b * p.tiles + (long)group * p.per_group) * tile + ((long)n * 2 + which) * p.T;
  int t[4];
  double s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = min(t0 + 32 * i, p.T - 1), s[i] = 0.0;
  int k = 0;
  for (; k + 8 <= p.per_group; k += 8, part += 8 * tile) {
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i][j] = part[j * tile + t[i]];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      s[i] += (double)(((v[i][0] + v[i][1]) + (v[i][2] + v[i][3])) + ((v[i][4] + v[i][5]) + (v[i][6] + v[i][7])));
  }
  for (; k < p.per_group; ++k, part += tile)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] += (double)part[t[i]];
  T* to = static_cast<T*>(which ? p.dc : p.db);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t0 + 32 * i < p.T) to[((b * p.T + t[i]) * p.G + group) * p.N + n] = from_f32<T>((float)s[i]);
}

struct StoreSums {  // dA, then dskip, then dbias
  float *da, *dskip, *dbias;
  long an;
  int D;
  __device__ __forceinline__ void operator()(long c, float x) const {
    if (c < an) da[c] = x;
    else if (c < an + D) {
      if (dskip) dskip[c - an] = x;
    } else if (dbias) {
      dbias[c - an - D] = x;
    }
  }
};

template <typename T, int GW, int MOST, int OCC, int W>
int launch_backward(const Problem& p, cudaStream_t stream) {
  const int warps = p.np / (2 * GW);
  const size_t smem = layout(warps, p.np, p.N, sizeof(T)).total * sizeof(float);
  const long units = (long)p.B * p.tiles;
  LaunchScope scope(kKindSelectiveScan, stream, p.segs > 1 ? 4 : 3);
  if (p.segs > 1) {
    auto kernel = scan_backward_kernel<T, GW, true, false, MOST, OCC, W>;
    GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<(unsigned)(units * (p.segs - 1)), 32 * warps, smem, stream>>>(p);
    GRU_CUDA_TRY(cudaGetLastError());
  }
  auto kernel = p.N == p.np ? scan_backward_kernel<T, GW, false, false, MOST, OCC, W> : scan_backward_kernel<T, GW, false, true, MOST, OCC, W>;
  GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<(unsigned)(units * p.segs), 32 * warps, smem, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  const long rows = (long)p.B * p.G * 2 * p.N, items = rows * ceil_div(p.T, kSumTokens);
  sum_tiles_kernel<T><<<(unsigned)((items + 7) / 8), 256, 0, stream>>>(p, rows);
  GRU_CUDA_TRY(cudaGetLastError());
  const long an = (long)p.D * p.N, cols = an + 2L * p.D;
  return sum_parts(p.part, p.B * p.segs, cols, cols, StoreSums{p.da, p.dskip, p.dbias, an, p.D}, stream);
}

// Two pairs of states a warp, one after the other, from 20 states on, where that many
// warps leave room for two CTAs (64 sequences of 512 tokens, 512 channels, 32 states:
// 954 us, 1081 with a pair a warp; 16 states 562 and 517).  As many CTAs an SM as
// shared memory and 128 registers a thread allow.
template <typename T>
int backward_of(const Problem& p, cudaStream_t stream) {
  if (p.np == 4) return launch_backward<T, 1, 64, 4, 2>(p, stream);
  if (p.np == 8) return launch_backward<T, 1, 128, 3, 4>(p, stream);
  if (p.np == 12) return launch_backward<T, 1, 192, 2, 6>(p, stream);
  if (p.np == 16) return launch_backward<T, 1, 256, 2, 8>(p, stream);
  if (p.np < 32) return launch_backward<T, 2, 224, 2, 0>(p, stream);
  if (p.np == 32) return launch_backward<T, 2, 256, 2, 8>(p, stream);
  if (p.np == 64) return launch_backward<T, 2, 512, 1, 16>(p, stream);
  return launch_backward<T, 2, 512, 1, 0>(p, stream);
}

}  // namespace

Fit backward_fit(int np) { return {np <= 16 ? np / 2 : np / 4, np == 4 ? 4 : np == 8 ? 3 : np <= 32 ? 2 : 1}; }

int backward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? backward_of<float>(p, stream) : backward_of<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
