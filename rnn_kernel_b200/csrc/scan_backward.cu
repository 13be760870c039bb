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
// each, and goes over blocks of 32 tokens from the last to the first, 8 tokens a
// warp.  The forward kept the state before each block.  For four states at a time a
// warp computes its tokens' decays once and from them its tokens' effect on the
// state (P h + S) and on what is handed back (P r + R); both meet the other
// warps' in shared memory, and the warp goes over its tokens forwards for h and
// backwards for the gradients.  Sums over channels are butterflies over the
// lanes in which each round halves the values: 64 values (8 tokens, 4 states, dB
// and dC) take 62 exchanges and leave a lane two sums.  The tiles' sums of dB and
// dC are added by a second launch, in a fixed order, as are those over sequences
// of dA, dskip and dbias.  Clusters share a sequence's blocks as in the forward.
// Bound by instructions: some 22 per token, channel and state.

#include <algorithm>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {

__device__ int g_backward_status = 0;

namespace {

constexpr int kTok = 8;            // tokens of a warp
constexpr int kRow = kTok + 4;     // floats between two states' tokens in shared memory
constexpr int kBlock = kWarps * kTok;
constexpr int kResident = 3;       // CTAs an SM holds, by registers
static_assert(kBlock == kMark, "the forward keeps the state before each block");

// Shared memory in floats; np: states, padded; elem: bytes of an element.
struct Lay {
  int bars, in, bs, cs, ex, carry, rate, da, rows, sums, total;
};
__host__ __device__ inline Lay layout(int np, int elem) {
  Lay l;
  int n = 0;
  l.bars = n, n += np;
  l.in = n, n += 2 * kWarps * 4 * kTok * kLanes * elem / 4;
  l.bs = n, n += kWarps * np * kRow;
  l.cs = n, n += kWarps * np * kRow;
  l.ex = n, n += 2 * kWarps * 3 * kLanes * 4;
  l.carry = n, n += 2 * np * kLanes;
  l.rate = n, n += np * kLanes;
  l.da = n, n += kWarps * np * kLanes;
  l.rows = n, n += kWarps * kTok * np * 2;
  l.sums = n, n += 2 * kWarps * kLanes;
  l.total = n;
  return l;
}

__device__ __forceinline__ float4 fma4(float4 x, float4 y, float4 z) {
  const float2 a = __ffma2_rn(make_float2(x.x, x.y), make_float2(y.x, y.y), make_float2(z.x, z.y));
  const float2 b = __ffma2_rn(make_float2(x.z, x.w), make_float2(y.z, y.w), make_float2(z.z, z.w));
  return make_float4(a.x, a.y, b.x, b.y);
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

// Q: several CTAs share a tile, as a cluster.
template <typename T, bool Q>
__global__ void __launch_bounds__(32 * kWarps, kResident) scan_backward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, ng = p.np / 4;
  const Lay l = layout(p.np, sizeof(T));
  const int rank = Q ? (int)cluster_rank() : 0, peers = Q ? (int)cluster_size() : 1;
  const int unit = blockIdx.x / peers, tile = unit % p.tiles, b = unit / p.tiles;
  const int group = tile / p.per_group, c0 = (tile - group * p.per_group) * kLanes;
  const int width = min(p.R - c0, kLanes), d0 = group * p.R + c0;
  const bool live = lane < width;
  const int d = d0 + (live ? lane : 0);
  constexpr int kTile = kTok * kLanes;
  T* in0 = reinterpret_cast<T*>(sm + l.in) + w * 8 * kTile;  // two buffers of x, dt, dout, z
  float* bs = sm + l.bs + w * p.np * kRow;
  float* cs = sm + l.cs + w * p.np * kRow;
  float* rows = sm + l.rows + w * kTok * p.np * 2;  // [token][dB, dC][state]
  float4* ex = reinterpret_cast<float4*>(sm + l.ex) + lane;
  float4* carry = reinterpret_cast<float4*>(sm + l.carry) + lane;
  float4* rate = reinterpret_cast<float4*>(sm + l.rate) + lane;
  float4* das = reinterpret_cast<float4*>(sm + l.da) + w * ng * kLanes + lane;
  const uint32_t bars = smem_at(sm + l.bars);

  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + d0;
  const T* dt = static_cast<const T*>(p.dt) + b * p.dts[0] + d0;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.zs[0] + d0 : nullptr;
  const T* bm = static_cast<const T*>(p.b) + b * p.bs[0] + group * p.bs[2];
  const T* cm = static_cast<const T*>(p.c) + b * p.cs[0] + group * p.cs[2];
  const T* dout = p.dout ? static_cast<const T*>(p.dout) + (long)b * p.T * p.D + d0 : nullptr;
  const int blocks = (p.T + kBlock - 1) / kBlock;
  const bool async = p.pairs && (sizeof(T) == 4 || width % 2 == 0);
  auto fetch = [&](int i, T* to) {
    const int t0 = i * kBlock + w * kTok, here = p.T - t0;
    if (here <= 0) return;
    fetch_rows<T, kTok>(x + t0 * p.xs[1], p.xs[1], here, width, async, to);
    fetch_rows<T, kTok>(dt + t0 * p.dts[1], p.dts[1], here, width, async, to + kTile);
    if (dout) fetch_rows<T, kTok>(dout + (long)t0 * p.D, p.D, here, width, async && p.dpairs, to + 2 * kTile);
    if (z) fetch_rows<T, kTok>(z + t0 * p.zs[1], p.zs[1], here, width, async, to + 3 * kTile);
  };
  fetch(blocks - 1 - rank, in0);
  copies_issued();

  const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
  for (int g = w; g < ng; g += kWarps) {
    float r[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = 4 * g + j;
      r[j] = live && n < p.N ? decay_rate(p.a[(long)d * p.N + n]) : 0.0f;
      s[j] = live && n < p.N && p.dlast ? p.dlast[((long)b * p.D + d) * p.N + n] : 0.0f;
    }
    rate[g * kLanes] = make_float4(r[0], r[1], r[2], r[3]);
    if (rank == 0) carry[g * kLanes] = make_float4(s[0], s[1], s[2], s[3]);
  }
  for (int g = 0; g < ng; ++g) das[g * kLanes] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (Q) {  // the barrier of slot k & 1 counts the bytes of what is handed back to this CTA's k-th block
    if (threadIdx.x == 0) {
      for (int i = 0; i < 2 * ng; ++i) bar_init(bars + 8 * i);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      for (int i = 0; i < 2 * ng; ++i)
        if (rank == 0 && i < ng) bar_arrive(bars + 8 * i);  // the last state's gradient is there
        else bar_expect(bars + 8 * i, kLanes * 16);
    }
    __syncthreads();
    cluster_sync();
  } else {
    __syncthreads();
  }
  float dskip = 0.0f, dbias = 0.0f;

  int turn = 0;
  bool ok = true;
  for (int from = rank, k = 0; from < blocks; from += peers, ++k) {
    const int i = blocks - 1 - from;
    const int t0 = i * kBlock + w * kTok, here = min(max(p.T - t0, 0), kTok);
    const T* in = in0 + (k & 1) * 4 * kTile;
    float2 step[kTok / 2], du[kTok / 2], gy[kTok / 2];
    float sdt = 0.0f;
    {
      FewRows<T, kTok, kRow> few;
      const T *pb = bm + t0 * p.bs[1], *pc = cm + t0 * p.cs[1];
      few.load(p, pb, pc, here, 0);
      copies_done<0>();
      __syncwarp();
      auto pair = [&](int which, int t) {
        const T* at = in + which * kTile + 2 * t * kLanes + lane;
        return make_float2(to_f32(at[0]), to_f32(at[kLanes]));
      };
#pragma unroll
      for (int t = 0; t < kTok / 2; ++t) {
        step[t] = step_of(p.softplus, pair(1, t), bias);
        du[t] = __fmul2_rn(step[t], pair(0, t));
        gy[t] = dout ? pair(2, t) : twice(0.0f);
        if (z) {
          const float2 v = pair(3, t);
          gy[t] = __fmul2_rn(gy[t], __fmul2_rn(v, sigmoid_of2(v)));
        }
        if (here < kTok) {
          if (2 * t >= here) step[t].x = du[t].x = gy[t].x = 0.0f;
          if (2 * t + 1 >= here) step[t].y = du[t].y = gy[t].y = 0.0f;
        }
        sdt += step[t].x + step[t].y;
      }
      few.store(p, bs, cs, p.np, 0);
      few.rest(p, pb, pc, here, bs, cs, p.np);
    }
    if (from + peers < blocks) fetch(i - peers, in0 + (~k & 1) * 4 * kTile);
    copies_issued();
    float2 y[kTok / 2], sb[kTok / 2], sa[kTok / 2];
#pragma unroll
    for (int t = 0; t < kTok / 2; ++t) y[t] = sb[t] = sa[t] = twice(0.0f);
    __syncwarp();
#pragma unroll 1
    for (int g = 0; g < ng; ++g, turn ^= 1) {
      const float4 rt4 = rate[g * kLanes];
      const float rt[4] = {rt4.x, rt4.y, rt4.z, rt4.w};
      float a[4][kTok], s[4], r[4], mark[4];
      const float* kept = p.marks + (((long)unit * p.nmarks + i) * p.np + 4 * g) * kLanes + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) mark[j] = 4 * g + j < p.N ? kept[j * kLanes] : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 r2 = twice(rt[j]);
        const float4* b4 = reinterpret_cast<const float4*>(bs + (4 * g + j) * kRow);
        const float4* c4 = reinterpret_cast<const float4*>(cs + (4 * g + j) * kRow);
        s[j] = r[j] = 0.0f;
#pragma unroll
        for (int t = 0; t < kTok / 4; ++t) {
          const float4 v = b4[t];
          const float2 e0 = __fmul2_rn(step[2 * t], r2), e1 = __fmul2_rn(step[2 * t + 1], r2);
          const float2 v0 = __fmul2_rn(du[2 * t], make_float2(v.x, v.y)), v1 = __fmul2_rn(du[2 * t + 1], make_float2(v.z, v.w));
          a[j][4 * t] = exp2_of(e0.x), a[j][4 * t + 1] = exp2_of(e0.y);
          a[j][4 * t + 2] = exp2_of(e1.x), a[j][4 * t + 3] = exp2_of(e1.y);
          s[j] = fmaf(a[j][4 * t], s[j], v0.x);
          s[j] = fmaf(a[j][4 * t + 1], s[j], v0.y);
          s[j] = fmaf(a[j][4 * t + 2], s[j], v1.x);
          s[j] = fmaf(a[j][4 * t + 3], s[j], v1.y);
        }
#pragma unroll
        for (int t = kTok / 4 - 1; t >= 0; --t) {
          const float4 v = c4[t];
          const float2 v0 = __fmul2_rn(gy[2 * t], make_float2(v.x, v.y)), v1 = __fmul2_rn(gy[2 * t + 1], make_float2(v.z, v.w));
          r[j] = a[j][4 * t + 3] * (v1.y + r[j]);
          r[j] = a[j][4 * t + 2] * (v1.x + r[j]);
          r[j] = a[j][4 * t + 1] * (v0.y + r[j]);
          r[j] = a[j][4 * t] * (v0.x + r[j]);
        }
      }
      float4* e = ex + turn * kWarps * 3 * kLanes;
      const float4 mine = make_float4(exp2_of(sdt * rt[0]), exp2_of(sdt * rt[1]), exp2_of(sdt * rt[2]), exp2_of(sdt * rt[3]));
      e[(w * 3 + 0) * kLanes] = mine;
      e[(w * 3 + 1) * kLanes] = make_float4(s[0], s[1], s[2], s[3]);
      e[(w * 3 + 2) * kLanes] = make_float4(r[0], r[1], r[2], r[3]);
      __syncthreads();
      float4 h4 = make_float4(mark[0], mark[1], mark[2], mark[3]);
      float4 q = make_float4(1.f, 1.f, 1.f, 1.f), v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int o = 0; o < kWarps - 1; ++o)
        if (o < w) h4 = fma4(e[(o * 3 + 0) * kLanes], h4, e[(o * 3 + 1) * kLanes]);
#pragma unroll
      for (int o = kWarps - 1; o > 0; --o)
        if (o > w) {  // what the warps behind make of what is handed to the block
          const float4 pr = e[(o * 3 + 0) * kLanes];
          v = fma4(pr, v, e[(o * 3 + 2) * kLanes]);
          q.x *= pr.x, q.y *= pr.y, q.z *= pr.z, q.w *= pr.w;
        }
      const int slot = (k & 1) * ng + g;
      if (Q && ok) ok = bar_wait(bars + 8 * slot, (k >> 1) & 1, &g_backward_status);
      const float4 back4 = fma4(q, carry[slot * kLanes], v);
      if (w == 0) {  // for the block before
        const float4 next = fma4(mine, back4, make_float4(r[0], r[1], r[2], r[3]));
        if (Q) {
          if (lane == 0 && from + 2 * peers < blocks) bar_expect(bars + 8 * slot, kLanes * 16);  // its use after the next
          __syncwarp();
          if (from + 1 < blocks) {
            const int to = (rank + 1) % peers, slot_to = (((from + 1) / peers) & 1) * ng + g;
            const uint32_t there = at_rank(smem_at(carry + slot_to * kLanes), to), bar = at_rank(bars + 8 * slot_to, to);
            send(there, make_float2(next.x, next.y), bar);
            send(there + 8, make_float2(next.z, next.w), bar);
          }
        } else {
          carry[(((k + 1) & 1) * ng + g) * kLanes] = next;
        }
      }
      const float h0[4] = {h4.x, h4.y, h4.z, h4.w};
      float h[4][kTok];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4* b4 = reinterpret_cast<const float4*>(bs + (4 * g + j) * kRow);
        float hv = h0[j];
#pragma unroll
        for (int t = 0; t < kTok / 4; ++t) {
          const float4 bv = b4[t];
          const float2 v0 = __fmul2_rn(du[2 * t], make_float2(bv.x, bv.y)), v1 = __fmul2_rn(du[2 * t + 1], make_float2(bv.z, bv.w));
          h[j][4 * t] = fmaf(a[j][4 * t], hv, v0.x);
          h[j][4 * t + 1] = fmaf(a[j][4 * t + 1], h[j][4 * t], v0.y);
          h[j][4 * t + 2] = fmaf(a[j][4 * t + 2], h[j][4 * t + 1], v1.x);
          hv = h[j][4 * t + 3] = fmaf(a[j][4 * t + 3], h[j][4 * t + 2], v1.y);
        }
      }
      const float4 da = das[g * kLanes];
      float2 da2[4] = {{da.x, 0.0f}, {da.y, 0.0f}, {da.z, 0.0f}, {da.w, 0.0f}};
      float sums[kTok], back[4] = {back4.x, back4.y, back4.z, back4.w};
#pragma unroll
      for (int t = kTok / 2 - 1; t >= 0; --t) {
        float lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 bv = *reinterpret_cast<const float2*>(bs + (4 * g + j) * kRow + 2 * t);
          const float2 cv = *reinterpret_cast<const float2*>(cs + (4 * g + j) * kRow + 2 * t);
          const float2 cg = __fmul2_rn(cv, gy[t]), hv = make_float2(h[j][2 * t], h[j][2 * t + 1]);
          float2 dh, rr;
          dh.y = cg.y + back[j];
          rr.y = a[j][2 * t + 1] * dh.y;
          dh.x = cg.x + rr.y;
          rr.x = back[j] = a[j][2 * t] * dh.x;
          const float2 wt = make_float2(rr.x * (t ? h[j][2 * t - 1] : h0[j]), rr.y * h[j][2 * t]);
          y[t] = __ffma2_rn(cv, hv, y[t]);
          sb[t] = __ffma2_rn(bv, dh, sb[t]);
          sa[t] = __ffma2_rn(twice(rt[j]), wt, sa[t]);
          da2[j] = __ffma2_rn(step[t], wt, da2[j]);
          const float2 vb = __fmul2_rn(dh, du[t]), vc = __fmul2_rn(gy[t], hv);
          lo[j] = vb.x, hi[j] = vb.y, lo[4 + j] = vc.x, hi[4 + j] = vc.y;
        }
        halve<4>(lo, 16, lane & 16), halve<4>(hi, 16, lane & 16);
        halve<2>(lo, 8, lane & 8), halve<2>(hi, 8, lane & 8);
        halve<1>(lo, 4, lane & 4), halve<1>(hi, 4, lane & 4);
        sums[2 * t] = lo[0], sums[2 * t + 1] = hi[0];
      }
      das[g * kLanes] = make_float4(da2[0].x + da2[0].y, da2[1].x + da2[1].y, da2[2].x + da2[2].y, da2[3].x + da2[3].y);
      // a lane holds dB (lane < 16) or dC of state (lane >> 2) & 3, for all tokens,
      // over a quarter of the lanes each
      halve<4>(sums, 2, lane & 2);
      halve<2>(sums, 1, lane & 1);
      {
        const int t = (lane & 2 ? 4 : 0) + (lane & 1 ? 2 : 0);
        float* to = rows + (t * 2 + (lane >> 4)) * p.np + 4 * g + ((lane >> 2) & 3);
        to[0] = sums[0], to[2 * p.np] = sums[1];
      }
      if (w == 0 && i == 0 && live && p.ds0) {
        float* ds0 = p.ds0 + ((long)b * p.D + d) * p.N + 4 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * g + j < p.N) ds0[j] = back[j];
      }
    }
    __syncwarp();
    {
      float4* part = reinterpret_cast<float4*>(p.part_bc + ((long)unit * p.T + t0) * p.np * 2);
      for (int e = lane; e < here * p.np / 2; e += 32) part[e] = reinterpret_cast<const float4*>(rows)[e];
    }
    if (live) {
      const long at0 = ((long)b * p.T + t0) * p.D + d;
      T* dx = static_cast<T*>(p.dx) + at0;
      T* ddt = static_cast<T*>(p.ddt) + at0;
      T* dz = z ? static_cast<T*>(p.dz) + at0 : nullptr;
#pragma unroll
      for (int t = 0; t < kTok / 2; ++t) {
        auto pair = [&](int which) {
          const T* at = in + which * kTile + 2 * t * kLanes + lane;
          return make_float2(to_f32(at[0]), to_f32(at[kLanes]));
        };
        const float2 xv = pair(0);
        const float2 gx = __ffma2_rn(step[t], sb[t], p.skip ? __fmul2_rn(twice(skip), gy[t]) : twice(0.0f));
        float2 raw = __ffma2_rn(xv, sb[t], __fmul2_rn(sa[t], twice(0.6931471805599453f)));  // rate is A / ln 2
        if (p.softplus) raw = __fmul2_rn(raw, sigmoid_of2(__fadd2_rn(pair(1), twice(bias))));
        float2 gz = twice(0.0f);
        if (z) {
          const float2 v = pair(3), s = sigmoid_of2(v), full = p.skip ? __ffma2_rn(twice(skip), xv, y[t]) : y[t];
          const float2 go = dout ? pair(2) : twice(0.0f), one = __ffma2_rn(v, make_float2(1.0f - s.x, 1.0f - s.y), twice(1.0f));
          gz = __fmul2_rn(__fmul2_rn(go, full), __fmul2_rn(s, one));
        }
        if (2 * t < here) {
          const long at = (long)(2 * t) * p.D;
          dx[at] = from_f32<T>(gx.x), ddt[at] = from_f32<T>(raw.x);
          if (z) dz[at] = from_f32<T>(gz.x);
          dbias += raw.x, dskip = fmaf(gy[t].x, xv.x, dskip);
        }
        if (2 * t + 1 < here) {
          const long at = (long)(2 * t + 1) * p.D;
          dx[at] = from_f32<T>(gx.y), ddt[at] = from_f32<T>(raw.y);
          if (z) dz[at] = from_f32<T>(gz.y);
          dbias += raw.y, dskip = fmaf(gy[t].y, xv.y, dskip);
        }
      }
    }
    __syncwarp();
  }
  float* sums = sm + l.sums;
  sums[w * kLanes + lane] = dskip;
  sums[(kWarps + w) * kLanes + lane] = dbias;
  __syncthreads();
  if (live) {
    const long at = (long)b * peers + rank;
    if (w < 2) {
      float s = 0.0f;
      for (int o = 0; o < kWarps; ++o) s += sums[(w * kWarps + o) * kLanes + lane];
      p.part_ch[(at * 2 + w) * p.D + d] = s;
    }
    const float4* all = reinterpret_cast<const float4*>(sm + l.da) + lane;
    for (int g = w; g < ng; g += kWarps) {
      float4 s = all[g * kLanes];
      for (int o = 1; o < kWarps; ++o) {
        const float4 v = all[(o * ng + g) * kLanes];
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
      float* part = p.part_a + (at * p.D + d) * p.N + 4 * g;
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * g + j < p.N) part[j] = v[j];
    }
  }
  if (Q) cluster_sync();  // no CTA leaves while another may still write to it
}

// dB and dC: the sums over a group's tiles of 32 channels, in their order.
template <typename T>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const Problem p) {
  const int np = p.np;
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
  const size_t smem = layout(p.np, sizeof(T)).total * sizeof(float);
  const int q = backward_sharing(p);
  LaunchScope scope(kKindSelectiveScan, stream, 4);
  const int rc = q > 1 ? launch_shared(scan_backward_kernel<T, true>, p, q, 32 * kWarps, smem, stream)
                       : launch_shared(scan_backward_kernel<T, false>, p, 1, 32 * kWarps, smem, stream);
  if (rc) return rc;
  const long sums = (long)p.B * p.T * p.G * 2 * p.np;
  sum_tiles_kernel<T><<<(unsigned)((sums + 255) / 256), 256, 0, stream>>>(p);
  GRU_CUDA_TRY(cudaGetLastError());
  const long an = (long)p.D * p.N;
  if (const int rc = sum_parts(p.part_a, p.B * q, an, an, StoreF32{p.da}, stream)) return rc;
  return sum_parts(p.part_ch, p.B * q, 2L * p.D, 2L * p.D, StoreChannels{p.dskip, p.dbias, p.D}, stream);
}

}  // namespace

int backward_sharing(const Problem& p) { return sharing(p, (p.T + kBlock - 1) / kBlock, kResident); }

int read_backward_status(int reset, int* status) {
  GRU_CUDA_TRY(cudaMemcpyFromSymbol(status, g_backward_status, sizeof(int)));
  if (reset) {
    const int zero = 0;
    GRU_CUDA_TRY(cudaMemcpyToSymbol(g_backward_status, &zero, sizeof(int)));
  }
  return GRU_OK;
}

int backward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? launch_backward<float>(p, stream) : launch_backward<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
