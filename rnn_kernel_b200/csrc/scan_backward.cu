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
// warp.  The forward kept the state before each block.  For two states at a time a
// warp computes its tokens' decays once and from them its tokens' effect on the
// state (P h + S) and on what is handed back (P r + R); both meet the other
// warps' in shared memory, and the warp goes over its tokens forwards for h and
// backwards for the gradients.  Sums over channels are butterflies over the
// lanes in which each round halves the values: 32 values (8 tokens, 2 states, dB
// and dC) take 31 exchanges and leave a lane one sum.  The tiles' sums of dB and
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
constexpr int kResident = 4;       // CTAs an SM holds, by registers
static_assert(kBlock == kMark, "the forward keeps the state before each block");

// Shared memory in floats.
struct Lay {
  int bars, bs, cs, ex, carry, rate, da, rows, sums, total;
};
__host__ __device__ inline Lay layout(int ng) {
  Lay l;
  int n = 0;
  l.bars = n, n += 2 * ng * 2;
  n = (n + 3) / 4 * 4;
  l.bs = n, n += kWarps * ng * 2 * kRow;
  l.cs = n, n += kWarps * ng * 2 * kRow;
  l.ex = n, n += 2 * kWarps * 3 * kLanes * 2;
  l.carry = n, n += 2 * ng * kLanes * 2;
  l.rate = n, n += ng * kLanes * 2;
  l.da = n, n += kWarps * ng * kLanes * 2;
  l.rows = n, n += kWarps * kTok * ng * 4;
  l.sums = n, n += 2 * kWarps * kLanes;
  l.total = n;
  return l;
}

__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }

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
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lay l = layout(p.ng);
  const int rank = Q ? (int)cluster_rank() : 0, peers = Q ? (int)cluster_size() : 1;
  const int unit = blockIdx.x / peers, tile = unit % p.tiles, b = unit / p.tiles;
  const int group = tile / p.per_group, local = (tile - group * p.per_group) * kLanes + lane;
  const bool live = local < p.R;
  const int d = group * p.R + (live ? local : 0);
  float* bs = sm + l.bs + w * p.ng * 2 * kRow;
  float* cs = sm + l.cs + w * p.ng * 2 * kRow;
  float* rows = sm + l.rows + w * kTok * p.ng * 4;  // [token][dB, dC][state]
  float2* ex = reinterpret_cast<float2*>(sm + l.ex) + lane;
  float2* carry = reinterpret_cast<float2*>(sm + l.carry) + lane;
  float2* rate = reinterpret_cast<float2*>(sm + l.rate) + lane;
  float2* das = reinterpret_cast<float2*>(sm + l.da) + w * p.ng * kLanes + lane;
  const uint32_t bars = smem_at(sm + l.bars);

  const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
  const int blocks = (p.T + kBlock - 1) / kBlock;
  for (int g = w; g < p.ng; g += kWarps) {
    float r[2], s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = 2 * g + j;
      r[j] = live && n < p.N ? decay_rate(p.a[(long)d * p.N + n]) : 0.0f;
      s[j] = live && n < p.N && p.dlast ? p.dlast[((long)b * p.D + d) * p.N + n] : 0.0f;
    }
    rate[g * kLanes] = make_float2(r[0], r[1]);
    if (rank == 0) carry[g * kLanes] = make_float2(s[0], s[1]);
  }
  for (int g = 0; g < p.ng; ++g) das[g * kLanes] = twice(0.0f);
  if (Q) {  // the barrier of slot k & 1 counts the bytes of what is handed back to this CTA's k-th block
    if (threadIdx.x == 0) {
      for (int i = 0; i < 2 * p.ng; ++i) bar_init(bars + 8 * i);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      for (int i = 0; i < 2 * p.ng; ++i)
        if (rank == 0 && i < p.ng) bar_arrive(bars + 8 * i);  // the last state's gradient is there
        else bar_expect(bars + 8 * i, kLanes * 8);
    }
    __syncthreads();
    cluster_sync();
  }
  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + d;
  const T* dt = static_cast<const T*>(p.dt) + b * p.dts[0] + d;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.zs[0] + d : nullptr;
  const T* bm = static_cast<const T*>(p.b) + b * p.bs[0] + group * p.bs[2];
  const T* cm = static_cast<const T*>(p.c) + b * p.cs[0] + group * p.cs[2];
  const long dense = (long)b * p.T * p.D + d;
  const T* dout = p.dout ? static_cast<const T*>(p.dout) + dense : nullptr;
  float dskip = 0.0f, dbias = 0.0f;
  if (!Q) __syncthreads();

  int turn = 0;
  bool ok = true;
  for (int step_i = rank, k = 0; step_i < blocks; step_i += peers, ++k) {
    const int i = blocks - 1 - step_i;
    const int t0 = i * kBlock + w * kTok, here = min(max(p.T - t0, 0), kTok);
    float2 step[kTok / 2], du[kTok / 2], gy[kTok / 2];
    float sdt = 0.0f;
    {
      float raw[kTok], xv[kTok], gv[kTok];
      const T *px = x + t0 * p.xs[1], *pd = dt + t0 * p.dts[1], *pg = dout + (dout ? (long)t0 * p.D : 0);
#pragma unroll
      for (int t = 0; t < kTok; ++t, px += p.xs[1], pd += p.dts[1], pg += p.D) {
        const bool in = live && t < here;
        xv[t] = in ? to_f32(*px) : 0.0f;
        raw[t] = in ? to_f32(*pd) : 0.0f;
        gv[t] = in && dout ? to_f32(*pg) : 0.0f;
      }
      if (z) {
        const T* pz = z + t0 * p.zs[1];
        float zv[kTok];
#pragma unroll
        for (int t = 0; t < kTok; ++t, pz += p.zs[1]) zv[t] = live && t < here ? to_f32(*pz) : 0.0f;
#pragma unroll
        for (int t = 0; t < kTok; ++t) gv[t] *= zv[t] * sigmoid_of(zv[t]);
      }
      __syncwarp();
      const int lanes = 1 << p.wide, n = lane & (lanes - 1);
#pragma unroll 4
      for (int e = lane; e < kTok << p.wide; e += 32) {
        const int t = e >> p.wide, m = lanes <= 32 ? n : e & (lanes - 1);
        const bool in = t < here && m < p.N;
        const float bv = in ? to_f32(bm[(t0 + t) * p.bs[1] + m]) : 0.0f;
        const float cv = in ? to_f32(cm[(t0 + t) * p.cs[1] + m]) : 0.0f;
        if (m < 2 * p.ng) bs[m * kRow + t] = bv, cs[m * kRow + t] = cv;
      }
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        raw[t] = live && t < here ? step_of(p, raw[t], bias) : 0.0f;
        sdt += raw[t];
      }
#pragma unroll
      for (int t = 0; t < kTok / 2; ++t) {
        step[t] = make_float2(raw[2 * t], raw[2 * t + 1]);
        du[t] = __fmul2_rn(step[t], make_float2(xv[2 * t], xv[2 * t + 1]));
        gy[t] = make_float2(gv[2 * t], gv[2 * t + 1]);
      }
    }
    float2 y[kTok / 2], sb[kTok / 2], sa[kTok / 2];
#pragma unroll
    for (int t = 0; t < kTok / 2; ++t) y[t] = sb[t] = sa[t] = twice(0.0f);
    __syncwarp();
#pragma unroll 1
    for (int g = 0; g < p.ng; ++g, turn ^= 1) {
      const float2 rt = rate[g * kLanes];
      const float2 mark = reinterpret_cast<const float2*>(p.marks)[(((long)unit * p.nmarks + i) * p.ng + g) * kLanes + lane];
      float a[2][kTok], s[2], r[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 r2 = twice(j ? rt.y : rt.x);
        const float4* b4 = reinterpret_cast<const float4*>(bs + (2 * g + j) * kRow);
        const float4* c4 = reinterpret_cast<const float4*>(cs + (2 * g + j) * kRow);
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
      float2* e = ex + turn * kWarps * 3 * kLanes;
      const float2 mine = make_float2(exp2_of(sdt * rt.x), exp2_of(sdt * rt.y));
      e[(w * 3 + 0) * kLanes] = mine;
      e[(w * 3 + 1) * kLanes] = make_float2(s[0], s[1]);
      e[(w * 3 + 2) * kLanes] = make_float2(r[0], r[1]);
      __syncthreads();
      float2 h2 = mark, q = twice(1.0f), v = twice(0.0f);
#pragma unroll
      for (int o = 0; o < kWarps - 1; ++o)
        if (o < w) h2 = __ffma2_rn(e[(o * 3 + 0) * kLanes], h2, e[(o * 3 + 1) * kLanes]);
#pragma unroll
      for (int o = kWarps - 1; o > 0; --o)
        if (o > w) {  // what the warps behind make of what is handed to the block
          const float2 pr = e[(o * 3 + 0) * kLanes];
          v = __ffma2_rn(pr, v, e[(o * 3 + 2) * kLanes]);
          q = __fmul2_rn(pr, q);
        }
      const int slot = (k & 1) * p.ng + g;
      if (Q && ok) ok = bar_wait(bars + 8 * slot, (k >> 1) & 1, &g_backward_status);
      const float2 first = carry[slot * kLanes];
      float2 back = __ffma2_rn(q, first, v);
      if (w == 0) {  // for the block before
        const float2 next = __ffma2_rn(mine, back, make_float2(r[0], r[1]));
        if (Q) {
          if (lane == 0 && step_i + 2 * peers < blocks) bar_expect(bars + 8 * slot, kLanes * 8);  // its use after the next
          __syncwarp();
          if (step_i + 1 < blocks) {
            const int to = (rank + 1) % peers, slot_to = (((step_i + 1) / peers) & 1) * p.ng + g;
            send(at_rank(smem_at(carry + slot_to * kLanes), to), next, at_rank(bars + 8 * slot_to, to));
          }
        } else {
          carry[(((k + 1) & 1) * p.ng + g) * kLanes] = next;
        }
      }
      float h[2][kTok];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4* b4 = reinterpret_cast<const float4*>(bs + (2 * g + j) * kRow);
        float hv = j ? h2.y : h2.x;
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
      const float2 da = das[g * kLanes];
      float2 da2[2] = {make_float2(da.x, 0.0f), make_float2(da.y, 0.0f)};
      float sums[kTok];
#pragma unroll
      for (int t = kTok / 2 - 1; t >= 0; --t) {
        float2 vb[2], vc[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 bv = *reinterpret_cast<const float2*>(bs + (2 * g + j) * kRow + 2 * t);
          const float2 cv = *reinterpret_cast<const float2*>(cs + (2 * g + j) * kRow + 2 * t);
          float& rj = j ? back.y : back.x;
          const float2 cg = __fmul2_rn(cv, gy[t]), hv = make_float2(h[j][2 * t], h[j][2 * t + 1]);
          float2 dh, rr;
          dh.y = cg.y + rj;
          rr.y = a[j][2 * t + 1] * dh.y;
          dh.x = cg.x + rr.y;
          rr.x = rj = a[j][2 * t] * dh.x;
          const float2 wt = make_float2(rr.x * (t ? h[j][2 * t - 1] : j ? h2.y : h2.x), rr.y * h[j][2 * t]);
          y[t] = __ffma2_rn(cv, hv, y[t]);
          sb[t] = __ffma2_rn(bv, dh, sb[t]);
          sa[t] = __ffma2_rn(twice(j ? rt.y : rt.x), wt, sa[t]);
          da2[j] = __ffma2_rn(step[t], wt, da2[j]);
          vb[j] = __fmul2_rn(dh, du[t]);
          vc[j] = __fmul2_rn(gy[t], hv);
        }
        float lo[4] = {vb[0].x, vb[1].x, vc[0].x, vc[1].x}, hi[4] = {vb[0].y, vb[1].y, vc[0].y, vc[1].y};
        halve<2>(lo, 16, lane & 16), halve<2>(hi, 16, lane & 16);
        halve<1>(lo, 8, lane & 8), halve<1>(hi, 8, lane & 8);
        sums[2 * t] = lo[0], sums[2 * t + 1] = hi[0];
      }
      das[g * kLanes] = make_float2(da2[0].x + da2[0].y, da2[1].x + da2[1].y);
      // a lane holds dB (lane < 16) or dC of state (lane >> 3) & 1, for all tokens,
      // over an eighth of the lanes each
      halve<4>(sums, 4, lane & 4);
      halve<2>(sums, 2, lane & 2);
      halve<1>(sums, 1, lane & 1);
      rows[((lane & 7) * 2 + (lane >> 4)) * p.ng * 2 + 2 * g + ((lane >> 3) & 1)] = sums[0];
      if (w == 0 && i == 0 && live && p.ds0) {
        float* ds0 = p.ds0 + ((long)b * p.D + d) * p.N + 2 * g;
        ds0[0] = back.x;
        if (2 * g + 1 < p.N) ds0[1] = back.y;
      }
    }
    __syncwarp();
    {
      float* part = p.part_bc + ((long)unit * p.T + t0) * p.ng * 4;
      for (int e = lane; e < here * p.ng * 4; e += 32) part[e] = rows[e];
    }
    if (!live) continue;
    const T *px = x + t0 * p.xs[1], *pd = dt + t0 * p.dts[1];
    long at = dense + (long)t0 * p.D;
#pragma unroll
    for (int t = 0; t < kTok; ++t, px += p.xs[1], pd += p.dts[1], at += p.D) {
      if (t >= here) continue;
      const float st = t & 1 ? step[t / 2].y : step[t / 2].x, gv = t & 1 ? gy[t / 2].y : gy[t / 2].x;
      const float sbt = t & 1 ? sb[t / 2].y : sb[t / 2].x, sat = t & 1 ? sa[t / 2].y : sa[t / 2].x;
      const float xt = to_f32(*px);
      static_cast<T*>(p.dx)[at] = from_f32<T>(fmaf(st, sbt, p.skip ? skip * gv : 0.0f));
      float raw = fmaf(xt, sbt, sat * 0.6931471805599453f);  // rate is A / ln 2
      if (p.softplus) raw *= sigmoid_of(to_f32(*pd) + bias);
      static_cast<T*>(p.ddt)[at] = from_f32<T>(raw);
      dbias += raw;
      dskip = fmaf(gv, xt, dskip);
      if (z) {
        const float v = to_f32(z[(t0 + t) * p.zs[1]]), g = sigmoid_of(v), yt = t & 1 ? y[t / 2].y : y[t / 2].x;
        const float full = p.skip ? fmaf(skip, xt, yt) : yt, go = dout ? to_f32(dout[(long)(t0 + t) * p.D]) : 0.0f;
        static_cast<T*>(p.dz)[at] = from_f32<T>(go * full * g * fmaf(v, 1.0f - g, 1.0f));
      }
    }
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
    const float2* all = reinterpret_cast<const float2*>(sm + l.da) + lane;
    for (int g = w; g < p.ng; g += kWarps) {
      float2 s = all[g * kLanes];
      for (int o = 1; o < kWarps; ++o) {
        const float2 v = all[(o * p.ng + g) * kLanes];
        s.x += v.x, s.y += v.y;
      }
      float* part = p.part_a + (at * p.D + d) * p.N + 2 * g;
      part[0] = s.x;
      if (2 * g + 1 < p.N) part[1] = s.y;
    }
  }
  if (Q) cluster_sync();  // no CTA leaves while another may still write to it
}

// dB and dC: the sums over a group's tiles of 32 channels, in their order.
template <typename T>
__global__ void __launch_bounds__(256) sum_tiles_kernel(const Problem p) {
  const int np = p.ng * 2;
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
  const int q = backward_sharing(p);
  LaunchScope scope(kKindSelectiveScan, stream, 4);
  const int rc = q > 1 ? launch_shared(scan_backward_kernel<T, true>, p, q, 32 * kWarps, smem, stream)
                       : launch_shared(scan_backward_kernel<T, false>, p, 1, 32 * kWarps, smem, stream);
  if (rc) return rc;
  const long sums = (long)p.B * p.T * p.G * 2 * p.ng * 2;
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
