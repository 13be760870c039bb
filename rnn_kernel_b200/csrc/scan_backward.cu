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
// each, a warp four states, and goes over blocks of 16 tokens from the last to the
// first.  The forward kept the state before each block; from it a warp computes its
// states at eight tokens, with the decays, in registers, and then goes over the
// tokens backwards, first for the later eight (for them it passes the earlier ones
// once more: half an exponential, where twice as many kept states would cost as
// much in memory traffic).  The warps' shares of y, sum_n B dh and sum_n A w meet in
// shared memory, where each warp finishes four tokens.  Sums over channels are
// butterflies over the lanes in which each round halves the values: 64 values (8
// tokens, 4 states, dB and dC) take 62 exchanges and leave a lane two sums.  The
// tiles' sums of dB and dC are added by a second launch, in a fixed order, as are
// those over sequences of dA, dskip and dbias.  Segments as in the forward.
// Bound by instructions, 8 of them per token, channel and state for the sums over
// channels.

#include <algorithm>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {

namespace {

constexpr int kHalf = kBlock / 2;

// Shared memory in floats.
struct Lay {
  int step, du, gy, xs, sg, gz, bs, cs, part, marks, in, few, sums, total;
};
__host__ __device__ inline Lay layout(int warps, int N, int elem) {
  const int np = warps * kStates;
  Lay l;
  int n = 0;
  l.step = n, n += kBlock * kLanes;
  l.du = n, n += kBlock * kLanes;  // dt x
  l.gy = n, n += kBlock * kLanes;  // gradient of y
  l.xs = n, n += kBlock * kLanes;
  l.sg = n, n += kBlock * kLanes;  // softplus'
  l.gz = n, n += kBlock * kLanes;  // dout silu'(z)
  l.bs = n, n += np * kRow;
  l.cs = n, n += np * kRow;
  l.part = n, n += warps * 3 * kBlock * kLanes;  // [quad][y, sum B dh, sum A w][warp][lane] float4
  l.marks = n, n += np * kLanes;
  l.in = n, n += 4 * kBlock * kLanes * elem / 4;
  l.few = n, n += 2 * kBlock * N * elem / 4;
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

// SUM: only what the segments hand back.  MOST and W as in the forward.
template <typename T, bool SUM, int MOST, int W>
__global__ void __launch_bounds__(MOST, MOST == 128 ? 3 : 1) scan_backward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int warps = W ? W : blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31, np = warps * kStates;
  const Lay l = layout(warps, p.N, sizeof(T));
  const Place q = place(p);
  if (SUM && q.seg == 0) return;
  const T* x = static_cast<const T*>(p.x) + q.b * p.xb + q.d0;
  const T* dt = static_cast<const T*>(p.dt) + q.b * p.dtb + q.d0;
  const T* z = p.z ? static_cast<const T*>(p.z) + q.b * p.zb + q.d0 : nullptr;
  const T* bm = static_cast<const T*>(p.b) + q.b * p.bb + q.group * p.bg;
  const T* cm = static_cast<const T*>(p.c) + q.b * p.cb + q.group * p.cg;
  const long dense = (long)q.b * p.T * p.D + q.d;
  const T* dout = p.dout ? static_cast<const T*>(p.dout) + (long)q.b * p.T * p.D + q.d0 : nullptr;
  const float bias = p.bias ? p.bias[q.d] : 0.0f, skip = p.skip ? p.skip[q.d] : 0.0f;
  const int lastt = q.end - 1, n0 = kStates * w;
  T* in = reinterpret_cast<T*>(sm + l.in);
  T* few = reinterpret_cast<T*>(sm + l.few);
  constexpr int kTile = kBlock * kLanes;
  auto fetch = [&](int t0) {
    fetch_rows(in, x, p.xst, t0, lastt, q.width, p.wide_rows);
    fetch_rows(in + kTile, dt, p.dtst, t0, lastt, q.width, p.wide_rows);
    if (z) fetch_rows(in + 2 * kTile, z, p.zst, t0, lastt, q.width, p.wide_rows);
    if (dout) fetch_rows(in + 3 * kTile, dout, p.ost, t0, lastt, q.width, p.wide_rows && p.wide_dout);
    fetch_few(few, bm, p.bst, t0, lastt, p.N, p.wide_few);
    fetch_few(few + kBlock * p.N, cm, p.cst, t0, lastt, p.N, p.wide_few);
  };
  auto fetch_marks = [&](int t0) {
    const float4* from = reinterpret_cast<const float4*>(p.marks + ((long)q.unit * p.nmarks + t0 / kBlock) * np * kLanes);
    for (int e = threadIdx.x; e < np * kLanes / 4; e += blockDim.x) copy16(reinterpret_cast<float4*>(sm + l.marks) + e, from + e);
  };
  const int start = q.first + (lastt - q.first) / kBlock * kBlock;  // the last block
  fetch(start);
  if (!SUM) fetch_marks(start);

  float rt[kStates], back[kStates], da[kStates];
#pragma unroll
  for (int j = 0; j < kStates; ++j) {
    const bool in = q.live && n0 + j < p.N;
    rt[j] = in ? decay_rate(p.a[(long)q.d * p.N + n0 + j]) : 0.0f;
    back[j] = !SUM && in && p.dlast ? p.dlast[((long)q.b * p.D + q.d) * p.N + n0 + j] : 0.0f;
    da[j] = 0.0f;
  }
  if (!SUM)
    for (int s = p.segs - 1; s > q.seg; --s) {
      const long at = (long)q.unit * p.segs + s;
      const float steps = p.seg_steps[at * kLanes + lane];
#pragma unroll
      for (int j = 0; j < kStates; ++j)
        back[j] = fmaf(exp2_of(rt[j] * steps), back[j], p.seg_sums[(at * p.np + n0 + j) * kLanes + lane]);
    }

  float4* rows = reinterpret_cast<float4*>(sm) + lane;  // [array][quad][lane]
  const int a_step = l.step / 4, a_du = l.du / 4, a_gy = l.gy / 4, a_xs = l.xs / 4, a_sg = l.sg / 4, a_gz = l.gz / 4;
  float4* shares = reinterpret_cast<float4*>(sm + l.part) + lane;
  // What four tokens have per channel.
  auto prepare = [&](int t0) {
    for (int u = w; u < kQuads; u += warps) {
      const int t = t0 + 4 * u;
      float s[4], v[4], g[4] = {0.0f, 0.0f, 0.0f, 0.0f}, xv[4], sg[4], gz[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      quad_of(in, u, lane, xv);
      quad_of(in + kTile, u, lane, s);
      if (dout) quad_of(in + 3 * kTile, u, lane, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sg[i] = p.softplus ? gate_of(s[i] + bias) : 1.0f;
        s[i] = step_of(p.softplus, s[i], bias);
        v[i] = s[i] * xv[i];
      }
      if (z) {
        float zv[4];
        quad_of(in + 2 * kTile, u, lane, zv);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float c = gate_of(zv[i]);
          gz[i] = g[i] * (c * fmaf(zv[i], 1.0f - c, 1.0f));
          g[i] *= zv[i] * c;
        }
      }
      if (!q.live || t + 3 > lastt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!q.live || t + i > lastt) s[i] = v[i] = g[i] = 0.0f;
      float4* to = rows + u * kLanes;
      to[a_step] = as4(s), to[a_du] = as4(v), to[a_gy] = as4(g);
      if (!SUM) to[a_xs] = as4(xv), to[a_sg] = as4(sg), to[a_gz] = as4(gz);
      if (W) break;
    }
    turn_few(p, few, few + kBlock * p.N, sm + l.bs, sm + l.cs, np, q.end - t0);
  };
  float dskip = 0.0f, dbias = 0.0f;
  // Four tokens' sums over the states, and what follows from them.
  auto finish_quad = [&](int u, int t) {
    float4 sum[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const float4* part = shares + (u * 3 + i) * warps * kLanes;
      sum[i] = part[0];
#pragma unroll (W ? W : 4)
      for (int k = 1; k < warps; ++k) sum[i] = add4(sum[i], part[k * kLanes]);
    }
    if (!q.live) return;
    const float4* of = rows + u * kLanes;
    const float4 s4 = of[a_step], g4 = of[a_gy], x4 = of[a_xs], sg4 = of[a_sg], gz4 = of[a_gz];
    const float y[4] = {sum[0].x, sum[0].y, sum[0].z, sum[0].w}, sb[4] = {sum[1].x, sum[1].y, sum[1].z, sum[1].w};
    const float sa[4] = {sum[2].x, sum[2].y, sum[2].z, sum[2].w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
    const float g[4] = {g4.x, g4.y, g4.z, g4.w}, xv[4] = {x4.x, x4.y, x4.z, x4.w}, sg[4] = {sg4.x, sg4.y, sg4.z, sg4.w};
    const float gz[4] = {gz4.x, gz4.y, gz4.z, gz4.w};
    T* dx = row_at(static_cast<T*>(p.dx) + dense, t, p.ost);
    T* ddt = row_at(static_cast<T*>(p.ddt) + dense, t, p.ost);
    T* dz = z ? row_at(static_cast<T*>(p.dz) + dense, t, p.ost) : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t + i > lastt) break;
      const float raw = fmaf(xv[i], sb[i], sa[i] * 0.6931471805599453f) * sg[i];  // rt is A / ln 2
      *row_at(dx, i, p.ost) = from_f32<T>(fmaf(s[i], sb[i], p.skip ? skip * g[i] : 0.0f));
      *row_at(ddt, i, p.ost) = from_f32<T>(raw);
      if (z) *row_at(dz, i, p.ost) = from_f32<T>(gz[i] * (p.skip ? fmaf(skip, xv[i], y[i]) : y[i]));
      dbias += raw, dskip = fmaf(g[i], xv[i], dskip);
    }
  };
  auto finish = [&](int t0) {
    for (int u = w; u < kQuads; u += warps) {
      finish_quad(u, t0 + 4 * u);
      if (W) break;
    }
  };

  const float* bs = sm + l.bs + n0 * kRow;
  const float* cs = sm + l.cs + n0 * kRow;
  float total = 0.0f;
  // the lanes' rows of partial sums
  float* bc = p.part_bc + (((long)q.unit * p.np + n0 + ((lane >> 2) & 3)) * 2 + (lane >> 4)) * p.T;
  const int mine = (lane & 2 ? 4 : 0) + (lane & 1 ? 2 : 0);
  copies_done();
  __syncthreads();
  prepare(start);
  __syncthreads();
  for (int t0 = start; t0 >= q.first; t0 -= kBlock) {
    const bool more = t0 > q.first;
    // what a quad's tokens make of the warp's states; their decays and states are kept at a, h
    float a[kStates][kHalf], h[kStates][kHalf];
    auto scan = [&](int t, float (&st)[kStates], bool keep, int at) {
      const float4 s = rows[a_step + t * kLanes], u = rows[a_du + t * kLanes];
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
        const float2 e0 = __fmul2_rn(lo(s), twice(rt[j])), e1 = __fmul2_rn(hi(s), twice(rt[j]));
        const float2 v0 = __fmul2_rn(lo(u), lo(bv)), v1 = __fmul2_rn(hi(u), hi(bv));
        const float c[4] = {exp2_of(e0.x), exp2_of(e0.y), exp2_of(e1.x), exp2_of(e1.y)}, v[4] = {v0.x, v0.y, v1.x, v1.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          st[j] = fmaf(c[i], st[j], v[i]);
          if (keep) a[j][at + i] = c[i], h[j][at + i] = st[j];
        }
      }
    };
    float h0[kStates];
    if (!SUM) {
#pragma unroll
      for (int j = 0; j < kStates; ++j) h0[j] = sm[l.marks + (n0 + j) * kLanes + lane];
    }
    if (more) fetch(t0 - kBlock);
#pragma unroll
    for (int half = 1; half >= 0; --half) {
      constexpr int kQ = kHalf / 4;
      float before[kStates];  // the state before these tokens
      if (!SUM) {
        float st[kStates];
#pragma unroll
        for (int j = 0; j < kStates; ++j) st[j] = h0[j];
        if (half)
#pragma unroll
          for (int t = 0; t < kQ; ++t) scan(t, st, false, 0);
#pragma unroll
        for (int j = 0; j < kStates; ++j) before[j] = st[j];
#pragma unroll
        for (int t = 0; t < kQ; ++t) scan(half * kQ + t, st, true, 4 * t);
      }
      float sums[kHalf];
      float2 da2[kStates];
#pragma unroll
      for (int j = 0; j < kStates; ++j) da2[j] = twice(0.0f);
#pragma unroll
      for (int tt = kQ - 1; tt >= 0; --tt) {
        const int t = half * kQ + tt;
        const float4 s = rows[a_step + t * kLanes], gv = rows[a_gy + t * kLanes];
        if (SUM) {
          total += (s.x + s.y) + (s.z + s.w);
#pragma unroll
          for (int j = 0; j < kStates; ++j) {
            const float4 cv = *reinterpret_cast<const float4*>(cs + j * kRow + 4 * t);
            back[j] = exp2_of(s.w * rt[j]) * fmaf(cv.w, gv.w, back[j]);
            back[j] = exp2_of(s.z * rt[j]) * fmaf(cv.z, gv.z, back[j]);
            back[j] = exp2_of(s.y * rt[j]) * fmaf(cv.y, gv.y, back[j]);
            back[j] = exp2_of(s.x * rt[j]) * fmaf(cv.x, gv.x, back[j]);
          }
          continue;
        }
        const float4 u = rows[a_du + t * kLanes];
        float2 y0 = twice(0.0f), y1 = y0, b0 = y0, b1 = y0, w0 = y0, w1 = y0;
        float v[kStates * 4];  // [state][token]: of dB in the lower lanes, of dC in the upper
#pragma unroll
        for (int j = 0; j < kStates; ++j) {
          const float4 cv = *reinterpret_cast<const float4*>(cs + j * kRow + 4 * t);
          const float4 bv = *reinterpret_cast<const float4*>(bs + j * kRow + 4 * t);
          const float* aj = &a[j][4 * tt];
          const float2 h01 = make_float2(h[j][4 * tt], h[j][4 * tt + 1]), h23 = make_float2(h[j][4 * tt + 2], h[j][4 * tt + 3]);
          const float2 g0 = __fmul2_rn(lo(cv), lo(gv)), g1 = __fmul2_rn(hi(cv), hi(gv));
          float2 d0, d1, r0, r1;
          d1.y = g1.y + back[j];
          r1.y = aj[3] * d1.y;
          d1.x = g1.x + r1.y;
          r1.x = aj[2] * d1.x;
          d0.y = g0.y + r1.x;
          r0.y = aj[1] * d0.y;
          d0.x = g0.x + r0.y;
          r0.x = back[j] = aj[0] * d0.x;
          r0.x *= tt ? h[j][tt ? 4 * tt - 1 : 0] : before[j];  // w
          r0.y *= h01.x, r1.x *= h01.y, r1.y *= h23.x;
          y0 = __ffma2_rn(lo(cv), h01, y0), y1 = __ffma2_rn(hi(cv), h23, y1);
          b0 = __ffma2_rn(lo(bv), d0, b0), b1 = __ffma2_rn(hi(bv), d1, b1);
          w0 = __ffma2_rn(twice(rt[j]), r0, w0), w1 = __ffma2_rn(twice(rt[j]), r1, w1);
          da2[j] = __ffma2_rn(lo(s), r0, da2[j]);
          da2[j] = __ffma2_rn(hi(s), r1, da2[j]);
          const float2 vb0 = __fmul2_rn(d0, lo(u)), vb1 = __fmul2_rn(d1, hi(u));
          const float2 vc0 = __fmul2_rn(lo(gv), h01), vc1 = __fmul2_rn(hi(gv), h23);
          float m[8] = {vb0.x, vb0.y, vb1.x, vb1.y, vc0.x, vc0.y, vc1.x, vc1.y};
          halve<4>(m, 16, lane & 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * j + i] = m[i];
        }
        shares[(3 * t + 0) * warps * kLanes + w * kLanes] = make_float4(y0.x, y0.y, y1.x, y1.y);
        shares[(3 * t + 1) * warps * kLanes + w * kLanes] = make_float4(b0.x, b0.y, b1.x, b1.y);
        shares[(3 * t + 2) * warps * kLanes + w * kLanes] = make_float4(w0.x, w0.y, w1.x, w1.y);
        halve<8>(v, 8, lane & 8);
        halve<4>(v, 4, lane & 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[4 * tt + i] = v[i];
      }
      if (SUM) continue;
#pragma unroll
      for (int j = 0; j < kStates; ++j) da[j] += da2[j].x + da2[j].y;  // short sums first
      // a lane holds dB (lane < 16) or dC of state (lane >> 2) & 3, for all eight
      // tokens, over a quarter of the lanes each
      halve<4>(sums, 2, lane & 2);
      halve<2>(sums, 1, lane & 1);
      const int t = t0 + half * kHalf + mine;
      if (t <= lastt) bc[t] = sums[0];
      if (t < lastt) bc[t + 1] = sums[1];
    }
    copies_done();
    __syncthreads();
    if (!SUM && more) fetch_marks(t0 - kBlock);
    if (!SUM) finish(t0);
    // finish() reads the quads of this block that prepare() overwrites: the warp's own
    if (more) prepare(t0 - kBlock);
    copies_done();
    __syncthreads();
  }
  if (SUM) {
    const long at = (long)q.unit * p.segs + q.seg;
#pragma unroll
    for (int j = 0; j < kStates; ++j) p.seg_sums[(at * p.np + n0 + j) * kLanes + lane] = back[j];
    if (w == 0) p.seg_steps[at * kLanes + lane] = total;
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
  for (int j = 0; j < kStates; ++j) {
    const int n = n0 + j;
    if (n >= p.N) continue;
    p.part_a[(at * p.D + q.d) * p.N + n] = da[j];
    if (q.seg == 0 && p.ds0) p.ds0[((long)q.b * p.D + q.d) * p.N + n] = back[j];
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

template <typename T, int MOST, int W>
int launch_backward(const Problem& p, cudaStream_t stream) {
  const int warps = p.np / kStates;
  const size_t smem = layout(warps, p.N, sizeof(T)).total * sizeof(float);
  const unsigned ctas = (unsigned)((long)p.B * p.tiles * p.segs);
  LaunchScope scope(kKindSelectiveScan, stream, p.segs > 1 ? 5 : 4);
  if (p.segs > 1) {
    auto kernel = scan_backward_kernel<T, true, MOST, W>;
    GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<ctas, 32 * warps, smem, stream>>>(p);
    GRU_CUDA_TRY(cudaGetLastError());
  }
  auto kernel = scan_backward_kernel<T, false, MOST, W>;
  GRU_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<ctas, 32 * warps, smem, stream>>>(p);
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
  if (p.np == 16) return launch_backward<T, 128, 4>(p, stream);
  return p.np < 16 ? launch_backward<T, 128, 0>(p, stream) : launch_backward<T, 512, 0>(p, stream);
}

}  // namespace

int backward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? backward_of<float>(p, stream) : backward_of<bf16>(p, stream);
}

}  // namespace scan
}  // namespace gru
