// Forward of the selective scan over all tokens.
//
//   h[n] = e^{dt A[n]} h[n] + dt x B[n];   y = sum_n C[n] h[n] + skip x;   out = y silu(z)
//
// A CTA owns 32 channels of one sequence, a lane each, and goes over the time in
// blocks of 64 tokens, 16 a warp.  For two states at a time a warp computes its
// tokens' decays once (kept in registers), and from them what its tokens make of
// a state: h -> P h + S with P = e^{A sum dt}.  The warps' P and S meet in shared
// memory; each warp then has the state before its first token from those ahead
// of it, and goes over its tokens again with that.  Two neighbouring tokens share
// each packed FP32 operation but the recurrence itself; B and C lie by state in
// shared memory, so that one broadcast read serves four tokens of 32 channels.
//
// Where sequences and channels do not fill the GPU, up to eight CTAs of a cluster
// share a sequence's channels and take its blocks in turn: a block's last state
// goes to the next CTA's shared memory (st.async, counted by a barrier of the
// receiver) as soon as the one before has come, two operations behind it; all
// else of a block runs beside the other CTAs'.
// One exponential per token, channel and state (16 a cycle and SM) is the bound.

#include <algorithm>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {

__device__ int g_forward_status = 0;

namespace {

constexpr int kTok = 16;           // tokens of a warp
constexpr int kRow = kTok + 4;     // floats between two states' tokens in shared memory
constexpr int kBlock = kWarps * kTok;
constexpr int kResident = 4;       // CTAs an SM holds, by registers

// Shared memory in floats; ng: pairs of states, elem: bytes of an element.
struct Lay {
  int bars, in, bs, cs, ex, carry, rate, total;
};
__host__ __device__ inline Lay layout(int ng, int elem) {
  Lay l;
  int n = 0;
  l.bars = n, n += (2 * ng * 2 + 3) / 4 * 4;
  l.in = n, n += kWarps * 3 * kTok * kLanes * elem / 4;
  l.bs = n, n += kWarps * ng * 2 * kRow;
  l.cs = n, n += kWarps * ng * 2 * kRow;
  l.ex = n, n += 2 * kWarps * kLanes * 4;
  l.carry = n, n += 2 * ng * kLanes * 2;
  l.rate = n, n += ng * kLanes * 2;
  l.total = n;
  return l;
}

// Q: several CTAs share a tile, as a cluster.
template <typename T, bool Q>
__global__ void __launch_bounds__(32 * kWarps, kResident) scan_forward_kernel(const __grid_constant__ Problem p) {
  extern __shared__ __align__(16) float sm[];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, ng = (p.N + 1) / 2;
  const Lay l = layout(ng, sizeof(T));
  const int rank = Q ? (int)cluster_rank() : 0, peers = Q ? (int)cluster_size() : 1;
  const int unit = blockIdx.x / peers, tile = unit % p.tiles, b = unit / p.tiles;
  const int group = tile / p.per_group, c0 = (tile - group * p.per_group) * kLanes;
  const int width = min(p.R - c0, kLanes), d0 = group * p.R + c0;
  const bool live = lane < width;
  const int d = d0 + (live ? lane : 0);
  T* xs = reinterpret_cast<T*>(sm + l.in) + w * 3 * kTok * kLanes;  // x, dt, z
  T *ds = xs + kTok * kLanes, *zs = ds + kTok * kLanes;
  float* bs = sm + l.bs + w * ng * 2 * kRow;
  float* cs = sm + l.cs + w * ng * 2 * kRow;
  float4* ex = reinterpret_cast<float4*>(sm + l.ex) + lane;
  float2* carry = reinterpret_cast<float2*>(sm + l.carry) + lane;
  float2* rate = reinterpret_cast<float2*>(sm + l.rate) + lane;
  const uint32_t bars = smem_at(sm + l.bars);

  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + d0;
  const T* dt = static_cast<const T*>(p.dt) + b * p.dts[0] + d0;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.zs[0] + d0 : nullptr;
  const T* bm = static_cast<const T*>(p.b) + b * p.bs[0] + group * p.bs[2];
  const T* cm = static_cast<const T*>(p.c) + b * p.cs[0] + group * p.cs[2];
  T* out = static_cast<T*>(p.out) + (long)b * p.T * p.D + d;
  const bool async = p.pairs && (sizeof(T) == 4 || width % 2 == 0);
  auto fetch = [&](const T* src, long stride, int i, T* dst) {
    const int t0 = i * kBlock + w * kTok;
    if (t0 < p.T) fetch_rows<T, kTok>(src + t0 * stride, stride, p.T - t0, width, async, dst);
  };
  fetch(x, p.xs[1], rank, xs);
  fetch(dt, p.dts[1], rank, ds);
  copies_issued();  // x and dt, then z, block after block: what is waited for is always the last but one
  if (z) fetch(z, p.zs[1], rank, zs);
  copies_issued();

  const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
  for (int g = w; g < ng; g += kWarps) {
    float r[2], s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = 2 * g + j;
      r[j] = live && n < p.N ? decay_rate(p.a[(long)d * p.N + n]) : 0.0f;
      s[j] = live && n < p.N && p.s0 ? p.s0[((long)b * p.D + d) * p.N + n] : 0.0f;
    }
    rate[g * kLanes] = make_float2(r[0], r[1]);
    if (rank == 0) carry[g * kLanes] = make_float2(s[0], s[1]);
  }
  if (Q) {  // the barrier of slot k & 1 counts the bytes of the state before this CTA's k-th block
    if (threadIdx.x == 0) {
      for (int i = 0; i < 2 * ng; ++i) bar_init(bars + 8 * i);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      for (int i = 0; i < 2 * ng; ++i)
        if (rank == 0 && i < ng) bar_arrive(bars + 8 * i);  // the initial state is there
        else bar_expect(bars + 8 * i, kLanes * 8);
    }
    __syncthreads();
    cluster_sync();
  } else {
    __syncthreads();
  }

  int turn = 0;
  bool ok = true;
  const int blocks = (p.T + kBlock - 1) / kBlock;
  for (int i = rank, k = 0; i < blocks; i += peers, ++k) {
    const int t0 = i * kBlock + w * kTok, here = min(max(p.T - t0, 0), kTok);
    float2 step[kTok / 2], du[kTok / 2], y[kTok / 2];
    float sdt = 0.0f;
    {
      FewRows<T, kTok, kRow> few;
      const T *pb = bm + t0 * p.bs[1], *pc = cm + t0 * p.cs[1];
      few.load(p, pb, pc, here, 0);
      copies_done<1>();
      __syncwarp();
#pragma unroll
      for (int t = 0; t < kTok / 2; ++t) {
        const float2 v = make_float2(to_f32(xs[2 * t * kLanes + lane]), to_f32(xs[(2 * t + 1) * kLanes + lane]));
        float2 s = step_of(p.softplus, make_float2(to_f32(ds[2 * t * kLanes + lane]), to_f32(ds[(2 * t + 1) * kLanes + lane])), bias);
        if (here < kTok) s.x = 2 * t < here ? s.x : 0.0f, s.y = 2 * t + 1 < here ? s.y : 0.0f;
        step[t] = s;
        du[t] = __fmul2_rn(s, v);
        if (here < kTok) du[t].x = 2 * t < here ? du[t].x : 0.0f, du[t].y = 2 * t + 1 < here ? du[t].y : 0.0f;
        y[t] = p.skip ? __fmul2_rn(twice(skip), v) : twice(0.0f);
        sdt += s.x + s.y;
      }
      few.store(p, bs, cs, 2 * ng, 0);
      few.rest(p, pb, pc, here, bs, cs, 2 * ng);
      __syncwarp();
      if (i + peers < blocks) {
        fetch(x, p.xs[1], i + peers, xs);
        fetch(dt, p.dts[1], i + peers, ds);
      }
      copies_issued();
    }
#pragma unroll 1
    for (int g = 0; g < ng; ++g, turn ^= 1) {
      const float2 rt = rate[g * kLanes];
      float a[2][kTok], s[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 r2 = twice(j ? rt.y : rt.x);
        const float4* b4 = reinterpret_cast<const float4*>(bs + (2 * g + j) * kRow);
        s[j] = 0.0f;
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
      }
      float4* e = ex + turn * kWarps * kLanes;
      const float2 mine = make_float2(exp2_of(sdt * rt.x), exp2_of(sdt * rt.y));
      e[w * kLanes] = make_float4(mine.x, mine.y, s[0], s[1]);
      __syncthreads();
      // what the warps ahead make of the block's first state
      float2 q = twice(1.0f), v = twice(0.0f);
#pragma unroll
      for (int r = 0; r < kWarps - 1; ++r)
        if (r < w) {
          const float4 o = e[r * kLanes];
          v = __ffma2_rn(make_float2(o.x, o.y), v, make_float2(o.z, o.w));
          q = __fmul2_rn(make_float2(o.x, o.y), q);
        }
      const int slot = (k & 1) * ng + g;
      if (Q && ok) ok = bar_wait(bars + 8 * slot, (k >> 1) & 1, &g_forward_status);
      const float2 first = carry[slot * kLanes];
      float2 h2 = __ffma2_rn(q, first, v);
      if (w == kWarps - 1) {  // the state behind the block, for the next
        const float2 next = __ffma2_rn(mine, h2, make_float2(s[0], s[1]));
        if (Q) {
          if (lane == 0 && i + 2 * peers < blocks) bar_expect(bars + 8 * slot, kLanes * 8);  // its use after the next
          __syncwarp();
          if (i + 1 < blocks) {
            const int to = (rank + 1) % peers, slot_to = (((i + 1) / peers) & 1) * ng + g;
            send(at_rank(smem_at(carry + slot_to * kLanes), to), next, at_rank(bars + 8 * slot_to, to));
          }
        } else {
          carry[(((k + 1) & 1) * ng + g) * kLanes] = next;
        }
      }
      if (p.marks && t0 % kMark == 0 && here > 0) {
        float* mark = p.marks + (((long)unit * p.nmarks + t0 / kMark) * p.np + 2 * g) * kLanes + lane;
        mark[0] = h2.x, mark[kLanes] = h2.y;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4* b4 = reinterpret_cast<const float4*>(bs + (2 * g + j) * kRow);
        const float4* c4 = reinterpret_cast<const float4*>(cs + (2 * g + j) * kRow);
        float h = j ? h2.y : h2.x;
#pragma unroll
        for (int t = 0; t < kTok / 4; ++t) {
          const float4 bv = b4[t], cv = c4[t];
          const float2 v0 = __fmul2_rn(du[2 * t], make_float2(bv.x, bv.y)), v1 = __fmul2_rn(du[2 * t + 1], make_float2(bv.z, bv.w));
          float2 h0, h1;
          h0.x = fmaf(a[j][4 * t], h, v0.x);
          h0.y = fmaf(a[j][4 * t + 1], h0.x, v0.y);
          h1.x = fmaf(a[j][4 * t + 2], h0.y, v1.x);
          h1.y = fmaf(a[j][4 * t + 3], h1.x, v1.y);
          h = h1.y;
          y[2 * t] = __ffma2_rn(make_float2(cv.x, cv.y), h0, y[2 * t]);
          y[2 * t + 1] = __ffma2_rn(make_float2(cv.z, cv.w), h1, y[2 * t + 1]);
        }
        s[j] = h;
      }
      if (w == kWarps - 1 && i == blocks - 1 && live) {
        float* last = p.last + ((long)b * p.D + d) * p.N + 2 * g;
        last[0] = s[0];
        if (2 * g + 1 < p.N) last[1] = s[1];
      }
    }
    copies_done<1>();
    __syncwarp();
    if (z) {
#pragma unroll
      for (int t = 0; t < kTok / 2; ++t) {
        const float2 v = make_float2(to_f32(zs[2 * t * kLanes + lane]), to_f32(zs[(2 * t + 1) * kLanes + lane]));
        y[t] = __fmul2_rn(y[t], __fmul2_rn(v, sigmoid_of2(v)));
      }
      __syncwarp();
      if (i + peers < blocks) fetch(z, p.zs[1], i + peers, zs);
    }
    copies_issued();
    if (live) {
      T* po = out + (long)t0 * p.D;
      if (here == kTok) {
#pragma unroll
        for (int t = 0; t < kTok; ++t, po += p.D) *po = from_f32<T>(t & 1 ? y[t / 2].y : y[t / 2].x);
      } else {
#pragma unroll
        for (int t = 0; t < kTok; ++t, po += p.D)
          if (t < here) *po = from_f32<T>(t & 1 ? y[t / 2].y : y[t / 2].x);
      }
    }
    __syncwarp();
  }
  if (Q) cluster_sync();  // no CTA leaves while another may still write to it
}

template <typename T>
int launch_forward(const Problem& p, cudaStream_t stream) {
  const size_t smem = layout((p.N + 1) / 2, sizeof(T)).total * sizeof(float);
  const int q = sharing(p, (p.T + kBlock - 1) / kBlock, kResident);
  LaunchScope scope(kKindSelectiveScan, stream);
  if (q > 1) return launch_shared(scan_forward_kernel<T, true>, p, q, 32 * kWarps, smem, stream);
  return launch_shared(scan_forward_kernel<T, false>, p, 1, 32 * kWarps, smem, stream);
}

}  // namespace

int forward(const Problem& p, int dtype, cudaStream_t stream) {
  return dtype == GRU_F32 ? launch_forward<float>(p, stream) : launch_forward<bf16>(p, stream);
}

int read_forward_status(int reset, int* status) {
  GRU_CUDA_TRY(cudaMemcpyFromSymbol(status, g_forward_status, sizeof(int)));
  if (reset) {
    const int zero = 0;
    GRU_CUDA_TRY(cudaMemcpyToSymbol(g_forward_status, &zero, sizeof(int)));
  }
  return GRU_OK;
}

}  // namespace scan
}  // namespace gru
