// The selective state space scan: what its kernels share (contract in
// include/rnn_kernel_b200.h).
#pragma once

#include "row_ops.cuh"

namespace gru {
namespace scan {

constexpr int kMaxStates = 64;
constexpr int kLanes = 32;       // channels of a CTA, one a lane
constexpr int kBlock = 16;       // tokens of a block
constexpr int kQuads = kBlock / 4;
constexpr int kStates = 4;       // states of a warp
constexpr int kRow = kBlock + 4; // floats between two states' tokens in shared memory

struct Problem {
  const void *x, *dt, *b, *c, *z;
  const float *a, *skip, *bias, *s0;
  long xb, dtb, zb, bb, cb, bg, cg;   // elements between batch rows, and groups
  int xst, dtst, zst, bst, cst, ost;  // bytes between tokens; ost: of dense rows
  void* out;
  float* last;
  float* marks;  // [B][tiles][mark][state, padded][32]: states before each block
  // gradient
  const void* dout;
  const float* dlast;
  void *dx, *ddt, *dz, *db, *dc;
  float *da, *dskip, *dbias, *ds0;
  float* part_bc;  // [B][tiles][padded N][dB, dC][T]
  float* part_a;   // [B][segment][D][N]
  float* part_ch;  // [B][segment][2][D]: of skip and dt_bias
  // a segment's effect on a state that passes it: S or R, and its sum of steps
  float* seg_sums;   // [B][tiles][segment][state, padded][32]
  float* seg_steps;  // [B][tiles][segment][32]
  int B, T, D, N, G, R;  // R: channels of a group
  int softplus;
  int wide_rows, wide_dout, wide_few;  // rows of x, dt and z, of dout, and of B and C lie on 16-byte boundaries
  int per_group, tiles;  // tiles of 32 channels in a group, and in all
  int np;                // states rounded up to a multiple of four
  int wide;              // log2 of the states rounded up to a power of two, at least 4
  int nmarks;
  int segs, len;         // segments of the time, and their tokens (a multiple of kBlock)
};

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A in powers of two, kept finite: a token that is not there has dt = 0, and
// 0 * infinity would make its decay NaN, not 1.
__device__ __forceinline__ float decay_rate(float a) {
  const float r = a * 1.4426950408889634f;
  return r < -3.0e38f ? -3.0e38f : r > 3.0e38f ? 3.0e38f : r;
}

__device__ __forceinline__ float rcp_of(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float x, float y) {  // NaN where either is
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}
__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x|.  With s = e / (2 + e), at
// most 1/3, log(1 + e) = 2 artanh(s) = 2 (s + s^3 / 3 + s^5 / 5 + ...), whose
// terms after s^15 sum to less than 2^-26 of it: as exact for small e as for
// large, in 2 special and some 16 plain operations (log1pf(expf(x)) takes about 60,
// which made a third of the forward's instructions).  Not packed: the constants
// would have to be moved into pairs of registers.
__device__ __forceinline__ float softplus_of(float x) {
  const float ax = fminf(fabsf(x), 120.0f), t = ax * -1.4426950408889634f;
  const float lost = fmaf(ax, -1.4426950408889634f, -t);  // of the exponent by its rounding
  float e = exp2_of(t);
  e = fmaf(e, lost * 0.6931471805599453f, e);
  const float s = e * rcp_of(e + 2.0f), q = s * s;
  float r = fmaf(q, 1.0f / 15.0f, 1.0f / 13.0f);
  r = fmaf(q, r, 1.0f / 11.0f);
  r = fmaf(q, r, 1.0f / 9.0f);
  r = fmaf(q, r, 1.0f / 7.0f);
  r = fmaf(q, r, 1.0f / 5.0f);
  r = fmaf(q, r, 1.0f / 3.0f);
  r = fmaf(q * r, s, s);
  return fmaf(2.0f, r, max_nan(x, 0.0f));
}
// The step size of a raw value.
__device__ __forceinline__ float step_of(int softplus, float raw, float bias) {
  raw += bias;
  return softplus ? softplus_of(raw) : raw;
}
// 1 / (1 + e^-x), as sigmoid_of but for the last bits
__device__ __forceinline__ float gate_of(float x) { return rcp_of(1.0f + exp2_of(x * -1.4426950408889634f)); }

// The tile of 32 channels and the range of tokens of a CTA.
struct Place {
  int seg, unit, b, group, d, local;  // local: the lane's channel in its group
  int first, end;                     // tokens
  int d0, width;                      // the tile's first channel, and its channels
  bool live;                          // the lane has a channel
};
__device__ __forceinline__ Place place(const Problem& p) {
  Place q;
  q.seg = blockIdx.x % p.segs, q.unit = blockIdx.x / p.segs;
  const int tile = q.unit % p.tiles;
  q.b = q.unit / p.tiles;
  q.group = tile / p.per_group;
  q.local = (tile - q.group * p.per_group) * kLanes + (threadIdx.x & 31);
  q.live = q.local < p.R;
  q.d0 = q.group * p.R + q.local - (int)(threadIdx.x & 31), q.width = min(p.R - (q.d0 - q.group * p.R), kLanes);
  q.d = q.live ? q.group * p.R + q.local : q.d0;
  q.first = q.seg * p.len, q.end = min(q.first + p.len, p.T);
  return q;
}

// Byte offset `token` rows of `stride` bytes on: one wide multiply-add.
template <typename T>
__device__ __forceinline__ T* row_at(T* base, int token, int stride) {
  return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(base) + (long)token * stride);
}

// ---- a block's inputs, as stored, in shared memory --------------------------------

__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from)
               : "memory");
}
// This thread's copies are there (other threads' after a barrier).
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Tokens t0 .. t0 + 15 of a tile's channels, from src (its first channel at token
// 0), to dst [token][32]; the last token again where there are no more.  Pieces of
// 16 bytes that arrive behind the CTA's work where all rows lie on their boundaries
// (wide), elements otherwise; channels from `width` on are not written.
template <typename T>
__device__ __forceinline__ void fetch_rows(T* dst, const T* src, int stride, int t0, int last, int width, bool wide) {
  if (wide) {
    constexpr int kPer = 16 / sizeof(T), kPieces = kLanes / kPer;
    for (int e = threadIdx.x; e < kBlock * kPieces; e += blockDim.x) {
      const int t = e / kPieces, c = (e % kPieces) * kPer;
      if (c < width) copy16(dst + t * kLanes + c, row_at(src + c, min(t0 + t, last), stride));
    }
  } else {
    for (int e = threadIdx.x; e < kBlock * kLanes; e += blockDim.x) {
      const int t = e / kLanes, c = e % kLanes;
      if (c < width) dst[e] = *row_at(src + c, min(t0 + t, last), stride);
    }
  }
}
// The same for N states of B or C: dst [token][N].
template <typename T>
__device__ __forceinline__ void fetch_few(T* dst, const T* src, int stride, int t0, int last, int N, bool wide) {
  if (wide) {
    const int pieces = N * (int)sizeof(T) / 16;
    for (int e = threadIdx.x; e < kBlock * pieces; e += blockDim.x) {
      const int t = e / pieces, c = (e - t * pieces) * (16 / (int)sizeof(T));
      copy16(dst + t * N + c, row_at(src + c, min(t0 + t, last), stride));
    }
  } else {
    for (int e = threadIdx.x; e < kBlock * N; e += blockDim.x) {
      const int t = e / N;
      dst[e] = *row_at(src + (e - t * N), min(t0 + t, last), stride);
    }
  }
}
// From there to FP32 rows by state (kRow floats apart): states from N on and tokens
// behind the last are zero.
template <typename T>
__device__ __forceinline__ void turn_few(const Problem& p, const T* b, const T* c, float* bs, float* cs, int np, int left) {
  for (int e = threadIdx.x; e < kBlock << p.wide; e += blockDim.x) {
    const int t = e >> p.wide, n = e & ((1 << p.wide) - 1);
    if (n >= np) continue;
    const bool in = t < left && n < p.N;
    bs[n * kRow + t] = in ? to_f32(b[t * p.N + n]) : 0.0f;
    cs[n * kRow + t] = in ? to_f32(c[t * p.N + n]) : 0.0f;
  }
}
// Four tokens of the lane's channel.
template <typename T>
__device__ __forceinline__ void quad_of(const T* rows, int u, int lane, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f32(rows[(4 * u + i) * kLanes + lane]);
}

__device__ __forceinline__ float4 as4(const float (&v)[4]) { return make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ float2 lo(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  const float2 x = __fadd2_rn(lo(a), lo(b)), y = __fadd2_rn(hi(a), hi(b));
  return make_float4(x.x, x.y, y.x, y.y);
}

}  // namespace scan
}  // namespace gru
