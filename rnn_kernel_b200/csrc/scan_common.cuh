// The selective state space scan: what its kernels share (contract in
// include/rnn_kernel_b200.h).
#pragma once

#include "row_ops.cuh"

namespace gru {
namespace scan {

constexpr int kMaxStates = 64;
constexpr int kLanes = 32;       // channels of a CTA, one a lane
constexpr int kBlock = 16;       // tokens of a block
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
  q.d = q.group * p.R + (q.live ? q.local : 0);
  q.first = q.seg * p.len, q.end = min(q.first + p.len, p.T);
  return q;
}

// Byte offset `token` rows of `stride` bytes on: one wide multiply-add.
template <typename T>
__device__ __forceinline__ T* row_at(T* base, int token, int stride) {
  return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(base) + (long)token * stride);
}

// Two neighbouring tokens of a lane's channel from src (the channel's first
// token), as stored; the last token again where there are no more (a load without
// a branch does not wait for its value).
template <typename T>
struct Pair {
  T x, y;
  __device__ __forceinline__ void load(const T* src, int stride, int t, int last) {
    x = *row_at(src, min(t, last), stride);
    y = *row_at(src, min(t + 1, last), stride);
  }
};
// A block's B and C [token][state], K elements of each a thread at most, from
// memory to rows of shared memory by state (kRow floats apart; states from N on and
// tokens behind the last are zero).
template <typename T, int K>
struct Few {
  const T *bm[K], *cm[K];  // this thread's state of the first token
  int token[K], to[K];     // of a block; where in shared memory, or -1
  T b[K], c[K];
  __device__ __forceinline__ void init(const Problem& p, const T* bm0, const T* cm0) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int e = threadIdx.x + i * blockDim.x, n = e & ((1 << p.wide) - 1);
      token[i] = e >> p.wide;
      to[i] = token[i] < kBlock && n < p.np ? n * kRow + token[i] : -1;
      bm[i] = bm0 + min(n, p.N - 1), cm[i] = cm0 + min(n, p.N - 1);
      if (n >= p.N) token[i] = 1 << 30;  // never there: zero
    }
  }
  __device__ __forceinline__ void load(const Problem& p, int t0, int last) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int t = min(t0 + token[i], last);
      b[i] = *row_at(bm[i], t, p.bst);
      c[i] = *row_at(cm[i], t, p.cst);
    }
  }
  __device__ __forceinline__ void store(float* bs, float* cs, int t0, int last) const {
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (to[i] >= 0) {
        const bool in = t0 + token[i] <= last;
        bs[to[i]] = in ? to_f32(b[i]) : 0.0f;
        cs[to[i]] = in ? to_f32(c[i]) : 0.0f;
      }
  }
};

// Rows of four tokens, [quad][lane] float4: the float2 of tokens t and t + 1.
__device__ __forceinline__ int pair_at(int t, int lane) { return ((t >> 2) * kLanes + lane) * 4 + (t & 2); }
__device__ __forceinline__ float2& pair_in(float* rows, int at) { return *reinterpret_cast<float2*>(rows + at); }

}  // namespace scan
}  // namespace gru
