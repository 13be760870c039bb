// The selective state space scan: what its kernels share (contract in
// include/rnn_kernel_b200.h).
#pragma once

#include <math_constants.h>

#include "row_ops.cuh"

namespace gru {
namespace scan {

constexpr int kMaxStates = 64;
constexpr int kLanes = 32;
constexpr int kTile = 64;        // channels of a CTA: two neighbours a lane
constexpr int kBlock = 16;       // tokens of a block
constexpr int kPairs = kBlock / 2;
constexpr int kRow = 2 * kBlock + 4;  // floats between two states' tokens in shared memory, each twice

struct Problem {
  const void *x, *dt, *b, *c, *z;
  const float *a, *skip, *bias, *s0;
  long xb, dtb, zb, bb, cb, bg, cg;   // elements between batch rows, and groups
  int xst, dtst, zst, bst, cst, ost;  // bytes between tokens; ost: of dense rows
  void* out;
  float* last;
  // what a training forward keeps
  float* marks;  // [B][tiles][block][state, padded][64]: states before each block
  float* sums;   // [B][T][D], with a gate: what it multiplies
  // gradient
  const void* dout;
  const float* dlast;
  void *dx, *ddt, *dz, *db, *dc;
  float *da, *dskip, *dbias, *ds0;
  float* part_bc;  // [B][tiles][padded N][dB, dC][T]
  float* part;     // [B][segment]: of dA [D][N], of dskip and dbias [2][D]
  // a segment's effect on a state that passes it: S or R, and its sum of steps
  float* seg_sums;   // [B][tiles][segment][state, padded][64]
  float* seg_steps;  // [B][tiles][segment][64]
  int B, T, D, N, G, R;  // R: channels of a group
  int softplus;
  // bytes of the pieces in which rows of x, dt and z, of dout, and of B and C are
  // copied: 16 or 4 where all lie on such boundaries, else 0 (single elements)
  int row_piece, dout_piece, sums_piece, few_piece;
  int even_out;   // neighbouring channels of dense tensors can be stored together
  int even_sums;  // and those of sums
  int per_group, tiles;  // tiles of 64 channels in a group, and in all
  int np;                // states rounded up to a multiple of four
  int wide;              // log2 of the states rounded up to a power of two, at least 4
  int nmarks;
  int segs, len;         // segments of the time, and their tokens (a multiple of kBlock)
};

__device__ __forceinline__ float max_nan(float x, float y) {  // NaN where either is
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}
__device__ __forceinline__ float min_nan(float x, float y) {
  float z;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// A in powers of two, kept finite: a token that is not there has dt = 0, and
// 0 * infinity would make its decay NaN, not 1.
__device__ __forceinline__ float decay_rate(float a) {
  return min_nan(max_nan(a * 1.4426950408889634f, -3.0e38f), 3.0e38f);
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
// The tile of channels and the range of tokens of a CTA.
struct Place {
  int seg, unit, b, group;
  int first, end;     // tokens
  int d0, width;      // the tile's first channel, and its channels
  int d;              // the lane's first channel (the tile's where it has none)
  bool live, second;  // the lane has a channel, and its neighbour
};
// segs: of them that the launch takes, from `from` on.
__device__ __forceinline__ Place place(const Problem& p, int segs, int from) {
  Place q;
  q.unit = blockIdx.x / segs, q.seg = from + blockIdx.x - q.unit * segs;
  const int tile = q.unit % p.tiles, c = 2 * (threadIdx.x & 31);
  q.b = q.unit / p.tiles;
  q.group = tile / p.per_group;
  const int in_group = (tile - q.group * p.per_group) * kTile;
  q.d0 = q.group * p.R + in_group;
  q.width = min(p.R - in_group, kTile);
  q.live = c < q.width, q.second = c + 1 < q.width;
  q.d = q.d0 + (q.live ? c : 0);
  q.first = q.seg * p.len, q.end = min(q.first + p.len, p.T);
  return q;
}
// A parameter [D] of the lane's channels; 0 where there are none.
__device__ __forceinline__ float2 two_of(const float* v, const Place& q) {
  return make_float2(v && q.live ? v[q.d] : 0.0f, v && q.second ? v[q.d + 1] : 0.0f);
}
// And a matrix [D, N]'s (or [B, D, N]'s from its batch row).
__device__ __forceinline__ float2 two_of(const float* v, const Place& q, int n, int N) {
  const bool in = v && n < N;
  return make_float2(in && q.live ? v[(long)q.d * N + n] : 0.0f, in && q.second ? v[(long)(q.d + 1) * N + n] : 0.0f);
}
__device__ __forceinline__ void put_two(float* v, const Place& q, int n, int N, float2 x) {
  if (n >= N) return;
  if (q.live) v[(long)q.d * N + n] = x.x;
  if (q.second) v[(long)(q.d + 1) * N + n] = x.y;
}

// Byte offset `token` rows of `stride` bytes on: one wide multiply-add.
template <typename T>
__device__ __forceinline__ T* row_at(T* base, int token, int stride) {
  return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(base) + (long)token * stride);
}

// ---- a block's inputs, as stored, in shared memory --------------------------------

template <int BYTES>
__device__ __forceinline__ void copy(void* to, const void* from) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}
// This thread's copies are there (other threads' after a barrier).
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Brings a block's rows of up to four tensors [token][channel] and of B and C
// [token][state] from memory to shared memory, as they are stored: [token][64] and
// [token][N]; the last token again where there are no more.  Pieces of 16 bytes, or
// of 4, that arrive behind the CTA's work, as all rows' boundaries allow; elements
// (16-bit ones at odd places), which do not, otherwise.  Channels past the tile's
// width are not written.
template <typename T>
struct Feed {
  bool few;            // B and C by pieces of 16 bytes, one a thread
  const T* few_src;
  int few_token, few_at, few_stride;
  bool few_has;
  __device__ __forceinline__ void init(const Problem& p, const T* bm, const T* cm) {
    constexpr int kPer = 16 / (int)sizeof(T);
    const int e = threadIdx.x, pieces = p.N / kPer;
    few = p.few_piece == 16 && (int)blockDim.x >= 2 * kBlock * pieces;
    few_has = false;
    if (few) {
      const bool c = e >= kBlock * pieces;
      const int f = c ? e - kBlock * pieces : e;
      few_has = f < kBlock * pieces;
      few_token = f / pieces;
      const int n = (f - few_token * pieces) * kPer;
      few_src = (c ? cm : bm) + n;
      few_stride = c ? p.cst : p.bst;
      few_at = (c ? kBlock * p.N : 0) + few_token * p.N + n;
    }
  }
  // BYTES of a piece; rows of kTile.
  template <int BYTES>
  __device__ __forceinline__ void pieces(T* dst, const T* src, int stride, int t0, int last, int width) const {
    constexpr int kPer = BYTES / (int)sizeof(T), kPieces = kTile / kPer;
    const int at = (threadIdx.x % kPieces) * kPer;  // blockDim is a multiple of 32, and so of kPieces or its half
    if (kPieces <= 32) {
      if (at < width)
        for (int t = threadIdx.x / kPieces; t < kBlock; t += blockDim.x / kPieces)
          copy<BYTES>(dst + t * kTile + at, row_at(src + at, min(t0 + t, last), stride));
    } else {
      for (int e = threadIdx.x; e < kBlock * kPieces; e += blockDim.x) {
        const int t = e / kPieces, c = (e % kPieces) * kPer;
        if (c < width) copy<BYTES>(dst + t * kTile + c, row_at(src + c, min(t0 + t, last), stride));
      }
    }
  }
  __device__ __forceinline__ void row(T* dst, const T* src, int stride, int t0, int last, int width, int piece) const {
    if (piece == 16) pieces<16>(dst, src, stride, t0, last, width);
    else if (piece == 4) pieces<4>(dst, src, stride, t0, last, width);
    else
#pragma unroll 4
      for (int e = threadIdx.x; e < kBlock * kTile; e += blockDim.x) {
        const int t = e / kTile, c = e % kTile;
        dst[e] = *row_at(src + min(c, width - 1), min(t0 + t, last), stride);
      }
  }
  __device__ __forceinline__ void bc(const Problem& p, T* dst, const T* bm, const T* cm, int t0, int last) const {
    if (few) {
      if (few_has) copy<16>(dst + few_at, row_at(few_src, min(t0 + few_token, last), few_stride));
      return;
    }
    const int each = p.few_piece ? 4 / (int)sizeof(T) : 1, count = p.N / each;
#pragma unroll 2
    for (int e = threadIdx.x; e < kBlock * count; e += blockDim.x) {
      const int t = e / count, n = (e - t * count) * each, from = min(t0 + t, last);
      const T *b = row_at(bm + n, from, p.bst), *c = row_at(cm + n, from, p.cst);
      T *tb = dst + t * p.N + n, *tc = tb + kBlock * p.N;
      if (p.few_piece) copy<4>(tb, b), copy<4>(tc, c);
      else tb[0] = *b, tc[0] = *c;
    }
  }
};
// B and C from there to FP32 rows by state, each number twice (an operand of two
// channels), kRow floats apart: states from N on and tokens behind the last are zero.
template <typename T>
__device__ __forceinline__ void turn_few(const Problem& p, const T* raw, float* bs, float* cs, int np, int left) {
  for (int e = threadIdx.x; e < kBlock << p.wide; e += blockDim.x) {
    const int t = e >> p.wide, n = e & ((1 << p.wide) - 1);
    if (n >= np) continue;
    const bool in = t < left && n < p.N;
    const float b = in ? to_f32(raw[t * p.N + n]) : 0.0f, c = in ? to_f32(raw[(kBlock + t) * p.N + n]) : 0.0f;
    *reinterpret_cast<float2*>(bs + n * kRow + 2 * t) = make_float2(b, b);
    *reinterpret_cast<float2*>(cs + n * kRow + 2 * t) = make_float2(c, c);
  }
}
// The lane's channels of one token, and of two.
__device__ __forceinline__ float2 both(const float* rows, int t, int lane) {
  return *reinterpret_cast<const float2*>(rows + t * kTile + 2 * lane);
}
__device__ __forceinline__ float2 both(const bf16* rows, int t, int lane) {
  const unsigned r = *reinterpret_cast<const unsigned*>(rows + t * kTile + 2 * lane);
  return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ void four(const T* rows, int u, int lane, float (&v)[4]) {
  const float2 a = both(rows, 2 * u, lane), b = both(rows, 2 * u + 1, lane);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
// Stores the lane's channels of one token of a dense tensor.
template <typename T>
__device__ __forceinline__ void put_both(T* at, float x, float y, const Place& q, bool even) {
  if (even) {
    if (q.live) {
      const float v[2] = {x, y};
      store_row<2>(at, v);
    }
  } else {
    if (q.live) at[0] = from_f32<T>(x);
    if (q.second) at[1] = from_f32<T>(y);
  }
}

__device__ __forceinline__ float4 as4(const float (&v)[4]) { return make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ float4 as4(float2 a, float2 b) { return make_float4(a.x, a.y, b.x, b.y); }
__device__ __forceinline__ float2 lo(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float4 add4(float4 a, float4 b) { return as4(__fadd2_rn(lo(a), lo(b)), __fadd2_rn(hi(a), hi(b))); }
using gru::exp2_of;
__device__ __forceinline__ float2 exp2_of(float2 v) { return make_float2(exp2_of(v.x), exp2_of(v.y)); }

constexpr float kMost = 3.0e38f;
// The decay over tokens whose steps sum to `steps`.  Finite: a state that is zero
// stays so, where each token's own decay would have left it zero.
__device__ __forceinline__ float2 passed(float2 rate, float2 steps) {
  const float2 d = exp2_of(__fmul2_rn(rate, steps));
  return make_float2(fminf(d.x, kMost), fminf(d.y, kMost));
}
// A state behind some tokens, its part from before them carried by `decay` and not
// by the product of the tokens' decays (unless that overflowed, where A is positive).
// An infinite state has no such difference (0 or a negative number of infinities is
// NaN): it stays as the tokens left it.
__device__ __forceinline__ float2 carried(float2 state, float2 before, float2 decay, float2 product) {
  const float2 d = __fadd2_rn(decay, make_float2(-product.x, -product.y)), r = __ffma2_rn(d, before, state);
  return make_float2(fabsf(r.x) <= kMost ? r.x : state.x, fabsf(r.y) <= kMost ? r.y : state.y);
}
// A state behind a segment that adds `sum` to it.  Its decay may be below the least FP32
// number where no token's is, so an infinity is not multiplied by it.
__device__ __forceinline__ float2 behind_segment(float2 state, float2 decay, float2 sum) {
  const float2 r = __ffma2_rn(decay, state, sum);
  return make_float2(fabsf(state.x) == CUDART_INF_F ? state.x + sum.x : r.x,
                     fabsf(state.y) == CUDART_INF_F ? state.y + sum.y : r.y);
}

}  // namespace scan
}  // namespace gru
