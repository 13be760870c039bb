// The selective state space scan: what its kernels share (contract in
// include/rnn_kernel_b200.h).
#pragma once

#include "row_ops.cuh"

namespace gru {
namespace scan {

constexpr int kMaxStates = 64;
constexpr int kLanes = 32;       // channels of a CTA, one a lane
constexpr int kWarps = 4;        // warps of a CTA, neighbouring pieces of the time
constexpr int kMark = 32;        // tokens between two states that the forward keeps for the gradient

struct Problem {
  const void *x, *dt, *b, *c, *z;
  const float *a, *skip, *bias, *s0;
  long xs[2], dts[2], zs[2], bs[3], cs[3];  // batch, token (, group)
  void* out;
  float* last;
  float* marks;  // [B][tiles][mark][state, padded][32]: states at the tokens 0, kMark, ...
  // gradient
  const void* dout;
  const float* dlast;
  void *dx, *ddt, *dz, *db, *dc;
  float *da, *dskip, *dbias, *ds0;
  float* part_bc;  // [B][tiles][T][2][padded N]
  float* part_a;   // [B][CTA of a tile][D][N]
  float* part_ch;  // [B][CTA of a tile][2][D]: of skip and dt_bias
  int B, T, D, N, G, R;  // R: channels of a group
  int softplus;
  int pairs, dpairs;  // rows of x, dt and z, and of dout, lie on 4-byte boundaries
  int per_group, tiles;  // tiles of 32 channels in a group, and in all
  int np;                // states rounded up to a multiple of four
  int wide;              // log2 of the states rounded up to a power of two, at least 4
  int nmarks;
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
// large, in 2 special and some 10 packed operations (log1pf(expf(x)) takes about
// 60, which made a third of the forward's instructions).
__device__ __forceinline__ float2 softplus_of(float2 x) {
  const float2 ax = make_float2(fminf(fabsf(x.x), 120.0f), fminf(fabsf(x.y), 120.0f));
  const float2 t = __fmul2_rn(ax, twice(-1.4426950408889634f));
  // what the exponent lost by its rounding
  const float2 lost = __ffma2_rn(ax, twice(-1.4426950408889634f), make_float2(-t.x, -t.y));
  float2 e = make_float2(exp2_of(t.x), exp2_of(t.y));
  e = __ffma2_rn(e, __fmul2_rn(lost, twice(0.6931471805599453f)), e);
  const float2 den = __fadd2_rn(e, twice(2.0f));
  const float2 s = __fmul2_rn(e, make_float2(rcp_of(den.x), rcp_of(den.y))), q = __fmul2_rn(s, s);
  float2 r = __ffma2_rn(q, twice(1.0f / 15.0f), twice(1.0f / 13.0f));
  r = __ffma2_rn(q, r, twice(1.0f / 11.0f));
  r = __ffma2_rn(q, r, twice(1.0f / 9.0f));
  r = __ffma2_rn(q, r, twice(1.0f / 7.0f));
  r = __ffma2_rn(q, r, twice(1.0f / 5.0f));
  r = __ffma2_rn(q, r, twice(1.0f / 3.0f));
  r = __ffma2_rn(__fmul2_rn(q, r), s, s);
  return __ffma2_rn(twice(2.0f), r, make_float2(max_nan(x.x, 0.0f), max_nan(x.y, 0.0f)));
}
// The step sizes of two raw values.
__device__ __forceinline__ float2 step_of(int softplus, float2 raw, float bias) {
  raw = __fadd2_rn(raw, twice(bias));
  return softplus ? softplus_of(raw) : raw;
}
// 1 / (1 + e^-x), as sigmoid_of
__device__ __forceinline__ float2 sigmoid_of2(float2 x) {
  const float2 t = __fmul2_rn(x, twice(-1.4426950408889634f));
  const float2 d = __fadd2_rn(make_float2(exp2_of(t.x), exp2_of(t.y)), twice(1.0f));
  return make_float2(rcp_of(d.x), rcp_of(d.y));
}

// ---- a warp's tokens of a tensor [token][channel], through shared memory ----

__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits for all but the last N issued.
template <int N>
__device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// TOK tokens x 32 channels from src (the tile's first channel of the first token,
// `stride` elements a token) to dst [TOK][32]; tokens from `here` on and channels
// from `width` on read as zero.  `async`: rows lie on 4-byte boundaries and the
// width fills 4-byte pieces, so the copy can run behind the warp's work (finished
// by copies_done() and a __syncwarp()); otherwise it is done at once.
template <typename T, int TOK>
__device__ __forceinline__ void fetch_rows(const T* src, long stride, int here, int width, bool async, T* dst) {
  const int lane = threadIdx.x & 31;
  constexpr int kPer = 4 / sizeof(T), kLanesRow = kLanes / kPer, kRows = 32 / kLanesRow;
  if (async) {
    const int row = lane / kLanesRow, c = (lane % kLanesRow) * kPer;
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst + row * kLanes + c));
#pragma unroll
    for (int t = 0; t < TOK; t += kRows) {
      const int at = t + row;
      const bool in = at < here && c < width;
      const T* from = in ? src + at * stride + c : src;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + t * kLanes * (int)sizeof(T)), "l"(from),
                   "r"(in ? 4 : 0)
                   : "memory");
    }
  } else {
#pragma unroll
    for (int t = 0; t < TOK; ++t)
      dst[t * kLanes + lane] = t < here && lane < width ? src[t * stride + lane] : from_f32<T>(0.0f);
  }
}

// A warp's rows of B and C [token][state], as FP32 by state: row n holds the
// tokens, ROW floats apart; states from N on are zero.  load() leaves them in
// registers, so that the loads run behind other work, up to store().
template <typename T, int TOK, int ROW>
struct FewRows {
  static constexpr int kMost = TOK * kMaxStates / 32;
  // states past the first 16 tokens x 16 are loaded and stored in turns
  static constexpr int kHeld = TOK / 2;
  T b[kHeld], c[kHeld];
  __device__ __forceinline__ void at(const Problem& p, int i, int* t, int* n) const {
    const int e = i * 32 + (threadIdx.x & 31);
    *t = e >> p.wide, *n = e & ((1 << p.wide) - 1);
  }
  __device__ __forceinline__ void load(const Problem& p, const T* bm, const T* cm, int here, int first) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      int t, n;
      at(p, first + i, &t, &n);
      const bool in = t < here && n < p.N;
      b[i] = in ? bm[t * p.bs[1] + n] : from_f32<T>(0.0f);
      c[i] = in ? cm[t * p.cs[1] + n] : from_f32<T>(0.0f);
    }
  }
  __device__ __forceinline__ void store(const Problem& p, float* bs, float* cs, int rows, int first) const {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      int t, n;
      at(p, first + i, &t, &n);
      if (t < TOK && n < rows) bs[n * ROW + t] = to_f32(b[i]), cs[n * ROW + t] = to_f32(c[i]);
    }
  }
  // what does not fit the registers
  __device__ __forceinline__ void rest(const Problem& p, const T* bm, const T* cm, int here, float* bs, float* cs, int rows) {
    for (int first = kHeld; first * 32 < TOK << p.wide; first += kHeld) {
      load(p, bm, cm, here, first);
      store(p, bs, cs, rows, first);
    }
  }
};

// ---- clusters: CTAs of one sequence and tile that take its blocks in turn ----

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void bar_init(uint32_t bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Eight bytes to another CTA's memory, counted by its barrier.
__device__ __forceinline__ void send(uint32_t to, float2 v, uint32_t bar) {
  const unsigned long long w = (unsigned long long)__float_as_uint(v.y) << 32 | __float_as_uint(v.x);
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to), "l"(w), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool bar_done(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits at most two seconds; after that the status word says so, the caller
// waits no more, and the launch's results are invalid.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int* status) {
  if (bar_done(bar, parity)) return true;
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if (bar_done(bar, parity)) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t - t0 > 2000000000ull) {
      atomicOr(status, GRU_STATUS_WAIT_TIMEOUT);
      return false;
    }
  }
}

}  // namespace scan
}  // namespace gru
