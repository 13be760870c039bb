// The selective state space scan: what its kernels share (contract in
// include/rnn_kernel_b200.h).
#pragma once

#include "row_ops.cuh"

namespace gru {
namespace scan {

constexpr int kMaxStates = 64;
constexpr int kGroup = 2;        // states a lane works on at a time
constexpr int kLanes = 32;       // channels of a CTA, one a lane
constexpr int kWarps = 4;        // warps of a CTA, neighbouring pieces of the time
constexpr int kMark = 32;        // tokens between two states that the forward keeps for the gradient

struct Problem {
  const void *x, *dt, *b, *c, *z;
  const float *a, *skip, *bias, *s0;
  long xs[2], dts[2], zs[2], bs[3], cs[3];  // batch, token (, group)
  void* out;
  float* last;
  float* marks;  // [B][tiles][mark][state group][32] float2: states at the tokens 0, kMark, ...
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
  int per_group, tiles;  // tiles of 32 channels in a group, and in all
  int ng;                // groups of states: ceil(N / 2)
  int wide;              // log2 of the states rounded up to a power of two
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

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x|.  With s = e / (2 + e), at
// most 1/3, log(1 + e) = 2 artanh(s) = 2 (s + s^3 / 3 + s^5 / 5 + ...), whose
// terms after s^13 sum to less than 2^-24 of it: as exact for small e as for
// large, in 2 special and some 14 plain operations (log1pf(expf(x)): about 60,
// which made a third of the forward's instructions).
__device__ __forceinline__ float softplus_of(float x) {
  const float ax = fminf(fabsf(x), 120.0f), t = ax * -1.4426950408889634f;
  const float lost = fmaf(ax, -1.4426950408889634f, -t);  // of the exponent by its rounding
  float e = exp2_of(t);
  e = fmaf(e, lost * 0.6931471805599453f, e);
  const float s = __fdividef(e, 2.0f + e), q = s * s;
  float r = fmaf(q, 1.0f / 15.0f, 1.0f / 13.0f);
  r = fmaf(q, r, 1.0f / 11.0f);
  r = fmaf(q, r, 1.0f / 9.0f);
  r = fmaf(q, r, 1.0f / 7.0f);
  r = fmaf(q, r, 1.0f / 5.0f);
  r = fmaf(q, r, 1.0f / 3.0f);
  r = fmaf(q * r, s, s);
  return x == x ? fmaxf(x, 0.0f) + 2.0f * r : x;
}

// The step size of a raw value.
__device__ __forceinline__ float step_of(const Problem& p, float raw, float bias) {
  raw += bias;
  return p.softplus ? softplus_of(raw) : raw;
}

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
