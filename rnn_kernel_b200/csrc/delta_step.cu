// The gated delta rule's single token (serving) and the C entry points of the
// whole rule (contract in include/rnn_kernel_b200.h).
//
// One token reads a state S [dk, dv] and writes it back:
//
//   a = e^g S^T k;  u = beta (v - a);  S <- e^g S + k u^T;  o = scale (e^g S_old^T q + (k . q) u)
//
// o comes from the sums over the OLD state, so that one pass of reads feeds one
// reduction over dk, for both sums, before the writes.  A CTA owns 32 value
// columns of one head: a warp takes four rows of 128 bytes at a time, a thread
// keeps its (up to four) float4 of the state in registers from read to write.
// HBM-bound: 8 dk dv bytes a head, which are loaded and stored as used once
// (64 sequences x 32 heads of 128 x 128: 47 to 49 us on different boards, 85 to 89 %
// of the copy rate).

#include <string>

#include "delta_common.cuh"

namespace gru {
namespace delta {
namespace {

constexpr int kMaxD = 128;

struct Step {
  const void *q, *k, *v;
  const float *g, *beta;
  float* s;
  void* o;
  long sq[2], sk[2], sv[2], sg[2], sb[2];  // batch, head
  int Hv, rep, dk, dv, slices, vec;
  float scale;
};

// ROWS: the rows of a thread where the key columns are that many times 32 and
// four value columns make an aligned access; 0: any sizes.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kThreads) delta_step_kernel(const Step a) {
  constexpr int R = ROWS ? ROWS : kMaxD / 32;
  __shared__ float ks[kMaxD], qs[kMaxD];
  __shared__ __align__(16) float part[2][8][kSlice];
  __shared__ __align__(16) float us[kSlice];
  const int slice = blockIdx.x % a.slices, bh = blockIdx.x / a.slices;
  const int hv = bh % a.Hv, b = bh / a.Hv, hk = hv / a.rep;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = slice * kSlice + (lane & 7) * 4;  // this thread's four columns
  const int row0 = warp * 4 + (lane >> 3);        // and rows row0, row0 + 32, ...
  float* s = a.s + (long)bh * a.dk * a.dv + c;
  const int left = a.dv - c;
  float4 x[R];
  if (ROWS) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      x[i] = left > 0 ? __ldcs(reinterpret_cast<const float4*>(s + (row0 + 32 * i) * a.dv)) : make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
    const float* safe = a.s + (long)bh * a.dk * a.dv;
#pragma unroll
    for (int i = 0; i < R; ++i)
      x[i] = load4_any(s + (row0 + 32 * i) * a.dv, safe, row0 + 32 * i < a.dk ? left : 0);
  }
  if (threadIdx.x < kMaxD) {
    const int d = threadIdx.x;
    const T* k = static_cast<const T*>(a.k) + b * a.sk[0] + hk * a.sk[1];
    const T* q = static_cast<const T*>(a.q) + b * a.sq[0] + hk * a.sq[1];
    ks[d] = d < a.dk ? as_float(k[d]) : 0.0f;
    qs[d] = d < a.dk ? as_float(q[d]) : 0.0f;
  }
  const float decay = expf(a.g[b * a.sg[0] + hv * a.sg[1]]);
  const float beta = a.beta[b * a.sb[0] + hv * a.sb[1]];
  __syncthreads();
  float4 sk = make_float4(0.f, 0.f, 0.f, 0.f), sq = sk;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float kr = ks[row0 + 32 * i], qr = qs[row0 + 32 * i];
    x[i].x *= decay, x[i].y *= decay, x[i].z *= decay, x[i].w *= decay;
    sk.x += x[i].x * kr, sk.y += x[i].y * kr, sk.z += x[i].z * kr, sk.w += x[i].w * kr;
    sq.x += x[i].x * qr, sq.y += x[i].y * qr, sq.z += x[i].z * qr, sq.w += x[i].w * qr;
  }
  float f[8] = {sk.x, sk.y, sk.z, sk.w, sq.x, sq.y, sq.z, sq.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] += __shfl_xor_sync(0xffffffffu, f[i], 8);
    f[i] += __shfl_xor_sync(0xffffffffu, f[i], 16);
  }
  if (lane < 8) {
    *reinterpret_cast<float4*>(&part[0][warp][lane * 4]) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(&part[1][warp][lane * 4]) = make_float4(f[4], f[5], f[6], f[7]);
  }
  __syncthreads();
  if (warp == 0) {
    float kv = 0.0f, qv = 0.0f, kq = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      kv += part[0][w][lane];
      qv += part[1][w][lane];
    }
#pragma unroll
    for (int i = 0; i < kMaxD / 32; ++i) kq += ks[lane + 32 * i] * qs[lane + 32 * i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, o);
    const int col = slice * kSlice + lane;
    float u = 0.0f;
    if (col < a.dv) {
      const float v = as_float((static_cast<const T*>(a.v) + b * a.sv[0] + hv * a.sv[1])[col]);
      u = beta * (v - kv);
      static_cast<T*>(a.o)[(long)bh * a.dv + col] = as_type<T>(a.scale * (qv + kq * u));
    }
    us[lane] = u;
  }
  __syncthreads();
  const float4 u = *reinterpret_cast<const float4*>(&us[(lane & 7) * 4]);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = row0 + 32 * i;
    const float kr = ks[r];
    const float4 y = make_float4(x[i].x + kr * u.x, x[i].y + kr * u.y, x[i].z + kr * u.z, x[i].w + kr * u.w);
    float* p = s + r * a.dv;
    if (ROWS) {
      if (left > 0) __stcs(reinterpret_cast<float4*>(p), y);
    } else if (r < a.dk) {
      if (left > 0) p[0] = y.x;
      if (left > 1) p[1] = y.y;
      if (left > 2) p[2] = y.z;
      if (left > 3) p[3] = y.w;
    }
  }
}

template <typename T>
int launch_step(const Step& a, unsigned ctas, cudaStream_t stream) {
  const int rows = a.vec && a.dk % 32 == 0 ? a.dk / 32 : 0;
  LaunchScope scope(kKindDeltaRule, stream);
  if (rows == 1) delta_step_kernel<T, 1><<<ctas, kThreads, 0, stream>>>(a);
  else if (rows == 2) delta_step_kernel<T, 2><<<ctas, kThreads, 0, stream>>>(a);
  else if (rows == 3) delta_step_kernel<T, 3><<<ctas, kThreads, 0, stream>>>(a);
  else if (rows == 4) delta_step_kernel<T, 4><<<ctas, kThreads, 0, stream>>>(a);
  else delta_step_kernel<T, 0><<<ctas, kThreads, 0, stream>>>(a);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

int bad(const char* what, const char* msg, int code = GRU_ERR_INVALID) {
  set_error(std::string(what) + ": " + msg);
  return code;
}

// Which of the tensors have to be there.
enum Needs { kSizesOnly, kDecays, kInputs };
int check_args(const char* what, const gru_delta_args* p, Needs needs) {
  if (!p) return bad(what, "null arguments");
  if (p->dtype != GRU_F32 && p->dtype != GRU_BF16)
    return bad(what, "dtype must be GRU_F32 or GRU_BF16", GRU_ERR_UNSUPPORTED);
  if (p->B < 0 || p->T < 0 || p->Hk < 1 || p->Hv < 1 || p->Hv % p->Hk != 0)
    return bad(what, "need B >= 0, T >= 0, and value heads a multiple of the key heads");
  if (p->dk < 1 || p->dk > kMaxD || p->dv < 1 || p->dv > kMaxD)
    return bad(what, "head sizes must be in [1, 128]", GRU_ERR_UNSUPPORTED);
  const uintptr_t es = p->dtype == GRU_F32 ? 4 : 2;
  if (((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) &
       (es - 1)) != 0 ||
      ((reinterpret_cast<uintptr_t>(p->g) | reinterpret_cast<uintptr_t>(p->beta) |
        reinterpret_cast<uintptr_t>(p->initial_state)) & 3) != 0)
    return bad(what, "a tensor is not aligned to its element size");
  const bool any = p->B > 0 && p->T > 0;
  if (any && ((needs != kSizesOnly && !p->g) || (needs == kInputs && (!p->q || !p->k || !p->v || !p->beta))))
    return bad(what, "null tensor");
  const long nc = ((long)p->T + kC - 1) / kC;
  if ((long)p->B * p->Hv > (1L << 28) || (long)p->B * p->Hv * (nc > 4 ? nc : 4) > 0x7fffffffL)
    return bad(what, "too many chunks for one launch", GRU_ERR_UNSUPPORTED);
  return GRU_OK;
}

size_t key_width(const gru_delta_args& p) { return p.dk <= 64 ? 64 : 128; }

// Hands out 256-byte aligned pieces of a buffer; with a null base it only
// counts.
struct Arena {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t n) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += align_up(n * sizeof(T), 256);
    return p;
  }
};

void fill(Problem& a, const gru_delta_args& p) {
  a.q = p.q, a.k = p.k, a.v = p.v, a.g = p.g, a.beta = p.beta, a.s0 = p.initial_state;
  for (int i = 0; i < 3; ++i) {
    a.sq[i] = p.q_stride[i], a.sk[i] = p.k_stride[i], a.sv[i] = p.v_stride[i];
    a.sg[i] = p.g_stride[i], a.sb[i] = p.beta_stride[i];
  }
  a.B = p.B, a.T = p.T, a.Hk = p.Hk, a.Hv = p.Hv, a.dk = p.dk, a.dv = p.dv;
  a.rep = p.Hv / p.Hk;
  a.nc = (p.T + kC - 1) / kC;
  a.dvp = (p.dv + kSlice - 1) / kSlice * kSlice;
  a.scale = p.scale;
}

// What the forward computes, and a training one keeps.
void lay_forward(Problem& a, const gru_delta_args& p, Arena& m) {
  const size_t nk = (size_t)a.B * a.Hk * a.nc, nv = (size_t)a.B * a.Hv * a.nc, w = key_width(p);
  const size_t np = p.dtype == GRU_F32 ? 2 : 1, groups = a.dvp / kGroup;
  a.kp = m.take<f16>(nk * np * kC * w);
  a.qp = m.take<f16>(nk * np * kC * w);
  a.wp = m.take<f16>(nv * 2 * kTile);
  a.pp = m.take<f16>(nv * 2 * kTile);
  a.gates = m.take<float>(nv * kGates * kC);
  a.states = m.take<f16>(nv * 2 * a.dvp * w);
  a.sscale = m.take<float>(nv * groups * 4);
  a.e = m.take<f16>(nv * 2 * a.dvp * kC);
  a.escale = m.take<float>(nv * groups * kC);
}

void lay_backward(Problem& a, const gru_delta_args& p, Arena& m) {
  const size_t nk = (size_t)a.B * a.Hk * a.nc, nv = (size_t)a.B * a.Hv * a.nc, w = key_width(p);
  const size_t np = p.dtype == GRU_F32 ? 2 : 1, groups = a.dvp / kGroup;
  a.z = m.take<f16>(nv * 2 * a.dvp * kC);
  a.zscale = m.take<float>(nv * groups * kC);
  a.dstates = m.take<f16>(nv * 2 * a.dvp * w);
  a.dsscale = m.take<float>(nv * groups * 4);
  a.dop = m.take<f16>(nv * np * a.dvp * kC);
  a.doscale = m.take<float>(nv * groups * kC);
  a.dqk = m.take<float>(a.rep > 1 ? nk * 2 * kC * w : 0);
}

}  // namespace
}  // namespace delta
}  // namespace gru

using namespace gru;
using namespace gru::delta;

extern "C" size_t gru_delta_stash_bytes(const gru_delta_args* p) {
  if (check_args("gru_delta_stash_bytes", p, kSizesOnly)) return 0;
  Problem a{};
  fill(a, *p);
  Arena m{nullptr};
  lay_forward(a, *p, m);
  return m.used;
}

extern "C" size_t gru_delta_workspace_bytes(const gru_delta_args* p, int backward) {
  if (check_args("gru_delta_workspace_bytes", p, kSizesOnly)) return 0;
  Problem a{};
  fill(a, *p);
  Arena m{nullptr};
  if (backward) lay_backward(a, *p, m);
  else lay_forward(a, *p, m);
  return m.used;
}

extern "C" int gru_delta_forward(const gru_delta_args* p, void* out, float* final_state, void* stash,
                                 size_t stash_bytes, void* workspace, size_t workspace_bytes, void* stream_) {
  clear_error();
  const char* me = "gru_delta_forward";
  if (const int rc = check_args(me, p, kInputs)) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (p->B == 0) return GRU_OK;
  if (!final_state || (reinterpret_cast<uintptr_t>(final_state) & 3)) return bad(me, "null or misaligned final_state");
  Problem a{};
  fill(a, *p);
  if (p->T == 0) {
    const size_t n = sizeof(float) * (size_t)p->B * p->Hv * p->dk * p->dv;
    if (!p->initial_state) GRU_CUDA_TRY(cudaMemsetAsync(final_state, 0, n, stream));
    else if (p->initial_state != final_state)
      GRU_CUDA_TRY(cudaMemcpyAsync(final_state, p->initial_state, n, cudaMemcpyDeviceToDevice, stream));
    return GRU_OK;
  }
  if (!out || (reinterpret_cast<uintptr_t>(out) & (p->dtype == GRU_F32 ? 3 : 1))) return bad(me, "null or misaligned out");
  Arena m{static_cast<char*>(stash ? stash : workspace)};
  lay_forward(a, *p, m);
  if (!m.base || (stash ? stash_bytes : workspace_bytes) < m.used || (reinterpret_cast<uintptr_t>(m.base) & 15))
    return bad(me, "stash (or workspace without one) too small or not 16-byte aligned");
  a.o = out;
  a.s_out = final_state;
  return forward(a, p->dtype, stream);
}

extern "C" int gru_delta_backward(const gru_delta_args* p, const void* dout, const float* dfinal, const void* stash,
                                  size_t stash_bytes, void* dq, void* dk, void* dv, float* dg, float* dbeta,
                                  float* dinitial, void* workspace, size_t workspace_bytes, void* stream_) {
  clear_error();
  const char* me = "gru_delta_backward";
  if (const int rc = check_args(me, p, kDecays)) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (p->B == 0) return GRU_OK;
  Problem a{};
  fill(a, *p);
  if (p->T == 0) {
    const size_t n = sizeof(float) * (size_t)p->B * p->Hv * p->dk * p->dv;
    if (dinitial && !dfinal) GRU_CUDA_TRY(cudaMemsetAsync(dinitial, 0, n, stream));
    else if (dinitial && dfinal != dinitial)
      GRU_CUDA_TRY(cudaMemcpyAsync(dinitial, dfinal, n, cudaMemcpyDeviceToDevice, stream));
    return GRU_OK;
  }
  const uintptr_t es = p->dtype == GRU_F32 ? 4 : 2;
  if (!dq || !dk || !dv || !dg || !dbeta ||
      ((reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk)) & (2 * es - 1)) ||
      (reinterpret_cast<uintptr_t>(dv) & (2 * es - 1)) || (reinterpret_cast<uintptr_t>(dout) & (es - 1)) ||
      ((reinterpret_cast<uintptr_t>(dg) | reinterpret_cast<uintptr_t>(dbeta) | reinterpret_cast<uintptr_t>(dinitial) |
        reinterpret_cast<uintptr_t>(dfinal)) & 3))
    return bad(me, "null gradient, or one not aligned to two of its elements");
  Arena s{static_cast<char*>(const_cast<void*>(stash))}, w{static_cast<char*>(workspace)};
  lay_forward(a, *p, s);
  lay_backward(a, *p, w);
  if (!stash || stash_bytes < s.used || !workspace || workspace_bytes < w.used ||
      ((reinterpret_cast<uintptr_t>(stash) | reinterpret_cast<uintptr_t>(workspace)) & 15))
    return bad(me, "stash or workspace too small or not 16-byte aligned");
  a.dout = dout, a.ds_out = dfinal;
  a.dq = dq, a.dk_ = dk, a.dv_ = dv, a.dg = dg, a.dbeta = dbeta, a.ds0 = dinitial;
  return backward(a, p->dtype, stream);
}

extern "C" int gru_delta_step(const gru_delta_args* p, float* state, void* out, void* stream_) {
  clear_error();
  const char* me = "gru_delta_step";
  if (const int rc = check_args(me, p, kInputs)) return rc;
  if (p->T != 1) return bad(me, "T must be 1");
  if (p->B == 0) return GRU_OK;
  if (!state || !out || (reinterpret_cast<uintptr_t>(state) & 3) ||
      (reinterpret_cast<uintptr_t>(out) & (p->dtype == GRU_F32 ? 3 : 1)))
    return bad(me, "null or misaligned state or out");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  Step a{p->q, p->k, p->v, p->g, p->beta, state, out,
         {p->q_stride[0], p->q_stride[2]}, {p->k_stride[0], p->k_stride[2]}, {p->v_stride[0], p->v_stride[2]},
         {p->g_stride[0], p->g_stride[2]}, {p->beta_stride[0], p->beta_stride[2]},
         p->Hv, p->Hv / p->Hk, p->dk, p->dv, (p->dv + kSlice - 1) / kSlice,
         p->dv % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0, p->scale};
  const unsigned ctas = (unsigned)((long)p->B * p->Hv * a.slices);
  return p->dtype == GRU_F32 ? launch_step<float>(a, ctas, stream) : launch_step<bf16>(a, ctas, stream);
}
