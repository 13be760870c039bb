// The selective scan's single token (serving) and the C entry points of the whole
// operator (contract in include/rnn_kernel_b200.h).
//
// One token reads a state [D, N] and writes it back.  A thread has four states
// of a channel in registers from read to write, the lanes of a channel lie side
// by side, and their sums of C h meet by shuffles.  Bound by memory, 8 N bytes a
// channel, loaded and stored as used once: 256 sequences of 4096 channels and 16
// states, 134 MB, take 32 us, 64 % of the copy rate; the rest is the latency of one
// round of loads per CTA (a channel a thread instead of four: 47 us).

#include <algorithm>
#include <initializer_list>
#include <utility>

#include "scan_common.cuh"
#include "scan_launch.cuh"

namespace gru {
namespace scan {
namespace {

constexpr int kStepThreads = 256;

// LP: lanes of a channel; K <= LP: channels a thread takes one after another, whose
// loads are in flight together.  The k-th lane of a channel's works out the step and
// the gate of the k-th channel for all.  vec: states, and groups of B and C, lie in
// aligned fours.
template <typename T, int LP, int K>
__global__ void __launch_bounds__(kStepThreads, 3) scan_step_kernel(const Problem p, float* state, int vec, int blocks) {
  static_assert(K <= LP, "a lane for every channel");
  constexpr int kSlots = kStepThreads / LP;
  const int b = blockIdx.x / blocks, part = threadIdx.x % LP, slot = threadIdx.x / LP, lane = threadIdx.x & 31;
  const int d0 = (blockIdx.x - b * blocks) * (kSlots * K) + slot;
  const int n0 = 4 * part, left = p.N - n0;
  const int mine = min(d0 + (part % K) * kSlots, p.D - 1);
  const float x = to_f32(static_cast<const T*>(p.x)[b * p.xb + mine]), raw = to_f32(static_cast<const T*>(p.dt)[b * p.dtb + mine]);
  const float z = to_f32(p.z ? static_cast<const T*>(p.z)[b * p.zb + mine] : static_cast<const T*>(p.x)[b * p.xb + mine]);
  const float bias = *(p.bias ? p.bias + mine : p.a), skip = *(p.skip ? p.skip + mine : p.a);
  float h[K][4], a[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int d = min(d0 + k * kSlots, p.D - 1);  // loads without a branch; the last channel is not written twice
    const float* s = state + ((long)b * p.D + d) * p.N + n0;
    const float* r = p.a + (long)d * p.N + n0;
    if (vec) {
      const int at = left > 0 ? 0 : -n0;  // lanes without states read the channel's first
      const float4 v = __ldcs(reinterpret_cast<const float4*>(s + at));
      const float4 u = __ldg(reinterpret_cast<const float4*>(r + at));
      h[k][0] = v.x, h[k][1] = v.y, h[k][2] = v.z, h[k][3] = v.w;
      a[k][0] = u.x, a[k][1] = u.y, a[k][2] = u.z, a[k][3] = u.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) h[k][j] = j < left ? s[j] : 0.0f, a[k][j] = j < left ? r[j] : 0.0f;
    }
  }
  const float step = step_of(p.softplus, raw, p.bias ? bias : 0.0f), du = step * x;
  float bv[4], cv[4], own = 0.0f;
  int group = -1;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int d = min(d0 + k * kSlots, p.D - 1);
    const int g = p.G == 1 ? 0 : d / p.R;
    if (g != group) {
      group = g;
      const T* bm = static_cast<const T*>(p.b) + b * p.bb + g * p.bg + n0;
      const T* cm = static_cast<const T*>(p.c) + b * p.cb + g * p.cg + n0;
      if (vec && left > 0) {
        load_row<4>(bm, bv);
        load_row<4>(cm, cv);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) bv[j] = j < left ? to_f32(bm[j]) : 0.0f, cv[j] = j < left ? to_f32(cm[j]) : 0.0f;
      }
    }
    const int from = (lane & ~(LP - 1)) + k;
    const float sk = __shfl_sync(0xffffffffu, step, from), uk = __shfl_sync(0xffffffffu, du, from);
    float y = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[k][j] = fmaf(exp2_of(sk * decay_rate(a[k][j])), h[k][j], uk * bv[j]);
      if (j < left) y = fmaf(cv[j], h[k][j], y);  // an infinite dt x makes NaN of states that are not there
    }
#pragma unroll
    for (int o = LP / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (part == k) own = y;
    if (d0 + k * kSlots >= p.D) continue;
    float* s = state + ((long)b * p.D + d) * p.N + n0;
    if (vec) {
      if (left > 0) __stcs(reinterpret_cast<float4*>(s), make_float4(h[k][0], h[k][1], h[k][2], h[k][3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) s[j] = h[k][j];
    }
  }
  if (part < K && d0 + part * kSlots < p.D) {
    if (p.skip) own = fmaf(skip, x, own);
    if (p.z) own *= z * sigmoid_of(z);
    static_cast<T*>(p.out)[(long)b * p.D + mine] = from_f32<T>(own);
  }
}

template <typename T, int LP, int K>
int launch_step(const Problem& p, float* state, int vec, cudaStream_t stream) {
  const int blocks = ceil_div(p.D, kStepThreads / LP * K);
  LaunchScope scope(kKindSelectiveScan, stream);
  scan_step_kernel<T, LP, K><<<(unsigned)((long)p.B * blocks), kStepThreads, 0, stream>>>(p, state, vec, blocks);
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

// Four channels a thread (as many as a channel has lanes, where those are fewer),
// where that still gives every SM four CTAs.
template <typename T>
int step(const Problem& p, float* state, int vec, cudaStream_t stream) {
  int lp = 1;
  while (lp * 4 < p.N) lp *= 2;
  const bool four = (long)p.B * p.D * lp / (kStepThreads * 4) >= 4L * 148;
#define GRU_STEP(LP, K) \
  if (lp == LP) return four ? launch_step<T, LP, K>(p, state, vec, stream) : launch_step<T, LP, 1>(p, state, vec, stream);
  GRU_STEP(1, 1)
  GRU_STEP(2, 2)
  GRU_STEP(4, 4)
  GRU_STEP(8, 4)
  GRU_STEP(16, 4)
#undef GRU_STEP
  return GRU_ERR_UNSUPPORTED;
}

enum Needs { kSizesOnly, kInputs };
int check(const char* me, const gru_scan_args* p, Needs needs) {
  if (!p) return refuse(me, "null arguments");
  if (!known(p->dtype)) return refuse(me, "dtype must be GRU_F32 or GRU_BF16", GRU_ERR_UNSUPPORTED);
  if (p->B < 0 || p->T < 0 || p->D < 1 || p->G < 1 || p->D % p->G != 0)
    return refuse(me, "need B >= 0, T >= 0, and channels a multiple of the groups");
  if (p->N < 1 || p->N > kMaxStates) return refuse(me, "the states must be in [1, 64]", GRU_ERR_UNSUPPORTED);
  if (p->dt_softplus != 0 && p->dt_softplus != 1) return refuse(me, "dt_softplus must be 0 or 1");
  const uintptr_t es = elem_size(p->dtype);
  if ((bits(p->x) | bits(p->dt) | bits(p->b) | bits(p->c) | bits(p->z)) & (es - 1) ||
      (bits(p->a) | bits(p->skip) | bits(p->dt_bias) | bits(p->initial_state)) & 3)
    return refuse(me, "a tensor is not aligned to its element size");
  if (needs == kInputs && p->B > 0 && p->T > 0 && (!p->x || !p->dt || !p->b || !p->c || !p->a)) return refuse(me, "null tensor");
  for (const long s : {p->x_stride[1], p->dt_stride[1], p->z_stride[1], p->b_stride[1], p->c_stride[1]})
    if (s < 0 || s * (long)es > 0x7fffffffL)
      return refuse(me, "tokens must be less than 2^31 bytes apart", GRU_ERR_UNSUPPORTED);
  const double tiles = (double)p->G * ((p->D / p->G + kTile - 1) / kTile);
  if (p->B * tiles > 2e9 || (double)p->B * p->D * 16 > 4e11 || (double)p->B * p->T * p->G > 4e9 || p->T > (1 << 30) ||
      p->D > (1 << 26))
    return refuse(me, "too large for one launch", GRU_ERR_UNSUPPORTED);
  return GRU_OK;
}

// The widest piece (16 or 4 bytes, else 0) whose boundaries all rows of the tensors
// lie on, and `inner` elements fill.
int piece_of(std::initializer_list<std::pair<const void*, const long*>> all, int strides, long inner, int es) {
  for (const int n : {16, 4}) {
    bool ok = inner * es % n == 0;
    for (const auto& t : all) {
      if (!t.first) continue;
      ok = ok && bits(t.first) % n == 0;
      for (int i = 0; i < strides; ++i) ok = ok && t.second[i] * es % n == 0;
    }
    if (ok) return n;
  }
  return 0;
}

void fill(Problem& a, const gru_scan_args& p) {
  a.x = p.x, a.dt = p.dt, a.b = p.b, a.c = p.c, a.z = p.z;
  a.a = p.a, a.skip = p.skip, a.bias = p.dt_bias, a.s0 = p.initial_state;
  const int es = (int)elem_size(p.dtype);
  a.xb = p.x_stride[0], a.dtb = p.dt_stride[0], a.zb = p.z_stride[0], a.bb = p.b_stride[0], a.cb = p.c_stride[0];
  a.bg = p.b_stride[2], a.cg = p.c_stride[2];
  a.xst = (int)(p.x_stride[1] * es), a.dtst = (int)(p.dt_stride[1] * es), a.zst = (int)(p.z_stride[1] * es);
  a.bst = (int)(p.b_stride[1] * es), a.cst = (int)(p.c_stride[1] * es), a.ost = p.D * es;
  a.row_piece = piece_of({{p.x, p.x_stride}, {p.dt, p.dt_stride}, {p.z, p.z_stride}}, 2, p.D / p.G, es);
  a.few_piece = piece_of({{p.b, p.b_stride}, {p.c, p.c_stride}}, 3, p.N, es);
  a.B = p.B, a.T = p.T, a.D = p.D, a.N = p.N, a.G = p.G, a.R = p.D / p.G;
  a.softplus = p.dt_softplus;
  a.per_group = ceil_div(a.R, kTile), a.tiles = a.per_group * a.G;
  a.np = ceil_div(a.N, 4) * 4;
  a.wide = 2;
  while ((1 << a.wide) < a.N) ++a.wide;
  a.nmarks = ceil_div(a.T, kBlock);
}

// Segments of the time: as many as take the least time, by what a pass measured.  An
// SM that is given c CTAs of w warps, r at once, takes c + 9.5 / w ceil(c / r) for a
// token of them (9.5 / w: the latencies that the warps beside do not hide), and a CTA
// takes 17 tokens' time to start, and a third of one's for each segment ahead of it.
// More than one segment needs a first pass over all but one, with `pre` of the work.
// (Fitted to some 100 forwards and 50 gradients of 1 to 128 segments, which it gives
// to about 5 %; its choices take at most 4 % more than the best ones.  16384 tokens of
// 512 channels, 1 / 8 / 64 segments: 2404 / 495 / 150 us; 4 sequences of 2048, 2048
// channels, 1 / 4 / 8 segments 332 / 250 / 246 us and 674 / 624 / 592 of the gradient;
// 64 of 512, 512 channels, 1 / 2 segments 168 / 217 and 514 / 561 us.)
void cut(Problem& a, Fit fit, double pre) {
  const long units = (long)a.B * a.tiles;
  const int few = std::max(1, ceil_div(a.T, kBlock)), most = std::min(few, 128);
  auto pass = [&](long ctas) {
    const long c = (ctas + 147) / 148;
    return (double)c + 9.5 / fit.warps * (double)((c + fit.resident - 1) / fit.resident);
  };
  double best = 0.0;
  a.segs = 1, a.len = few * kBlock;
  for (int i = 0, s = 1, tried = 0; a.T > 0 && tried < most; ++i, s = i % 2 ? 2 << i / 2 : 3 << (i / 2 - 1)) {  // 1, 2, 3, 4, 6, 8, 12 ...
    tried = std::min(s, most);
    const int len = ceil_div(ceil_div(a.T, tried), kBlock) * kBlock, segs = ceil_div(a.T, len);
    double cost = (len + 17.0 + 0.3 * (segs - 1)) * pass(units * segs);
    if (segs > 1) cost += 10.0 + pre * (len + 17.0) * pass(units * (segs - 1));
    if (i == 0 || cost < 1.03 * best) a.segs = segs, a.len = len;  // of as good ones the finer, which balances better
    if (i == 0 || cost < best) best = cost;
  }
}

// Whether the lanes' two channels of dense tensors start on a boundary of two elements.
int even(const Problem& a, int dtype, uintptr_t all) { return a.R % 2 == 0 && (all & (2 * elem_size(dtype) - 1)) == 0; }

void lay_stash(Problem& a, Pieces& m) {
  a.marks = m.floats((size_t)a.B * a.tiles * a.nmarks * a.np * kTile);
  a.sums = a.z ? m.floats((size_t)a.B * a.T * a.D) : nullptr;
  a.even_sums = a.R % 2 == 0;
  const long rows[2] = {a.D, a.D};
  a.sums_piece = piece_of({{a.sums, rows}}, 2, a.R, sizeof(float));
}
void lay_segments(Problem& a, Pieces& m) {
  const size_t n = a.segs > 1 ? (size_t)a.B * a.tiles * a.segs * kTile : 0;
  a.seg_sums = m.floats(n * a.np);
  a.seg_steps = m.floats(n);
}
void lay_forward(Problem& a, Pieces& m) {
  cut(a, forward_fit(a.np), 0.56);
  lay_segments(a, m);
}
void lay_backward(Problem& a, Pieces& m) {
  cut(a, backward_fit(a.np), 0.22);
  lay_segments(a, m);
  a.part_bc = m.floats((size_t)a.B * a.tiles * a.T * 2 * a.np);
  a.part = m.floats((size_t)a.segs * a.B * a.D * (a.N + 2));
}

}  // namespace
}  // namespace scan
}  // namespace gru

using namespace gru;
using namespace gru::scan;

extern "C" size_t gru_scan_stash_bytes(const gru_scan_args* p) {
  if (check("gru_scan_stash_bytes", p, kSizesOnly)) return 0;
  Problem a{};
  fill(a, *p);
  Pieces m{nullptr};
  lay_stash(a, m);
  return m.used;
}

extern "C" size_t gru_scan_workspace_bytes(const gru_scan_args* p, int backward) {
  if (check("gru_scan_workspace_bytes", p, kSizesOnly)) return 0;
  Problem a{};
  fill(a, *p);
  Pieces m{nullptr};
  if (backward) lay_backward(a, m);
  else lay_forward(a, m);
  return m.used;
}

extern "C" int gru_scan_forward(const gru_scan_args* p, void* out, float* final_state, void* stash, size_t stash_bytes,
                                void* workspace, size_t workspace_bytes, void* stream_) {
  clear_error();
  const char* me = "gru_scan_forward";
  if (const int rc = check(me, p, kInputs)) return rc;
  if (p->B == 0) return GRU_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!final_state || bits(final_state) & 3) return refuse(me, "null or misaligned final_state");
  Problem a{};
  fill(a, *p);
  if (p->T == 0) {
    const size_t n = sizeof(float) * (size_t)p->B * p->D * p->N;
    if (!p->initial_state) GRU_CUDA_TRY(cudaMemsetAsync(final_state, 0, n, stream));
    else if (p->initial_state != final_state)
      GRU_CUDA_TRY(cudaMemcpyAsync(final_state, p->initial_state, n, cudaMemcpyDeviceToDevice, stream));
    return GRU_OK;
  }
  // several segments read the one while the last writes the other
  if (p->initial_state == final_state) return refuse(me, "final_state must not be the initial state");
  if (!out || bits(out) & (elem_size(p->dtype) - 1)) return refuse(me, "null or misaligned out");
  if (stash) {
    Pieces m{static_cast<char*>(stash)};
    lay_stash(a, m);
    if (stash_bytes < m.used || bits(stash) & 15) return refuse(me, "stash too small or not 16-byte aligned");
  }
  Pieces m{static_cast<char*>(workspace)};
  lay_forward(a, m);
  if (m.used && (!workspace || workspace_bytes < m.used || bits(workspace) & 15))
    return refuse(me, "workspace too small or not 16-byte aligned");
  a.out = out, a.last = final_state;
  a.even_out = even(a, p->dtype, bits(out));
  return forward(a, p->dtype, stream);
}

extern "C" int gru_scan_backward(const gru_scan_args* p, const void* dout, const float* dfinal, const void* stash,
                                 size_t stash_bytes, void* dx, void* ddt, float* da, void* db, void* dc, float* dskip,
                                 void* dz, float* ddt_bias, float* dinitial, void* workspace, size_t workspace_bytes,
                                 void* stream_) {
  clear_error();
  const char* me = "gru_scan_backward";
  if (const int rc = check(me, p, kInputs)) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const uintptr_t es = elem_size(p->dtype);
  if (!da || (bits(da) | bits(dskip) | bits(ddt_bias) | bits(dinitial) | bits(dfinal)) & 3 ||
      (bits(dx) | bits(ddt) | bits(db) | bits(dc) | bits(dz) | bits(dout)) & (es - 1))
    return refuse(me, "null or misaligned gradient");
  Problem a{};
  fill(a, *p);
  if (p->B == 0 || p->T == 0) {
    const size_t n = sizeof(float) * (size_t)p->B * p->D * p->N, wide = sizeof(float) * (size_t)p->D;
    GRU_CUDA_TRY(cudaMemsetAsync(da, 0, wide * p->N, stream));
    if (dskip) GRU_CUDA_TRY(cudaMemsetAsync(dskip, 0, wide, stream));
    if (ddt_bias) GRU_CUDA_TRY(cudaMemsetAsync(ddt_bias, 0, wide, stream));
    if (n && dinitial && !dfinal) GRU_CUDA_TRY(cudaMemsetAsync(dinitial, 0, n, stream));
    else if (n && dinitial && dfinal != dinitial)
      GRU_CUDA_TRY(cudaMemcpyAsync(dinitial, dfinal, n, cudaMemcpyDeviceToDevice, stream));
    return GRU_OK;
  }
  if (!dx || !ddt || !db || !dc || (p->z && !dz)) return refuse(me, "null gradient");
  if (dinitial && dinitial == dfinal) return refuse(me, "dinitial must not be dfinal");
  Pieces m{static_cast<char*>(const_cast<void*>(stash))}, w{static_cast<char*>(workspace)};
  lay_stash(a, m);
  lay_backward(a, w);
  if (!stash || stash_bytes < m.used || !workspace || workspace_bytes < w.used || (bits(stash) | bits(workspace)) & 15)
    return refuse(me, "stash or workspace too small or not 16-byte aligned");
  a.dout = dout, a.dlast = dfinal;
  a.even_out = even(a, p->dtype, bits(dx) | bits(ddt) | bits(dz));
  const long rows[2] = {p->D, p->D};  // with the groups' channels, all that dout's rows add up from
  a.dout_piece = piece_of({{dout, rows}}, 2, p->D / p->G, (int)es);
  a.dx = dx, a.ddt = ddt, a.da = da, a.db = db, a.dc = dc, a.dskip = dskip, a.dz = dz, a.dbias = ddt_bias, a.ds0 = dinitial;
  return backward(a, p->dtype, stream);
}

extern "C" int gru_scan_step(const gru_scan_args* p, float* state, void* out, void* stream_) {
  clear_error();
  const char* me = "gru_scan_step";
  if (const int rc = check(me, p, kInputs)) return rc;
  if (p->T != 1) return refuse(me, "T must be 1");
  if (p->B == 0) return GRU_OK;
  if (!state || !out || bits(state) & 3 || bits(out) & (elem_size(p->dtype) - 1))
    return refuse(me, "null or misaligned state or out");
  Problem a{};
  fill(a, *p);
  a.out = out;
  const uintptr_t four = 4 * elem_size(p->dtype) - 1;
  const int vec = p->N % 4 == 0 && ((bits(state) | bits(p->a)) & 15) == 0 && ((bits(p->b) | bits(p->c)) & four) == 0 &&
                  (p->b_stride[0] | p->b_stride[2] | p->c_stride[0] | p->c_stride[2]) % 4 == 0;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return p->dtype == GRU_F32 ? step<float>(a, state, vec, stream) : step<bf16>(a, state, vec, stream);
}
