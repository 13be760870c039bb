// The short causal convolution of each channel with its own W weights, its
// gradient and its single token (contract in include/rnn_kernel_b200.h).
//
//   p_t = bias + sum_j w_j x_{t-W+1+j};  y = p, or silu(p) = p sigmoid(p)
//   e = dy silu'(p);  dx_t = sum_j w_j e_{t+W-1-j};  dw_j = sum_t e_t x_{t-W+1+j};  db = sum_t e_t
//
// Tokens before the first come from a state of W - 1 inputs.  A thread takes a
// few neighbouring channels through a run of tokens with the last W inputs in
// registers (the loop goes W tokens at a time, so that none of them is moved), so x
// is read once, but for the W - 1 tokens that two runs share.  The gradient keeps
// the last W errors too: e_t is final when x_t is read, and with it dx_{t-W+1}.
// Sums of dw and db go from a thread's registers over the CTA's runs and then over
// the CTAs, in a fixed order.  Loads have no branch around them, which would wait for
// each: rows past the ends are the last one again, and their numbers dropped.
//
// 4 x 2048 tokens of 4096 channels, 4 weights, bf16: forward 32 us (134 MB, 64 % of the
// copy rate), gradient 62 us (201 MB, 49 %).  Memory is the floor; instructions and their
// latencies bound it, with what a window takes of the registers (issue slots 53 and
// 48 %).  Two channels a thread and more warps: 13 % and 15 % slower or more.

#include <algorithm>
#include <type_traits>

#include "row_ops.cuh"

namespace gru {
namespace {

constexpr int kMinConv = 2, kMaxConv = 8;
constexpr int kGradRuns = 8;    // runs of tokens of a gradient's CTA

struct Conv {
  const void *x, *w, *bias, *s0;
  void *y, *last;
  // gradient
  const void *dy, *dlast;
  void *dx, *ds0;
  float* part;  // [CTA of tokens][W + 1][D]
  long xb, xt;  // elements between x's batch rows and tokens
  int B, T, D, W, wtype, wvec, silu, run, runs;  // wvec: weights lie on boundaries of V elements
};

// a[e] b[e] + c[e], neighbours packed.
template <int V>
__device__ __forceinline__ void fma_into(float (&c)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 r = __ffma2_rn(make_float2(a[e], a[e + 1]), make_float2(b[e], b[e + 1]), make_float2(c[e], c[e + 1]));
      c[e] = r.x, c[e + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = fmaf(a[e], b[e], c[e]);
  }
}

// a[e] *= b[e], neighbours packed.
template <int V>
__device__ __forceinline__ void mul_into(float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 r = __fmul2_rn(make_float2(a[e], a[e + 1]), make_float2(b[e], b[e + 1]));
      a[e] = r.x, a[e + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) a[e] *= b[e];
  }
}

// The weights of channels c .. c + V - 1.
template <int W, int V>
__device__ __forceinline__ void weights(const Conv& a, int c, float (&w)[W][V], float (&bias)[V]) {
  float flat[W][V];  // V channels x W weights, as they lie
#pragma unroll
  for (int i = 0; i < W; ++i) get_row<V>(a.w, (long)c * W + i * V, a.wtype, a.wvec, flat[i]);
  get_row<V>(a.bias ? a.bias : a.w, c, a.wtype, a.wvec, bias);
#pragma unroll
  for (int e = 0; e < V; ++e) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e] = flat[(e * W + j) / V][(e * W + j) % V];
    if (!a.bias) bias[e] = 0.0f;
  }
}

// A thread's channels c .. c + V - 1 of batch row b.
template <typename T, int W, int V>
struct Run {
  const T *x, *s0;  // rows of tokens 0
  float w[W][V], bias[V], win[W][V];  // the input of token t at win[t mod W], counted from the run's first
  __device__ __forceinline__ Run(const Conv& a, int b, int c) {
    x = static_cast<const T*>(a.x) + b * a.xb + c;
    s0 = a.s0 ? static_cast<const T*>(a.s0) + ((long)b * (W - 1) + W - 1) * a.D + c : nullptr;
    weights<W, V>(a, c, w, bias);
  }
  // Token t, which may lie before the first.
  __device__ __forceinline__ void any(const Conv& a, int t, float (&v)[V]) const {
    const T* at = t < 0 && s0 ? s0 + (long)t * a.D : x + (long)min(max(t, 0), a.T - 1) * a.xt;
    load_row<V>(at, v);
    if (t < 0 && !s0)
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = 0.0f;
  }
  __device__ __forceinline__ void start(const Conv& a, int t0) {
#pragma unroll
    for (int j = 1; j < W; ++j) any(a, t0 - W + j, win[j]);
  }
  // The sum for token u of a turn.
  __device__ __forceinline__ void sum(int u, float (&p)[V]) const {
#pragma unroll
    for (int e = 0; e < V; ++e) p[e] = bias[e];
#pragma unroll
    for (int j = 0; j < W; ++j) fma_into(p, w[j], win[(u + 1 + j) % W]);
  }
};

template <typename T, int W, int V>
__global__ void __launch_bounds__(256, V > 2 ? 3 : 2) conv_forward_kernel(const Conv a) {
  const int vecs = a.D / V;
  const long item = blockIdx.x * 256L + threadIdx.x;
  const long rest = item / vecs;
  const int c = (int)(item - rest * vecs) * V;
  const int b = (int)(rest / a.runs);
  if (b >= a.B) return;
  const int t0 = (int)(rest - (long)b * a.runs) * a.run, t1 = min(t0 + a.run, a.T);
  Run<T, W, V> r(a, b, c);
  r.start(a, t0);
  T* y = static_cast<T*>(a.y) + ((long)b * a.T + t0) * a.D + c;
  Raw<T, V> next[2][W];  // two turns ahead
  auto load = [&](int t, Raw<T, V>(&to)[W]) {
#pragma unroll
    for (int u = 0; u < W; ++u) to[u].load(r.x + (long)min(t + u, a.T - 1) * a.xt);
  };
  load(t0, next[0]);
  load(t0 + W, next[1]);
  // Each input goes where the oldest of the window was, and the one that follows it two
  // turns later is asked for.
  auto turn = [&](int t, Raw<T, V>(&raw)[W]) {
    const bool more = t + 2 * W < t1;
#pragma unroll
    for (int u = 0; u < W; ++u) {
      raw[u].get(r.win[u]);
      if (more) raw[u].load(r.x + (long)min(t + 2 * W + u, a.T - 1) * a.xt);
      float p[V];
      r.sum(u, p);
      if (a.silu) {
        float g[V];
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = sigmoid_of(p[e]);
        mul_into(p, g);
      }
      if (t + u < t1) store_row<V>(y, p);
      y += a.D;
    }
  };
  for (int t = t0; t < t1; t += 2 * W) {
    turn(t, next[0]);
    if (t + W < t1) turn(t + W, next[1]);
  }
  if (t1 == a.T) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      float v[V];
      r.any(a, a.T - (W - 1) + j, v);
      store_row<V>(static_cast<T*>(a.last) + ((long)b * (W - 1) + j) * a.D + c, v);
    }
  }
}

// A CTA: 32 lanes x V channels, kGradRuns runs of tokens, one a warp.
template <typename T, int W, int V>
__global__ void __launch_bounds__(32 * kGradRuns, W <= 4 ? 2 : 1) conv_backward_kernel(const Conv a) {
  extern __shared__ __align__(16) float sums[];  // [run][W + 1][32 V]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = (a.D + 32 * V - 1) / (32 * V);
  const int cb = blockIdx.x % blocks;
  const long rest = blockIdx.x / blocks;  // batch row and run group
  const int groups = (a.runs + kGradRuns - 1) / kGradRuns;
  const int b = (int)(rest / groups), run = (int)(rest - (long)b * groups) * kGradRuns + warp;
  const int c = (cb * 32 + lane) * V;
  float dw[W][V], db[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    db[e] = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j][e] = 0.0f;
  }
  if (c < a.D && run < a.runs) {
    const int t0 = run * a.run, t1 = min(t0 + a.run, a.T);
    Run<T, W, V> r(a, b, c);
    r.start(a, t0);
    float err[W][V];  // the error of token t at err[t mod W]
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) err[j][e] = 0.0f;
    const long dense = (long)b * a.T * a.D + c;
    const T* dy = a.dy ? static_cast<const T*>(a.dy) + dense : nullptr;
    Raw<T, V> xn[W], dn[W];  // a turn ahead
    auto load = [&](int t, int u) {
      const long at = min(t + u, a.T - 1);
      xn[u].load(r.x + at * a.xt);
      if (dy) dn[u].load(dy + at * a.D);
    };
#pragma unroll
    for (int u = 0; u < W; ++u) load(t0, u);
    // Errors of the W - 1 tokens behind the run belong to its dx; the first run's
    // errors also go to the state.
    const int end = t1 + W - 1;
    // W tokens from t on.  INNER: all of them, and those that their dx belongs to, are
    // this run's, and no state's; and there is a dy.
    auto turn = [&](int t, auto inner) {
      constexpr bool INNER = decltype(inner)::value;
      const bool more = t + W < end;
      T* dx = static_cast<T*>(a.dx) + dense + (long)(t - (W - 1)) * a.D;
#pragma unroll
      for (int u = 0; u < W; ++u, dx += a.D) {
        const int now = t + u;
        xn[u].get(r.win[u]);
        float (&q)[V] = err[u];
        dn[u].get(q);
        if (more) load(t + W, u);
        if (!INNER && !dy)
#pragma unroll
          for (int e = 0; e < V; ++e) q[e] = 0.0f;
        if (a.silu) {  // s + p s (1 - s)
          float p[V], s[V], n[V];
          r.sum(u, p);
#pragma unroll
          for (int e = 0; e < V; ++e) s[e] = sigmoid_of(p[e]), n[e] = 1.0f - s[e];
          mul_into(p, s);
          fma_into(s, p, n);
          mul_into(q, s);
        }
        if (!INNER && now >= a.T)
#pragma unroll
          for (int e = 0; e < V; ++e) q[e] = 0.0f;
        if (INNER || now < t1) {
#pragma unroll
          for (int e = 0; e < V; ++e) db[e] += q[e];
#pragma unroll
          for (int j = 0; j < W; ++j) fma_into(dw[j], q, r.win[(u + 1 + j) % W]);
        }
        float g[V];
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) fma_into(g, r.w[W - 1 - j], err[(u + 1 + j) % W]);
        if (INNER) {
          store_row<V>(dx, g);
          continue;
        }
        // dx of token now - W + 1
        const int to = now - (W - 1);
        if (now >= end || (to < t0 && t0 > 0)) continue;  // past the run, or an earlier one's
        if (a.dlast && to >= a.T - (W - 1)) {
          float s[V];
          load_row<V>(static_cast<const T*>(a.dlast) + ((long)b * (W - 1) + to - (a.T - (W - 1))) * a.D + c, s);
#pragma unroll
          for (int e = 0; e < V; ++e) g[e] += s[e];
        }
        if (to >= 0) store_row<V>(dx, g);
        else if (a.ds0) store_row<V>(static_cast<T*>(a.ds0) + ((long)b * (W - 1) + (W - 1) + to) * a.D + c, g);
      }
    };
    turn(t0, std::false_type{});
    int t = t0 + W;
    if (dy)
      for (; t + W <= t1 && t + W <= a.T - (W - 1); t += W) turn(t, std::true_type{});
    for (; t < end; t += W) turn(t, std::false_type{});
  }
  constexpr int C = 32 * V;
#pragma unroll
  for (int j = 0; j < W; ++j) store_row<V>(sums + (warp * (W + 1) + j) * C + lane * V, dw[j]);
  store_row<V>(sums + (warp * (W + 1) + W) * C + lane * V, db);
  __syncthreads();
  for (int i = threadIdx.x; i < (W + 1) * C; i += 32 * kGradRuns) {
    const int col = cb * C + i % C;
    if (col >= a.D) continue;
    float s = sums[i];
#pragma unroll
    for (int r = 1; r < kGradRuns; ++r) s += sums[r * (W + 1) * C + i];
    a.part[(rest * (W + 1) + i / C) * a.D + col] = s;
  }
}

// One token: the state moves on by one input.  A thread has its channels' weights for
// ROWS sequences, whose loads are in flight together.
template <typename T, int W, int V, int ROWS>
__global__ void __launch_bounds__(128) conv_step_kernel(const Conv a) {
  const int vecs = a.D / V;
  const long item = blockIdx.x * 128L + threadIdx.x;
  const long group = item / vecs;
  const int b0 = (int)group * ROWS, c = (int)(item - group * vecs) * V;
  if (b0 >= a.B) return;
  float w[W][V], bias[V];
  Raw<T, V> in[ROWS][W];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int b = min(b0 + k, a.B - 1);
    const T* s = static_cast<const T*>(a.last) + (long)b * (W - 1) * a.D + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) in[k][j].load(s + (long)j * a.D);
    in[k][W - 1].load(static_cast<const T*>(a.x) + b * a.xb + c);
  }
  weights<W, V>(a, c, w, bias);
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    if (k > 0 && b0 + k >= a.B) break;
    T* s = static_cast<T*>(a.last) + (long)(b0 + k) * (W - 1) * a.D + c;
    float p[V];
#pragma unroll
    for (int e = 0; e < V; ++e) p[e] = bias[e];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float v[V];
      in[k][j].get(v);
      fma_into(p, w[j], v);
      if (j > 0) store_row<V>(s + (long)(j - 1) * a.D, v);
    }
    if (a.silu) {
      float g[V];
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = sigmoid_of(p[e]);
      mul_into(p, g);
    }
    store_row<V>(static_cast<T*>(a.y) + (long)(b0 + k) * a.D + c, p);
  }
}

template <typename T, int W, int V, int ROWS>
void launch_step(const Conv& a, cudaStream_t stream) {
  const long threads = (long)((a.B + ROWS - 1) / ROWS) * (a.D / V);
  conv_step_kernel<T, W, V, ROWS><<<(unsigned)((threads + 127) / 128), 128, 0, stream>>>(a);
}

struct StoreConv {
  void *dw, *db;
  int D, W, dtype;
  __device__ __forceinline__ void operator()(long i, float x) const {
    const long j = i / D, c = i - j * D;
    if (j < W) put(dw, c * W + j, dtype, x);
    else if (db) put(db, c, dtype, x);
  }
};

enum Way { kForward, kBackward, kStep };

template <typename T, int W, int V>
int launch(const Conv& a, Way way, const StoreConv& store, cudaStream_t stream) {
  if (way == kStep) {
    LaunchScope scope(kKindCausalConv, stream);
    // four sequences a thread where that leaves three CTAs for an SM (4096 channels, 4
    // weights, bf16, one and four a thread: 256 sequences 5.5 and 3.7 us, 512 8.8 and 5.4)
    if ((long)a.B * (a.D / V) >= 4L * 128 * 3 * 148) launch_step<T, W, V, 4>(a, stream);
    else launch_step<T, W, V, 1>(a, stream);
  } else if (way == kForward) {
    LaunchScope scope(kKindCausalConv, stream);
    conv_forward_kernel<T, W, V><<<(unsigned)(((long)a.B * a.runs * (a.D / V) + 255) / 256), 256, 0, stream>>>(a);
  } else {
    LaunchScope scope(kKindCausalConv, stream, 2);
    const int parts = a.B * ceil_div(a.runs, kGradRuns);
    const size_t smem = sizeof(float) * kGradRuns * (W + 1) * 32 * V;
    conv_backward_kernel<T, W, V><<<(unsigned)((long)parts * ceil_div(a.D, 32 * V)), 32 * kGradRuns, smem, stream>>>(a);
    GRU_CUDA_TRY(cudaGetLastError());
    const long cols = (W + 1L) * a.D;
    return sum_parts(a.part, parts, cols, cols, store, stream);
  }
  GRU_CUDA_TRY(cudaGetLastError());
  return GRU_OK;
}

// V: elements a thread; two where the window is long, for its registers' sake.  (Four were
// chosen by bf16 times.  In FP32 W = 4 spills 108 bytes in the forward and 360 in the gradient:
// 4 x 2048 tokens of 4096 channels 70 and 130 us, timed with the launches, where bytes take
// 41 and 62.)
template <typename T>
int launch_any(const Conv& a, bool vec, Way way, const StoreConv& store, cudaStream_t stream) {
#define GRU_CONV(WIDTH, V)                                                             \
  if (a.W == WIDTH)                                                                  \
    return vec ? launch<T, WIDTH, V>(a, way, store, stream) : launch<T, WIDTH, 1>(a, way, store, stream);
  GRU_CONV(2, 4)
  GRU_CONV(3, 4)
  GRU_CONV(4, 4)
  GRU_CONV(5, 2)
  GRU_CONV(6, 2)
  GRU_CONV(7, 2)
  GRU_CONV(8, 2)
#undef GRU_CONV
  return GRU_ERR_UNSUPPORTED;
}

// The tokens of a run, of T that `units` pieces of work each have: of the runs that
// fill the GPU once, twice and so on, those that take the least, at `extra` tokens'
// time besides its own for a run.  side: runs of a CTA; resident: CTAs of an SM.  Not
// above `longest`, and not more runs than eighths of T, so of 5 tokens at least where T
// is more.  (4 x 2048 tokens of 4096 channels, bf16, timed with the launches and the sum, which
// the file's head leaves out: forward in runs of 76, once the GPU, 37 us, of 32 39, of 64
// or 128 43; gradient in runs of 128, once, 71 us, of 32 or 64 77.)
int run_of(long units, int side, int resident, int T, int longest, int extra) {
  const long slots = 148L * resident, most = (T + 7) / 8, least = (T + longest - 1) / longest;
  long best = 0;
  int run = T;
  for (long k = 1; k <= 8; ++k) {
    const long runs = std::min(std::max(k * slots * side / units, least), most);
    const int len = (int)((T + runs - 1) / runs);
    const long ctas = (units * ceil_div(T, len) + side - 1) / side;
    const long cost = (ctas + slots - 1) / slots * (len + extra);
    if (k == 1 || cost < best) best = cost, run = len;
  }
  return run;
}
// A gradient's: its CTAs take 8 runs of one batch row and 32 lanes, so that short sequences
// have runs down to a token, one for each warp (4096 channels, bf16: 64 x 8 tokens 42 us in
// runs of 1 or of 8, 64 x 72 75 us in runs of 9, 114 in runs of 8, whose last one takes a
// CTA).  The same whether
// or not the tensors' boundaries let a lane have several channels.  A thread adds up
// at most 512 tokens of dw in FP32 (an error of about 256^0.5 2^-25 = 5e-7 of it).
int grad_run(const gru_conv_args& p) {
  const long units = (long)p.B * ceil_div(p.D, p.W <= 4 ? 128 : 64);
  return run_of(units, 1, p.W <= 4 ? 2 : 1, ceil_div(p.T, kGradRuns), 512, p.W + 3);
}
long grad_parts(const gru_conv_args& p) {
  return p.T > 0 && p.B > 0 ? (long)p.B * ceil_div(ceil_div(p.T, grad_run(p)), kGradRuns) : 0;
}

int check(const char* me, const gru_conv_args* p) {
  if (!p) return refuse(me, "null arguments");
  if (!known(p->dtype) || !known(p->weight_dtype)) return refuse(me, "types must be GRU_F32 or GRU_BF16", GRU_ERR_UNSUPPORTED);
  if (p->weight_dtype != p->dtype && p->weight_dtype != GRU_F32)
    return refuse(me, "the weights must be FP32 or of x's type", GRU_ERR_UNSUPPORTED);
  if (p->B < 0 || p->T < 0 || p->D < 1) return refuse(me, "need B >= 0, T >= 0 and D >= 1");
  if (p->T > (1 << 30) || p->D > (1 << 24)) return refuse(me, "too many tokens or channels", GRU_ERR_UNSUPPORTED);
  if (p->W < kMinConv || p->W > kMaxConv) return refuse(me, "the width must be in [2, 8]", GRU_ERR_UNSUPPORTED);
  if (p->activation != 0 && p->activation != 1) return refuse(me, "activation must be 0 or 1", GRU_ERR_UNSUPPORTED);
  // CTAs of the smallest pieces that a launch cuts the work into
  const long runs = std::max(1L, (p->T + 7L) / 8);
  if ((double)p->B * runs * p->D / 128 > 2e9) return refuse(me, "too large for one launch", GRU_ERR_UNSUPPORTED);
  if (bits(p->x) & (elem_size(p->dtype) - 1) || bits(p->initial_state) & (elem_size(p->dtype) - 1) ||
      bits(p->weight) & (elem_size(p->weight_dtype) - 1) || bits(p->bias) & (elem_size(p->weight_dtype) - 1))
    return refuse(me, "a tensor is not aligned to its element size");
  return GRU_OK;
}

void fill(Conv& a, const gru_conv_args& p) {
  a.x = p.x, a.w = p.weight, a.bias = p.bias, a.s0 = p.initial_state;
  a.xb = p.x_stride[0], a.xt = p.x_stride[1];
  a.B = p.B, a.T = p.T, a.D = p.D, a.W = p.W, a.wtype = p.weight_dtype, a.silu = p.activation;
  const int v = p.W <= 4 ? 4 : 2;
  a.wvec = ((bits(p.weight) | bits(p.bias)) & (v * elem_size(p.weight_dtype) - 1)) == 0;
}

// Whether every row of the dense tensors and of x starts on the boundary that V
// elements need.
bool vectors(const gru_conv_args& p, uintptr_t all) {
  const int v = p.W <= 4 ? 4 : 2;
  return p.D % v == 0 && p.x_stride[0] % v == 0 && p.x_stride[1] % v == 0 && (all & (v * elem_size(p.dtype) - 1)) == 0;
}

}  // namespace
}  // namespace gru

using namespace gru;

extern "C" size_t gru_conv_workspace_bytes(const gru_conv_args* p) {
  if (check("gru_conv_workspace_bytes", p)) return 0;
  return align_up(sizeof(float) * (size_t)grad_parts(*p) * (p->W + 1) * p->D, 256);
}

extern "C" int gru_conv_forward(const gru_conv_args* p, void* out, void* final_state, void* stream_) {
  clear_error();
  const char* me = "gru_conv_forward";
  if (const int rc = check(me, p)) return rc;
  if (p->B == 0) return GRU_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const uintptr_t es = elem_size(p->dtype);
  if (!final_state || bits(final_state) & (es - 1)) return refuse(me, "null or misaligned final_state");
  if (p->T == 0) {
    const size_t n = es * p->B * (p->W - 1) * p->D;
    if (!p->initial_state) GRU_CUDA_TRY(cudaMemsetAsync(final_state, 0, n, stream));
    else if (p->initial_state != final_state)
      GRU_CUDA_TRY(cudaMemcpyAsync(final_state, p->initial_state, n, cudaMemcpyDeviceToDevice, stream));
    return GRU_OK;
  }
  if (!p->x || !p->weight || !out || bits(out) & (es - 1)) return refuse(me, "null tensor or misaligned out");
  if (p->initial_state && p->initial_state == final_state) return refuse(me, "final_state must not be the initial state");
  Conv a{};
  fill(a, *p);
  a.y = out, a.last = final_state;
  const bool vec = vectors(*p, bits(p->x) | bits(p->initial_state) | bits(out) | bits(final_state));
  const int v = vec ? (p->W <= 4 ? 4 : 2) : 1;
  a.run = run_of((long)p->B * (p->D / v), 256, v > 2 ? 3 : 2, p->T, p->T, p->W + 3);
  a.runs = ceil_div(p->T, a.run);
  return p->dtype == GRU_F32 ? launch_any<float>(a, vec, kForward, {}, stream) : launch_any<bf16>(a, vec, kForward, {}, stream);
}

extern "C" int gru_conv_backward(const gru_conv_args* p, const void* dout, const void* dfinal, void* dx, void* dweight,
                                 void* dbias, void* dinitial, void* workspace, size_t workspace_bytes, void* stream_) {
  clear_error();
  const char* me = "gru_conv_backward";
  if (const int rc = check(me, p)) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const uintptr_t es = elem_size(p->dtype), ws = elem_size(p->weight_dtype);
  if (!dweight || bits(dweight) & (ws - 1) || bits(dbias) & (ws - 1))
    return refuse(me, "null or misaligned gradient of the weight");
  if (bits(dout) & (es - 1) || bits(dfinal) & (es - 1) || bits(dx) & (es - 1) || bits(dinitial) & (es - 1))
    return refuse(me, "a tensor is not aligned to its element size");
  if (p->B == 0 || p->T == 0) {
    GRU_CUDA_TRY(cudaMemsetAsync(dweight, 0, ws * p->D * p->W, stream));
    if (dbias) GRU_CUDA_TRY(cudaMemsetAsync(dbias, 0, ws * p->D, stream));
    const size_t n = es * p->B * (p->W - 1) * p->D;
    if (n && dinitial && !dfinal) GRU_CUDA_TRY(cudaMemsetAsync(dinitial, 0, n, stream));
    else if (n && dinitial && dfinal != dinitial)
      GRU_CUDA_TRY(cudaMemcpyAsync(dinitial, dfinal, n, cudaMemcpyDeviceToDevice, stream));
    return GRU_OK;
  }
  if (!p->x || !p->weight || !dx) return refuse(me, "null tensor");
  if (!workspace || bits(workspace) & 15 || workspace_bytes < gru_conv_workspace_bytes(p))
    return refuse(me, "workspace too small or not 16-byte aligned");
  Conv a{};
  fill(a, *p);
  a.dy = dout, a.dlast = dfinal, a.dx = dx, a.ds0 = dinitial, a.part = static_cast<float*>(workspace);
  a.run = grad_run(*p), a.runs = ceil_div(p->T, a.run);
  const bool vec = vectors(*p, bits(p->x) | bits(p->initial_state) | bits(dout) | bits(dfinal) | bits(dx) | bits(dinitial));
  const StoreConv store{dweight, dbias, p->D, p->W, p->weight_dtype};
  return p->dtype == GRU_F32 ? launch_any<float>(a, vec, kBackward, store, stream)
                             : launch_any<bf16>(a, vec, kBackward, store, stream);
}

extern "C" int gru_conv_step(const gru_conv_args* p, void* state, void* out, void* stream_) {
  clear_error();
  const char* me = "gru_conv_step";
  if (const int rc = check(me, p)) return rc;
  if (p->T != 1) return refuse(me, "T must be 1");
  if (p->B == 0) return GRU_OK;
  const uintptr_t es = elem_size(p->dtype);
  if (!p->x || !p->weight || !state || !out || (bits(state) | bits(out)) & (es - 1))
    return refuse(me, "null or misaligned tensor");
  Conv a{};
  fill(a, *p);
  a.y = out, a.last = state;
  const bool vec = vectors(*p, bits(p->x) | bits(state) | bits(out));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return p->dtype == GRU_F32 ? launch_any<float>(a, vec, kStep, {}, stream) : launch_any<bf16>(a, vec, kStep, {}, stream);
}
