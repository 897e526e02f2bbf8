// Gated linear recurrence over the frames of ragged utterances, channels last:
//
//   f_t = sigmoid(gate_t),  h_t = f_t h_{t-1} + (1 - f_t) x_t,  y_t = h_t        (per utterance and channel)
//
// t runs over the utterance's own frames, first to last or (reverse) last to first; frames behind its end are never
// read and their outputs are zero.  The state is held in the accumulation type (float; double for double) whatever the
// tensors' type, and so are the states kept for backward: one every kStateStride frames (kRows for long utterances).
//
// Backward, with gh_t the whole gradient of h_t and m_t = f_{t+1} gh_{t+1} what the frames after t pass back:
//
//   gh_t = gy_t + m_t,  m_{t-1} = f_t gh_t,  gx_t = (1 - f_t) gh_t,  ggate_t = f_t (1 - f_t) gh_t (h_{t-1} - x_t)
//
// h_{t-1} is recomputed from the kept states: y is not read (it may be rounded to 16 bits, and it would be one more
// tensor to fetch).
#include <cooperative_groups.h>

#include <algorithm>

#include "sequence_common.cuh"

namespace mellin {
namespace {

using namespace seq;

constexpr int kStateStride = 16;
constexpr int kWalkThreads = 128;
constexpr int kWalkFrames = 4;    // up to so many frames: one thread per channel

template <typename T>
struct RecurrenceArgs {
  Frames<const T> x, gate, grad_y;
  Frames<T> y, grad_x, grad_gate;
  const Acc<T> *initial = nullptr, *grad_final = nullptr;  // (batch, channels), or null: zeros
  Acc<T> *final = nullptr, *grad_initial = nullptr;        // (batch, channels), or null
  Acc<T> *states = nullptr;                                // (batch, ceil(frames / kStateStride), channels), or null
  const int *lens = nullptr;
  int batch = 0, frames = 0, channels = 0, reverse = 0;
  int tiles = 0, cluster = 1;  // blocks across the channels; blocks of a cluster across the frames
};

// One thread per (utterance, channel), frame after frame: for a few frames a call, where there is nothing to split, and
// for tensors whose frames lie 2^31 elements or more apart.
template <typename T>
__global__ void __launch_bounds__(kWalkThreads) recurrence_walk_kernel(const RecurrenceArgs<T> a) {
  begin<false>();
  using A = Acc<T>;
  const long long i = blockIdx.x * (long long)kWalkThreads + threadIdx.x;
  if (i >= (long long)a.batch * a.channels) return;
  const long long n = i / a.channels, c = i - n * a.channels;
  const int len = live_frames(a.lens, n, a.frames);
  const long long slots = (a.frames + kStateStride - 1) / kStateStride;
  const T *x = a.x.p + n * a.x.sn + c, *gate = a.gate.p + n * a.gate.sn + c;
  T *y = a.y.p + n * a.y.sn + c;
  A h = a.initial != nullptr ? a.initial[i] : A(0);
  for (int s = 0; s < len; ++s) {
    if (a.states != nullptr && s % kStateStride == 0) a.states[(n * slots + s / kStateStride) * a.channels + c] = h;
    const long long t = a.reverse ? len - 1 - s : s;
    A f, keep;
    sigmoid_pair<true>(to_acc(gate[t * a.gate.st]), f, keep);
    h = f * h + keep * to_acc(x[t * a.x.st]);
    y[t * a.y.st] = from_acc<T>(h);
  }
  for (long long t = len; t < a.frames; ++t) y[t * a.y.st] = from_acc<T>(A(0));
  if (a.final != nullptr) a.final[i] = h;
}

template <typename T>
__global__ void __launch_bounds__(kWalkThreads) recurrence_walk_backward_kernel(const RecurrenceArgs<T> a) {
  begin<false>();
  using A = Acc<T>;
  const long long i = blockIdx.x * (long long)kWalkThreads + threadIdx.x;
  if (i >= (long long)a.batch * a.channels) return;
  const long long n = i / a.channels, c = i - n * a.channels;
  const int len = live_frames(a.lens, n, a.frames);
  const long long slots = (a.frames + kStateStride - 1) / kStateStride;
  const T *x = a.x.p + n * a.x.sn + c, *gate = a.gate.p + n * a.gate.sn + c;
  const T *gy = a.grad_y.p == nullptr ? nullptr : a.grad_y.p + n * a.grad_y.sn + c;
  T *gx = a.grad_x.p + n * a.grad_x.sn + c, *gg = a.grad_gate.p + n * a.grad_gate.sn + c;
  A m = a.grad_final != nullptr ? a.grad_final[i] : A(0);
  for (int first = (len - 1) / kStateStride * kStateStride; len > 0 && first >= 0; first -= kStateStride) {
    A f[kStateStride], keep[kStateStride], d[kStateStride];  // d = h_{t-1} - x_t
    A h = a.states[(n * slots + first / kStateStride) * a.channels + c];
#pragma unroll
    for (int k = 0; k < kStateStride; ++k) {
      if (first + k < len) {
        const long long t = a.reverse ? len - 1 - (first + k) : first + k;
        const A xv = to_acc(x[t * a.x.st]);
        sigmoid_pair<true>(to_acc(gate[t * a.gate.st]), f[k], keep[k]);
        d[k] = h - xv;
        h = f[k] * h + keep[k] * xv;
      }
    }
#pragma unroll
    for (int k = kStateStride - 1; k >= 0; --k) {
      if (first + k < len) {
        const long long t = a.reverse ? len - 1 - (first + k) : first + k;
        const A gh = m + (gy != nullptr ? to_acc(gy[t * a.grad_y.st]) : A(0));
        m = f[k] * gh;
        gx[t * a.grad_x.st] = from_acc<T>(keep[k] * gh);
        gg[t * a.grad_gate.st] = from_acc<T>(keep[k] * m * d[k]);
      }
    }
  }
  for (long long t = len; t < a.frames; ++t) gx[t * a.grad_x.st] = gg[t * a.grad_gate.st] = from_acc<T>(A(0));
  if (a.grad_initial != nullptr) a.grad_initial[i] = m;
}

// ---- scan over pieces of the time axis -----------------------------------------------------------------------------
//
// A block has CT = CL * V adjacent channels of one utterance and walks its frames W * kStateStride at a time.  A warp has
// kStateStride of them, a thread S frames of V channels, in registers: TL = 32 / CL threads of a warp split its frames.
// A run of frames maps the state before it to the state after it, h -> A h + B with A the product of its f; the runs'
// (A, B) are joined across a warp by shuffles and across the block's warps through shared memory.  Then every thread
// knows the state before its first frame and walks its own frames.  Each input is read once, each output written once;
// the next frames' loads are in flight while the present ones are joined.  The order of all sums is fixed.
//
// Frames that do not exist are gates of +infinity on values of zero: f = 1, keep = 0, the state passes through.

// V values of the accumulation type by accesses of at most 16 bytes
template <int V, typename A>
__device__ __forceinline__ void store_acc(A *to, const A (&from)[V]) {
  store_raw<A, V>(to, rounded<A, V>(from));
}
template <int V, typename A>
__device__ __forceinline__ void load_acc(A (&to)[V], const A *from) {
  constexpr int W = V * sizeof(A) <= 16 ? V : 16 / (int)sizeof(A);
  struct alignas(W * sizeof(A)) Part {
    A v[W];
  };
#pragma unroll
  for (int v = 0; v < V; v += W) {
    const Part p = *reinterpret_cast<const Part *>(from + v);
#pragma unroll
    for (int i = 0; i < W; ++i) to[v + i] = p.v[i];
  }
}

template <typename A, int CT, int W>
struct alignas(16) ScanShared {
  A a[2][W][CT], b[2][W][CT], carry[2][CT];
};
template <typename T, int V, int CL, int W, int MB>
__global__ void __launch_bounds__(32 * W, MB) recurrence_scan_kernel(const RecurrenceArgs<T> a) {
  begin<false>();
  using A = Acc<T>;
  constexpr int TL = 32 / CL, S = kStateStride / TL, CT = CL * V, SPAN = W * kStateStride;
  __shared__ ScanShared<A, CT, W> sh;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, cl = lane % CL, tl = lane / CL, at = cl * V;
  const int unit = (int)blockIdx.x;
  const Utterance whose = utterance_of(a.lens, a.batch, a.frames, unit / a.tiles);
  const long long n = whose.n;
  const int c = unit % a.tiles * CT + at;
  const bool on = c < a.channels;
  const int len = whose.len, steps = (len + SPAN - 1) / SPAN;
  const int slots = (a.frames + kStateStride - 1) / kStateStride;
  const int mine = w * kStateStride + tl * S;  // this thread's first frame of step 0
  const T *x = a.x.p + n * a.x.sn + c, *gate = a.gate.p + n * a.gate.sn + c;
  T *y = a.y.p + n * a.y.sn + c;

  if (w == 0 && tl == 0) {
    A h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = a.initial != nullptr && on ? a.initial[n * a.channels + c + v] : A(0);
    store_acc<V>(&sh.carry[0][at], h);
  }
  Raw<T, V> xr[S], gr[S];
  // strides between frames are below 2^31 elements here: one widening multiply-add makes a frame's address
  const int way = a.reverse ? -1 : 1, xs = way * (int)a.x.st, gs = way * (int)a.gate.st, ys = way * (int)a.y.st;
  const int ahead = kStateStride - tl * S;  // the warp's frames from this thread's first one on
  auto fetch = [&](int k) {
    const int s0 = k * SPAN + mine, t0 = a.reverse ? len - 1 - s0 : s0;
    const T *px = x + t0 * a.x.st, *pg = gate + t0 * a.gate.st;
    if (on && s0 + ahead <= len) {
#pragma unroll
      for (int j = 0; j < S; ++j) xr[j] = load_raw<T, V>(px + (long long)xs * j), gr[j] = load_raw<T, V>(pg + (long long)gs * j);
    } else {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        xr[j] = zeros<T, V>(), gr[j] = infinities<T, V>();
        if (on && s0 + j < len) xr[j] = load_raw<T, V>(px + (long long)xs * j), gr[j] = load_raw<T, V>(pg + (long long)gs * j);
      }
    }
  };
  if (steps > 0) fetch(0);
  for (int k = 0; k < steps; ++k) {
    const int buffer = k & 1, s0 = k * SPAN + mine;
    A f[S][V], u[S][V], pa[V], pb[V];
#pragma unroll
    for (int j = 0; j < S; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        A keep;
        sigmoid_pair<true>(element(gr[j], v), f[j][v], keep);
        u[j][v] = keep * element(xr[j], v);
      }
    if (k + 1 < steps) fetch(k + 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      pa[v] = f[0][v], pb[v] = u[0][v];
#pragma unroll
      for (int j = 1; j < S; ++j) pb[v] = f[j][v] * pb[v] + u[j][v], pa[v] *= f[j][v];
    }
#pragma unroll
    for (int o = CL; o < 32; o *= 2)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A qa = __shfl_up_sync(0xffffffffu, pa[v], o), qb = __shfl_up_sync(0xffffffffu, pb[v], o);
        if (lane >= o) pb[v] = pa[v] * qb + pb[v], pa[v] *= qa;
      }
    if (tl == TL - 1) store_acc<V>(&sh.a[buffer][w][at], pa), store_acc<V>(&sh.b[buffer][w][at], pb);
    __syncthreads();
    A h[V], next[V];
    load_acc<V>(h, &sh.carry[buffer][at]);
    for (int i = 0; i < w; ++i) {
      A qa[V], qb[V];
      load_acc<V>(qa, &sh.a[buffer][i][at]), load_acc<V>(qb, &sh.b[buffer][i][at]);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = qa[v] * h[v] + qb[v];
    }
    if (w == W - 1 && tl == TL - 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) next[v] = pa[v] * h[v] + pb[v];
      store_acc<V>(&sh.carry[buffer ^ 1][at], next);
    }
    // before the warp's frames: h; before this thread's: what the threads with the warp's earlier frames make of it
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const A qa = __shfl_up_sync(0xffffffffu, pa[v], TL > 1 ? CL : 0), qb = __shfl_up_sync(0xffffffffu, pb[v], TL > 1 ? CL : 0);
      if (tl > 0) h[v] = qa * h[v] + qb;
    }
    if (on) {
      if (a.states != nullptr && tl == 0 && s0 < len)
        store_acc<V>(a.states + (n * slots + s0 / kStateStride) * (long long)a.channels + c, h);
      T *py = y + (a.reverse ? len - 1 - s0 : s0) * a.y.st;
      if (s0 + ahead <= len) {
#pragma unroll
        for (int j = 0; j < S; ++j) {
#pragma unroll
          for (int v = 0; v < V; ++v) h[v] = f[j][v] * h[v] + u[j][v];
          store_raw<T, V>(py + (long long)ys * j, rounded<T, V>(h));
        }
      } else {
#pragma unroll
        for (int j = 0; j < S; ++j) {
          const int s = s0 + j;
#pragma unroll
          for (int v = 0; v < V; ++v) h[v] = f[j][v] * h[v] + u[j][v];
          if (s < len) store_raw<T, V>(py + (long long)ys * j, rounded<T, V>(h));
          else if (s < a.frames) store_raw<T, V>(y + s * a.y.st, zeros<T, V>());
        }
      }
    }
  }
  if (on)
    for (int k = steps; k * SPAN < a.frames; ++k) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const int t = k * SPAN + mine + j;
        if (t < a.frames) store_raw<T, V>(y + t * a.y.st, zeros<T, V>());
      }
    }
  __syncthreads();
  if (a.final != nullptr && on && w == 0 && tl == 0) {
    A h[V];
    load_acc<V>(h, &sh.carry[steps & 1][at]);
#pragma unroll
    for (int v = 0; v < V; ++v) a.final[n * a.channels + c + v] = h[v];
  }
}

// Backward: the same walk from the last frames to the first, joining the runs' maps of m (what later frames pass back)
// from the end: m -> A m + B.  The states before a warp's frames are the kept ones; those inside it are joined forward
// by shuffles.
template <typename T, int V, int CL, int W, int MB>
__global__ void __launch_bounds__(32 * W, MB) recurrence_scan_backward_kernel(const RecurrenceArgs<T> a) {
  begin<false>();
  using A = Acc<T>;
  constexpr int TL = 32 / CL, S = kStateStride / TL, CT = CL * V, SPAN = W * kStateStride;
  __shared__ ScanShared<A, CT, W> sh;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, cl = lane % CL, tl = lane / CL, at = cl * V;
  const int unit = (int)blockIdx.x;
  const Utterance whose = utterance_of(a.lens, a.batch, a.frames, unit / a.tiles);
  const long long n = whose.n;
  const int c = unit % a.tiles * CT + at;
  const bool on = c < a.channels;
  const int len = whose.len, steps = (len + SPAN - 1) / SPAN;
  const int slots = (a.frames + kStateStride - 1) / kStateStride;
  const int mine = w * kStateStride + tl * S;
  const T *x = a.x.p + n * a.x.sn + c, *gate = a.gate.p + n * a.gate.sn + c;
  const T *gy = a.grad_y.p + n * a.grad_y.sn + c;
  T *gx = a.grad_x.p + n * a.grad_x.sn + c, *gg = a.grad_gate.p + n * a.grad_gate.sn + c;

  if (w == 0 && tl == 0) {
    A m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) m[v] = a.grad_final != nullptr && on ? a.grad_final[n * a.channels + c + v] : A(0);
    store_acc<V>(&sh.carry[0][at], m);
  }
  Raw<T, V> xr[S], gr[S], yr[S];
  A before[V];  // the state before the warp's frames, in the threads that have the first of them
  const int way = a.reverse ? -1 : 1, xs = way * (int)a.x.st, gs = way * (int)a.gate.st, ys = way * (int)a.grad_y.st;
  const int gxs = way * (int)a.grad_x.st, ggs = way * (int)a.grad_gate.st;
  const int ahead = kStateStride - tl * S;
  auto fetch = [&](int k) {
    const int s0 = k * SPAN + mine, t0 = a.reverse ? len - 1 - s0 : s0;
    const T *px = x + t0 * a.x.st, *pg = gate + t0 * a.gate.st, *py = gy + t0 * a.grad_y.st;
    if (on && s0 + ahead <= len && a.grad_y.p != nullptr) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        xr[j] = load_raw<T, V>(px + (long long)xs * j), gr[j] = load_raw<T, V>(pg + (long long)gs * j);
        yr[j] = load_raw<T, V>(py + (long long)ys * j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        xr[j] = yr[j] = zeros<T, V>(), gr[j] = infinities<T, V>();
        if (on && s0 + j < len) {
          xr[j] = load_raw<T, V>(px + (long long)xs * j), gr[j] = load_raw<T, V>(pg + (long long)gs * j);
          if (a.grad_y.p != nullptr) yr[j] = load_raw<T, V>(py + (long long)ys * j);
        }
      }
    }
    if (on && tl == 0 && s0 < len) {
      load_acc<V>(before, a.states + (n * slots + s0 / kStateStride) * (long long)a.channels + c);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) before[v] = 0;
    }
  };
  if (steps > 0) fetch(steps - 1);
  for (int k = steps - 1, turn = 0; k >= 0; --k, ++turn) {
    const int buffer = turn & 1, s0 = k * SPAN + mine;
    A f[S][V], keep[S][V], d[S][V], pa[V], pb[V], h[V];
    Raw<T, V> yc[S];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      pa[v] = A(1), pb[v] = A(0);
#pragma unroll
      for (int j = 0; j < S; ++j) {
        sigmoid_pair<true>(element(gr[j], v), f[j][v], keep[j][v]);
        d[j][v] = element(xr[j], v);
        pb[v] = f[j][v] * pb[v] + keep[j][v] * d[j][v], pa[v] *= f[j][v];
      }
    }
    // the state before this thread's frames
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A ia = pa[v], ib = pb[v];
#pragma unroll
      for (int o = CL; o < 32; o *= 2) {
        const A qa = __shfl_up_sync(0xffffffffu, ia, o), qb = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) ib = ia * qb + ib, ia *= qa;
      }
      h[v] = __shfl_sync(0xffffffffu, before[v], cl);
      const A qa = __shfl_up_sync(0xffffffffu, ia, TL > 1 ? CL : 0), qb = __shfl_up_sync(0xffffffffu, ib, TL > 1 ? CL : 0);
      if (tl > 0) h[v] = qa * h[v] + qb;
    }
#pragma unroll
    for (int j = 0; j < S; ++j) {
      yc[j] = yr[j];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A xv = d[j][v];
        d[j][v] = h[v] - xv;
        h[v] = f[j][v] * h[v] + keep[j][v] * xv;
      }
    }
    if (k > 0) fetch(k - 1);
    // this thread's map of m
#pragma unroll
    for (int v = 0; v < V; ++v) {
      pb[v] = A(0);
#pragma unroll
      for (int j = S - 1; j >= 0; --j) pb[v] = f[j][v] * (pb[v] + element(yc[j], v));
    }
#pragma unroll
    for (int o = CL; o < 32; o *= 2)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A qa = __shfl_down_sync(0xffffffffu, pa[v], o), qb = __shfl_down_sync(0xffffffffu, pb[v], o);
        if (lane + o < 32) pb[v] = pa[v] * qb + pb[v], pa[v] *= qa;
      }
    if (tl == 0) store_acc<V>(&sh.a[buffer][w][at], pa), store_acc<V>(&sh.b[buffer][w][at], pb);
    __syncthreads();
    A m[V], next[V];
    load_acc<V>(m, &sh.carry[buffer][at]);
    for (int i = W - 1; i > w; --i) {
      A qa[V], qb[V];
      load_acc<V>(qa, &sh.a[buffer][i][at]), load_acc<V>(qb, &sh.b[buffer][i][at]);
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = qa[v] * m[v] + qb[v];
    }
    if (w == 0 && tl == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) next[v] = pa[v] * m[v] + pb[v];
      store_acc<V>(&sh.carry[buffer ^ 1][at], next);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const A qa = __shfl_down_sync(0xffffffffu, pa[v], TL > 1 ? CL : 0), qb = __shfl_down_sync(0xffffffffu, pb[v], TL > 1 ? CL : 0);
      if (tl < TL - 1) m[v] = qa * m[v] + qb;
    }
    if (on) {
      const int t0 = a.reverse ? len - 1 - s0 : s0;
      T *px = gx + t0 * a.grad_x.st, *pg = gg + t0 * a.grad_gate.st;
      const bool whole = s0 + ahead <= len;
#pragma unroll
      for (int j = S - 1; j >= 0; --j) {
        const int s = s0 + j;
        A ox[V], og[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const A gh = m[v] + element(yc[j], v);
          m[v] = f[j][v] * gh;
          ox[v] = keep[j][v] * gh;
          og[v] = keep[j][v] * m[v] * d[j][v];
        }
        if (whole || s < len) {
          store_raw<T, V>(px + (long long)gxs * j, rounded<T, V>(ox));
          store_raw<T, V>(pg + (long long)ggs * j, rounded<T, V>(og));
        } else if (s < a.frames) {
          store_raw<T, V>(gx + s * a.grad_x.st, zeros<T, V>());
          store_raw<T, V>(gg + s * a.grad_gate.st, zeros<T, V>());
        }
      }
    }
  }
  if (on)
    for (int k = steps; k * SPAN < a.frames; ++k) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const int t = k * SPAN + mine + j;
        if (t < a.frames) {
          store_raw<T, V>(gx + t * a.grad_x.st, zeros<T, V>());
          store_raw<T, V>(gg + t * a.grad_gate.st, zeros<T, V>());
        }
      }
    }
  __syncthreads();
  if (a.grad_initial != nullptr && on && w == 0 && tl == 0) {
    A m[V];
    load_acc<V>(m, &sh.carry[steps & 1][at]);
#pragma unroll
    for (int v = 0; v < V; ++v) a.grad_initial[n * a.channels + c + v] = m[v];
  }
}

// ---- long utterances, few of them --------------------------------------------------------------------------------------
//
// Where utterances and channels alone do not fill the device, a cluster of blocks shares CL * V = 16 channels of one
// utterance: every CL lanes have one run of adjacent frames, kLongWarps * 32 / CL runs a block.  First each run's (A, B)
// is formed by walking it once; these are joined in the warp, the block and the cluster, one exchange in all; then the
// run is walked again from the state that is now known.  The second walk finds its inputs in L2 (so few utterances and
// channels are small), and no step waits for another block, as the single walk above would have to every SPAN frames.
// 16384 frames of 2 x 256 channels in bfloat16: 26 us forward, 31 us backward (bytes alone: 8 and 13); 31 and 41 with
// the single walk and an exchange in the cluster every 1024 frames; 37 and 47 with 32 channels a cluster, which leaves
// half the multiprocessors without one.

constexpr int kMaxCluster = 8;  // the portable limit
constexpr int kLongWarps = 8;   // two blocks fit a multiprocessor, so that every cluster of eight finds its place at once
constexpr int kRows = 8;        // frames fetched together, and between two kept states

template <typename A, int CT>
struct alignas(16) LongShared {
  A a[kLongWarps][CT], b[kLongWarps][CT];      // of the block's warps
  A ca[kMaxCluster][CT], cb[kMaxCluster][CT];  // of the cluster's blocks
};

// The frames of one run and the join of all runs.  FORWARD: runs before this one; else those after it.
template <typename A, int V, int CL, bool FORWARD>
__device__ __forceinline__ void join_runs(LongShared<A, V * CL> &sh, int size, int rank, A (&pa)[V], A (&pb)[V], A (&state)[V],
                                          A (&last)[V]) {
  constexpr int TL = 32 / CL;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, tl = lane / CL, at = lane % CL * V;
  auto shift = [&](A value, int by) {
    return FORWARD ? __shfl_up_sync(0xffffffffu, value, by) : __shfl_down_sync(0xffffffffu, value, by);
  };
  const int order = FORWARD ? tl : TL - 1 - tl;  // runs of the warp that go before this one
#pragma unroll
  for (int o = 1; o < TL; o *= 2)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const A qa = shift(pa[v], o * CL), qb = shift(pb[v], o * CL);
      if (order >= o) pb[v] = pa[v] * qb + pb[v], pa[v] *= qa;
    }
  if (order == TL - 1) store_acc<V>(&sh.a[w][at], pa), store_acc<V>(&sh.b[w][at], pb);
  __syncthreads();
  auto cluster = cooperative_groups::this_cluster();
  if (w == 0) {
    A ta[V], tb[V], qa[V], qb[V];
#pragma unroll
    for (int v = 0; v < V; ++v) ta[v] = A(1), tb[v] = A(0);
#pragma unroll 4
    for (int i = 0; i < kLongWarps; ++i) {
      const int from = FORWARD ? i : kLongWarps - 1 - i;
      load_acc<V>(qa, &sh.a[from][at]), load_acc<V>(qb, &sh.b[from][at]);
#pragma unroll
      for (int v = 0; v < V; ++v) tb[v] = qa[v] * tb[v] + qb[v], ta[v] *= qa[v];
    }
    for (int r = tl; r < size; r += TL) {
      store_acc<V>(size > 1 ? cluster.map_shared_rank(&sh.ca[rank][at], r) : &sh.ca[rank][at], ta);
      store_acc<V>(size > 1 ? cluster.map_shared_rank(&sh.cb[rank][at], r) : &sh.cb[rank][at], tb);
    }
  }
  if (size > 1) cluster.sync();
  else __syncthreads();
  // `state`: from what is given outside to what this run meets; `last`: to what is after all runs
  A qa[V], qb[V];
  for (int i = 0; i < size; ++i) {
    const int from = FORWARD ? i : size - 1 - i;
    load_acc<V>(qa, &sh.ca[from][at]), load_acc<V>(qb, &sh.cb[from][at]);
    const bool before = FORWARD ? from < rank : from > rank;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      last[v] = qa[v] * last[v] + qb[v];
      if (before) state[v] = last[v];
    }
  }
#pragma unroll 4
  for (int i = 0; i < (FORWARD ? w : kLongWarps - 1 - w); ++i) {
    const int from = FORWARD ? i : kLongWarps - 1 - i;
    load_acc<V>(qa, &sh.a[from][at]), load_acc<V>(qb, &sh.b[from][at]);
#pragma unroll
    for (int v = 0; v < V; ++v) state[v] = qa[v] * state[v] + qb[v];
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const A ea = shift(pa[v], TL > 1 ? CL : 0), eb = shift(pb[v], TL > 1 ? CL : 0);
    if (order > 0) state[v] = ea * state[v] + eb;
  }
}

// kRows frames from logical frame `first` on, those from `end` on filled
template <typename T, int V>
__device__ __forceinline__ void fetch_rows(Raw<T, V> (&to)[kRows], const T *base, long long st, int first, int end, int len,
                                           bool reverse, const Raw<T, V> &fill) {
  const T *p = base + (reverse ? len - 1 - first : first) * st;
  const int step = (reverse ? -1 : 1) * (int)st;
  if (first + kRows <= end) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) to[j] = load_raw<T, V>(p + (long long)step * j);
  } else {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      to[j] = fill;
      if (first + j < end) to[j] = load_raw<T, V>(p + (long long)step * j);
    }
  }
}

struct Run {
  int unit, n, c, rank, size, begin, end, len, index, count;
  bool on;
};
template <typename T, int V, int CL>
__device__ __forceinline__ Run run_of(const RecurrenceArgs<T> &a) {
  constexpr int TL = 32 / CL;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  Run r;
  r.size = a.cluster, r.rank = (int)(blockIdx.x % a.cluster), r.unit = (int)(blockIdx.x / a.cluster);
  r.n = r.unit / a.tiles, r.c = r.unit % a.tiles * (V * CL) + lane % CL * V;
  r.on = r.c < a.channels;
  r.len = live_frames(a.lens, r.n, a.frames);
  r.count = r.size * kLongWarps * TL, r.index = (r.rank * kLongWarps + w) * TL + lane / CL;
  const int frames = ((r.len + r.count - 1) / r.count + kRows - 1) / kRows * kRows;  // of a run
  const long long begin = (long long)r.index * frames;
  r.begin = begin < r.len ? (int)begin : r.len;
  r.end = r.on ? (r.len - r.begin < frames ? r.len : r.begin + frames) : r.begin;
  return r;
}

template <typename T, int V, int CL>
__global__ void __launch_bounds__(32 * kLongWarps, 16 / kLongWarps) recurrence_long_kernel(const RecurrenceArgs<T> a) {
  begin<false>();
  using A = Acc<T>;
  __shared__ LongShared<A, V * CL> sh;
  const Run r = run_of<T, V, CL>(a);
  if (r.size > 1) cooperative_groups::this_cluster().sync();  // no block writes to one that has not started
  const T *x = a.x.p + r.n * a.x.sn + r.c, *gate = a.gate.p + r.n * a.gate.sn + r.c;
  T *y = a.y.p + r.n * a.y.sn + r.c;
  const long long row = (long long)r.n * a.channels + r.c;

  Raw<T, V> xr[kRows], gr[kRows];
  A pa[V], pb[V], h[V], last[V];
#pragma unroll
  for (int v = 0; v < V; ++v) pa[v] = A(1), pb[v] = A(0);
  for (int s = r.begin; s < r.end; s += kRows) {
    fetch_rows(xr, x, a.x.st, s, r.end, r.len, a.reverse, zeros<T, V>());
    fetch_rows(gr, gate, a.gate.st, s, r.end, r.len, a.reverse, infinities<T, V>());
#pragma unroll
    for (int j = 0; j < kRows; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        A f, keep;
        sigmoid_pair<true>(element(gr[j], v), f, keep);
        pb[v] = f * pb[v] + keep * element(xr[j], v), pa[v] *= f;
      }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = last[v] = a.initial != nullptr && r.on ? a.initial[row + v] : A(0);
  join_runs<A, V, CL, true>(sh, r.size, r.rank, pa, pb, h, last);

  const int slots = (a.frames + kRows - 1) / kRows, step = (a.reverse ? -1 : 1) * (int)a.y.st;
  for (int s = r.begin; s < r.end; s += kRows) {
    fetch_rows(xr, x, a.x.st, s, r.end, r.len, a.reverse, zeros<T, V>());
    fetch_rows(gr, gate, a.gate.st, s, r.end, r.len, a.reverse, infinities<T, V>());
    if (a.states != nullptr) store_acc<V>(a.states + ((long long)r.n * slots + s / kRows) * a.channels + r.c, h);
    T *py = y + (a.reverse ? r.len - 1 - s : s) * a.y.st;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        A f, keep;
        sigmoid_pair<true>(element(gr[j], v), f, keep);
        h[v] = f * h[v] + keep * element(xr[j], v);
      }
      if (s + j < r.end) store_raw<T, V>(py + (long long)step * j, rounded<T, V>(h));
    }
  }
  if (r.on) {
    for (long long t = (long long)r.len + r.index; t < a.frames; t += r.count) store_raw<T, V>(y + t * a.y.st, zeros<T, V>());
    if (a.final != nullptr && r.index == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) a.final[row + v] = last[v];
    }
  }
}

template <typename T, int V, int CL>
__global__ void __launch_bounds__(32 * kLongWarps, 16 / kLongWarps) recurrence_long_backward_kernel(const RecurrenceArgs<T> a) {
  begin<false>();
  using A = Acc<T>;
  __shared__ LongShared<A, V * CL> sh;
  const Run r = run_of<T, V, CL>(a);
  if (r.size > 1) cooperative_groups::this_cluster().sync();
  const T *x = a.x.p + r.n * a.x.sn + r.c, *gate = a.gate.p + r.n * a.gate.sn + r.c;
  const T *gy = a.grad_y.p + r.n * a.grad_y.sn + r.c;
  T *gx = a.grad_x.p + r.n * a.grad_x.sn + r.c, *gg = a.grad_gate.p + r.n * a.grad_gate.sn + r.c;
  const long long row = (long long)r.n * a.channels + r.c;
  const int blocks = (r.end - r.begin + kRows - 1) / kRows;  // of kRows frames in this run
  const bool has_gy = a.grad_y.p != nullptr;

  Raw<T, V> xr[kRows], gr[kRows], yr[kRows];
  A pa[V], pb[V], m[V], last[V];
#pragma unroll
  for (int v = 0; v < V; ++v) pa[v] = A(1), pb[v] = A(0);
  for (int i = blocks - 1; i >= 0; --i) {
    const int s = r.begin + i * kRows;
    fetch_rows(gr, gate, a.gate.st, s, r.end, r.len, a.reverse, infinities<T, V>());
    fetch_rows(yr, gy, a.grad_y.st, s, has_gy ? r.end : s, r.len, a.reverse, zeros<T, V>());
#pragma unroll
    for (int j = kRows - 1; j >= 0; --j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        A f, keep;
        sigmoid_pair<true>(element(gr[j], v), f, keep);
        pb[v] = f * (pb[v] + element(yr[j], v)), pa[v] *= f;
      }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = last[v] = a.grad_final != nullptr && r.on ? a.grad_final[row + v] : A(0);
  join_runs<A, V, CL, false>(sh, r.size, r.rank, pa, pb, m, last);

  const int slots = (a.frames + kRows - 1) / kRows, way = a.reverse ? -1 : 1;
  for (int i = blocks - 1; i >= 0; --i) {
    const int s = r.begin + i * kRows, t0 = a.reverse ? r.len - 1 - s : s;
    A h[V], f[kRows][V], keep[kRows][V], d[kRows][V];
    load_acc<V>(h, a.states + ((long long)r.n * slots + s / kRows) * a.channels + r.c);
    fetch_rows(xr, x, a.x.st, s, r.end, r.len, a.reverse, zeros<T, V>());
    fetch_rows(gr, gate, a.gate.st, s, r.end, r.len, a.reverse, infinities<T, V>());
    fetch_rows(yr, gy, a.grad_y.st, s, has_gy ? r.end : s, r.len, a.reverse, zeros<T, V>());
#pragma unroll
    for (int j = 0; j < kRows; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A xv = element(xr[j], v);
        sigmoid_pair<true>(element(gr[j], v), f[j][v], keep[j][v]);
        d[j][v] = h[v] - xv;
        h[v] = f[j][v] * h[v] + keep[j][v] * xv;
      }
    T *px = gx + t0 * a.grad_x.st, *pg = gg + t0 * a.grad_gate.st;
#pragma unroll
    for (int j = kRows - 1; j >= 0; --j) {
      A ox[V], og[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A gh = m[v] + element(yr[j], v);
        m[v] = f[j][v] * gh;
        ox[v] = keep[j][v] * gh;
        og[v] = keep[j][v] * m[v] * d[j][v];
      }
      if (s + j < r.end) {
        store_raw<T, V>(px + (long long)(way * (int)a.grad_x.st) * j, rounded<T, V>(ox));
        store_raw<T, V>(pg + (long long)(way * (int)a.grad_gate.st) * j, rounded<T, V>(og));
      }
    }
  }
  if (r.on) {
    for (long long t = (long long)r.len + r.index; t < a.frames; t += r.count) {
      store_raw<T, V>(gx + t * a.grad_x.st, zeros<T, V>());
      store_raw<T, V>(gg + t * a.grad_gate.st, zeros<T, V>());
    }
    if (a.grad_initial != nullptr && r.index == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) a.grad_initial[row + v] = last[v];
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------

template <typename T>
int check(const char *who, const RecurrenceArgs<T> &a, int64_t batch, int64_t frames, int64_t channels, bool backward) {
  const int rc = check_extents(who, batch, frames, channels);
  if (rc != MELLIN_OK) return rc;
  if (batch == 0 || channels == 0) return MELLIN_OK;
  if (frames > 0) {
    if (a.x.p == nullptr || a.gate.p == nullptr || (!backward && a.y.p == nullptr) ||
        (backward && (a.grad_x.p == nullptr || a.grad_gate.p == nullptr)))
      return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": null pointer");
    if (backward && a.states == nullptr)
      return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": the states that the forward call keeps are needed");
  }
  return MELLIN_OK;
}

// Every tensor can be moved V elements at a time.
template <typename T>
bool packed(const RecurrenceArgs<T> &a, int64_t channels, int V) {
  auto ok = [V](const auto &f) {
    return f.p == nullptr || (aligned_to(f.p, V * sizeof(T)) && f.sn % V == 0 && f.st % V == 0);
  };
  return channels % V == 0 && ok(a.x) && ok(a.gate) && ok(a.grad_y) && ok(a.y) && ok(a.grad_x) && ok(a.grad_gate) &&
         aligned_to(a.states, 16);
}

// Few tiles of 32 channels and many frames: the time axis has to be shared by a cluster.  By shape alone, so that a
// forward call and its backward agree on the kept states.  Below 148 tiles (one block a multiprocessor) the long form
// wins from about 256 frames on: 8 x 800 x 512 channels 12 / 15 us against 12 / 19, 1 x 2000 x 128 6 / 7 against 25 / 37,
// 1 x 300 x 512 6 / 7 against 7 / 8; at 256 tiles (8 x 800 x 1024) it loses, 23 / 27 against 17 / 23.
bool is_long(int64_t batch, int64_t frames, int64_t channels) {
  return frames >= 256 && batch * ((channels + 31) / 32) < 148;
}

template <typename K, typename T>
int launch(const char *who, K kernel, const RecurrenceArgs<T> &a, long long blocks, int threads, void *stream) {
  if (blocks > 0x7fffffffLL) return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many utterances times channels");
  const cudaError_t err = launch_kernel(kernel, dim3((unsigned)blocks), threads, 0, a.cluster, stream, a);
  if (err != cudaSuccess) return fail(MELLIN_ERR_LAUNCH, std::string(who) + ": " + cudaGetErrorString(err));
  return launched(who);
}

template <typename T, int V, int CL, int W, int MB, bool BACKWARD>
int launch_scan(const char *who, RecurrenceArgs<T> a, void *stream) {
  a.tiles = (a.channels + CL * V - 1) / (CL * V);
  if constexpr (BACKWARD)
    return launch(who, recurrence_scan_backward_kernel<T, V, CL, W, MB>, a, (long long)a.batch * a.tiles, 32 * W, stream);
  else return launch(who, recurrence_scan_kernel<T, V, CL, W, MB>, a, (long long)a.batch * a.tiles, 32 * W, stream);
}

template <typename T, int V, int CL, bool BACKWARD>
int launch_long(const char *who, RecurrenceArgs<T> a, void *stream) {
  a.tiles = (a.channels + V * CL - 1) / (V * CL);
  // blocks for every multiprocessor, as long as each run has its kRows frames
  const long long units = (long long)a.batch * a.tiles;
  while (a.cluster < kMaxCluster && units * a.cluster < 148 && a.cluster * kLongWarps * (32 / CL) * kRows < a.frames)
    a.cluster *= 2;
  if constexpr (BACKWARD)
    return launch(who, recurrence_long_backward_kernel<T, V, CL>, a, units * a.cluster, 32 * kLongWarps, stream);
  else return launch(who, recurrence_long_kernel<T, V, CL>, a, units * a.cluster, 32 * kLongWarps, stream);
}

template <typename T, bool BACKWARD>
int run(const char *who, RecurrenceArgs<T> a, int64_t batch, int64_t frames, int64_t channels, void *stream) {
  return guarded(who, [&]() -> int {
    const int rc = check(who, a, batch, frames, channels, BACKWARD);
    if (rc != MELLIN_OK || batch == 0 || channels == 0) return rc;
    a.batch = (int)batch, a.frames = (int)frames, a.channels = (int)channels;
    const bool lengthy = is_long(batch, frames, channels);
    auto near = [](const auto &f) { return f.st < 0x7fffffffLL && f.st > -0x7fffffffLL; };
    if (frames <= kWalkFrames || !(near(a.x) && near(a.gate) && near(a.grad_y) && near(a.y) && near(a.grad_x) && near(a.grad_gate))) {
      if (lengthy)  // 1 TB in 16 bits: no device has them
        return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": 256 frames or more with 2^31 elements between them");
      const long long blocks = (batch * channels + kWalkThreads - 1) / kWalkThreads;
      if constexpr (BACKWARD) return launch(who, recurrence_walk_backward_kernel<T>, a, blocks, kWalkThreads, stream);
      else return launch(who, recurrence_walk_kernel<T>, a, blocks, kWalkThreads, stream);
    }
    if (lengthy) {
      if (packed(a, channels, 2)) return launch_long<T, 2, 8, BACKWARD>(who, a, stream);
      return launch_long<T, 1, 16, BACKWARD>(who, a, stream);
    }
    // V, CL, W and blocks a multiprocessor, measured at 32 utterances of 200 to 800 frames and 1024 channels (us, forward
    // / backward): 16 bits <4, 16, 4, 4> 30 / 73, <4, 16, 4, 2> 35 / 47, <4, 8, 4, 4> 31 / 45, <4, 16, 8, 2> 29 / 66 (39
    // against 35 forward where all have 800 frames); float <4, 8, 4, 4> 44 / 78, <4, 8, 4, 3> 50 / 77, <4, 16, 4, 2>
    // 45 / 68.  Bytes alone: 18 / 31 and 36 / 62.  What is left goes to the joins (a barrier every step), to 26
    // instructions an element, and to 3.5 blocks a multiprocessor; packed multiply-adds changed nothing.
    constexpr int V = sizeof(T) == 8 ? 2 : 4;
    if (!packed(a, channels, V)) {
      // an even number of channels: pairs, 16 bits 35 / 53; else one by one, 44 / 86
      if (V > 2 && packed(a, channels, 2)) return launch_scan<T, 2, 16, 4, 4, BACKWARD>(who, a, stream);
      return launch_scan<T, 1, 32, 4, BACKWARD ? 3 : 4, BACKWARD>(who, a, stream);
    }
    if constexpr (sizeof(T) == 2 && !BACKWARD) return launch_scan<T, V, 16, 4, 4, BACKWARD>(who, a, stream);
    else if constexpr (sizeof(T) == 4 && BACKWARD) return launch_scan<T, V, 16, 4, 2, BACKWARD>(who, a, stream);
    else return launch_scan<T, V, 8, 4, 4, BACKWARD>(who, a, stream);
  });
}

template <typename T, typename P, typename S>
int forward_entry(const P *x, int64_t x_sn, int64_t x_st, const P *gate, int64_t gate_sn, int64_t gate_st,
                  const S *initial, const int *lens, int reverse, int64_t batch, int64_t frames, int64_t channels, P *y,
                  int64_t y_sn, int64_t y_st, S *final, S *states, void *stream) {
  RecurrenceArgs<T> a;
  a.x = {static_cast<const T *>(x), x_sn, x_st}, a.gate = {static_cast<const T *>(gate), gate_sn, gate_st};
  a.y = {static_cast<T *>(y), y_sn, y_st};
  a.initial = initial, a.final = final, a.states = states, a.lens = lens, a.reverse = reverse;
  return run<T, false>("gated_recurrence", a, batch, frames, channels, stream);
}

template <typename T, typename P, typename S>
int backward_entry(const P *x, int64_t x_sn, int64_t x_st, const P *gate, int64_t gate_sn, int64_t gate_st,
                   const S *states, const int *lens, int reverse, int64_t batch, int64_t frames, int64_t channels,
                   const P *grad_y, int64_t grad_y_sn, int64_t grad_y_st, const S *grad_final, P *grad_x,
                   int64_t grad_x_sn, int64_t grad_x_st, P *grad_gate, int64_t grad_gate_sn, int64_t grad_gate_st,
                   S *grad_initial, void *stream) {
  RecurrenceArgs<T> a;
  a.x = {static_cast<const T *>(x), x_sn, x_st}, a.gate = {static_cast<const T *>(gate), gate_sn, gate_st};
  a.grad_y = {static_cast<const T *>(grad_y), grad_y_sn, grad_y_st};
  a.grad_x = {static_cast<T *>(grad_x), grad_x_sn, grad_x_st};
  a.grad_gate = {static_cast<T *>(grad_gate), grad_gate_sn, grad_gate_st};
  a.states = const_cast<S *>(states), a.grad_final = grad_final, a.grad_initial = grad_initial;
  a.lens = lens, a.reverse = reverse;
  return run<T, true>("backward of gated_recurrence", a, batch, frames, channels, stream);
}

}  // namespace

}  // namespace mellin

using namespace mellin;

#define RECURRENCE_ENTRIES(SUFFIX, T, P, S)                                                                           \
  int mellin_gated_recurrence_##SUFFIX(const P *x, int64_t x_sn, int64_t x_st, const P *gate, int64_t gate_sn,        \
                                       int64_t gate_st, const S *initial, const int *lens, int reverse,              \
                                       int64_t batch, int64_t frames, int64_t channels, P *y, int64_t y_sn,          \
                                       int64_t y_st, S *final, S *states, void *stream) {                            \
    return forward_entry<T, P, S>(x, x_sn, x_st, gate, gate_sn, gate_st, initial, lens, reverse, batch, frames,      \
                                  channels, y, y_sn, y_st, final, states, stream);                                   \
  }                                                                                                                  \
  int mellin_gated_recurrence_backward_##SUFFIX(                                                                     \
      const P *x, int64_t x_sn, int64_t x_st, const P *gate, int64_t gate_sn, int64_t gate_st, const S *states,      \
      const int *lens, int reverse, int64_t batch, int64_t frames, int64_t channels, const P *grad_y,                \
      int64_t grad_y_sn, int64_t grad_y_st, const S *grad_final, P *grad_x, int64_t grad_x_sn, int64_t grad_x_st,    \
      P *grad_gate, int64_t grad_gate_sn, int64_t grad_gate_st, S *grad_initial, void *stream) {                     \
    return backward_entry<T, P, S>(x, x_sn, x_st, gate, gate_sn, gate_st, states, lens, reverse, batch, frames,      \
                                   channels, grad_y, grad_y_sn, grad_y_st, grad_final, grad_x, grad_x_sn, grad_x_st, \
                                   grad_gate, grad_gate_sn, grad_gate_st, grad_initial, stream);                     \
  }

extern "C" {

int64_t mellin_gated_recurrence_state_count(int64_t batch, int64_t frames, int64_t channels) {
  if (batch < 0 || frames < 0 || channels < 0) return 0;
  const int64_t every = is_long(batch, frames, channels) ? kRows : kStateStride;
  return batch * ((frames + every - 1) / every) * channels;
}

RECURRENCE_ENTRIES(f32, float, float, float)
RECURRENCE_ENTRIES(f64, double, double, double)
RECURRENCE_ENTRIES(f16, __half, void, float)
RECURRENCE_ENTRIES(bf16, __nv_bfloat16, void, float)

}  // extern "C"
