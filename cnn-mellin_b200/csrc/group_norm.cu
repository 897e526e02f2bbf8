// Group norm over the frames of ragged utterances followed by an activation, channels last:
//
//   xhat = (x - mean) * rstd,   y = act(xhat * weight[c] + bias[c])
//
// mean and the (biased) variance are taken over an utterance's own frames and the channels / groups adjacent channels of
// a group; rstd = 1 / sqrt(var + eps).  Frames behind the end are never read, their outputs are zero.
//
// Backward, with gz = gy * act'(z) and M = frames * channels of a group:
//   P1[n, c] = sum_t gz,  P2[n, c] = sum_t gz * xhat;   gbias = sum_n P1,  gweight = sum_n P2
//   gx = rstd * (weight gz - (sum_c weight P1 + xhat * sum_c weight P2) / M)
//
// All sums in a fixed order: two runs give the same bits.
//
// ReLU's slope is 1 where z as computed is positive.  z next to zero is the difference of terms as large as the bias, so in
// float which side it falls on is certain to about 2e-8: of 16.4 million elements (32 utterances of 200 to 800 frames, 1024
// channels) one was on the other side than in 64 bits in 11 of 120 draws, never at |z| above 2.2e-8; the same formula written
// out in elementary operations, 15 of 120.  Statistics rounded to float alone would leave 7.
#include <cooperative_groups.h>

#include <algorithm>

#include "sequence_common.cuh"

namespace mellin {
namespace {

using namespace seq;

constexpr int kThreads = 256;
constexpr int kMaxRanks = 8;    // blocks of a cluster: the portable limit

enum Activation { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

__device__ __forceinline__ float exp_of(float v) { return __expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float erf_of(float v) { return erff(v); }
__device__ __forceinline__ double erf_of(double v) { return erf(v); }

template <int ACT>
using ActTag = std::integral_constant<int, ACT>;
// calls body(ActTag<act>): what depends on the activation is compiled once for each
template <typename F>
__device__ __forceinline__ void by_act(int act, F &&body) {
  if (act == kRelu) body(ActTag<kRelu>{});
  else if (act == kSilu) body(ActTag<kSilu>{});
  else if (act == kGelu) body(ActTag<kGelu>{});
  else body(ActTag<kNone>{});
}

// SiLU and its slope vanish far below zero, where z sigmoid(z) as a product would not: the least sigmoid in float is
// 2^-126, which z beyond 1e30 makes visible, and infinity times zero is none.  z sigmoid(z) at the floor is below 2e-36 in
// size (float) and zero (double).
template <typename A>
__device__ __forceinline__ A silu_floor(A z) {
  return max_nan(z, sizeof(A) == 4 ? A(-128) : A(-1024));
}

template <typename A>
__device__ __forceinline__ A act_value(A z, int act) {
  if (act == kRelu) return max_nan(z, A(0));
  if (act == kSilu) {
    A f, keep;
    z = silu_floor(z);
    sigmoid_pair(z, f, keep);
    return z * f;
  }
  if (act == kGelu) return A(0.5) * z * (A(1) + erf_of(z * A(0.70710678118654752440)));
  return z;
}
template <typename A>
__device__ __forceinline__ A act_slope(A z, int act) {
  if (act == kRelu) return z > A(0) ? A(1) : A(0);
  if (act == kSilu) {
    A f, keep;
    z = silu_floor(z);
    sigmoid_pair(z, f, keep);
    return f * (A(1) + z * keep);
  }
  if (act == kGelu)
    return A(0.5) * (A(1) + erf_of(z * A(0.70710678118654752440))) +
           z * exp_of(A(-0.5) * z * z) * A(0.39894228040143267794);
  return A(1);
}

template <typename T>
struct NormArgs {
  Frames<const T> x, grad_y;
  Frames<T> y, grad_x;
  const Acc<T> *weight = nullptr, *bias = nullptr;            // (channels), or null: ones / zeros
  const Acc<T> *stats = nullptr;                              // (batch, groups, 2): mean, rstd
  Acc<T> *stats_out = nullptr;
  Acc<T> *grad_weight = nullptr, *grad_bias = nullptr;        // (channels), or null
  const int *lens = nullptr;
  int batch = 0, frames = 0, channels = 0, groups = 0, act = 0;
  Acc<T> eps = 0;
  // the fused kernels
  int team = 0, col_ranks = 1, row_ranks = 1;  // threads that share a group in a block; blocks of a cluster across both
  int team_log2 = 0, packs = 1, rows = 1;      // packs of a group's frame, frames a block (team) has at a time
  unsigned packs_magic = 0;                    // ceil(2^20 / packs of a frame in a block)
  int kept = 0;                                // most frames of a thread in shared memory
  int per_block = 1;                           // utterances a backward block takes one after the other
  int parts = 1;                               // sets of parameter sums: (parts, channels, 2) at `part`
  // the kernels for large groups: `tx` packs of `slabs` blocks make a frame of a group, `chunks` of `chunk_rows` its frames
  Acc<T> *part = nullptr;   // forward (batch, groups, entries, 3): mean, m2, count; backward (batch, chunks, channels, 2)
  Acc<T> *gsums = nullptr;  // (batch, groups, entries, 2): sums of weight * P1, weight * P2
  int chunks = 0, tx = 0, slabs = 0, chunk_rows = 0, entries = 0;
};

// (mean, sum of squared deviations, count) of two sets of values, joined
template <typename A>
__device__ __forceinline__ void join(A &mean, A &m2, A &count, A mean_b, A m2_b, A count_b) {
  if (count_b == A(0)) return;
  if (count == A(0)) {  // taken over as they are: the square of a mean far from zero may pass the type's range
    mean = mean_b, m2 = m2_b, count = count_b;
    return;
  }
  const A total = count + count_b, delta = mean_b - mean, share = count_b * reciprocal_unit(total);
  mean += delta * share;
  m2 += m2_b + delta * delta * count * share;
  count = total;
}

// Sums of count * mean are formed 2^32 times smaller: that changes no bit of them (unless the mean is below 1e-28) and keeps
// those of large groups within the type's range where the mean is.
template <typename A>
constexpr A kShrink = A(1) / A(4294967296.0);
template <typename A>
constexpr A kGrow = A(4294967296.0);

// ---- one pass: a group's values stay in shared memory between the sums and the result ---------------------------------
//
// `team` threads of a block (or the blocks of a cluster, team = all threads of each) share one utterance's group.  A
// thread has V adjacent channels, always the same, of every `rows`-th frame; these are copied to its own slots in shared
// memory, all copies issued at once, so x (and grad_y) is read once.  Teams are as small as the group allows, down to
// four threads, so that groups of a single frame share a warp.  Bound by HBM: two or more blocks a multiprocessor overlap one's sums
// with another's loads and stores.  Measured with 32 utterances of 200 to 800 frames, 1024 channels, 32 groups: float32
// and ReLU 32 us forward and 55 us backward (bytes alone: 26 and 36), bfloat16 and SiLU 26 and 43 (13 and 18: the special
// function unit and the conversions count there).  Values kept in registers instead, 64 a thread: 68 and 151 us (fewer
// bytes in flight, more clusters, code beyond the instruction cache).  Utterances are taken as they come: sorting them
// costs every block more than the shorter tail gains (float32 backward 60 us).

struct Seat {  // a thread's place
  int n, len, g, c, rank, size, team_id, j, tx, ty, rows, row_rank, cols;
  bool some, live;  // there are columns for this rank; this thread has one
};
template <typename T, int V>
__device__ __forceinline__ Seat seat_of(const NormArgs<T> &a) {
  Seat s;
  s.size = a.col_ranks * a.row_ranks;  // powers of two
  s.rank = (int)(blockIdx.x & (s.size - 1));
  s.row_rank = s.rank >> (31 - __clz(a.col_ranks));
  const unsigned col_rank = s.rank & (a.col_ranks - 1), block = blockIdx.x >> (31 - __clz(s.size));
  const unsigned turn = blockIdx.z * 65535u + blockIdx.y;
  s.n = (int)turn, s.len = a.per_block == 1 && s.n < a.batch ? live_frames(a.lens, s.n, a.frames) : 0;
  s.team_id = (int)(threadIdx.x >> a.team_log2), s.j = (int)(threadIdx.x & ((1u << a.team_log2) - 1));
  s.g = (int)(block * (kThreads >> a.team_log2)) + s.team_id;
  s.cols = a.packs, s.rows = a.rows, s.some = true;
  if (a.col_ranks > 1) {
    const int left = a.packs - (int)col_rank * a.team;  // none for the last ranks where the ranks are not a multiple
    s.some = left > 0;
    s.cols = left < 1 ? 1 : (left < a.team ? left : a.team);
    s.rows = a.team / s.cols;
    s.ty = s.j / s.cols;
  } else {
    s.ty = (int)((unsigned)s.j * a.packs_magic >> 20);  // j / packs, exact for j and packs up to 512
  }
  s.tx = s.j - s.ty * s.cols;
  s.live = s.g < a.groups && s.ty < s.rows && s.some;
  s.c = (s.g * a.packs + (int)col_rank * a.team + s.tx) * V;
  return s;
}
struct Span {
  int begin, end;
};
__device__ __forceinline__ Span span_of(int len, int rank, int ranks) {
  if (ranks == 1) return {0, len};
  const int rows = (int)((unsigned)(len + ranks - 1) / (unsigned)ranks);
  const long long begin = (long long)rows * rank;
  Span s;
  s.begin = begin < len ? (int)begin : len;
  s.end = len - s.begin < rows ? len : s.begin + rows;
  return s;
}

// Zeros in the frames first, first + step, ... behind an utterance's end
template <typename T, int V>
__device__ __forceinline__ void clear_from(const Frames<T> &f, long long n, int c, int first, int step, int frames) {
  T *p = f.p + n * f.sn + first * f.st + c;
  const long long jump = step * f.st;
  for (int t = first; t < frames; t += step, p += jump) store_raw<T, V>(p, zeros<T, V>());
}

// count, mean and sum of squared deviations of a thread's values, taken in a few frames at a time relative to the first of
// them: a pivot that is one of n values costs the squares at most n units in the last place
template <typename A>
struct Moments {
  A mean = 0, m2 = 0, count = 0;
};
// `n` (1 to B) frames
template <typename T, int V, int B, typename F>
__device__ __forceinline__ void add_batch(Moments<Acc<T>> &m, int n, F &&frame) {
  using A = Acc<T>;
  A pivot = 0, sum = 0, squares = 0;
#pragma unroll
  for (int i = 0; i < B; ++i) {
    if (i < n) {
      const Raw<T, V> r = frame(i);
      if (i == 0) pivot = element(r, 0);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A d = element(r, v) - pivot;
        sum += d, squares += d * d;
      }
    }
  }
  const A count = A(n * V), off = sum * reciprocal_unit(count);
  // squares beyond the type's range become NaN here, not a variance of zero
  join(m.mean, m.m2, m.count, pivot + off, max_nan(squares - sum * off, A(0)), count);
}

// A cluster's barrier in two halves: what lies between them does not wait for blocks that have not started
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// Sum over a team, the same bits in all its threads; `slots` (one a warp) is not used again before the next block barrier
// but one.
template <typename A, int Q>
__device__ __forceinline__ void team_sum(A (&v)[Q], int team_id, int team, A (*slots)[kThreads / 32]) {
#pragma unroll
  for (int o = 1; o < 32; o *= 2)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const A other = __shfl_xor_sync(0xffffffffu, v[q], o);
      if (o < team) v[q] += other;
    }
  if (team > 32) {
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int q = 0; q < Q; ++q) slots[q][threadIdx.x >> 5] = v[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (team == kThreads) {
        A all[kThreads / 32];
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) all[i] = slots[q][i];
#pragma unroll
        for (int o = kThreads / 64; o > 0; o /= 2)
#pragma unroll
          for (int i = 0; i < o; ++i) all[i] += all[i + o];
        v[q] = all[0];
      } else {
        v[q] = 0;
        for (int i = 0; i < team / 32; ++i) v[q] += slots[q][team_id * (team / 32) + i];
      }
    }
  }
}

template <typename T, int V, int MB>
__global__ void __launch_bounds__(kThreads, MB) norm_fused_kernel(const NormArgs<T> a) {
  begin<true>();
  using A = Acc<T>;
  extern __shared__ __align__(16) unsigned char shared_raw[];
  __shared__ __align__(16) A slots[2][kThreads / 32];
  __shared__ A ranks[kMaxRanks][3];
  const Seat s = seat_of<T, V>(a);
  if (s.n >= a.batch) return;  // the last plane of the grid is not full
  if (s.size > 1) cluster_arrive();
  const int len = s.len;
  const Span span = span_of(len, s.row_rank, a.row_ranks);
  const int first = span.begin + s.ty, end = s.live ? span.end : 0;
  const int kept = first < end ? (int)((unsigned)(end - first + s.rows - 1) / (unsigned)s.rows) : 0;
  const T *x = a.x.p + s.n * a.x.sn + first * a.x.st + s.c;
  const long long jump = s.rows * a.x.st;
  T *mine = reinterpret_cast<T *>(shared_raw) + threadIdx.x * V;  // frame i at mine + i * kThreads * V
  const T *from = x;
  for (int i = 0; i < kept; ++i, from += jump) copy_async<T, V>(mine + i * (kThreads * V), from);
  if (s.live) clear_from<T, V>(a.y, s.n, s.c, len + s.row_rank * s.rows + s.ty, a.row_ranks * s.rows, a.frames);
  A scale[V], shift[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    scale[v] = a.weight != nullptr && s.live ? a.weight[s.c + v] : A(1);
    shift[v] = a.bias != nullptr && s.live ? a.bias[s.c + v] : A(0);
  }
  Moments<A> m;
  copies_done();
  constexpr int kBatch = 16;
  for (int i0 = 0; i0 < kept; i0 += kBatch)
    add_batch<T, V, kBatch>(m, min(kBatch, kept - i0), [&](int i) { return load_shared<T, V>(mine + (i0 + i) * (kThreads * V)); });

  // the block's: sum of the values, then of the squared deviations from their mean
  A count = A(span.end - span.begin) * A(s.some ? s.cols * V : 0);
  A total[1] = {m.count * (m.mean * kShrink<A>)};
  team_sum(total, s.team_id, a.team, &slots[0]);
  A mean = count > A(0) ? total[0] / count * kGrow<A> : A(0);
  const A d = m.mean - mean;
  A squares[1] = {m.m2 + m.count * d * d};
  team_sum(squares, s.team_id, a.team, &slots[1]);
  A m2 = squares[0];
  if (s.size > 1) {
    auto cluster = cooperative_groups::this_cluster();
    cluster_wait();  // no block writes to one that has not started
    if (threadIdx.x < s.size) {
      A *to = cluster.map_shared_rank(&ranks[s.rank][0], threadIdx.x);
      to[0] = mean, to[1] = m2, to[2] = count;
    }
    cluster.sync();
    mean = ranks[0][0], m2 = ranks[0][1], count = ranks[0][2];
    for (int i = 1; i < s.size; ++i) join(mean, m2, count, ranks[i][0], ranks[i][1], ranks[i][2]);
  }
  if (!s.live) return;
  const A rstd = count > A(0) ? A(1) / sqrt(m2 / count + a.eps) : A(0);  // no frames: nothing to scale, no 0 * inf
  if (a.stats_out != nullptr && s.j == 0 && s.rank == 0) {
    A *out = a.stats_out + stats_offset(s.n, a.groups, s.g);
    out[0] = mean, out[1] = rstd;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) scale[v] *= rstd;
  T *y = a.y.p + s.n * a.y.sn + first * a.y.st + s.c;
  const long long leap = s.rows * a.y.st;
  by_act(a.act, [&](auto act) {
    auto result = [&](const Raw<T, V> &r, int i) {
      A o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = act_value((element(r, v) - mean) * scale[v] + shift[v], decltype(act)::value);
      store_raw<T, V>(y + i * leap, rounded<T, V>(o));
    };
#pragma unroll 4
    for (int i = 0; i < kept; ++i) result(load_shared<T, V>(mine + i * (kThreads * V)), i);
  });
}

// Backward: the same seats.  MANY: a block takes `per_block` utterances, all of whose frames fit, one after the other and
// keeps each channel's P1, P2 over all of them, so that few sets of parameter sums are left to be added (none, where one
// block has all utterances).
template <typename T, int V, int MB, bool MANY>
__global__ void __launch_bounds__(kThreads, MB) norm_fused_backward_kernel(const NormArgs<T> a) {
  begin<true>();
  using A = Acc<T>;
  extern __shared__ __align__(16) unsigned char shared_raw[];
  __shared__ __align__(16) A slots[2][2][kThreads / 32];
  __shared__ A ranks[2][kMaxRanks][2];
  const Seat s = seat_of<T, V>(a);
  // with one utterance a block, `chunk` is that utterance, else a run of them
  const long long chunk = s.n, n_first = MANY ? chunk * a.per_block : chunk;
  const long long n_end = MANY ? min(n_first + a.per_block, (long long)a.batch) : n_first + 1;
  if (n_first >= a.batch) return;  // the last plane of the grid is not full
  if (s.size > 1) cluster_arrive();
  bool met = false;
  A weight[V], bias[V], p1[V], p2[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    weight[v] = a.weight != nullptr && s.live ? a.weight[s.c + v] : A(1);
    bias[v] = a.bias != nullptr && s.live ? a.bias[s.c + v] : A(0);
    p1[v] = p2[v] = 0;
  }
  T *mine = reinterpret_cast<T *>(shared_raw) + threadIdx.x * V, *mine_y = mine + a.kept * (kThreads * V);
  int buffer = 0;
  for (long long n = n_first; n < n_end; ++n, buffer ^= 1) {
    const int len = MANY ? live_frames(a.lens, n, a.frames) : s.len;
    const Span span = span_of(len, s.row_rank, a.row_ranks);
    const int first = span.begin + s.ty, end = s.live ? span.end : 0;
    const int kept = first < end ? (int)((unsigned)(end - first + s.rows - 1) / (unsigned)s.rows) : 0;
    const T *x = a.x.p + n * a.x.sn + first * a.x.st + s.c, *gy = a.grad_y.p + n * a.grad_y.sn + first * a.grad_y.st + s.c;
    const long long jump = s.rows * a.x.st, jump_y = s.rows * a.grad_y.st, leap = s.rows * a.grad_x.st;
    const T *from = x, *from_y = gy;
    for (int i = 0; i < kept; ++i, from += jump, from_y += jump_y) {
      copy_async<T, V>(mine + i * (kThreads * V), from);
      copy_async<T, V>(mine_y + i * (kThreads * V), from_y);
    }
    if (s.live) clear_from<T, V>(a.grad_x, n, s.c, len + s.row_rank * s.rows + s.ty, a.row_ranks * s.rows, a.frames);
    A mean = 0, rstd = 0, scale[V], q1[V], q2[V], sums[2] = {A(0), A(0)};
    if (s.live) {
      const A *st = a.stats + stats_offset(n, a.groups, s.g);
      mean = st[0], rstd = st[1];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) q1[v] = q2[v] = 0, scale[v] = rstd * weight[v];
    by_act(a.act, [&](auto act) {
      auto add = [&](const Raw<T, V> &xq, const Raw<T, V> &yq) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const A d = element(xq, v) - mean, gz = element(yq, v) * act_slope(d * scale[v] + bias[v], decltype(act)::value);
          q1[v] += gz, q2[v] += gz * d;
        }
      };
      copies_done();
#pragma unroll 2
      for (int i = 0; i < kept; ++i)
        add(load_shared<T, V>(mine + i * (kThreads * V)), load_shared<T, V>(mine_y + i * (kThreads * V)));
    });
#pragma unroll
    for (int v = 0; v < V; ++v) {
      q2[v] *= rstd;  // of gz * xhat
      if constexpr (MANY) p1[v] += q1[v], p2[v] += q2[v];
      else p1[v] = q1[v], p2[v] = q2[v];
      sums[0] += weight[v] * q1[v], sums[1] += weight[v] * q2[v];
    }
    team_sum(sums, s.team_id, a.team, slots[buffer]);
    A s1 = sums[0], s2 = sums[1];
    if (s.size > 1) {
      auto cluster = cooperative_groups::this_cluster();
      if (!met) cluster_wait();
      met = true;
      if (threadIdx.x < s.size) {
        A *to = cluster.map_shared_rank(&ranks[buffer][s.rank][0], threadIdx.x);
        to[0] = s1, to[1] = s2;
      }
      cluster.sync();
      s1 = s2 = 0;
      for (int i = 0; i < s.size; ++i) s1 += ranks[buffer][i][0], s2 += ranks[buffer][i][1];
    }
    const A count = A(len) * A(a.channels / a.groups), inv = count > A(0) ? A(1) / count : A(0);
    s1 *= inv * rstd, s2 *= inv * rstd * rstd;  // gx = scale gz - s1 - (x - mean) s2
    if (!s.live) continue;
    T *gx = a.grad_x.p + n * a.grad_x.sn + first * a.grad_x.st + s.c;
    by_act(a.act, [&](auto act) {
      auto result = [&](const Raw<T, V> &xq, const Raw<T, V> &yq, int i) {
        A o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const A d = element(xq, v) - mean, gz = element(yq, v) * act_slope(d * scale[v] + bias[v], decltype(act)::value);
          o[v] = gz * scale[v] - (d * s2 + s1);
        }
        store_raw<T, V>(gx + i * leap, rounded<T, V>(o));
      };
#pragma unroll 2
      for (int i = 0; i < kept; ++i)
        result(load_shared<T, V>(mine + i * (kThreads * V)), load_shared<T, V>(mine_y + i * (kThreads * V)), i);
    });
  }
  if (a.grad_weight == nullptr && a.grad_bias == nullptr) return;
  // every channel's sums over the threads that have it, in the order of their frames
  __syncthreads();  // the slots of the last utterance's frames are taken for them
  A *columns = reinterpret_cast<A *>(shared_raw);  // [2 V][kThreads]
#pragma unroll
  for (int v = 0; v < V; ++v) columns[2 * v * kThreads + threadIdx.x] = p1[v], columns[(2 * v + 1) * kThreads + threadIdx.x] = p2[v];
  __syncthreads();
  if (s.g >= a.groups || !s.some) return;
  const int base = threadIdx.x - s.j;
  for (int q = s.j; q < 2 * V * s.cols; q += a.team) {
    const int v = q / s.cols, tx = q - v * s.cols, c = s.c + (tx - s.tx) * V + v / 2;
    A sum = 0;
#pragma unroll 8
    for (int r = 0; r < s.rows; ++r) sum += columns[v * kThreads + base + r * s.cols + tx];
    if (a.parts > 1) a.part[((chunk * a.row_ranks + s.row_rank) * a.channels + c) * 2 + v % 2] = sum;
    else if (v % 2 == 0 && a.grad_bias != nullptr) a.grad_bias[c] = sum;
    else if (v % 2 == 1 && a.grad_weight != nullptr) a.grad_weight[c] = sum;
  }
}

// gweight and gbias of 32 channels: P2 and P1 of the `parts` sets at a.part added, 8 threads a channel, whose sums are
// joined in order.  All threads of a block call it.
template <typename T>
__device__ __forceinline__ void add_parts(const NormArgs<T> &a, int parts, int block) {
  using A = Acc<T>;
  __shared__ A s1[kThreads], s2[kThreads];
  const int c = block * 32 + (int)(threadIdx.x & 31);
  A p1 = 0, p2 = 0;
  if (c < a.channels) {
#pragma unroll 4
    for (long long n = threadIdx.x >> 5; n < parts; n += kThreads / 32) {
      const A *in = a.part + (n * a.channels + c) * 2;
      p1 += in[0], p2 += in[1];
    }
  }
  s1[threadIdx.x] = p1, s2[threadIdx.x] = p2;
  __syncthreads();
  if (threadIdx.x >= 32 || c >= a.channels) return;
  for (int i = 1; i < kThreads / 32; ++i) p1 += s1[i * 32 + threadIdx.x], p2 += s2[i * 32 + threadIdx.x];
  if (a.grad_weight != nullptr) a.grad_weight[c] = p2;
  if (a.grad_bias != nullptr) a.grad_bias[c] = p1;
}

// ---- large groups: sums and result in two launches ---------------------------------------------------------------------
//
// Groups that a cluster's shared memory does not hold.  A block has `tx` packs of channels of one group and `chunk_rows`
// of its utterance's frames; `slabs` blocks side by side have a frame of the group, `chunks` one after the other its
// frames.  The first launch writes every block's sums; in the second every
// block adds its group's and normalises its part, read from L2 as a rule.  4 x 16384 x 256 channels, 8 groups, SiLU,
// bfloat16: 26 us forward and 44 us backward (bytes alone: 10 and 15); 12 x 548..2191 x 549 float32, one group: 39 and 55
// (12 and 22).

// frames of a thread fetched together: 8, or 4 where two tensors of 16 bytes a thread would fill the registers (four with
// the next four in flight were slower, 27 / 53 us below)
template <int BYTES, bool BOTH>
constexpr int kSpreadRows = BOTH && BYTES >= 16 ? 4 : 8;

struct Part {  // a block's part of a group, and a thread's place in it
  int n, len, g, c, ty, begin, end, entry, cols;
  bool live;
};
template <typename T, int V>
__device__ __forceinline__ Part part_of(const NormArgs<T> &a) {
  Part s;
  s.n = (int)(blockIdx.z * 65535u + blockIdx.y);
  s.len = s.n < a.batch ? live_frames(a.lens, s.n, a.frames) : 0;
  const unsigned across = (unsigned)(a.groups * a.slabs), chunk = blockIdx.x / across, rest = blockIdx.x - chunk * across;
  s.g = (int)(rest / (unsigned)a.slabs);
  const int slab = (int)rest - s.g * a.slabs, left = a.packs - slab * a.tx;
  s.cols = left < a.tx ? left : a.tx;
  s.ty = (int)(threadIdx.x * a.packs_magic >> 20);  // threadIdx.x / tx
  const int tx = (int)threadIdx.x - s.ty * a.tx;
  s.live = s.ty < a.rows && tx < s.cols;
  s.c = (s.g * a.packs + slab * a.tx + tx) * V;
  s.begin = (int)chunk * a.chunk_rows;
  s.end = s.begin + a.chunk_rows;  // of the frames there are room for; those of the utterance end at len
  s.entry = (int)chunk * a.slabs + slab;
  return s;
}

// A thread's frames first, first + step, ... below `end`, U at a time: body(x, grad_y, frame, n) with n frames in x (and,
// BOTH, in grad_y)
template <typename T, int V, bool BOTH, int U, typename F>
__device__ __forceinline__ void walk(const Frames<const T> &xf, const Frames<const T> &yf, int n, int c, int first, int step,
                                     int end, F &&body) {
  const T *x = xf.p + n * xf.sn + c, *gy = yf.p + n * yf.sn + c;
  for (int t = first; t < end; t += U * step) {
    Raw<T, V> xq[U], yq[BOTH ? U : 1];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (t + i * step < end) {
        xq[i] = load_raw<T, V>(x + (t + i * step) * xf.st);
        if constexpr (BOTH) yq[i] = load_raw<T, V>(gy + (t + i * step) * yf.st);
      }
    body(xq, yq, t, min(U, (int)((unsigned)(end - t + step - 1) / (unsigned)step)));
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) norm_moments_kernel(const NormArgs<T> a) {
  begin<true>();
  using A = Acc<T>;
  constexpr int U = kSpreadRows<Raw<T, V>::kBytes, false>;
  __shared__ __align__(16) A slots[2][kThreads / 32];
  const Part s = part_of<T, V>(a);
  if (s.n >= a.batch) return;
  const int end = min(s.end, s.len);
  Moments<A> m;
  walk<T, V, false, U>(a.x, a.grad_y, s.n, s.c, s.begin + s.ty, a.rows, s.live ? end : 0,
                    [&](Raw<T, V> (&xq)[U], Raw<T, V> (&)[1], int, int n) {
                      add_batch<T, V, U>(m, n, [&](int i) { return xq[i]; });
                    });
  const A count = A(max(end - s.begin, 0)) * A(s.cols * V);
  A total[1] = {m.count * (m.mean * kShrink<A>)};
  team_sum(total, 0, kThreads, &slots[0]);
  const A mean = count > A(0) ? total[0] / count * kGrow<A> : A(0), d = m.mean - mean;
  A squares[1] = {m.m2 + m.count * d * d};
  team_sum(squares, 0, kThreads, &slots[1]);
  if (threadIdx.x == 0) {
    A *to = a.part + (((long long)s.n * a.groups + s.g) * a.entries + s.entry) * 3;
    to[0] = mean, to[1] = squares[0], to[2] = count;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) norm_apply_kernel(const NormArgs<T> a) {
  begin<true>();
  using A = Acc<T>;
  constexpr int U = kSpreadRows<Raw<T, V>::kBytes, false>;
  __shared__ __align__(16) A slots[3][kThreads / 32];
  const Part s = part_of<T, V>(a);
  const int end = min(s.end, s.len), first = s.begin + s.ty, step = a.rows;
  A scale[V], shift[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    scale[v] = a.weight != nullptr && s.live ? a.weight[s.c + v] : A(1);
    shift[v] = a.bias != nullptr && s.live ? a.bias[s.c + v] : A(0);
  }
  if (s.n >= a.batch) return;
  const A *in = a.part + ((long long)s.n * a.groups + s.g) * a.entries * 3;
  A sums[2] = {A(0), A(0)}, squares[1] = {A(0)};
  for (int e = threadIdx.x; e < a.entries; e += kThreads) sums[0] += in[3 * e + 2], sums[1] += in[3 * e + 2] * (in[3 * e] * kShrink<A>);
  team_sum(sums, 0, kThreads, &slots[0]);
  const A count = sums[0], mean = count > A(0) ? sums[1] / count * kGrow<A> : A(0);
  for (int e = threadIdx.x; e < a.entries; e += kThreads) {
    const A d = in[3 * e] - mean;
    squares[0] += in[3 * e + 1] + in[3 * e + 2] * d * d;
  }
  team_sum(squares, 0, kThreads, &slots[2]);
  const A rstd = count > A(0) ? A(1) / sqrt(squares[0] / count + a.eps) : A(0);
  if (a.stats_out != nullptr && s.entry == 0 && threadIdx.x == 0) {
    A *out = a.stats_out + stats_offset(s.n, a.groups, s.g);
    out[0] = mean, out[1] = rstd;
  }
  if (!s.live) return;
#pragma unroll
  for (int v = 0; v < V; ++v) scale[v] *= rstd;
  T *y = a.y.p + s.n * a.y.sn + s.c;
  by_act(a.act, [&](auto act) {
    walk<T, V, false, U>(a.x, a.grad_y, s.n, s.c, first, step, end,
                      [&](Raw<T, V> (&xq)[U], Raw<T, V> (&)[1], int t, int n) {
#pragma unroll
                        for (int i = 0; i < U; ++i) {
                          if (i < n) {
                            A o[V];
#pragma unroll
                            for (int v = 0; v < V; ++v)
                              o[v] = act_value((element(xq[i], v) - mean) * scale[v] + shift[v], decltype(act)::value);
                            store_raw<T, V>(y + (t + i * step) * a.y.st, rounded<T, V>(o));
                          }
                        }
                      });
  });
  const int room = min(s.end, a.frames), from = max(s.len - s.begin, 0);  // frames behind the utterance's end
  clear_from<T, V>(a.y, s.n, s.c, first + (from > s.ty ? (from - s.ty + step - 1) / step * step : 0), step, room);
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 2) norm_sums_kernel(const NormArgs<T> a) {
  begin<true>();
  using A = Acc<T>;
  constexpr int U = kSpreadRows<Raw<T, V>::kBytes, true>;
  __shared__ __align__(16) A slots[2][kThreads / 32];
  __shared__ A columns[2 * V][kThreads];
  const Part s = part_of<T, V>(a);
  if (s.n >= a.batch) return;
  const int end = s.live ? min(s.end, s.len) : 0, first = s.begin + s.ty;
  const A *st = a.stats + stats_offset(s.n, a.groups, s.g), mean = st[0], rstd = st[1];
  A scale[V], weight[V], bias[V], q1[V], q2[V], sums[2] = {A(0), A(0)};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    weight[v] = a.weight != nullptr && s.live ? a.weight[s.c + v] : A(1);
    bias[v] = a.bias != nullptr && s.live ? a.bias[s.c + v] : A(0);
    q1[v] = q2[v] = 0, scale[v] = rstd * weight[v];
  }
  by_act(a.act, [&](auto act) {
    walk<T, V, true, U>(a.x, a.grad_y, s.n, s.c, first, a.rows, end,
                     [&](Raw<T, V> (&xq)[U], Raw<T, V> (&yq)[U], int, int n) {
#pragma unroll
                       for (int i = 0; i < U; ++i)
                         if (i < n)
#pragma unroll
                           for (int v = 0; v < V; ++v) {
                             const A d = element(xq[i], v) - mean;
                             const A gz = element(yq[i], v) * act_slope(d * scale[v] + bias[v], decltype(act)::value);
                             q1[v] += gz, q2[v] += gz * d;
                           }
                     });
  });
#pragma unroll
  for (int v = 0; v < V; ++v) {
    q2[v] *= rstd;
    sums[0] += weight[v] * q1[v], sums[1] += weight[v] * q2[v];
    columns[2 * v][threadIdx.x] = q1[v], columns[2 * v + 1][threadIdx.x] = q2[v];
  }
  team_sum(sums, 0, kThreads, slots);  // its barrier is the columns' too
  if (threadIdx.x == 0) {
    A *to = a.gsums + (((long long)s.n * a.groups + s.g) * a.entries + s.entry) * 2;
    to[0] = sums[0], to[1] = sums[1];
  }
  const int chunk = s.entry / a.slabs, first_pack = s.g * a.packs + (s.entry - chunk * a.slabs) * a.tx;
  A *to = a.part + ((long long)s.n * a.chunks + chunk) * a.channels * 2;
  for (int q = threadIdx.x; q < 2 * V * s.cols; q += kThreads) {
    const int v = q / s.cols, tx = q - v * s.cols;
    A sum = 0;
#pragma unroll 8
    for (int r = 0; r < a.rows; ++r) sum += columns[v][r * a.tx + tx];
    to[((first_pack + tx) * V + v / 2) * 2 + v % 2] = sum;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 2) norm_grad_input_kernel(const NormArgs<T> a) {
  begin<true>();
  using A = Acc<T>;
  constexpr int U = kSpreadRows<Raw<T, V>::kBytes, true>;
  __shared__ __align__(16) A slots[2][kThreads / 32];
  const int parts_of_all = a.groups * a.slabs * a.chunks;
  if ((int)blockIdx.x >= parts_of_all) {  // the blocks behind the parts of the first utterance add the parameters' sums
    if (blockIdx.y != 0 || blockIdx.z != 0) return;
    add_parts(a, a.batch * a.chunks, (int)blockIdx.x - parts_of_all);
    return;
  }
  const Part s = part_of<T, V>(a);
  if (s.n >= a.batch) return;
  const int end = s.live ? min(s.end, s.len) : 0, first = s.begin + s.ty;
  const A *st = a.stats + stats_offset(s.n, a.groups, s.g), mean = st[0], rstd = st[1];
  A scale[V], bias[V], sums[2] = {A(0), A(0)};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    scale[v] = rstd * (a.weight != nullptr && s.live ? a.weight[s.c + v] : A(1));
    bias[v] = a.bias != nullptr && s.live ? a.bias[s.c + v] : A(0);
  }
  const A *in = a.gsums + ((long long)s.n * a.groups + s.g) * a.entries * 2;
  for (int e = threadIdx.x; e < a.entries; e += kThreads) sums[0] += in[2 * e], sums[1] += in[2 * e + 1];
  team_sum(sums, 0, kThreads, slots);
  const A count = A(s.len) * A(a.channels / a.groups), inv = count > A(0) ? A(1) / count : A(0);
  const A s1 = sums[0] * inv * rstd, s2 = sums[1] * inv * rstd * rstd;  // gx = scale gz - s1 - (x - mean) s2
  if (!s.live) return;
  T *gx = a.grad_x.p + s.n * a.grad_x.sn + s.c;
  by_act(a.act, [&](auto act) {
    walk<T, V, true, U>(a.x, a.grad_y, s.n, s.c, first, a.rows, end,
                     [&](Raw<T, V> (&xq)[U], Raw<T, V> (&yq)[U], int t, int n) {
#pragma unroll
                       for (int i = 0; i < U; ++i) {
                         if (i < n) {
                           A o[V];
#pragma unroll
                           for (int v = 0; v < V; ++v) {
                             const A d = element(xq[i], v) - mean;
                             const A gz = element(yq[i], v) * act_slope(d * scale[v] + bias[v], decltype(act)::value);
                             o[v] = gz * scale[v] - (d * s2 + s1);
                           }
                           store_raw<T, V>(gx + (t + i * a.rows) * a.grad_x.st, rounded<T, V>(o));
                         }
                       }
                     });
  });
  const int room = min(s.end, a.frames), from = max(s.len - s.begin, 0), step = a.rows;
  clear_from<T, V>(a.grad_x, s.n, s.c, first + (from > s.ty ? (from - s.ty + step - 1) / step * step : 0), step, room);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_grad_params_kernel(const NormArgs<T> a, int parts) {
  begin<true>();
  add_parts(a, parts, (int)blockIdx.x);
}

// ---- host ---------------------------------------------------------------------------------------------------------

// Shared memory of a fused kernel's block: two fit a multiprocessor, or three of a forward call in 16 bits (32 utterances
// of 200 to 800 frames, 1024 channels, 32 groups, SiLU: 27 us against 31; float32 would need twice the clusters, 45
// against 39, and so would backward)
constexpr int kept_bytes(int tensors, size_t element) { return (tensors == 1 && element == 2 ? 72 : 108) * 1024; }

// Elements a thread moves at once: a power of two that divides a group's channels, so that they share its statistics
template <typename T>
int vector_width(const NormArgs<T> &a) {
  auto ok = [](const auto &f, int V) {
    return f.p == nullptr || (aligned_to(f.p, V * sizeof(T)) && f.sn % V == 0 && f.st % V == 0);
  };
  for (int V : {16 / (int)sizeof(T), 2})
    if (a.channels / a.groups % V == 0 && ok(a.x, V) && ok(a.grad_y, V) && ok(a.y, V) && ok(a.grad_x, V)) return V;
  return 1;
}

struct FusedPlan {
  bool use = false;  // a cluster holds a group
  int team = 0, col_ranks = 1, row_ranks = 1, kept = 0;
  long long blocks_per_utterance = 0;
};

// The fused kernels' division of a group of `per` channels, V at a time, keeping `tensors` tensors (1 forward, 2 backward)
FusedPlan plan_fused(int64_t batch, int64_t frames, int64_t groups, int64_t per, int V, int tensors, size_t element) {
  const int most = kept_bytes(tensors, element) / (int)(kThreads * V * element * tensors);  // frames a thread can keep
  FusedPlan p;
  const int64_t packs = per / V;
  p.team = 4;
  while (p.team < kThreads && (p.team < packs || (frames + p.team / packs - 1) / (p.team / packs) > 8)) p.team *= 2;
  while (p.col_ranks * (int64_t)p.team < packs && p.col_ranks < kMaxRanks) p.col_ranks *= 2;
  if (p.col_ranks * (int64_t)p.team < packs) return p;
  const int64_t rows = std::max<int64_t>(1, p.team / packs);
  auto kept = [&] { return ((frames + p.row_ranks - 1) / p.row_ranks + rows - 1) / rows; };
  while (p.team == kThreads && p.col_ranks * p.row_ranks < kMaxRanks && kept() > most) p.row_ranks *= 2;
  p.kept = (int)std::min<int64_t>(kept(), most);
  const int teams = kThreads / p.team;
  p.blocks_per_utterance = (groups + teams - 1) / teams * p.col_ranks * p.row_ranks;
  // clusters of eight, which find few places at a time, lose to the two launches above about one round of them: 20 x 5000
  // x 128, 4 groups, float32 33 us against 23 forward; 8 x 1200 x 512, 8 groups, backward 19 against 25
  const bool many = p.col_ranks * p.row_ranks == kMaxRanks && (size_t)(batch * frames * groups * per) * element > (24u << 20);
  p.use = kept() <= most && !many;
  return p;
}

// The division of groups that do not fit: up to 64 packs a block; as many chunks of frames as fill the multiprocessors
// (three blocks each forward, two backward) a whole number of times (a last round of a few blocks costs as much as a full one), with 16 to about 64
// frames a thread and at most about 1024 parts of a group
struct SpreadPlan {
  int tx, slabs, rows, chunks, chunk_rows;
};
SpreadPlan plan_spread(int64_t batch, int64_t frames, int64_t groups, int64_t per, int V, bool backward) {
  SpreadPlan p;
  const int64_t packs = per / V;
  p.slabs = (int)((packs + 63) / 64), p.tx = (int)((packs + p.slabs - 1) / p.slabs), p.rows = kThreads / p.tx;
  const int64_t base = batch * groups * p.slabs, slots = (backward ? 2 : 3) * 148, each = frames / p.rows;  // frames of a thread in all chunks
  const int64_t rounds = std::max<int64_t>(1, (int64_t)((long double)each * base / (64 * slots) + 0.999L));
  int64_t want = std::min(rounds * slots / std::max<int64_t>(base, 1), (each + 15) / 16);
  want = std::max<int64_t>(1, std::min<int64_t>(want, std::max(1, 1024 / p.slabs)));
  p.chunk_rows = (int)((frames + want - 1) / want);
  p.chunks = p.chunk_rows > 0 ? (int)((frames + p.chunk_rows - 1) / p.chunk_rows) : 1;
  return p;
}

// Utterances a backward block takes: all of them where that is little (one launch less), one where that leaves few sets
// of parameter sums, else as many as leave about three rounds of two blocks a multiprocessor
int64_t utterances_a_block(int64_t batch, int64_t frames, int64_t channels, const FusedPlan &p, size_t element) {
  if (batch <= 8 && (size_t)(frames * channels) * element <= (512u << 10)) return batch;
  if (batch * p.row_ranks <= 512) return 1;
  return std::max<int64_t>(1, batch * p.blocks_per_utterance / (148 * 6));
}

// Workspace in elements of the accumulation type, for whichever width the tensors' alignment allows
size_t workspace_elements(int64_t batch, int64_t frames, int64_t channels, int64_t groups, size_t element, bool backward) {
  if (batch <= 0 || frames < 0 || channels <= 0 || groups <= 0 || channels % groups != 0) return 0;
  const int64_t per = channels / groups;
  size_t need = 0;
  for (int V : {1, 2, 16 / (int)element}) {
    if (per % V != 0) continue;
    const FusedPlan p = plan_fused(batch, frames, groups, per, V, backward ? 2 : 1, element);
    if (p.use) {  // sets of parameter sums
      const int64_t each = utterances_a_block(batch, frames, channels, p, element);
      if (backward) need = std::max(need, (size_t)((batch + each - 1) / each) * p.row_ranks * (size_t)channels * 2);
    } else {
      const SpreadPlan q = plan_spread(batch, frames, groups, per, V, backward);
      const size_t entries = (size_t)batch * groups * q.chunks * q.slabs;
      need = std::max(need, backward ? (size_t)batch * q.chunks * channels * 2 + entries * 2 : entries * 3);
    }
  }
  return need;
}

template <typename T>
int prepare(const char *who, NormArgs<T> &a, int64_t batch, int64_t frames, int64_t channels, int64_t groups, int act,
            bool backward, void *workspace, size_t workspace_bytes) {
  const int rc = check_extents(who, batch, frames, channels);
  if (rc != MELLIN_OK) return rc;
  if (groups <= 0 || channels % groups != 0)
    return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": the channels are not a multiple of the groups");
  if (act < kNone || act > kGelu) return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": unknown activation");
  if (batch * std::max(groups, channels) > 0x7fffffffLL || batch > 0x7fff0000LL)
    return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many utterances times channels");
  a.batch = (int)batch, a.frames = (int)frames, a.channels = (int)channels, a.groups = (int)groups, a.act = act;
  if (batch == 0 || channels == 0) return MELLIN_OK;
  const size_t need = workspace_elements(batch, frames, channels, groups, sizeof(T), backward) * sizeof(Acc<T>);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(MELLIN_ERR_WORKSPACE, std::string(who) + ": workspace smaller than mellin_group_norm_act_workspace_bytes_*()");
  if (!aligned_to(workspace, 16)) return fail(MELLIN_ERR_WORKSPACE, std::string(who) + ": workspace must be 16-byte aligned");
  a.part = static_cast<Acc<T> *>(workspace);
  return MELLIN_OK;
}

template <typename T>
SpreadPlan take_spread(NormArgs<T> &a, int V, bool backward) {
  const SpreadPlan p = plan_spread(a.batch, a.frames, a.groups, a.channels / a.groups, V, backward);
  a.packs = a.channels / a.groups / V;
  a.tx = p.tx, a.slabs = p.slabs, a.rows = p.rows, a.chunks = p.chunks, a.chunk_rows = p.chunk_rows;
  a.entries = p.chunks * p.slabs, a.packs_magic = ((1u << 20) + p.tx - 1) / p.tx;
  a.gsums = a.part + (size_t)a.batch * a.chunks * a.channels * 2;
  return p;
}

template <typename K, typename T>
int launch(const char *who, K kernel, const NormArgs<T> &a, long long blocks, int cluster, size_t shared, cudaStream_t st,
           long long utterances) {
  const unsigned planes = (unsigned)((utterances + 65534) / 65535);  // the grid's second extent ends at 65535
  if (blocks > 0x7fffffffLL || planes > 65535) return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many blocks");
  if (shared > 44 * 1024) {  // with the static arrays beside it: beyond what a launch may have without asking
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 4096);
    if (err != cudaSuccess) return fail(MELLIN_ERR_LAUNCH, std::string(who) + ": " + cudaGetErrorString(err));
  }
  const dim3 grid((unsigned)blocks, (unsigned)std::min<long long>(utterances, 65535), planes);
  const cudaError_t err = launch_kernel(kernel, grid, kThreads, shared, cluster, st, a);
  if (err != cudaSuccess) return fail(MELLIN_ERR_LAUNCH, std::string(who) + ": " + cudaGetErrorString(err));
  return launched(who);
}

// body(V) for the widths there are of a type
template <typename T, typename F>
int by_width(int V, F &&body) {
  if (V == 1) return body(std::integral_constant<int, 1>{});
  if (V == 2) return body(std::integral_constant<int, 2>{});
  return body(std::integral_constant<int, 16 / (int)sizeof(T)>{});
}

template <typename T>
void take_plan(NormArgs<T> &a, const FusedPlan &p, int V) {
  a.team = p.team, a.col_ranks = p.col_ranks, a.row_ranks = p.row_ranks, a.kept = p.kept;
  a.team_log2 = 0;
  while ((1 << a.team_log2) < p.team) ++a.team_log2;
  a.packs = a.channels / a.groups / V, a.rows = std::max(1, p.team / a.packs);
  a.packs_magic = ((1u << 20) + a.packs - 1) / a.packs;
}
template <typename T, int V, int MB>
int launch_fused(const char *who, NormArgs<T> a, const FusedPlan &p, cudaStream_t st) {
  take_plan(a, p, V);
  return launch(who, norm_fused_kernel<T, V, MB>, a, p.blocks_per_utterance, p.col_ranks * p.row_ranks,
                (size_t)p.kept * kThreads * V * sizeof(T), st, a.batch);
}
template <typename T, int V, int MB>
int launch_fused_backward(const char *who, NormArgs<T> &a, const FusedPlan &p, cudaStream_t st) {
  take_plan(a, p, V);
  a.per_block = (int)utterances_a_block(a.batch, a.frames, a.channels, p, sizeof(T));
  const long long chunks = (a.batch + a.per_block - 1) / a.per_block;
  a.parts = (int)(chunks * p.row_ranks);
  const size_t shared = std::max((size_t)p.kept * kThreads * V * sizeof(T) * 2, kThreads * V * 2 * sizeof(Acc<T>));
  const int cluster = p.col_ranks * p.row_ranks;
  if (a.per_block == 1)
    return launch(who, norm_fused_backward_kernel<T, V, MB, false>, a, p.blocks_per_utterance, cluster, shared, st, chunks);
  return launch(who, norm_fused_backward_kernel<T, V, MB, true>, a, p.blocks_per_utterance, cluster, shared, st, chunks);
}

template <typename T>
int run_forward(NormArgs<T> a, int64_t batch, int64_t frames, int64_t channels, int64_t groups, int act, double eps,
                void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "group_norm_act";
  return guarded(who, [&]() -> int {
    if (!(eps >= 0)) return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": eps must not be negative or NaN");
    int rc = prepare(who, a, batch, frames, channels, groups, act, false, workspace, workspace_bytes);
    if (rc != MELLIN_OK || batch == 0 || channels == 0) return rc;
    if (frames > 0 && (a.x.p == nullptr || a.y.p == nullptr))
      return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": null pointer");
    a.eps = (Acc<T>)eps;
    auto st = static_cast<cudaStream_t>(stream);
    return by_width<T>(vector_width(a), [&](auto width) -> int {
      constexpr int V = decltype(width)::value;
      const FusedPlan p = plan_fused(batch, frames, groups, channels / groups, V, 1, sizeof(T));
      if (p.use) return launch_fused<T, V, sizeof(T) == 2 ? 3 : 2>(who, a, p, st);
      if (frames == 0) return MELLIN_OK;  // no statistics either: backward does not look at them
      const SpreadPlan q = take_spread(a, V, false);
      const long long blocks = groups * q.slabs * q.chunks;
      if ((rc = launch(who, norm_moments_kernel<T, V>, a, blocks, 1, 0, st, batch)) != MELLIN_OK) return rc;
      return launch(who, norm_apply_kernel<T, V>, a, blocks, 1, 0, st, batch);
    });
  });
}

template <typename T>
int run_backward(NormArgs<T> a, int64_t batch, int64_t frames, int64_t channels, int64_t groups, int act,
                 void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "backward of group_norm_act";
  return guarded(who, [&]() -> int {
    int rc = prepare(who, a, batch, frames, channels, groups, act, true, workspace, workspace_bytes);
    if (rc != MELLIN_OK || channels == 0) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    int parts = 0;
    if (batch > 0) {
      if (a.stats == nullptr || (frames > 0 && (a.x.p == nullptr || a.grad_y.p == nullptr || a.grad_x.p == nullptr)))
        return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": null pointer");
      rc = by_width<T>(vector_width(a), [&](auto width) -> int {
        constexpr int V = decltype(width)::value;
        const FusedPlan p = plan_fused(batch, frames, groups, channels / groups, V, 2, sizeof(T));
        if (p.use) {
          rc = launch_fused_backward<T, V, 2>(who, a, p, st);
          parts = a.parts;
          return rc;
        }
        if (frames == 0) {  // no sets of sums: zeros
          parts = a.parts = 0;
          return MELLIN_OK;
        }
        const SpreadPlan q = take_spread(a, V, true);
        const long long blocks = groups * q.slabs * q.chunks;
        if (batch * q.chunks > 0x7fffffffLL) return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many utterances times frames");
        a.parts = 1;  // the second launch adds the sets of sums itself
        const long long more = a.grad_weight != nullptr || a.grad_bias != nullptr ? (channels + 31) / 32 : 0;
        if ((rc = launch(who, norm_sums_kernel<T, V>, a, blocks, 1, 0, st, batch)) != MELLIN_OK) return rc;
        return launch(who, norm_grad_input_kernel<T, V>, a, blocks + more, 1, 0, st, batch);
      });
      if (rc != MELLIN_OK || a.parts == 1) return rc;
    }
    if (a.grad_weight == nullptr && a.grad_bias == nullptr) return MELLIN_OK;
    const cudaError_t err = launch_kernel(norm_grad_params_kernel<T>, dim3((unsigned)((channels + 31) / 32)), kThreads, 0, 1, st, a, parts);
    if (err != cudaSuccess) return fail(MELLIN_ERR_LAUNCH, std::string(who) + ": " + cudaGetErrorString(err));
    return launched(who);
  });
}

}  // namespace
}  // namespace mellin

using namespace mellin;

#define NORM_ENTRIES(SUFFIX, T, P, S)                                                                                  \
  size_t mellin_group_norm_act_workspace_bytes_##SUFFIX(int64_t batch, int64_t frames, int64_t channels,               \
                                                        int64_t groups, int backward) {                                \
    return workspace_elements(batch, frames, channels, groups, sizeof(T), backward != 0) * sizeof(S);                  \
  }                                                                                                                    \
  int mellin_group_norm_act_##SUFFIX(const P *x, int64_t x_sn, int64_t x_st, const S *weight, const S *bias,           \
                                     const int *lens, int64_t batch, int64_t frames, int64_t channels, int64_t groups, \
                                     double eps, int act, P *y, int64_t y_sn, int64_t y_st, S *stats,                  \
                                     void *workspace, size_t workspace_bytes, void *stream) {                          \
    NormArgs<T> a;                                                                                                     \
    a.x = {static_cast<const T *>(x), x_sn, x_st}, a.y = {static_cast<T *>(y), y_sn, y_st};                            \
    a.weight = weight, a.bias = bias, a.lens = lens, a.stats_out = stats;                                              \
    return run_forward<T>(a, batch, frames, channels, groups, act, eps, workspace, workspace_bytes, stream);           \
  }                                                                                                                    \
  int mellin_group_norm_act_backward_##SUFFIX(                                                                         \
      const P *x, int64_t x_sn, int64_t x_st, const S *weight, const S *bias, const S *stats, const int *lens,         \
      int64_t batch, int64_t frames, int64_t channels, int64_t groups, int act, const P *grad_y, int64_t grad_y_sn,    \
      int64_t grad_y_st, P *grad_x, int64_t grad_x_sn, int64_t grad_x_st, S *grad_weight, S *grad_bias,                \
      void *workspace, size_t workspace_bytes, void *stream) {                                                         \
    NormArgs<T> a;                                                                                                     \
    a.x = {static_cast<const T *>(x), x_sn, x_st}, a.grad_y = {static_cast<const T *>(grad_y), grad_y_sn, grad_y_st};  \
    a.grad_x = {static_cast<T *>(grad_x), grad_x_sn, grad_x_st};                                                       \
    a.weight = weight, a.bias = bias, a.stats = stats, a.lens = lens;                                                  \
    a.grad_weight = grad_weight, a.grad_bias = grad_bias;                                                              \
    return run_backward<T>(a, batch, frames, channels, groups, act, workspace, workspace_bytes, stream);               \
  }

extern "C" {

NORM_ENTRIES(f32, float, float, float)
NORM_ENTRIES(f64, double, double, double)
NORM_ENTRIES(f16, __half, void, float)
NORM_ENTRIES(bf16, __nv_bfloat16, void, float)

}  // extern "C"
