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
#include <algorithm>

#include "sequence_common.cuh"

namespace mellin {
namespace {

using namespace seq;

constexpr int kThreads = 256;
constexpr int kMaxChunks = 64;  // pieces of an utterance's frames in the kernels that pass over the tensor twice

enum Activation { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

__device__ __forceinline__ float exp_of(float v) { return __expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float erf_of(float v) { return erff(v); }
__device__ __forceinline__ double erf_of(double v) { return erf(v); }

template <typename A>
__device__ __forceinline__ A act_value(A z, int act) {
  if (act == kRelu) return z > A(0) ? z : (z <= A(0) ? A(0) : z);  // NaN stays
  if (act == kSilu) {
    A f, keep;
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
  // the kernels that pass over the tensor twice
  Acc<T> *part = nullptr;    // (batch, chunks, channels, 2)
  Acc<T> *sums = nullptr;    // (batch, channels, 2): P1, P2
  Acc<T> *gsums = nullptr;   // (batch, groups, 2): sums of weight * P1, weight * P2, over M
  int chunks = 0, tx = 0, slabs = 0;
};

// ---- any size: pass over the tensor for the sums, pass again to normalise ------------------------------------------

struct ChunkSpan {
  long long n, begin, end;  // frames of utterance n this block has
  int k, c;                 // chunk, first channel of the thread
};
template <typename T, int V>
__device__ __forceinline__ ChunkSpan chunk_span(const NormArgs<T> &a, long long upto) {
  long long b = blockIdx.x;
  ChunkSpan s;
  const int slab = (int)(b % a.slabs);
  b /= a.slabs;
  s.k = (int)(b % a.chunks), s.n = b / a.chunks;
  const long long rows = ((long long)a.frames + a.chunks - 1) / a.chunks;
  s.begin = s.k * rows;
  s.end = s.begin + rows < upto ? s.begin + rows : upto;
  s.c = (slab * a.tx + (int)(threadIdx.x % a.tx)) * V;
  return s;
}

// (mean, sum of squared deviations, count) of two sets of values, joined
template <typename A>
__device__ __forceinline__ void join(A &mean, A &m2, A &count, A mean_b, A m2_b, A count_b) {
  if (count_b == A(0)) return;
  const A total = count + count_b, delta = mean_b - mean, share = count_b / total;
  mean += delta * share;
  m2 += m2_b + delta * delta * count * share;
  count = total;
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_moments_kernel(const NormArgs<T> a) {
  using A = Acc<T>;
  __shared__ A mean_s[kThreads][V], m2_s[kThreads][V], count_s[kThreads];
  const long long upto = live_frames(a.lens, blockIdx.x / ((long long)a.slabs * a.chunks), a.frames);
  const ChunkSpan s = chunk_span<T, V>(a, upto);
  const int ty = threadIdx.x / a.tx, rows = kThreads / a.tx;
  A mean[V], m2[V], count = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0;
  if (s.c < a.channels) {
    for (long long t = s.begin + ty; t < s.end; t += rows) {
      const Raw<T, V> p = load_raw<T, V>(a.x.p + s.n * a.x.sn + t * a.x.st + s.c);
      count += A(1);
      const A inv = A(1) / count;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A value = element(p, v), delta = value - mean[v];
        mean[v] += delta * inv;
        m2[v] += delta * (value - mean[v]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) mean_s[threadIdx.x][v] = mean[v], m2_s[threadIdx.x][v] = m2[v];
  count_s[threadIdx.x] = count;
  __syncthreads();
  if (ty == 0 && s.c < a.channels) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A total = count;
      for (int r = 1; r < rows; ++r) {
        const int o = r * a.tx + threadIdx.x;
        join(mean[v], m2[v], total, mean_s[o][v], m2_s[o][v], count_s[o]);
      }
      A *out = a.part + (((long long)s.n * a.chunks + s.k) * a.channels + s.c + v) * 2;
      out[0] = mean[v], out[1] = m2[v];
    }
  }
}

// mean and rstd of one (utterance, group) from the chunks' moments
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(const NormArgs<T> a) {
  using A = Acc<T>;
  __shared__ A mean_s[kThreads], m2_s[kThreads], count_s[kThreads];
  const long long n = blockIdx.x / a.groups;
  const int g = (int)(blockIdx.x % a.groups), per = a.channels / a.groups;
  const long long upto = live_frames(a.lens, n, a.frames), rows = ((long long)a.frames + a.chunks - 1) / a.chunks;
  A mean = 0, m2 = 0, count = 0;
  for (long long i = threadIdx.x; i < (long long)a.chunks * per; i += kThreads) {
    const long long k = i / per, begin = k * rows, end = begin + rows < upto ? begin + rows : upto;
    const A *in = a.part + ((n * a.chunks + k) * a.channels + (long long)g * per + i % per) * 2;
    if (end > begin) join(mean, m2, count, in[0], in[1], A(end - begin));
  }
  mean_s[threadIdx.x] = mean, m2_s[threadIdx.x] = m2, count_s[threadIdx.x] = count;
  __syncthreads();
  for (int half = kThreads / 2; half > 0; half >>= 1) {
    if (threadIdx.x < half) {
      join(mean, m2, count, mean_s[threadIdx.x + half], m2_s[threadIdx.x + half], count_s[threadIdx.x + half]);
      mean_s[threadIdx.x] = mean, m2_s[threadIdx.x] = m2, count_s[threadIdx.x] = count;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    a.stats_out[2 * (long long)blockIdx.x] = mean;
    a.stats_out[2 * (long long)blockIdx.x + 1] = A(1) / sqrt((count > A(0) ? m2 / count : A(0)) + a.eps);
  }
}

// the statistics and parameters of a thread's V channels
template <typename T, int V>
struct ChannelParams {
  Acc<T> mean[V], rstd[V], weight[V], bias[V];
  __device__ __forceinline__ void load(const NormArgs<T> &a, long long n, int c) {
    const int per = a.channels / a.groups;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Acc<T> *st = a.stats + (n * a.groups + (c + v) / per) * 2;
      mean[v] = st[0], rstd[v] = st[1];
      weight[v] = a.weight != nullptr ? a.weight[c + v] : Acc<T>(1);
      bias[v] = a.bias != nullptr ? a.bias[c + v] : Acc<T>(0);
    }
  }
};

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(const NormArgs<T> a) {
  using A = Acc<T>;
  const ChunkSpan s = chunk_span<T, V>(a, a.frames);
  if (s.c >= a.channels) return;
  const long long upto = live_frames(a.lens, s.n, a.frames);
  ChannelParams<T, V> q;
  q.load(a, s.n, s.c);
  for (long long t = s.begin + threadIdx.x / a.tx; t < s.end; t += kThreads / a.tx) {
    A o[V];
    if (t < upto) {
      const Raw<T, V> p = load_raw<T, V>(a.x.p + s.n * a.x.sn + t * a.x.st + s.c);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A xhat = (element(p, v) - q.mean[v]) * q.rstd[v];
        o[v] = act_value(xhat * q.weight[v] + q.bias[v], a.act);
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = A(0);
    }
    store_raw<T, V>(a.y.p + s.n * a.y.sn + t * a.y.st + s.c, rounded<T, V>(o));
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_sums_kernel(const NormArgs<T> a) {
  using A = Acc<T>;
  __shared__ A sum_s[kThreads][2 * V];
  const long long upto = live_frames(a.lens, blockIdx.x / ((long long)a.slabs * a.chunks), a.frames);
  const ChunkSpan s = chunk_span<T, V>(a, upto);
  const int ty = threadIdx.x / a.tx, rows = kThreads / a.tx;
  A sum[2 * V];
#pragma unroll
  for (int v = 0; v < 2 * V; ++v) sum[v] = 0;
  if (s.c < a.channels) {
    ChannelParams<T, V> q;
    q.load(a, s.n, s.c);
    for (long long t = s.begin + ty; t < s.end; t += rows) {
      const Raw<T, V> p = load_raw<T, V>(a.x.p + s.n * a.x.sn + t * a.x.st + s.c);
      const Raw<T, V> gy = load_raw<T, V>(a.grad_y.p + s.n * a.grad_y.sn + t * a.grad_y.st + s.c);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A xhat = (element(p, v) - q.mean[v]) * q.rstd[v];
        const A gz = element(gy, v) * act_slope(xhat * q.weight[v] + q.bias[v], a.act);
        sum[2 * v] += gz, sum[2 * v + 1] += gz * xhat;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < 2 * V; ++v) sum_s[threadIdx.x][v] = sum[v];
  __syncthreads();
  if (ty == 0 && s.c < a.channels) {
    A *out = a.part + (((long long)s.n * a.chunks + s.k) * a.channels + s.c) * 2;
#pragma unroll
    for (int v = 0; v < 2 * V; ++v) {
      for (int r = 1; r < rows; ++r) sum[v] += sum_s[r * a.tx + threadIdx.x][v];
      out[v] = sum[v];
    }
  }
}

// P1, P2 of every channel of one (utterance, group), and the group's two weighted sums over M
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_group_sums_kernel(const NormArgs<T> a) {
  using A = Acc<T>;
  __shared__ A s1[kThreads], s2[kThreads];
  const long long n = blockIdx.x / a.groups;
  const int g = (int)(blockIdx.x % a.groups), per = a.channels / a.groups;
  A w1 = 0, w2 = 0;
  for (int j = threadIdx.x; j < per; j += kThreads) {
    const int c = g * per + j;
    A p1 = 0, p2 = 0;
    for (int k = 0; k < a.chunks; ++k) {
      const A *in = a.part + ((n * a.chunks + k) * a.channels + c) * 2;
      p1 += in[0], p2 += in[1];
    }
    a.sums[(n * a.channels + c) * 2] = p1, a.sums[(n * a.channels + c) * 2 + 1] = p2;
    const A w = a.weight != nullptr ? a.weight[c] : A(1);
    w1 += w * p1, w2 += w * p2;
  }
  s1[threadIdx.x] = w1, s2[threadIdx.x] = w2;
  __syncthreads();
  for (int half = kThreads / 2; half > 0; half >>= 1) {
    if (threadIdx.x < half) s1[threadIdx.x] += s1[threadIdx.x + half], s2[threadIdx.x] += s2[threadIdx.x + half];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const A count = A(live_frames(a.lens, n, a.frames)) * A(per);
    a.gsums[2 * (long long)blockIdx.x] = count > A(0) ? s1[0] / count : A(0);
    a.gsums[2 * (long long)blockIdx.x + 1] = count > A(0) ? s2[0] / count : A(0);
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) norm_grad_input_kernel(const NormArgs<T> a) {
  using A = Acc<T>;
  const ChunkSpan s = chunk_span<T, V>(a, a.frames);
  if (s.c >= a.channels) return;
  const long long upto = live_frames(a.lens, s.n, a.frames);
  const int per = a.channels / a.groups;
  ChannelParams<T, V> q;
  q.load(a, s.n, s.c);
  A s1[V], s2[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const A *in = a.gsums + (s.n * a.groups + (s.c + v) / per) * 2;
    s1[v] = in[0], s2[v] = in[1];
  }
  for (long long t = s.begin + threadIdx.x / a.tx; t < s.end; t += kThreads / a.tx) {
    A o[V];
    if (t < upto) {
      const Raw<T, V> p = load_raw<T, V>(a.x.p + s.n * a.x.sn + t * a.x.st + s.c);
      const Raw<T, V> gy = load_raw<T, V>(a.grad_y.p + s.n * a.grad_y.sn + t * a.grad_y.st + s.c);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const A xhat = (element(p, v) - q.mean[v]) * q.rstd[v];
        const A gz = element(gy, v) * act_slope(xhat * q.weight[v] + q.bias[v], a.act);
        o[v] = q.rstd[v] * (gz * q.weight[v] - s1[v] - xhat * s2[v]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = A(0);
    }
    store_raw<T, V>(a.grad_x.p + s.n * a.grad_x.sn + t * a.grad_x.st + s.c, rounded<T, V>(o));
  }
}

// gweight and gbias: P2 and P1 summed over the utterances, in order
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_grad_params_kernel(const NormArgs<T> a) {
  using A = Acc<T>;
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.channels) return;
  A p1 = 0, p2 = 0;
  for (long long n = 0; n < a.batch; ++n) {
    const A *in = a.sums + (n * a.channels + c) * 2;
    p1 += in[0], p2 += in[1];
  }
  if (a.grad_weight != nullptr) a.grad_weight[c] = p2;
  if (a.grad_bias != nullptr) a.grad_bias[c] = p1;
}

// ---- host ---------------------------------------------------------------------------------------------------------

int chunks_for(int64_t batch, int64_t frames, int64_t channels) {
  // enough blocks to fill the device a few times over, at least 32 frames in each
  const int64_t slabs = (channels + 31) / 32;
  const int64_t want = (148 * 16 + batch * slabs - 1) / std::max<int64_t>(batch * slabs, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, (frames + 31) / 32, (int64_t)kMaxChunks}));
}

// workspace in elements of the accumulation type: partial sums, then (batch, channels, 2), then (batch, groups, 2)
size_t workspace_elements(int64_t batch, int64_t frames, int64_t channels) {
  if (batch <= 0 || frames < 0 || channels <= 0) return 0;
  return (size_t)batch * (size_t)channels * 2 * ((size_t)chunks_for(batch, frames, channels) + 2);
}

template <typename T>
int vector_width(const NormArgs<T> &a) {
  constexpr int V = 16 / sizeof(T);
  auto ok = [&](const auto &f) {
    return f.p == nullptr || (aligned_to(f.p, 16) && f.sn % V == 0 && f.st % V == 0);
  };
  return a.channels % V == 0 && ok(a.x) && ok(a.grad_y) && ok(a.y) && ok(a.grad_x) ? V : 1;
}

template <typename T>
int prepare(const char *who, NormArgs<T> &a, int64_t batch, int64_t frames, int64_t channels, int64_t groups, int act,
            void *workspace, size_t workspace_bytes) {
  const int rc = check_extents(who, batch, frames, channels);
  if (rc != MELLIN_OK) return rc;
  if (groups <= 0 || channels % groups != 0)
    return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": the channels are not a multiple of the groups");
  if (act < kNone || act > kGelu) return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": unknown activation");
  if (batch * (groups > channels ? groups : channels) > 0x7fffffffLL)
    return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many utterances times channels");
  a.batch = (int)batch, a.frames = (int)frames, a.channels = (int)channels, a.groups = (int)groups, a.act = act;
  if (batch == 0 || channels == 0) return MELLIN_OK;
  const size_t need = workspace_elements(batch, frames, channels) * sizeof(Acc<T>);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(MELLIN_ERR_WORKSPACE, std::string(who) + ": workspace smaller than mellin_group_norm_act_workspace_bytes_*()");
  if (!aligned_to(workspace, sizeof(Acc<T>) * 2))
    return fail(MELLIN_ERR_WORKSPACE, std::string(who) + ": workspace must be 16-byte aligned");
  a.chunks = chunks_for(batch, frames, channels);
  a.part = static_cast<Acc<T> *>(workspace);
  a.sums = a.part + (size_t)batch * a.chunks * channels * 2;
  a.gsums = a.sums + (size_t)batch * channels * 2;
  return MELLIN_OK;
}

template <typename T>
long long grid_for(NormArgs<T> &a, int V) {
  int tx = 1;
  while (tx < 32 && tx * V < a.channels) tx *= 2;
  a.tx = tx, a.slabs = (a.channels + tx * V - 1) / (tx * V);
  return (long long)a.batch * a.chunks * a.slabs;
}

template <typename T>
int run_forward(NormArgs<T> a, int64_t batch, int64_t frames, int64_t channels, int64_t groups, int act, double eps,
                void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "group_norm_act";
  return guarded(who, [&]() -> int {
    int rc = prepare(who, a, batch, frames, channels, groups, act, workspace, workspace_bytes);
    if (rc != MELLIN_OK || batch == 0 || channels == 0) return rc;
    if (frames > 0 && (a.x.p == nullptr || a.y.p == nullptr))
      return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": null pointer");
    a.eps = (Acc<T>)eps;
    if (a.stats_out == nullptr) a.stats_out = a.gsums;
    a.stats = a.stats_out;
    auto st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto width) -> int {
      constexpr int V = decltype(width)::value;
      const long long blocks = grid_for(a, V);
      if (blocks > 0x7fffffffLL) return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many blocks");
      norm_moments_kernel<T, V><<<(unsigned)blocks, kThreads, 0, st>>>(a);
      if ((rc = launched(who)) != MELLIN_OK) return rc;
      norm_stats_kernel<T><<<(unsigned)(batch * groups), kThreads, 0, st>>>(a);
      if ((rc = launched(who)) != MELLIN_OK || frames == 0) return rc;
      norm_apply_kernel<T, V><<<(unsigned)blocks, kThreads, 0, st>>>(a);
      return launched(who);
    };
    constexpr int V = 16 / sizeof(T);
    return vector_width(a) == V ? go(std::integral_constant<int, V>{}) : go(std::integral_constant<int, 1>{});
  });
}

template <typename T>
int run_backward(NormArgs<T> a, int64_t batch, int64_t frames, int64_t channels, int64_t groups, int act,
                 void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "backward of group_norm_act";
  return guarded(who, [&]() -> int {
    int rc = prepare(who, a, batch, frames, channels, groups, act, workspace, workspace_bytes);
    if (rc != MELLIN_OK || channels == 0) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    const unsigned param_blocks = (unsigned)((channels + kThreads - 1) / kThreads);
    if (batch > 0) {
      if (a.stats == nullptr || (frames > 0 && (a.x.p == nullptr || a.grad_y.p == nullptr || a.grad_x.p == nullptr)))
        return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": null pointer");
      auto go = [&](auto width) -> int {
        constexpr int V = decltype(width)::value;
        const long long blocks = grid_for(a, V);
        if (blocks > 0x7fffffffLL) return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many blocks");
        norm_sums_kernel<T, V><<<(unsigned)blocks, kThreads, 0, st>>>(a);
        if ((rc = launched(who)) != MELLIN_OK) return rc;
        norm_group_sums_kernel<T><<<(unsigned)(batch * groups), kThreads, 0, st>>>(a);
        if ((rc = launched(who)) != MELLIN_OK || frames == 0) return rc;
        norm_grad_input_kernel<T, V><<<(unsigned)blocks, kThreads, 0, st>>>(a);
        return launched(who);
      };
      constexpr int V = 16 / sizeof(T);
      rc = vector_width(a) == V ? go(std::integral_constant<int, V>{}) : go(std::integral_constant<int, 1>{});
      if (rc != MELLIN_OK) return rc;
    }
    if (a.grad_weight == nullptr && a.grad_bias == nullptr) return MELLIN_OK;
    norm_grad_params_kernel<T><<<param_blocks, kThreads, 0, st>>>(a);
    return launched(who);
  });
}

}  // namespace
}  // namespace mellin

using namespace mellin;

#define NORM_ENTRIES(SUFFIX, T, P, S)                                                                                  \
  size_t mellin_group_norm_act_workspace_bytes_##SUFFIX(int64_t batch, int64_t frames, int64_t channels) {             \
    return workspace_elements(batch, frames, channels) * sizeof(S);                                                    \
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
