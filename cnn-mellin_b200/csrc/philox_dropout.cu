// Dropout whose mask is a function of (seed, element offset) and is never stored, with an optional residual added in the
// same pass:
//
//   y[i] = (word(i) >= round(p * 2^32) ? x[i] / (1 - p) : 0) + residual[i]
//
// word(i) is word i % 4 of Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw: Parallel random numbers:
// as easy as 1, 2, 3; SC 2011) with counter i / 4 and the 64-bit seed as key, i the element's offset in row-major order.
// Backward is the same pass over the gradient with the same seed and no residual.
#include <algorithm>
#include <cmath>

#include "sequence_common.cuh"

namespace mellin {
namespace {

using namespace seq;

constexpr int kThreads = 256;

struct Words {
  unsigned w[4];
};

__device__ __forceinline__ Words philox4x32_10(unsigned long long counter, unsigned long long key) {
  unsigned c0 = (unsigned)counter, c1 = (unsigned)(counter >> 32), c2 = 0, c3 = 0;
  unsigned k0 = (unsigned)key, k1 = (unsigned)(key >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const unsigned h0 = __umulhi(0xD2511F53u, c0), l0 = 0xD2511F53u * c0, h1 = __umulhi(0xCD9E8D57u, c2), l1 = 0xCD9E8D57u * c2;
    c0 = h1 ^ c1 ^ k0, c1 = l1, c2 = h0 ^ c3 ^ k1, c3 = l0;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

template <typename T>
struct DropoutArgs {
  const T *x = nullptr, *residual = nullptr;  // residual may be null
  T *y = nullptr;
  long long rows = 0, cols = 0, x_stride = 0, r_stride = 0;  // y is dense; strides between rows, in elements
  bool drop = false;       // round(p * 2^32) > 0; without it no word is drawn
  unsigned threshold = 0;  // kept where word > threshold = round(p * 2^32) - 1
  Acc<T> scale = 1;
  unsigned long long seed = 0;
  const long long *seed_device = nullptr;  // read instead of `seed` when there is one
};

// Two accesses of 16 bytes a thread are in flight before the generator's work, which is half of 16-bit tensors' time: a call
// for four elements has 38 instructions of the multiplier's pipe and 47 of the integer pipe, each of which takes one every
// second clock, 17 us of 26.2 M elements.  The other half is the beginning and end of blocks, which others cover in part only
// (integer pipe busy 60 %, issue slots 65 %).  26.2 M elements: float32 36 us = 5830 GB/s (0.89 of the measured copy rate),
// bfloat16 31 us = 3380 GB/s, with a residual 37 us = 4240 GB/s.  With whole 64-bit products 40 / 33 / 41 us; with one or four groups a thread 43 / 35 /
// 40 and 41 / 34 / 41 us.
//
// V elements a group, a multiple of 4; U groups a thread, kThreads groups apart, whose loads are issued together.  VEC:
// whole groups by packed accesses (aligned; one row of any length, or rows a multiple of V long); the group that ends a
// row which is no multiple of V, and everything without VEC, element by element.
template <typename T, int V, int U, bool VEC, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads) philox_dropout_kernel(const DropoutArgs<T> a) {
  begin<true>();
  using A = Acc<T>;
  const unsigned long long key = a.seed_device != nullptr ? (unsigned long long)*a.seed_device : a.seed;
  const long long total = a.rows * a.cols;
  const long long first = (blockIdx.x * (long long)(kThreads * U) + threadIdx.x) * V;
  Raw<T, V> xr[U], rr[U];
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const long long i = first + (long long)q * (kThreads * V);
      xr[q] = zeros<T, V>();
      if constexpr (RESIDUAL) rr[q] = zeros<T, V>();
      if (i + V <= total) {
        const long long row = a.rows == 1 ? 0 : i / a.cols, col = i - row * a.cols;
        xr[q] = load_raw<T, V>(a.x + row * a.x_stride + col);
        if constexpr (RESIDUAL) rr[q] = load_raw<T, V>(a.residual + row * a.r_stride + col);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < U; ++q) {
    const long long i = first + (long long)q * (kThreads * V);
    if (i >= total) return;
    A x[V], r[V];
    const bool whole = VEC && i + V <= total;
    if (whole) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = element(xr[q], v);
        if constexpr (RESIDUAL) r[v] = element(rr[q], v);
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = r[v] = A(0);
        if (i + v < total) {
          const long long row = a.rows == 1 ? 0 : (i + v) / a.cols, col = i + v - row * a.cols;
          x[v] = to_acc(a.x[row * a.x_stride + col]);
          if constexpr (RESIDUAL) r[v] = to_acc(a.residual[row * a.r_stride + col]);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < V / 4; ++g) {
      if (a.drop) {
        const Words w = philox4x32_10((unsigned long long)(i / 4 + g), key);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[g * 4 + j] = w.w[j] > a.threshold ? x[g * 4 + j] * a.scale : A(0);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[g * 4 + j] *= a.scale;  // 1, or what double sees of a p that drops nothing
      }
      if constexpr (RESIDUAL) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[g * 4 + j] += r[g * 4 + j];
      }
    }
    if (whole) {
      store_raw<T, V>(a.y + i, rounded<T, V>(x));
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (i + v < total) a.y[i + v] = from_acc<T>(x[v]);
    }
  }
}

template <typename T>
int run(DropoutArgs<T> a, double p, void *stream) {
  const char *who = "philox_dropout";
  return guarded(who, [&]() -> int {
    if (a.rows < 0 || a.cols < 0) return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": negative extent");
    if (!(p >= 0.0 && p <= 1.0)) return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": p outside [0, 1]");
    if ((long double)a.rows * (long double)a.cols > 4.0e18L)
      return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": more than 2^62 elements");
    const long long total = a.rows * a.cols;
    if (total == 0) return MELLIN_OK;
    if (a.x == nullptr || a.y == nullptr) return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": null pointer");
    const double threshold = std::floor(p * 4294967296.0 + 0.5);
    a.drop = threshold >= 1.0, a.threshold = a.drop ? (unsigned)(threshold - 1.0) : 0;
    a.scale = p < 1.0 ? (Acc<T>)(1.0 / (1.0 - p)) : Acc<T>(0);
    if (a.x_stride == a.cols && (a.residual == nullptr || a.r_stride == a.cols)) a.cols = total, a.rows = 1;
    constexpr int V = sizeof(T) == 2 ? 8 : 4, U = 2;
    constexpr size_t bytes = sizeof(T) == 8 ? 16 : sizeof(T) * V;
    const bool vec = aligned_to(a.x, bytes) && aligned_to(a.y, bytes) && aligned_to(a.residual, bytes) &&
                     (a.rows == 1 || (a.cols % V == 0 && a.x_stride % V == 0 && a.r_stride % V == 0));
    const long long per_block = (long long)V * U * kThreads, blocks = (total + per_block - 1) / per_block;
    if (blocks > 0x7fffffffLL) return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": more than 2^42 elements");
    cudaError_t err = cudaSuccess;
    auto go = [&](auto vector, auto residual) {
      err = launch_kernel(philox_dropout_kernel<T, V, U, decltype(vector)::value, decltype(residual)::value>,
                          dim3((unsigned)blocks), kThreads, 0, 1, stream, a);
    };
    if (vec && a.residual != nullptr) go(std::true_type{}, std::true_type{});
    else if (vec) go(std::true_type{}, std::false_type{});
    else if (a.residual != nullptr) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
    if (err != cudaSuccess) return fail(MELLIN_ERR_LAUNCH, std::string(who) + ": " + cudaGetErrorString(err));
    return launched(who);
  });
}

}  // namespace
}  // namespace mellin

using namespace mellin;

#define DROPOUT_ENTRY(SUFFIX, T, P)                                                                                  \
  int mellin_philox_dropout_##SUFFIX(const P *x, int64_t x_stride, const P *residual, int64_t residual_stride,       \
                                     int64_t rows, int64_t cols, double p, uint64_t seed, const int64_t *seed_device, \
                                     P *y, void *stream) {                                                           \
    DropoutArgs<T> a;                                                                                                \
    a.x = static_cast<const T *>(x), a.residual = static_cast<const T *>(residual), a.y = static_cast<T *>(y);       \
    a.rows = rows, a.cols = cols, a.x_stride = x_stride, a.r_stride = residual_stride, a.seed = seed;                \
    a.seed_device = reinterpret_cast<const long long *>(seed_device);                                                \
    return run<T>(a, p, stream);                                                                                     \
  }

extern "C" {

DROPOUT_ENTRY(f32, float, float)
DROPOUT_ENTRY(f64, double, double)
DROPOUT_ENTRY(f16, __half, void)
DROPOUT_ENTRY(bf16, __nv_bfloat16, void)

}  // extern "C"
