// Shared by the sequence operators (recurrence.cu, group_norm.cu, philox_dropout.cu): storage and accumulation types,
// packed accesses, the guard around their C entry points.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <exception>
#include <string>

#include "../../include/mellin_b200.h"
#include "mellin_internal.h"

namespace mellin {
namespace seq {

// What sums, states and statistics of a tensor of T are held in.
template <typename T>
struct AccOf {
  using type = float;
};
template <>
struct AccOf<double> {
  using type = double;
};
template <typename T>
using Acc = typename AccOf<T>::type;

__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ float to_acc(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_acc(Acc<T> v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_acc<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// V consecutive elements moved by one access; the address is a multiple of the pack's size.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

inline bool aligned_to(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// A (batch, frames, channels) tensor whose channels are adjacent; the other two strides are free.
template <typename T>
struct Frames {
  T *p = nullptr;
  long long sn = 0, st = 0;
};

// frames of utterance n that exist: lens[n] held inside [0, frames]; all of them without lens
__device__ __forceinline__ long long live_frames(const int *lens, long long n, long long frames) {
  if (lens == nullptr) return frames;
  const long long v = lens[n];
  return v < 0 ? 0 : (v > frames ? frames : v);
}

// sigmoid(g) and 1 - sigmoid(g), each to a few units in its own last place: the exponential never overflows, and the
// complement is not formed by a subtraction
__device__ __forceinline__ void sigmoid_pair(float g, float &f, float &keep) {
  const float e = __expf(-fabsf(g)), r = __fdividef(1.f, 1.f + e), q = e * r;
  f = g < 0.f ? q : r;
  keep = g < 0.f ? r : q;
}
__device__ __forceinline__ void sigmoid_pair(double g, double &f, double &keep) {
  const double e = exp(-fabs(g)), r = 1.0 / (1.0 + e), q = e * r;
  f = g < 0.0 ? q : r;
  keep = g < 0.0 ? r : q;
}

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(const char *who, F &&body) {
  try {
    return body();
  } catch (const std::exception &e) {
    return fail(MELLIN_ERR_LAUNCH, std::string(who) + ": " + e.what());
  } catch (...) {
    return fail(MELLIN_ERR_LAUNCH, std::string(who) + ": unknown error");
  }
}

inline int launched(const char *who) {
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return fail(MELLIN_ERR_LAUNCH, std::string(who) + ": " + cudaGetErrorString(err));
  count_launch();
  return MELLIN_OK;
}

// Extents of a (batch, frames, channels) tensor the kernels index: non-negative, the product below 2^62, each below
// 2^31 (coordinates are 32-bit, offsets 64-bit).
inline int check_extents(const char *who, int64_t batch, int64_t frames, int64_t channels) {
  if (batch < 0 || frames < 0 || channels < 0) return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": negative extent");
  if (batch > 0x7fffffffLL || frames > 0x7fffffffLL || channels > 0x7fffffffLL)
    return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": extent above 2^31 - 1");
  if ((long double)batch * (long double)frames * (long double)channels > 4.0e18L)
    return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": more than 2^62 elements");
  return MELLIN_OK;
}

}  // namespace seq
}  // namespace mellin
