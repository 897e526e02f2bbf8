// Shared by the sequence operators (recurrence.cu, group_norm.cu, philox_dropout.cu): storage and accumulation types,
// packed accesses, the guard around their C entry points.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <exception>
#include <string>
#include <type_traits>

#include "../../include/mellin_b200.h"
#include "mellin_internal.h"
#include "sequence_index.h"
#include "tc_ptx.cuh"

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

inline bool aligned_to(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// frames of utterance n that exist: lens[n] held inside [0, frames]; all of them without lens
__device__ __forceinline__ int live_frames(const int *lens, long long n, int frames) {
  if (lens == nullptr) return frames;
  const int v = lens[n];
  return v < 0 ? 0 : (v > frames ? frames : v);
}

// Which utterance a block takes that is `turn`th in launch order, and its frames: the longest first, so that the last
// blocks to start are short ones (recurrence, 32 utterances of 200 to 800 frames, 1024 channels, bfloat16: forward
// 36 -> 32 us, backward 55 -> 47).  Every warp sorts for itself, lane i counting what goes before utterance i (one warp
// and a block barrier: 5 % slower); batches above 32, whose blocks are many enough to even out, are taken as they come.
struct Utterance {
  int n, len;
};
__device__ __forceinline__ Utterance utterance_of(const int *lens, int batch, int frames, int turn) {
  if (lens == nullptr) return {turn, frames};
  if (batch > 32 || batch == 1) return {turn, turn < batch ? live_frames(lens, turn, frames) : 0};
  const int lane = threadIdx.x & 31, mine = lane < batch ? lens[lane] : INT_MIN;
  int place = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const int other = __shfl_sync(0xffffffffu, mine, j);
    place += other > mine || (other == mine && j < lane);
  }
  const int n = __ffs(__ballot_sync(0xffffffffu, place == turn)) - 1, len = __shfl_sync(0xffffffffu, mine, n);
  return {n, len < 0 ? 0 : (len > frames ? frames : len)};
}

// V consecutive elements as the 32-bit words they lie in, moved by accesses of up to 16 bytes (one address, a multiple of
// the access); elements are taken out of the words only where they are used, so that loads can stay in flight.
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = (int)sizeof(T) * V, kWords = kBytes < 4 ? 1 : kBytes / 4;
  unsigned w[kWords];
};

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T *p) {
  Raw<T, V> r;
  constexpr int BYTES = Raw<T, V>::kBytes;
  if constexpr (BYTES == 2) {
    r.w[0] = __ldg(reinterpret_cast<const unsigned short *>(p));
  } else if constexpr (BYTES == 4) {
    r.w[0] = __ldg(reinterpret_cast<const unsigned *>(p));
  } else if constexpr (BYTES == 8) {
    const uint2 q = __ldg(reinterpret_cast<const uint2 *>(p));
    r.w[0] = q.x, r.w[1] = q.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 q = __ldg(reinterpret_cast<const uint4 *>(p) + i);
      r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
    }
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_raw(T *p, const Raw<T, V> &r) {
  constexpr int BYTES = Raw<T, V>::kBytes;
  if constexpr (BYTES == 2) {
    *reinterpret_cast<unsigned short *>(p) = (unsigned short)r.w[0];
  } else if constexpr (BYTES == 4) {
    *reinterpret_cast<unsigned *>(p) = r.w[0];
  } else if constexpr (BYTES == 8) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(r.w[0], r.w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      reinterpret_cast<uint4 *>(p)[i] = make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
  }
}

// element v in the accumulation type
template <int V>
__device__ __forceinline__ float element(const Raw<float, V> &r, int v) {
  return __uint_as_float(r.w[v]);
}
template <int V>
__device__ __forceinline__ double element(const Raw<double, V> &r, int v) {
  return __hiloint2double((int)r.w[2 * v + 1], (int)r.w[2 * v]);
}
template <int V>
__device__ __forceinline__ float element(const Raw<__nv_bfloat16, V> &r, int v) {
  return __uint_as_float(v & 1 ? r.w[v / 2] & 0xffff0000u : r.w[v / 2] << 16);
}
template <int V>
__device__ __forceinline__ float element(const Raw<__half, V> &r, int v) {
  return __half2float(__ushort_as_half((unsigned short)(v & 1 ? r.w[v / 2] >> 16 : r.w[v / 2])));
}

// V elements from global to shared memory without a register between; complete after copies_done() in the same thread.
// Two-byte packs, which the asynchronous copy does not know, are loaded and stored.
template <typename T, int V>
__device__ __forceinline__ void copy_async(T *to, const T *from) {
  constexpr int BYTES = Raw<T, V>::kBytes;
  if constexpr (BYTES == 2) {
    store_raw<T, V>(to, load_raw<T, V>(from));
  } else {
    const unsigned dst = (unsigned)__cvta_generic_to_shared(to);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(BYTES) : "memory");
  }
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_shared(const T *p) {
  Raw<T, V> r;
  constexpr int BYTES = Raw<T, V>::kBytes;
  static_assert(BYTES <= 16, "one access");
  if constexpr (BYTES == 2) {
    r.w[0] = *reinterpret_cast<const unsigned short *>(p);
  } else if constexpr (BYTES == 4) {
    r.w[0] = *reinterpret_cast<const unsigned *>(p);
  } else if constexpr (BYTES == 8) {
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    r.w[0] = q.x, r.w[1] = q.y;
  } else {
    const uint4 q = *reinterpret_cast<const uint4 *>(p);
    r.w[0] = q.x, r.w[1] = q.y, r.w[2] = q.z, r.w[3] = q.w;
  }
  return r;
}

// V values rounded to T
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> rounded(const Acc<T> (&a)[V]) {
  Raw<T, V> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int v = 0; v < V; ++v) r.w[v] = __float_as_uint(a[v]);
  } else if constexpr (sizeof(T) == 8) {
#pragma unroll
    for (int v = 0; v < V; ++v) r.w[2 * v] = (unsigned)__double2loint(a[v]), r.w[2 * v + 1] = (unsigned)__double2hiint(a[v]);
  } else if constexpr (V == 1) {
    if constexpr (std::is_same<T, __half>::value) r.w[0] = __half_as_ushort(__float2half_rn(a[0]));
    else r.w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(a[0]));
  } else {
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 q = __floats2half2_rn(a[v], a[v + 1]);
        r.w[v / 2] = *reinterpret_cast<const unsigned *>(&q);
      } else {
        const __nv_bfloat162 q = __floats2bfloat162_rn(a[v], a[v + 1]);
        r.w[v / 2] = *reinterpret_cast<const unsigned *>(&q);
      }
    }
  }
  return r;
}

// the same value V times, as bits
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> zeros() {
  Raw<T, V> r;
#pragma unroll
  for (int i = 0; i < Raw<T, V>::kWords; ++i) r.w[i] = 0;
  return r;
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> infinities() {
  Raw<T, V> r;
#pragma unroll
  for (int i = 0; i < Raw<T, V>::kWords; ++i) {
    if constexpr (sizeof(T) == 8) r.w[i] = i & 1 ? 0x7ff00000u : 0u;
    else if constexpr (sizeof(T) == 4) r.w[i] = 0x7f800000u;
    else if constexpr (std::is_same<T, __half>::value) r.w[i] = 0x7c007c00u;
    else r.w[i] = 0x7f807f80u;
  }
  return r;
}

// A (batch, frames, channels) tensor whose channels are adjacent; the other two strides are free.
template <typename T>
struct Frames {
  T *p = nullptr;
  long long sn = 0, st = 0;
};

// 2^v and 1 / v by the special function unit alone, without the scaling around it that results below 2^-126 need
__device__ __forceinline__ float exp2_unit(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_unit(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ double reciprocal_unit(double v) { return 1.0 / v; }
// the larger one; NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ double max_nan(double a, double b) { return a > b ? a : (a <= b ? b : a + b); }

// sigmoid(g) and 1 - sigmoid(g), each to 8 + 1.25 |g| units of 2^-24 relative to itself at most: the complement is
// e sigmoid(g) with e = exp(-g), not a difference, and e is as exact as the product of g and log2(e) is after its rounding to
// one float (63 units at |g| = 80 as emulated).  e is held at 2^126, so that the quotient stays a normal number (the least
// sigmoid is 2^-126); NaN stays NaN.  SHUT: where e is held, sigmoid is 0, so that a shut gate lets nothing of a state
// through whatever its size (2^-126 of 3e38 would be 4); 1 % of the recurrence's time.
template <bool SHUT = false>
__device__ __forceinline__ void sigmoid_pair(float g, float &f, float &keep) {
  float t;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(t) : "f"(g * -1.4426950408889634f), "f"(126.f));
  const float e = exp2_unit(t), r = reciprocal_unit(1.f + e);
  keep = e * r;
  f = SHUT && t >= 126.f ? 0.f : r;
}
template <bool SHUT = false>
__device__ __forceinline__ void sigmoid_pair(double g, double &f, double &keep) {
  const double e = exp(-fabs(g)), r = 1.0 / (1.0 + e), q = e * r;
  f = g < 0.0 ? q : r;
  keep = g < 0.0 ? r : q;
}

// Every kernel here is launched programmatically dependent: its launch is under way while the kernel before it runs out,
// and begin() waits for that one before it touches memory.  With EARLY the next kernel's blocks may also take their
// places as this one's blocks leave: good for many short blocks (dropout 78 -> 76 us, norm 91 -> 88 of the training
// cases), bad where few long ones should spread evenly (recurrence, decoding: 31 -> 34 us).
template <bool EARLY>
__device__ __forceinline__ void begin() {
  if constexpr (EARLY) tc::launch_dependents();
  tc::grid_dependency_wait();
}
template <typename... KernelArgs, typename... Args>
cudaError_t launch_kernel(void (*kernel)(KernelArgs...), dim3 grid, int threads, size_t shared, int cluster, void *stream,
                          Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = dim3((unsigned)threads), cfg.dynamicSmemBytes = shared;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr, cfg.numAttrs = 0;
  if (dependent_launch_enabled()) {  // without it: an ordinary launch
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kernel, KernelArgs(args)...);
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

// Extents of a (batch, frames, channels) tensor the kernels index: non-negative, the product below 2^62, batch below
// 2^31, frames and channels at most 2^30 (coordinates are 32-bit, a step past the end included; offsets are 64-bit).
inline int check_extents(const char *who, int64_t batch, int64_t frames, int64_t channels) {
  if (batch < 0 || frames < 0 || channels < 0) return fail(MELLIN_ERR_BAD_ARGUMENT, std::string(who) + ": negative extent");
  if (batch > 0x7fffffffLL || frames > 0x40000000LL || channels > 0x40000000LL)
    return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": batch above 2^31 - 1, or frames or channels above 2^30");
  if ((long double)batch * (long double)frames * (long double)channels > 4.0e18L)
    return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": more than 2^62 elements");
  return MELLIN_OK;
}

}  // namespace seq
}  // namespace mellin
