// Offsets into the small tensors of the sequence operators, for device and host code: plain arithmetic without CUDA types,
// so that a test without a GPU can hold it to extents that no test would allocate.
#pragma once

#ifdef __CUDACC__
#define MELLIN_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define MELLIN_HOST_DEVICE inline
#endif

namespace mellin {
namespace seq {

// Where mean and rstd of (utterance, group) lie in the (batch, groups, 2) statistics.  batch * groups goes up to
// 2^31 - 1, so the offset needs 64 bits whatever the operands have.
MELLIN_HOST_DEVICE long long stats_offset(long long utterance, long long groups, long long group) {
  return (utterance * groups + group) * 2;
}

}  // namespace seq
}  // namespace mellin
