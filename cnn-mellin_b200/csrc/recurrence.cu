// Gated linear recurrence over the frames of ragged utterances, channels last:
//
//   f_t = sigmoid(gate_t),  h_t = f_t h_{t-1} + (1 - f_t) x_t,  y_t = h_t        (per utterance and channel)
//
// t runs over the utterance's own frames, first to last or (reverse) last to first; frames behind its end are never
// read and their outputs are zero.  The state is held in the accumulation type (float; double for double) whatever the
// tensors' type, and so are the states kept for backward: one every kStateStride frames.
//
// Backward, with gh_t the whole gradient of h_t and m_t = f_{t+1} gh_{t+1} what the frames after t pass back:
//
//   gh_t = gy_t + m_t,  m_{t-1} = f_t gh_t,  gx_t = (1 - f_t) gh_t,  ggate_t = f_t (1 - f_t) gh_t (h_{t-1} - x_t)
//
// h_{t-1} is recomputed from the kept states: y is not read (it may be rounded to 16 bits, and it would be one more
// tensor to fetch).
#include <algorithm>

#include "sequence_common.cuh"

namespace mellin {
namespace {

using namespace seq;

constexpr int kStateStride = 16;
constexpr int kWalkThreads = 128;

template <typename T>
struct RecurrenceArgs {
  Frames<const T> x, gate, grad_y;
  Frames<T> y, grad_x, grad_gate;
  const Acc<T> *initial = nullptr, *grad_final = nullptr;  // (batch, channels), or null: zeros
  Acc<T> *final = nullptr, *grad_initial = nullptr;        // (batch, channels), or null
  Acc<T> *states = nullptr;                                // (batch, ceil(frames / kStateStride), channels), or null
  const int *lens = nullptr;
  int batch = 0, frames = 0, channels = 0, reverse = 0;
};

// One thread per (utterance, channel), frame after frame.
template <typename T>
__global__ void __launch_bounds__(kWalkThreads) recurrence_walk_kernel(const RecurrenceArgs<T> a) {
  using A = Acc<T>;
  const long long i = blockIdx.x * (long long)kWalkThreads + threadIdx.x;
  if (i >= (long long)a.batch * a.channels) return;
  const long long n = i / a.channels, c = i - n * a.channels;
  const int len = (int)live_frames(a.lens, n, a.frames);
  const long long slots = (a.frames + kStateStride - 1) / kStateStride;
  const T *x = a.x.p + n * a.x.sn + c, *gate = a.gate.p + n * a.gate.sn + c;
  T *y = a.y.p + n * a.y.sn + c;
  A h = a.initial != nullptr ? a.initial[i] : A(0);
  for (int s = 0; s < len; ++s) {
    if (a.states != nullptr && s % kStateStride == 0) a.states[(n * slots + s / kStateStride) * a.channels + c] = h;
    const long long t = a.reverse ? len - 1 - s : s;
    A f, keep;
    sigmoid_pair(to_acc(gate[t * a.gate.st]), f, keep);
    h = f * h + keep * to_acc(x[t * a.x.st]);
    y[t * a.y.st] = from_acc<T>(h);
  }
  for (long long t = len; t < a.frames; ++t) y[t * a.y.st] = from_acc<T>(A(0));
  if (a.final != nullptr) a.final[i] = h;
}

template <typename T>
__global__ void __launch_bounds__(kWalkThreads) recurrence_walk_backward_kernel(const RecurrenceArgs<T> a) {
  using A = Acc<T>;
  const long long i = blockIdx.x * (long long)kWalkThreads + threadIdx.x;
  if (i >= (long long)a.batch * a.channels) return;
  const long long n = i / a.channels, c = i - n * a.channels;
  const int len = (int)live_frames(a.lens, n, a.frames);
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
        sigmoid_pair(to_acc(gate[t * a.gate.st]), f[k], keep[k]);
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

template <typename T>
int run_forward(RecurrenceArgs<T> a, int64_t batch, int64_t frames, int64_t channels, void *stream) {
  const char *who = "gated_recurrence";
  return guarded(who, [&] {
    const int rc = check(who, a, batch, frames, channels, false);
    if (rc != MELLIN_OK || batch == 0 || channels == 0) return rc;
    a.batch = (int)batch, a.frames = (int)frames, a.channels = (int)channels;
    const long long blocks = (batch * channels + kWalkThreads - 1) / kWalkThreads;
    if (blocks > 0x7fffffffLL) return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many rows");
    recurrence_walk_kernel<T><<<(unsigned)blocks, kWalkThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return launched(who);
  });
}

template <typename T>
int run_backward(RecurrenceArgs<T> a, int64_t batch, int64_t frames, int64_t channels, void *stream) {
  const char *who = "backward of gated_recurrence";
  return guarded(who, [&] {
    const int rc = check(who, a, batch, frames, channels, true);
    if (rc != MELLIN_OK || batch == 0 || channels == 0) return rc;
    a.batch = (int)batch, a.frames = (int)frames, a.channels = (int)channels;
    const long long blocks = (batch * channels + kWalkThreads - 1) / kWalkThreads;
    if (blocks > 0x7fffffffLL) return fail(MELLIN_ERR_UNSUPPORTED, std::string(who) + ": too many rows");
    recurrence_walk_backward_kernel<T><<<(unsigned)blocks, kWalkThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return launched(who);
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
  return run_forward<T>(a, batch, frames, channels, stream);
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
  return run_backward<T>(a, batch, frames, channels, stream);
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
  return batch * ((frames + kStateStride - 1) / kStateStride) * channels;
}

RECURRENCE_ENTRIES(f32, float, float, float)
RECURRENCE_ENTRIES(f64, double, double, double)
RECURRENCE_ENTRIES(f16, __half, void, float)
RECURRENCE_ENTRIES(bf16, __nv_bfloat16, void, float)

}  // extern "C"
