// The gated linear recurrence over the steps of a batch of sequences,
//   h[t] = a[t] h[t-1] + w[t] x[t],   w = 1 or (mixed form) 1 - a,
// and its gradients.  With e[t] = a[t] c[t] the gradient c[t] of h[t] follows the same recurrence backwards:
//   c[t] = dh[t] + e[t+1],  e[t] = a[t] c[t];   dx = w c,  da = c (h[t-1] - (mixed) x),  dstate = e[0].
// Behind a sequence's length the state is kept and nothing is read: whatever stands there cannot reach a result.
#include "recurrence.hpp"
#include "device.hpp"
#include "seq_types.hpp"
#include <algorithm>

namespace lga {

namespace {

constexpr int kThreads = 256;

enum GateKind { kNoGate, kOwnGate, kSharedGate };

// One lane walks a sequence's channel through all steps.
template <typename T, typename G, GateKind K>
__global__ __launch_bounds__(kThreads) void scan_walk_kernel(ScanArgs a) {
  typedef Wide<T> W;
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.batch * a.width) return;
  const int64_t b = c / a.width, d = c - b * a.width;
  const T* x = (const T*)a.x + b * a.x_b + d;
  const G* gate = K == kNoGate ? nullptr : (const G*)a.gate + b * a.gate_b + d / (a.width / a.groups);
  T* out = (T*)a.states + b * a.steps * a.width + d;
  const int64_t len = a.lengths ? std::min<int64_t>(((const int32_t*)a.lengths)[b], a.steps) : a.steps;
  W h = a.state ? ((const W*)a.state)[c] : (W)0;
  int64_t t = 0;
  for (; t < len; ++t) {
    W v = (W)x[t * a.x_t];
    if constexpr (K == kNoGate) {
      h += v;
    } else {
      const W g = (W)gate[t * a.gate_t];
      if (a.mix) v *= (W)1 - g;
      h = fma_wide(g, h, v);
    }
    out[t * a.width] = (T)h;
  }
  for (; t < a.steps; ++t) out[t * a.width] = (T)(W)0;
  ((W*)a.last)[c] = h;
}

template <typename T, typename G, GateKind K>
__global__ __launch_bounds__(kThreads) void scan_grad_walk_kernel(ScanGradArgs a) {
  typedef Wide<T> W;
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.batch * a.width) return;
  const int64_t b = c / a.width, d = c - b * a.width;
  const T* dh = (const T*)a.grad_states + b * a.g_b + d;
  const T* hs = (const T*)a.states + b * a.h_b + d;
  const T* x = a.mix ? (const T*)a.x + b * a.x_b + d : nullptr;
  const G* gate = K == kNoGate ? nullptr : (const G*)a.gate + b * a.gate_b + d / (a.width / a.groups);
  T* dx = (T*)a.grad_x + b * a.steps * a.width + d;
  W* slope = (W*)a.work + b * a.steps * a.width + d;        // the gate's gradient, value by value
  const int64_t len = a.lengths ? std::max<int64_t>(0, std::min<int64_t>(((const int32_t*)a.lengths)[b], a.steps)) : a.steps;
  W e = a.grad_last ? ((const W*)a.grad_last)[c] : (W)0;
  int64_t t = a.steps;
  for (; t > len; --t) {
    dx[(t - 1) * a.width] = (T)(W)0;
    if (K != kNoGate) slope[(t - 1) * a.width] = 0;
  }
  for (; t > 0; --t) {
    const W cc = (W)dh[(t - 1) * a.g_t] + e;
    W v = cc;
    if constexpr (K == kNoGate) {
      e = cc;
    } else {
      const W g = (W)gate[(t - 1) * a.gate_t];
      W before = t > 1 ? (W)hs[(t - 2) * a.h_t] : (a.state ? ((const W*)a.state)[c] : (W)0);
      if (a.mix) {
        before -= (W)x[(t - 1) * a.x_t];
        v *= (W)1 - g;
      }
      slope[(t - 1) * a.width] = cc * before;
      e = g * cc;
    }
    dx[(t - 1) * a.width] = (T)v;
  }
  ((W*)a.grad_state)[c] = e;
}

// grad_gate[q][t][g] = sum of the slopes of the sequences and channels that share the gate, in a fixed order:
// lanes over them, then a tree.
template <typename W, typename G>
__global__ __launch_bounds__(kThreads) void gate_sum_kernel(const W* __restrict__ slope, G* __restrict__ out, int64_t batch, int64_t steps,
                                                            int64_t width, int64_t groups, int64_t gate_batch) {
  __shared__ W part[kThreads];
  const int64_t per = width / groups, shared = gate_batch == batch ? 1 : batch;
  for (int64_t o = blockIdx.x; o < gate_batch * steps * groups; o += gridDim.x) {
    const int64_t q = o / (steps * groups), t = o / groups % steps, g = o % groups;
    W sum = 0;
    for (int64_t k = threadIdx.x; k < shared * per; k += kThreads) {
      const int64_t b = q + k / per, d = g * per + k % per;
      sum += slope[(b * steps + t) * width + d];
    }
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int s = kThreads / 2; s; s >>= 1) {
      if ((int)threadIdx.x < s) part[threadIdx.x] += part[threadIdx.x + s];
      __syncthreads();
    }
    if (threadIdx.x == 0) out[o] = (G)part[0];
    __syncthreads();
  }
}

unsigned lanes(int64_t n) { return (unsigned)((n + kThreads - 1) / kThreads); }

template <typename T, typename G> void run_scan(const ScanArgs& a) {
  const dim3 grid(lanes(a.batch * a.width)), block(kThreads);
  const hipStream_t s = (hipStream_t)a.stream;
  if (!a.gate) hipLaunchKernelGGL((scan_walk_kernel<T, G, kNoGate>), grid, block, 0, s, a);
  else if (a.groups == a.width) hipLaunchKernelGGL((scan_walk_kernel<T, G, kOwnGate>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((scan_walk_kernel<T, G, kSharedGate>), grid, block, 0, s, a);
  LGA_HIP_CHECK(hipGetLastError());
}

template <typename T, typename G> void run_scan_grad(const ScanGradArgs& a) {
  typedef Wide<T> W;
  const dim3 grid(lanes(a.batch * a.width)), block(kThreads);
  const hipStream_t s = (hipStream_t)a.stream;
  if (!a.gate) hipLaunchKernelGGL((scan_grad_walk_kernel<T, G, kNoGate>), grid, block, 0, s, a);
  else if (a.groups == a.width) hipLaunchKernelGGL((scan_grad_walk_kernel<T, G, kOwnGate>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((scan_grad_walk_kernel<T, G, kSharedGate>), grid, block, 0, s, a);
  LGA_HIP_CHECK(hipGetLastError());
  if (a.gate && a.steps) {
    const int64_t sums = a.gate_batch * a.steps * a.groups;
    hipLaunchKernelGGL((gate_sum_kernel<W, G>), dim3((unsigned)std::min<int64_t>(sums, 1 << 20)), block, 0, s, (const W*)a.work, (G*)a.grad_gate,
                       a.batch, a.steps, a.width, a.groups, a.gate_batch);
    LGA_HIP_CHECK(hipGetLastError());
  }
}

template <typename A> void check_args(const A& a) {
  if (a.batch < 0 || a.steps < 0 || a.width < 0) throw std::runtime_error("gated_scan: a negative size");
  if (a.batch * a.width > 2147483647LL * 64 || a.steps > 2147483647LL) throw std::runtime_error("gated_scan: the tensor is too large");
  if (a.gate && (a.groups <= 0 || a.width % a.groups)) throw std::runtime_error("gated_scan: the width is not a multiple of the gate's groups");
}

// type and gate_type -> template arguments
template <typename F> void by_types(int64_t type, int64_t gate_type, bool gate, F f) {
  if (!gate) gate_type = type;
  if (type == kBf16 && gate_type == kBf16) return f((__bf16)0, (__bf16)0);
  if (type == kBf16 && gate_type == kF32) return f((__bf16)0, (float)0);
  if (type == kF16 && gate_type == kF16) return f((_Float16)0, (_Float16)0);
  if (type == kF16 && gate_type == kF32) return f((_Float16)0, (float)0);
  if (type == kF32 && gate_type == kF32) return f((float)0, (float)0);
  if (type == kF64 && gate_type == kF64) return f((double)0, (double)0);
  throw std::runtime_error("gated_scan: unknown pair of types");
}

}  // namespace

int64_t scan_workspace(const ScanArgs& a) { return 0; }

void gated_scan(const ScanArgs& a) {
  check_args(a);
  if (a.batch * a.width == 0) return;
  DeviceScope scope(a.device);
  by_types(a.type, a.gate_type, a.gate != 0, [&](auto t, auto g) { run_scan<decltype(t), decltype(g)>(a); });
}

int64_t scan_grad_workspace(const ScanGradArgs& a) {
  return a.gate ? a.batch * a.steps * a.width * (a.type == kF64 ? 8 : 4) : 0;
}

void gated_scan_grad(const ScanGradArgs& a) {
  check_args(a);
  if (a.batch * a.width == 0) return;
  DeviceScope scope(a.device);
  by_types(a.type, a.gate_type, a.gate != 0, [&](auto t, auto g) { run_scan_grad<decltype(t), decltype(g)>(a); });
}

}  // namespace lga
