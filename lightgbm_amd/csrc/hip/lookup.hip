// out[i, :] = scale * table[ids[i], :] and its gradient dtable[v, :] = scale * sum over {i : ids[i] = v} of grad[i, :].
// An id outside the table is padding: its row is zero and it takes no gradient.
#include "lookup.hpp"
#include "device.hpp"
#include "seq_types.hpp"
#include <algorithm>

namespace lga {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t load_id(const void* ids, int64_t at, int ids64) {
  return ids64 ? reinterpret_cast<const int64_t*>(ids)[at] : (int64_t)reinterpret_cast<const int32_t*>(ids)[at];
}

// One lane per element of the output, for every width and alignment.
template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_elements_kernel(const T* __restrict__ table, const void* __restrict__ ids, T* __restrict__ out,
                                                                   int64_t rows, int64_t width, int64_t table_stride, int64_t n1, int64_t s0,
                                                                   int64_t s1, int ids64, int64_t total, Wide<T> scale) {
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kThreads) {
    const int64_t token = e / width, col = e - token * width;
    const int64_t i = token / n1, j = token - i * n1;
    const int64_t id = load_id(ids, i * s0 + j * s1, ids64);
    Wide<T> v = 0;
    if (id >= 0 && id < rows) v = (Wide<T>)table[id * table_stride + col] * scale;
    out[e] = (T)v;
  }
}

constexpr int kOwnRows = 8;       // table rows a workgroup owns
constexpr int kListSize = 1024;   // tokens it collects before it adds them up

// A workgroup owns kOwnRows rows of the table and 256 columns: it reads all ids, collects the tokens of its rows in their
// order (ballot compaction) and adds their gradients up in that order, so sums do not depend on timing.
template <typename T, typename O>
__global__ __launch_bounds__(kThreads) void lookup_grad_owned_kernel(const T* __restrict__ grad, const void* __restrict__ ids, O* __restrict__ out,
                                                                     int64_t rows, int64_t width, int64_t tokens, int64_t n1, int64_t s0, int64_t s1,
                                                                     int64_t g0, int64_t g1, int ids64, Wide<T> scale) {
  __shared__ int32_t list_token[kListSize + kThreads];
  __shared__ uint8_t list_row[kListSize + kThreads];
  __shared__ int wave_count[kThreads / 64];
  __shared__ Wide<T> acc[kOwnRows][kThreads];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t first = (int64_t)blockIdx.x * kOwnRows;
  const int64_t col = (int64_t)blockIdx.y * kThreads + t;
  for (int r = 0; r < kOwnRows; ++r) acc[r][t] = 0;
  int filled = 0;     // the same in every lane
  for (int64_t base = 0; base < tokens; base += kThreads) {
    const int64_t token = base + t;
    int64_t row = -1;
    if (token < tokens) {
      const int64_t i = token / n1, j = token - i * n1;
      row = load_id(ids, i * s0 + j * s1, ids64) - first;
      if (row < 0 || row >= kOwnRows || row + first >= rows) row = -1;
    }
    const uint64_t hit = __ballot(row >= 0);
    if (lane == 0) wave_count[wave] = __popcll(hit);
    __syncthreads();
    int before = filled, all = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
      if (w < wave) before += wave_count[w];
      all += wave_count[w];
    }
    if (row >= 0) {
      const int at = before + __popcll(hit & ((1ull << lane) - 1));
      list_token[at] = (int32_t)token;
      list_row[at] = (uint8_t)row;
    }
    filled += all;
    __syncthreads();
    if (filled >= kListSize || base + kThreads >= tokens) {
      if (col < width)
        for (int k = 0; k < filled; ++k) {
          const int64_t tk = list_token[k], i = tk / n1, j = tk - i * n1;
          acc[list_row[k]][t] += (Wide<T>)grad[i * g0 + j * g1 + col];
        }
      filled = 0;
      __syncthreads();
    }
  }
  if (col < width)
    for (int r = 0; r < kOwnRows; ++r)
      if (first + r < rows) out[(first + r) * width + col] = (O)(acc[r][t] * scale);
}

template <typename T> void run_lookup(const LookupArgs& a) {
  const int64_t total = a.n0 * a.n1 * a.width;
  const int blocks = (int)std::min<int64_t>((total + kThreads - 1) / kThreads, 1 << 20);
  hipLaunchKernelGGL(lookup_elements_kernel<T>, dim3(blocks), dim3(kThreads), 0, (hipStream_t)a.stream, (const T*)a.table, (const void*)a.ids,
                     (T*)a.out, a.rows, a.width, a.table_stride, a.n1, a.s0, a.s1, (int)a.ids64, total, (Wide<T>)a.scale);
  LGA_HIP_CHECK(hipGetLastError());
}

template <typename T, typename O> void run_lookup_grad(const LookupGradArgs& a) {
  const dim3 grid((unsigned)((a.rows + kOwnRows - 1) / kOwnRows), (unsigned)((a.width + kThreads - 1) / kThreads));
  hipLaunchKernelGGL((lookup_grad_owned_kernel<T, O>), grid, dim3(kThreads), 0, (hipStream_t)a.stream, (const T*)a.grad, (const void*)a.ids,
                     (O*)a.out, a.rows, a.width, a.n0 * a.n1, a.n1, a.s0, a.s1, a.g0, a.g1, (int)a.ids64, (Wide<T>)a.scale);
  LGA_HIP_CHECK(hipGetLastError());
}

void check_sizes(int64_t rows, int64_t width, int64_t n0, int64_t n1) {
  if (rows < 0 || width < 0 || n0 < 0 || n1 < 0) throw std::runtime_error("embedding: a negative size");
  if (n0 * n1 > 2147483647LL || rows > 2147483646LL) throw std::runtime_error("embedding: 2^31 tokens or rows, or more");
  if (width > (int64_t)kThreads * 65535) throw std::runtime_error("embedding: the rows are too wide");
}

}  // namespace

void lookup(const LookupArgs& a) {
  check_sizes(a.rows, a.width, a.n0, a.n1);
  if (a.n0 * a.n1 == 0 || a.width == 0) return;
  DeviceScope scope(a.device);
  switch (a.type) {
    case kBf16: return run_lookup<__bf16>(a);
    case kF16: return run_lookup<_Float16>(a);
    case kF32: return run_lookup<float>(a);
    case kF64: return run_lookup<double>(a);
    default: throw std::runtime_error("embedding: unknown type");
  }
}

int64_t lookup_grad_workspace(const LookupGradArgs& a) { return 0; }

void lookup_grad(const LookupGradArgs& a) {
  check_sizes(a.rows, a.width, a.n0, a.n1);
  if (a.rows == 0 || a.width == 0) return;
  DeviceScope scope(a.device);
  if (a.type == kBf16 && a.out_type == kBf16) return run_lookup_grad<__bf16, __bf16>(a);
  if (a.type == kBf16 && a.out_type == kF32) return run_lookup_grad<__bf16, float>(a);
  if (a.type == kF16 && a.out_type == kF16) return run_lookup_grad<_Float16, _Float16>(a);
  if (a.type == kF16 && a.out_type == kF32) return run_lookup_grad<_Float16, float>(a);
  if (a.type == kF32 && a.out_type == kF32) return run_lookup_grad<float, float>(a);
  if (a.type == kF64 && a.out_type == kF64) return run_lookup_grad<double, double>(a);
  throw std::runtime_error("embedding_grad: unknown pair of types");
}

}  // namespace lga
