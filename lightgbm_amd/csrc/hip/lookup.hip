// out[i, :] = scale * table[ids[i], :] and its gradient dtable[v, :] = scale * sum over {i : ids[i] = v} of grad[i, :].
// An id outside the table is padding: its row is zero and it takes no gradient.
#include "lookup.hpp"
#include "device.hpp"
#include "seq_types.hpp"
#include "token_sort.hpp"
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

// Sorted path.  The sorted tokens are cut into pieces of equal length.  A run (the tokens of one row) that lies within a
// piece is added up there; of a run that crosses pieces every piece leaves a partial sum - `tail` where the run begins,
// `head` in the pieces behind - which the join adds up in order.
struct Runs {
  const uint32_t* keys;     // sorted ids, `rows` for tokens that take no part
  const void* payload;      // token numbers, or (narrow kernel) the gradients themselves
  int64_t count;            // a multiple of the piece length
  int64_t rows, width, n1, g0, g1;
};
constexpr uint32_t kNobody = ~0u;

__device__ __forceinline__ bool has_tokens(const Runs& r, uint32_t row) {
  int64_t lo = 0, hi = r.count;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (r.keys[mid] < row) lo = mid + 1;
    else hi = mid;
  }
  return lo < r.count && r.keys[lo] == row;
}

constexpr int kZeroRows = 16;      // rows a wave looks after

// Zeros in the rows that no token names.  One wave, kZeroRows rows.
template <typename O> __device__ __forceinline__ void zero_rows(const Runs& r, O* __restrict__ out, int64_t wave, int lane) {
  const int64_t first = wave * kZeroRows;
  if (first >= r.rows) return;
  const bool absent = lane < kZeroRows && first + lane < r.rows && !has_tokens(r, (uint32_t)(first + lane));
  uint64_t todo = __ballot(absent);
  constexpr int kWords = 16 / sizeof(O);
  const bool whole = r.width % kWords == 0;
  while (todo) {
    O* row = out + (first + __ffsll((unsigned long long)todo) - 1) * r.width;
    todo &= todo - 1;
    if (whole) {
      for (int64_t c = (int64_t)lane * kWords; c < r.width; c += 64 * kWords) {
        Pack<O, kWords> z;
        for (int v = 0; v < kWords; ++v) z.v[v] = (O)0.f;
        store_pack<O, kWords>(row + c, z);
      }
    } else {
      for (int64_t c = lane; c < r.width; c += 64) row[c] = (O)0.f;
    }
  }
}

// Rows of more than kNarrow values: `group` lanes walk a piece, V columns a lane.
template <typename T, typename O, int V>
__global__ __launch_bounds__(kThreads) void lookup_grad_runs_kernel(Runs r, const T* __restrict__ grad, O* __restrict__ out, Wide<T>* __restrict__ head,
                                                                    Wide<T>* __restrict__ tail, int zero_blocks, int group, int piece_tokens, Wide<T> scale) {
  typedef Wide<T> W;
  if ((int)blockIdx.x < zero_blocks) {
    if (blockIdx.y == 0) zero_rows(r, out, (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), threadIdx.x & 63);
    return;
  }
  constexpr int kAhead = 8;
  const int64_t piece = ((int64_t)blockIdx.x - zero_blocks) * (kThreads / group) + threadIdx.x / group;
  const int64_t col = ((int64_t)blockIdx.y * group + threadIdx.x % group) * V;
  const int64_t begin = piece * piece_tokens, end = begin + piece_tokens;
  if (begin >= r.count || col >= r.width) return;
  uint32_t cur = r.keys[begin];
  if (cur >= (uint32_t)r.rows) return;
  const uint32_t* token = (const uint32_t*)r.payload;
  bool inside = begin == 0 || r.keys[begin - 1] != cur;
  W acc[V];
  for (int v = 0; v < V; ++v) acc[v] = 0;
  auto close = [&] {
    if (inside) {
      Pack<O, V> o;
      for (int v = 0; v < V; ++v) o.v[v] = (O)(acc[v] * scale);
      store_pack<O, V>(out + (int64_t)cur * r.width + col, o);
    } else {
      for (int v = 0; v < V; ++v) head[piece * r.width + col + v] = acc[v];
    }
  };
  for (int64_t at = begin; at < end; at += kAhead) {
    uint32_t key[kAhead];
    Pack<T, V> g[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) key[u] = r.keys[at + u];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (key[u] < (uint32_t)r.rows) {
        const uint32_t tk = token[at + u], i = tk / (uint32_t)r.n1, j = tk - i * (uint32_t)r.n1;
        g[u] = load_pack<T, V>(grad + i * r.g0 + j * r.g1 + col);
      }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (key[u] != cur) {
        close();
        if (key[u] >= (uint32_t)r.rows) return;
        cur = key[u];
        inside = true;
        for (int v = 0; v < V; ++v) acc[v] = 0;
      }
      for (int v = 0; v < V; ++v) acc[v] += (W)g[u].v[v];
    }
  }
  if (end >= r.count || r.keys[end] != cur) {
    close();
  } else {
    W* part = inside ? tail : head;
    for (int v = 0; v < V; ++v) part[piece * r.width + col + v] = acc[v];
  }
}

constexpr int kNarrow = 16, kNarrowItems = 8, kNarrowPiece = kThreads * kNarrowItems;

// Rows of up to kNarrow values: a workgroup takes a piece, a lane 8 neighbouring tokens; a segmented scan over the lanes
// carries a run's sum on.  kValues: the payload is the gradient itself (rows of one value).
template <typename T, typename O, bool kValues>
__global__ __launch_bounds__(kThreads) void lookup_grad_narrow_kernel(Runs r, const T* __restrict__ grad, O* __restrict__ out, Wide<T>* __restrict__ head,
                                                                      Wide<T>* __restrict__ tail, int zero_blocks, Wide<T> scale) {
  typedef Wide<T> W;
  if ((int)blockIdx.x < zero_blocks) {
    const int64_t row = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (row < r.rows && !has_tokens(r, (uint32_t)row))
      for (int64_t c = 0; c < r.width; ++c) out[row * r.width + c] = (O)0.f;
    return;
  }
  __shared__ W wave_sum[kThreads / 64];
  __shared__ int wave_break[kThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t piece = (int64_t)blockIdx.x - zero_blocks, begin = piece * kNarrowPiece, at = begin + threadIdx.x * kNarrowItems;
  const uint32_t rows = (uint32_t)r.rows;
  if (r.keys[begin] >= rows) return;
  uint32_t key[kNarrowItems + 1];     // [0]: the token before
  key[0] = at ? r.keys[at - 1] : kNobody;
  const Pack<uint32_t, kNarrowItems> here = load_pack<uint32_t, kNarrowItems>(r.keys + at);
#pragma unroll
  for (int u = 0; u < kNarrowItems; ++u) key[u + 1] = here.v[u];
  const uint32_t before_piece = begin ? r.keys[begin - 1] : kNobody;
  const uint32_t behind = begin + kNarrowPiece < r.count ? r.keys[begin + kNarrowPiece] : kNobody;
  Pack<T, kNarrowItems> values;
  Pack<uint32_t, kNarrowItems> tokens;
  if constexpr (kValues) values = load_pack<T, kNarrowItems>((const T*)r.payload + at);
  else tokens = load_pack<uint32_t, kNarrowItems>((const uint32_t*)r.payload + at);
  bool breaks = false;                // a run begins in this lane
#pragma unroll
  for (int u = 0; u < kNarrowItems; ++u) breaks |= key[u] != key[u + 1];
  for (int64_t c = 0; c < r.width; ++c) {
    W v[kNarrowItems], open = 0;      // open: the sum since the last beginning
#pragma unroll
    for (int u = 0; u < kNarrowItems; ++u) {
      v[u] = 0;
      if constexpr (kValues) v[u] = (W)values.v[u];
      else if (key[u + 1] < rows) {
        const uint32_t i = tokens.v[u] / (uint32_t)r.n1, j = tokens.v[u] - i * (uint32_t)r.n1;
        v[u] = (W)grad[i * r.g0 + j * r.g1 + c];
      }
    }
#pragma unroll
    for (int u = 0; u < kNarrowItems; ++u) open = key[u] != key[u + 1] ? v[u] : open + v[u];
    // inclusive segmented scan over the wave, then over the waves
    W sum = open;
    bool broken = breaks;
    for (int d = 1; d < 64; d <<= 1) {
      const W s = __shfl_up(sum, d);
      const bool b = __shfl_up((int)broken, d);
      if (lane >= d) {
        if (!broken) sum = s + sum;
        broken |= b;
      }
    }
    if (lane == 63) wave_sum[wave] = sum, wave_break[wave] = broken;
    W carry = __shfl_up(sum, 1);
    const bool cut = __shfl_up((int)broken, 1);
    __syncthreads();
    W from_waves = 0;
    for (int w = 0; w < wave; ++w) from_waves = wave_break[w] ? wave_sum[w] : from_waves + wave_sum[w];
    if (lane == 0) carry = from_waves;
    else if (!cut) carry = from_waves + carry;
    auto close = [&](uint32_t row, W total) {
      if (row >= rows) return;
      if (row == before_piece) head[piece * r.width + c] = total;
      else out[(int64_t)row * r.width + c] = (O)(total * scale);
    };
#pragma unroll
    for (int u = 0; u < kNarrowItems; ++u) {
      if (key[u] != key[u + 1] && at + u > begin) close(key[u], carry);
      carry = key[u] != key[u + 1] ? v[u] : carry + v[u];
    }
    if (threadIdx.x == kThreads - 1 && key[kNarrowItems] < rows) {
      const uint32_t last = key[kNarrowItems];
      if (last != behind) close(last, carry);
      else (last == before_piece ? head : tail)[piece * r.width + c] = carry;
    }
    __syncthreads();
  }
}

// A workgroup for every piece: if a run begins in it and goes on behind it, its partial sums are added up - 64 columns
// side by side, the chain of pieces in four parts.
template <typename W, typename O>
__global__ __launch_bounds__(kThreads) void lookup_grad_join_kernel(Runs r, O* __restrict__ out, const W* __restrict__ head, const W* __restrict__ tail,
                                                                    int64_t piece_tokens, W scale) {
  const int64_t piece = blockIdx.x, pieces = r.count / piece_tokens, begin = piece * piece_tokens;
  if (piece + 1 >= pieces) return;
  const uint32_t row = r.keys[begin + piece_tokens];
  if (row >= (uint32_t)r.rows || r.keys[begin + piece_tokens - 1] != row || (begin && r.keys[begin - 1] == row)) return;
  // the run covers the beginnings of pieces piece + 1 .. piece + chain
  int64_t chain = 1, step = 1;
  while (piece + chain + step < pieces && r.keys[(piece + chain + step) * piece_tokens] == row) chain += step, step *= 2;
  while (step >= 1) {
    if (piece + chain + step < pieces && r.keys[(piece + chain + step) * piece_tokens] == row) chain += step;
    step /= 2;
  }
  constexpr int kParts = kThreads / 64;
  __shared__ W parts[kParts][64];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
  const int64_t each = (chain + kParts - 1) / kParts, from = part * each, to = min(chain, from + each);
  for (int64_t base = 0; base < r.width; base += 64) {
    const int64_t col = base + lane;
    W sum = 0;
    if (col < r.width) {
      if (part == 0) sum = tail[piece * r.width + col];
      const W* h = head + (piece + 1) * r.width + col;
#pragma unroll 8
      for (int64_t q = from; q < to; ++q) sum += h[q * r.width];
    }
    parts[part][lane] = sum;
    __syncthreads();
    if (part == 0 && col < r.width) {
      for (int k = 1; k < kParts; ++k) sum += parts[k][lane];
      out[(int64_t)row * r.width + col] = (O)(sum * scale);
    }
    __syncthreads();
  }
}

template <typename T> void run_lookup(const LookupArgs& a) {
  const int64_t total = a.n0 * a.n1 * a.width;
  const int blocks = (int)std::min<int64_t>((total + kThreads - 1) / kThreads, 1 << 20);
  hipLaunchKernelGGL(lookup_elements_kernel<T>, dim3(blocks), dim3(kThreads), 0, (hipStream_t)a.stream, (const T*)a.table, (const void*)a.ids,
                     (T*)a.out, a.rows, a.width, a.table_stride, a.n1, a.s0, a.s1, (int)a.ids64, total, (Wide<T>)a.scale);
  LGA_HIP_CHECK(hipGetLastError());
}

// Up to this many tokens every workgroup looks through all ids for its own rows; above, they are sorted.
constexpr int64_t kOwnedTokens = 2048;

struct GradPlan {
  TokenGrid grid;
  int64_t g0, g1;
  int payload, vec, group;
  bool values;
  int64_t piece_tokens, pieces, sort_bytes, parts_bytes;
};

GradPlan plan_grad(const LookupGradArgs& a) {
  const int64_t size = a.type == kF64 ? 8 : a.type == kF32 ? 4 : 2, wide = a.type == kF64 ? 8 : 4;
  GradPlan p;
  p.grid.ids = (const void*)a.ids;
  p.grid.ids64 = (int)a.ids64;
  p.grid.rows = a.rows;
  p.grid.n0 = a.n0, p.grid.n1 = a.n1, p.grid.s0 = a.s0, p.grid.s1 = a.s1;
  p.g0 = a.g0, p.g1 = a.g1;
  if (a.n0 > 1 && a.g1 > a.g0) {      // the axis along which gradients are neighbours runs fastest
    std::swap(p.grid.n0, p.grid.n1);
    std::swap(p.grid.s0, p.grid.s1);
    std::swap(p.g0, p.g1);
  }
  p.values = a.width == 1 && size >= 4;
  p.payload = p.values ? (int)size : 4;
  const TokenTiles tiles = token_tiles(p.grid);
  p.vec = 1;
  p.group = 64;
  if (a.width <= kNarrow) {
    p.piece_tokens = kNarrowPiece;
  } else {
    for (int v = (int)(16 / size); v > 1; v /= 2)
      if (a.width % v == 0 && a.g0 % v == 0 && a.g1 % v == 0 && a.grad % (v * size) == 0) {
        p.vec = v;
        break;
      }
    while (p.group > 8 && p.group / 2 * p.vec >= a.width) p.group /= 2;
    p.piece_tokens = 32;
    while (p.piece_tokens < 1024 && tiles.count / p.piece_tokens > 16384) p.piece_tokens *= 2;
  }
  p.pieces = tiles.count / p.piece_tokens;
  p.sort_bytes = token_sort_workspace(p.grid, p.payload);
  p.parts_bytes = p.pieces * a.width * wide;
  return p;
}

bool owned(const LookupGradArgs& a) { return a.n0 * a.n1 <= kOwnedTokens; }

template <typename T, typename O, int V> void launch_runs(const LookupGradArgs& a, const GradPlan& p, const Runs& r, Wide<T>* head, Wide<T>* tail) {
  const int64_t zero_blocks = (a.rows + kZeroRows * (kThreads / 64) - 1) / (kZeroRows * (kThreads / 64));
  const int64_t run_blocks = (p.pieces * p.group + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(zero_blocks + run_blocks), (unsigned)((a.width + p.group * V - 1) / (p.group * V)));
  hipLaunchKernelGGL((lookup_grad_runs_kernel<T, O, V>), grid, dim3(kThreads), 0, (hipStream_t)a.stream, r, (const T*)a.grad, (O*)a.out, head, tail,
                     (int)zero_blocks, p.group, (int)p.piece_tokens, (Wide<T>)a.scale);
}

template <typename T, typename O> void run_lookup_grad(const LookupGradArgs& a) {
  typedef Wide<T> W;
  const hipStream_t s = (hipStream_t)a.stream;
  if (owned(a)) {
    const dim3 grid((unsigned)((a.rows + kOwnRows - 1) / kOwnRows), (unsigned)((a.width + kThreads - 1) / kThreads));
    hipLaunchKernelGGL((lookup_grad_owned_kernel<T, O>), grid, dim3(kThreads), 0, s, (const T*)a.grad, (const void*)a.ids, (O*)a.out, a.rows, a.width,
                       a.n0 * a.n1, a.n1, a.s0, a.s1, a.g0, a.g1, (int)a.ids64, (W)a.scale);
    LGA_HIP_CHECK(hipGetLastError());
    return;
  }
  const GradPlan p = plan_grad(a);
  const SortedTokens t = token_sort(p.grid, p.values ? (const void*)a.grad : nullptr, p.g0, p.g1, p.payload, (void*)a.work, s);
  const Runs r{t.keys, t.payload, t.count, a.rows, a.width, p.grid.n1, p.g0, p.g1};
  W* head = (W*)((char*)a.work + p.sort_bytes);
  W* tail = (W*)((char*)head + p.parts_bytes);
  if (a.width <= kNarrow) {
    const int zero_blocks = (int)((a.rows + kThreads - 1) / kThreads);
    const dim3 grid((unsigned)(zero_blocks + p.pieces));
    if constexpr (sizeof(T) >= 4) {
      if (p.values)
        hipLaunchKernelGGL((lookup_grad_narrow_kernel<T, O, true>), grid, dim3(kThreads), 0, s, r, (const T*)a.grad, (O*)a.out, head, tail, zero_blocks, (W)a.scale);
    }
    if (!p.values)
      hipLaunchKernelGGL((lookup_grad_narrow_kernel<T, O, false>), grid, dim3(kThreads), 0, s, r, (const T*)a.grad, (O*)a.out, head, tail, zero_blocks, (W)a.scale);
  } else if (p.vec == 1) {
    launch_runs<T, O, 1>(a, p, r, head, tail);
  } else if (p.vec == 2) {
    launch_runs<T, O, 2>(a, p, r, head, tail);
  } else if constexpr (sizeof(T) <= 4) {
    if (p.vec == 4) {
      launch_runs<T, O, 4>(a, p, r, head, tail);
    } else if constexpr (sizeof(T) == 2) {
      launch_runs<T, O, 8>(a, p, r, head, tail);
    }
  }
  LGA_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL((lookup_grad_join_kernel<W, O>), dim3((unsigned)p.pieces), dim3(kThreads), 0, s, r, (O*)a.out, head, tail, p.piece_tokens, (W)a.scale);
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

int64_t lookup_grad_workspace(const LookupGradArgs& a) {
  check_sizes(a.rows, a.width, a.n0, a.n1);
  if (owned(a)) return 0;
  const GradPlan p = plan_grad(a);
  return p.sort_bytes + 2 * p.parts_bytes;
}

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
