// out[i, :] = scale * table[ids[i], :] and its gradient dtable[v, :] = scale * sum over {i : ids[i] = v} of grad[i, :].
// An id outside the table is padding: its row is zero and it takes no gradient.
#include "lookup.hpp"
#include "device.hpp"
#include "seq_types.hpp"
#include "token_sort.hpp"
#include <algorithm>
#include <cmath>

namespace lga {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = 1 << 22;      // a launch has fewer than 2^32 lanes along an axis

__device__ __forceinline__ int64_t load_id(const void* ids, int64_t at, int ids64) {
  return ids64 ? reinterpret_cast<const int64_t*>(ids)[at] : (int64_t)reinterpret_cast<const int32_t*>(ids)[at];
}

// Rows of up to this many values go through a tile of tokens, wider ones are copied and summed by groups of lanes (1 M tokens of
// 70000 rows, tile against groups: 12 bf16 values 22 against 12 us, their gradient 102 against 78; 9 fp32 values 22 against 17 and 109
// against 76; below eight 16-bit values a row is shorter than a pack).
constexpr int kNarrow = 8;

// Rows of more than kNarrow values: `group` lanes copy a row in packs of V, four in flight.  Bound by HBM: 32768 rows of 4096
// bf16 values, 85 us (one lane per value took 366).
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void lookup_rows_kernel(const T* __restrict__ table, const void* __restrict__ ids, T* __restrict__ out,
                                                               int64_t rows, int64_t width, int64_t table_stride, int64_t n1, int64_t s0,
                                                               int64_t s1, int ids64, int64_t tokens, int group, Wide<T> scale) {
  typedef Wide<T> W;
  for (int64_t token = (int64_t)blockIdx.x * (kThreads / group) + threadIdx.x / group; token < tokens; token += (int64_t)gridDim.x * (kThreads / group)) {
    const uint32_t i = (uint32_t)token / (uint32_t)n1, j = (uint32_t)token - i * (uint32_t)n1;
    const int64_t id = load_id(ids, i * s0 + j * s1, ids64);
    const bool named = id >= 0 && id < rows;
    const T* from = table + (named ? id * table_stride : 0);
    T* to = out + token * width;
    const int packs = (int)((width + V - 1) / V), end = (int)(width - V);
    int c = threadIdx.x % group;
    constexpr int kAhead = 4;
    for (; c + (kAhead - 1) * group < packs; c += kAhead * group) {
      Pack<T, V> x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (named) x[u] = load_pack<T, V>(from + min((c + u * group) * V, end));
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        for (int v = 0; v < V; ++v) x[u].v[v] = named ? (T)((W)x[u].v[v] * scale) : (T)(W)0;
        store_pack<T, V>(to + min((c + u * group) * V, end), x[u]);
      }
    }
    for (; c < packs; c += group) {
      Pack<T, V> x;
      if (named) x = load_pack<T, V>(from + min(c * V, end));
      for (int v = 0; v < V; ++v) x.v[v] = named ? (T)((W)x.v[v] * scale) : (T)(W)0;
      store_pack<T, V>(to + min(c * V, end), x);
    }
  }
}

// Narrow rows: a workgroup takes a tile of tokens, reads its ids along the axis on which they are neighbours, and writes
// along the axis on which the results are.  300 trees x 45800 rows of one fp64 value, ids by row: 57 us (2.9 TB/s; what bounds it has
// not been taken apart: ids come in pieces of 256 bytes, and a tile gathers from 64 trees' values), 198 us with one lane per value.
template <typename T, typename I, int kBits>
__global__ __launch_bounds__(kThreads) void lookup_tile_kernel(const T* __restrict__ table, const I* __restrict__ ids, T* __restrict__ out, int64_t rows,
                                                               int width, int64_t table_stride, TokenGrid grid, TokenTiles tiles, Wide<T> scale) {
  constexpr int kSize = 1 << kBits, kItems = kSize / kThreads;
  __shared__ int32_t id_of[kSize];
  const int shift1 = tiles.shift1, side1 = 1 << shift1, shift0 = kBits - shift1;
  const int64_t ti = blockIdx.x / tiles.across, i0 = ti << shift0, j0 = (blockIdx.x - ti * tiles.across) << shift1;
  const bool along0 = grid.s0 < grid.s1;
  const int live1 = (int)min((int64_t)side1, grid.n1 - j0), live0 = (int)min((int64_t)1 << shift0, grid.n0 - i0);
  // A lane's items are kThreads apart, which is a fixed way in both walks unless an axis is longer than that and not all.
  const bool whole = live0 == 1 << shift0 && live1 == side1 && (shift1 <= 8 || shift1 == kBits) && (!along0 || shift0 <= 8);
  const int t = threadIdx.x;
  if (whole) {
    const int i = along0 ? t & ((1 << shift0) - 1) : t >> shift1, j = along0 ? t >> shift0 : t & (side1 - 1);
    const int64_t next = along0 ? (int64_t)(kThreads >> shift0) * grid.s1 : shift1 <= 8 ? (int64_t)(kThreads >> shift1) * grid.s0 : kThreads * grid.s1;
    const I* from = ids + (i0 + i) * grid.s0 + (j0 + j) * grid.s1;
    I id[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) id[k] = from[k * next];
    int at = i << shift1 | j;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      id_of[tile_slot(at)] = id[k] >= 0 && id[k] < rows ? (int32_t)id[k] : -1;
      at += along0 ? kThreads >> shift0 : kThreads;
    }
  } else {
    for (int n = t; n < kSize; n += kThreads) {
      const int i = along0 ? n & ((1 << shift0) - 1) : n >> shift1, j = along0 ? n >> shift0 : n & (side1 - 1);
      int32_t id = -1;
      if (i < live0 && j < live1) {
        const I v = ids[(i0 + i) * grid.s0 + (j0 + j) * grid.s1];
        if (v >= 0 && v < rows) id = (int32_t)v;
      }
      id_of[tile_slot(i << shift1 | j)] = id;
    }
  }
  __syncthreads();
  auto value = [&](int32_t id, int col) { return id >= 0 ? (T)((Wide<T>)table[id * table_stride + col] * scale) : (T)(Wide<T>)0; };
  if (width == 1) {
    if (whole) {
      T* to = out + (i0 + (t >> shift1)) * grid.n1 + j0 + (t & (side1 - 1));
      const int64_t next = shift1 <= 8 ? (int64_t)(kThreads >> shift1) * grid.n1 : kThreads;
      T v[kItems];
#pragma unroll
      for (int k = 0; k < kItems; ++k) v[k] = value(id_of[tile_slot(t + k * kThreads)], 0);
#pragma unroll
      for (int k = 0; k < kItems; ++k) to[k * next] = v[k];
      return;
    }
    for (int n = t; n < kSize; n += kThreads) {
      const int i = n >> shift1, j = n & (side1 - 1);
      if (i < live0 && j < live1) out[(i0 + i) * grid.n1 + j0 + j] = value(id_of[tile_slot(n)], 0);
    }
    return;
  }
  // divisions by multiplication: exact, as no n times its divisor reaches 2^32
  const uint32_t line = live1 * width, total = live0 * line, by_line = (uint32_t)((1ull << 32) / line + 1), by_width = (uint32_t)((1ull << 32) / width + 1);
#pragma unroll 4
  for (uint32_t n = t; n < total; n += kThreads) {
    const uint32_t i = __umulhi(n, by_line), e = n - i * line, j = __umulhi(e, by_width);
    out[((i0 + i) * grid.n1 + j0) * width + e] = value(id_of[tile_slot(i << shift1 | j)], e - j * width);
  }
}

constexpr int kOwnRows = 8;       // table rows a workgroup owns
constexpr int kListSize = 1024;   // tokens it collects before it adds them up
constexpr int kAhead = 16;        // gradients loaded before they are added

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
        for (int k = 0; k < filled; k += kAhead) {
          T g[kAhead];
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const uint32_t tk = list_token[min(k + u, filled - 1)], i = tk / (uint32_t)n1, j = tk - i * (uint32_t)n1;
            g[u] = grad[i * g0 + j * g1 + col];
          }
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
            if (k + u < filled) acc[list_row[k + u]][t] += (Wide<T>)g[u];
        }
      filled = 0;
      __syncthreads();
    }
  }
  if (col < width)
    for (int r = 0; r < kOwnRows; ++r)
      if (first + r < rows) out[(first + r) * width + col] = (O)(acc[r][t] * scale);
}

// Few rows, many tokens: every wave keeps sums of one column of the table in LDS and adds its tokens to them, kGroup x 64 at a
// time; the waves' sums are added up in order afterwards.  LDS accesses of one wave run in their order, so the additions
// have a fixed order as long as no two lanes touch one row at a time:  tag[row] = lane, read back, tells whether lanes share
// a row (whichever of two lanes is read back, the other one sees it); if so, they find each other with ballots and
// take turns.  LDS float atomics would need no reading back, but take about 200 cycles for 64 lanes: 130 us for the 13.7 M
// tokens of 300 trees x 45800 rows, where this takes 63 us (a third of it waits for loads: LDS holds three waves a CU).
constexpr int kPrivateItems = 32;     // tokens a lane holds
constexpr int kGroup = 4;             // of which so many are added at a time

// A step: 64 x kPrivateItems tokens; lanes along axis 0, items along axis 1 or (few tokens there) along axis 0 too.  A step
// is loaded while the one before is added up.  Every step runs the same straight code, which a wave of few steps mostly waits
// for: places behind an edge are read at the edge and take no part.  kWhole: gradients of one value that are neighbours along
// axis 1.
template <typename T, typename I, bool kAlong0, bool kWhole>
__global__ __launch_bounds__(64) void lookup_grad_private_kernel(const T* __restrict__ grad, TokenGrid grid, int64_t g0, int64_t g1, int width, int row_bits,
                                                                 int lines, int steps, int each, Wide<T>* __restrict__ parts) {
  grad += blockIdx.y;                 // the wave's column
  typedef Wide<T> W;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  W* sums = (W*)lds;                  // one row more than the table has: tokens that take no part
  const int rows = (int)grid.rows, lane = threadIdx.x;
  uint8_t* tag = (uint8_t*)(sums + rows + 1);
  for (int k = lane; k <= rows; k += 64) sums[k] = 0;
  __syncthreads();
  constexpr int item_i = kAlong0 ? 64 : 0, item_j = kAlong0 ? 0 : 1;
  const I* ids = (const I*)grid.ids;
  // Where a step's items begin; its first `again` items belong to the step before (the last step of a line is moved back).
  auto place = [&](int step, int64_t& i0, int64_t& j0, int& again) {
    const int si = step / lines, line = step - si * lines;
    i0 = (int64_t)si * 64 * (kAlong0 ? kPrivateItems : 1) + lane;
    j0 = (int64_t)line * (kAlong0 ? 1 : kPrivateItems);
    again = 0;
    if constexpr (!kAlong0) {
      again = (int)max((int64_t)0, j0 + kPrivateItems - grid.n1);
      j0 -= again;
    }
  };
  int32_t row[kPrivateItems];
  I next_id[kPrivateItems];
  T g[kPrivateItems], next_g[kPrivateItems];
  const int first = blockIdx.x * each, end = min(steps, first + each);
  for (int ahead = first; ahead <= end; ++ahead) {      // the step that is loaded; the one before is added up
    const int step = ahead - 1;
    int64_t i0 = 0, j0 = 0;
    int again = 0;
    if (step >= first) {
      place(step, i0, j0, again);
#pragma unroll
      for (int u = 0; u < kPrivateItems; ++u) {
        const int limit = i0 + u * item_i < grid.n0 && u >= again ? rows : 0;
        row[u] = next_id[u] >= 0 && next_id[u] < limit ? (int32_t)next_id[u] : rows;
        g[u] = next_g[u];
      }
    }
    if (ahead < end) {
      int64_t i, j;
      int skip;
      place(ahead, i, j, skip);
      if constexpr (kAlong0) {
#pragma unroll
        for (int u = 0; u < kPrivateItems; ++u) {
          const int64_t at = min(i + u * 64, grid.n0 - 1);
          next_id[u] = ids[at * grid.s0 + j * grid.s1];
          next_g[u] = grad[at * g0 + j * g1];
        }
      } else {
        i = min(i, grid.n0 - 1);
        const I* at = ids + i * grid.s0 + j * grid.s1;
        const T* from = grad + i * g0 + j * g1;
#pragma unroll
        for (int u = 0; u < kPrivateItems; ++u) next_id[u] = at[u * grid.s1];
        if constexpr (kWhole) {
          constexpr int V = 16 / sizeof(T);
#pragma unroll
          for (int u = 0; u < kPrivateItems; u += V) {
            const Pack<T, V> x = load_pack<T, V>(from + u);
#pragma unroll
            for (int v = 0; v < V; ++v) next_g[u + v] = x.v[v];
          }
        } else {
#pragma unroll
          for (int u = 0; u < kPrivateItems; ++u) next_g[u] = from[u * g1];
        }
      }
    }
    if (step < first) continue;
    uint32_t meets = 0;               // groups of items in which lanes share a row: later, read once more
#pragma unroll
    for (int u0 = 0; u0 < kPrivateItems; u0 += kGroup) {
      uint8_t seen[kGroup];
      W sum[kGroup];
#pragma unroll
      for (int k = 0; k < kGroup; ++k) tag[row[u0 + k]] = (uint8_t)lane;
      in_order();
#pragma unroll
      for (int k = 0; k < kGroup; ++k) seen[k] = tag[row[u0 + k]];
#pragma unroll
      for (int k = 0; k < kGroup; ++k) sum[k] = sums[row[u0 + k]];
      bool other = false;
#pragma unroll
      for (int k = 0; k < kGroup; ++k) other |= row[u0 + k] < rows && seen[k] != (uint8_t)lane;
      if (__any(other)) {
        meets |= 1u << u0;
      } else {
        // a lane's own items of one row follow each other in registers; the last one is stored last
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
#pragma unroll
          for (int e = 0; e < k; ++e) sum[k] = row[u0 + e] == row[u0 + k] ? sum[e] : sum[k];
          sum[k] += (W)g[u0 + k];
        }
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
          sums[row[u0 + k]] = sum[k];
          in_order();
        }
      }
      in_order();
    }
    for (; meets; meets &= meets - 1) {
      const int u0 = __ffs(meets) - 1;
      for (int u = u0; u < u0 + kGroup; ++u) {
        const int64_t i = i0 + u * item_i, j = j0 + u * item_j;
        const bool there = i < grid.n0 && u >= again;
        const I id = there ? ids[i * grid.s0 + j * grid.s1] : (I)-1;
        const W value = there ? (W)grad[i * g0 + j * g1] : (W)0;
        const int at = id >= 0 && id < rows ? (int)id : rows;
        uint64_t same = ~0ull;
        for (int bit = 0; bit < row_bits; ++bit) {
          const bool one = at >> bit & 1;
          const uint64_t ones = __ballot(one);
          same &= one ? ones : ~ones;
        }
        const int turn = at < rows ? __popcll(same & ((1ull << lane) - 1)) : -1;
        for (int k = 0; __any(turn >= k); ++k) {
          if (turn == k) sums[at] += value;
          in_order();
        }
      }
    }
    in_order();
  }
  __syncthreads();
  for (int k = lane; k < rows; k += 64) parts[((int64_t)blockIdx.x * rows + k) * width + blockIdx.y] = sums[k];
}

// out = scale * the waves' sums, 64 values side by side, the waves in kTotalThreads / 64 parts.
constexpr int kTotalThreads = 1024;

template <typename W, typename O>
__global__ __launch_bounds__(kTotalThreads) void lookup_grad_total_kernel(const W* __restrict__ parts, O* __restrict__ out, int64_t values, int waves, W scale) {
  constexpr int kParts = kTotalThreads / 64;
  __shared__ W of_part[kParts][64];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
  const int64_t at = (int64_t)blockIdx.x * 64 + lane;
  const int each = (waves + kParts - 1) / kParts, from = part * each, to = min(waves, from + each);
  W sum = 0;
  if (at < values) {
#pragma unroll 16
    for (int w = from; w < to; ++w) sum += parts[(int64_t)w * values + at];
  }
  of_part[part][lane] = sum;
  __syncthreads();
  if (part == 0 && at < values) {
    for (int k = 1; k < kParts; ++k) sum += of_part[k][lane];
    out[at] = (O)(sum * scale);
  }
}

// Sorted path.  The sorted tokens are cut into pieces of equal length.  A run (the tokens of one row) that lies within a
// piece is added up there; of a run that crosses pieces every piece leaves a partial sum - `tail` where the run begins,
// `head` in the pieces behind - which the join adds up in order.
struct Runs {
  const uint32_t* keys;     // sorted ids, `rows` for tokens that take no part
  const void* payload;      // token numbers, or (narrow kernel) the gradients themselves
  const uint8_t* named;     // [rows]
  int64_t count;            // a multiple of the piece length
  int64_t rows, width, n1, g0, g1;
};
constexpr uint32_t kNobody = ~0u;

constexpr int kZeroRows = 16;      // rows a wave looks after

// Zeros in the rows that no token names.  One wave, kZeroRows rows.
template <typename O> __device__ __forceinline__ void zero_rows(const Runs& r, O* __restrict__ out, int64_t wave, int lane) {
  const int64_t first = wave * kZeroRows;
  if (first >= r.rows) return;
  const bool absent = lane < kZeroRows && first + lane < r.rows && !r.named[first + lane];
  uint64_t todo = __ballot(absent);
  constexpr int kWords = 16 / sizeof(O);
  while (todo) {
    O* row = out + (first + __ffsll((unsigned long long)todo) - 1) * r.width;
    todo &= todo - 1;
    for (int64_t c = (int64_t)lane * kWords; c < r.width; c += 64 * kWords) {
      Pack<O, kWords> z;
      for (int v = 0; v < kWords; ++v) z.v[v] = (O)0.f;
      store_pack<O, kWords>(row + min(c, r.width - kWords), z);
    }
  }
}

// Rows of more than kNarrow values: `group` lanes walk a strip of `length` tokens, V columns a lane; the strips of a workgroup
// are a piece, and what crosses strips is joined in LDS.  65537 tokens of 1024 bf16 values in 50000 rows: 49 us for the 237 MB of
// gradients, sums and zeros (4.8 TB/s).
constexpr int kRunThreads = 512, kStage = 32;     // ids and tokens of a strip wait in LDS, kStage at a time
enum { kHasHead = 1, kThrough = 2, kHasTail = 4 };      // of a strip: ends / passes on the run it begins in, begins the run it ends in

template <typename T, typename O, int V>
__global__ __launch_bounds__(kRunThreads) void lookup_grad_runs_kernel(Runs r, const T* __restrict__ grad, O* __restrict__ out, Wide<T>* __restrict__ head,
                                                                       Wide<T>* __restrict__ tail, int zero_blocks, int group, int length, Wide<T> scale) {
  typedef Wide<T> W;
  if ((int)blockIdx.x < zero_blocks) {
    if (blockIdx.y == 0)
      for (int64_t wave = (int64_t)blockIdx.x * (kRunThreads / 64) + (threadIdx.x >> 6); wave * kZeroRows < r.rows; wave += (int64_t)zero_blocks * (kRunThreads / 64))
        zero_rows(r, out, wave, threadIdx.x & 63);
    return;
  }
  constexpr int kAhead = 4;
  __shared__ W shead[kRunThreads * V], stail[kRunThreads * V];
  __shared__ uint32_t skey[kRunThreads / 8 * kStage], stoken[kRunThreads / 8 * kStage];
  __shared__ int flags[kRunThreads / 8];
  const int strips = kRunThreads / group, strip = threadIdx.x / group, lane = threadIdx.x % group;
  const int64_t piece = (int64_t)blockIdx.x - zero_blocks;
  const int64_t pack = ((int64_t)blockIdx.y * group + lane) * V, col = min(pack, r.width - V);
  const int64_t begin = (piece * strips + strip) * length, end = begin + length;      // lengths divide kSortTile
  const uint32_t rows = (uint32_t)r.rows, *token = (const uint32_t*)r.payload;
  const bool live = pack < r.width;
  uint32_t cur = begin < r.count ? r.keys[begin] : rows;
  int flag = 0;
  auto write = [&](uint32_t row, const W (&sum)[V]) {
    Pack<O, V> o;
    for (int v = 0; v < V; ++v) o.v[v] = (O)(sum[v] * scale);
    store_pack<O, V>(out + (int64_t)row * r.width + col, o);
  };
  if (cur < rows) {
    const uint32_t ahead = begin ? r.keys[begin - 1] : kNobody, behind = end < r.count ? r.keys[end] : kNobody;
    bool inside = ahead != cur;
    W acc[V];
    for (int v = 0; v < V; ++v) acc[v] = 0;
    auto close = [&] {
      if (!inside) {
        flag |= kHasHead;
        for (int v = 0; v < V; ++v) shead[threadIdx.x * V + v] = acc[v];
      } else if (live) {
        write(cur, acc);
      }
    };
    uint32_t *keys = skey + strip * kStage, *tokens = stoken + strip * kStage;
    const int stage = min(kStage, length);
    for (int64_t at = begin; at < end && cur < rows; at += stage) {
      in_order();                     // the strip's lanes are of one wave
      for (int n = lane; n < stage; n += group) {
        keys[n] = r.keys[at + n];
        tokens[n] = token[at + n];
      }
      in_order();
#pragma unroll 1
      for (int from = 0; from < stage && cur < rows; from += kAhead) {
        uint32_t key[kAhead];
        Pack<T, V> g[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          key[u] = keys[from + u];
          if (key[u] < rows && live) {
            const uint32_t tk = tokens[from + u], i = tk / (uint32_t)r.n1, j = tk - i * (uint32_t)r.n1;
            g[u] = load_pack<T, V>(grad + i * r.g0 + j * r.g1 + col);
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (key[u] != cur) {
            if (cur < rows) close();
            cur = key[u];
            inside = true;
            for (int v = 0; v < V; ++v) acc[v] = 0;
          }
          if (cur < rows)
            for (int v = 0; v < V; ++v) acc[v] += (W)g[u].v[v];
        }
      }
    }
    if (cur < rows) {
      if (behind != cur) {
        close();
      } else {
        flag |= inside ? kHasTail : kHasHead | kThrough;
        W* part = inside ? stail : shead;
        for (int v = 0; v < V; ++v) part[threadIdx.x * V + v] = acc[v];
      }
    }
  }
  if (lane == 0) flags[strip] = flag;
  __syncthreads();
  if (!live) return;
  // the run that begins in this strip and goes on, or (first strip) the one that the piece begins in
  const bool first = strip == 0 && (flag & kHasHead);
  for (int from_before = first ? 1 : 0; from_before >= 0; --from_before) {
    if (!from_before && !(flag & kHasTail)) continue;
    W sum[V];
    for (int v = 0; v < V; ++v) sum[v] = (from_before ? shead : stail)[threadIdx.x * V + v];
    bool open = from_before ? (flag & kThrough) != 0 : true;
    int q = strip;
    while (open && q + 1 < strips) {
      ++q;
      for (int v = 0; v < V; ++v) sum[v] += shead[(q * group + lane) * V + v];
      open = (flags[q] & kThrough) != 0;
    }
    if (!open && !from_before) write(cur, sum);
    else
      for (int v = 0; v < V; ++v) (from_before ? head : tail)[piece * r.width + col + v] = sum[v];
  }
}

constexpr int kNarrowItems = 8, kNarrowPiece = kThreads * kNarrowItems;

// Rows of up to kNarrow values: a workgroup takes a piece, a lane 8 neighbouring tokens; a segmented scan over the lanes
// carries a run's sum on.  kValues: the payload is the gradient itself (rows of one value).
template <typename T, typename O, bool kValues, int C>
__global__ __launch_bounds__(kThreads) void lookup_grad_narrow_kernel(Runs r, const T* __restrict__ grad, O* __restrict__ out, Wide<T>* __restrict__ head,
                                                                      Wide<T>* __restrict__ tail, int zero_blocks, Wide<T> scale) {
  typedef Wide<T> W;
  if ((int)blockIdx.x < zero_blocks) {
    const int64_t row = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (row < r.rows && !r.named[row])
      for (int64_t c = 0; c < r.width; ++c) out[row * r.width + c] = (O)0.f;
    return;
  }
  __shared__ W wave_sum[kThreads / 64][C];
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
  const T* from[kNarrowItems];
#pragma unroll
  for (int u = 0; u < kNarrowItems; ++u) {
    from[u] = grad;
    if constexpr (!kValues) {
      const uint32_t tk = key[u + 1] < rows ? tokens.v[u] : 0, i = tk / (uint32_t)r.n1, j = tk - i * (uint32_t)r.n1;
      from[u] = grad + i * r.g0 + j * r.g1;
    }
  }
  // C columns at a time; the last ones may be some of those before once more, with the same sums
  for (int64_t base = 0; base < r.width; base += C) {
    const int64_t c0 = min(base, r.width - C);
    Pack<T, C> x[kNarrowItems];
    if constexpr (!kValues) {
#pragma unroll
      for (int u = 0; u < kNarrowItems; ++u) x[u] = load_pack<T, C>(from[u] + c0);
    }
    auto value = [&](int u, int e) -> W {
      if constexpr (kValues) return (W)values.v[u];
      else return key[u + 1] < rows ? (W)x[u].v[e] : (W)0;
    };
    W carry[C];
    bool broken = breaks;
#pragma unroll
    for (int e = 0; e < C; ++e) {     // the sum since the lane's last beginning
      carry[e] = 0;
#pragma unroll
      for (int u = 0; u < kNarrowItems; ++u) carry[e] = key[u] != key[u + 1] ? value(u, e) : carry[e] + value(u, e);
    }
    // inclusive segmented scan over the wave, then over the waves
    for (int d = 1; d < 64; d <<= 1) {
      const bool b = __shfl_up((int)broken, d);
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const W s = __shfl_up(carry[e], d);
        if (lane >= d && !broken) carry[e] = s + carry[e];
      }
      if (lane >= d) broken |= b;
    }
    if (lane == 63) {
      for (int e = 0; e < C; ++e) wave_sum[wave][e] = carry[e];
      wave_break[wave] = broken;
    }
    const bool cut = __shfl_up((int)broken, 1);
#pragma unroll
    for (int e = 0; e < C; ++e) carry[e] = __shfl_up(carry[e], 1);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < C; ++e) {
      const int64_t c = c0 + e;
      W from_waves = 0;
      for (int w = 0; w < wave; ++w) from_waves = wave_break[w] ? wave_sum[w][e] : from_waves + wave_sum[w][e];
      W sum = lane == 0 ? from_waves : cut ? carry[e] : from_waves + carry[e];
      auto close = [&](uint32_t row, W total) {
        if (row >= rows) return;
        if (row == before_piece) head[piece * r.width + c] = total;
        else out[(int64_t)row * r.width + c] = (O)(total * scale);
      };
#pragma unroll
      for (int u = 0; u < kNarrowItems; ++u) {
        if (key[u] != key[u + 1] && at + u > begin) close(key[u], sum);
        sum = key[u] != key[u + 1] ? value(u, e) : sum + value(u, e);
      }
      if (threadIdx.x == kThreads - 1 && key[kNarrowItems] < rows) {
        const uint32_t last = key[kNarrowItems];
        if (last != behind) close(last, sum);
        else (last == before_piece ? head : tail)[piece * r.width + c] = sum;
      }
    }
    __syncthreads();
  }
}

// A workgroup for every piece: if a run begins in it and goes on behind it, its partial sums are added up - 64 columns
// side by side, the chain of pieces in four parts.
template <typename W, typename O>
__global__ __launch_bounds__(kThreads) void lookup_grad_join_kernel(Runs r, O* __restrict__ out, const W* __restrict__ head, const W* __restrict__ tail,
                                                                    int64_t piece_tokens, W scale) {
  const int64_t piece = blockIdx.x, pieces = (r.count + piece_tokens - 1) / piece_tokens, begin = piece * piece_tokens;
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
  for (int64_t base = (int64_t)blockIdx.y * 64; base < r.width; base += (int64_t)gridDim.y * 64) {
    const int64_t col = base + lane;
    W sum = 0;
    if (col < r.width) {
      if (part == 0) sum = tail[piece * r.width + col];
      const W* h = head + (piece + 1) * r.width + col;
#pragma unroll 16
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

// Elements of a row a lane loads at a time.
template <typename T> constexpr int kPack = 16 / sizeof(T);

template <typename T> void run_lookup(const LookupArgs& a) {
  const int64_t tokens = a.n0 * a.n1;
  if (a.width <= kNarrow) {
    TokenGrid grid;
    grid.ids64 = (int)a.ids64;
    grid.n0 = a.n0, grid.n1 = a.n1, grid.s0 = a.s0, grid.s1 = a.s1;
    grid.rows = a.rows;
    // Small tiles until there are enough for every CU: 300 trees of fp64 leaf values, tiles of 1024 against 4096: 10000 rows (3125 small
    // tiles) 13.6 against 17.7 us, 20000 rows (6250) 27 against 29, 45800 rows (14315) 70 against 58; 100 trees x 45800 rows of three fp32
    // values (5728) 32 against 31.
    TokenTiles tiles = token_tiles(grid, 10);
    if (tiles.blocks > 4096) tiles = token_tiles(grid);
    auto run = [&](auto kernel, auto* ids) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)tiles.blocks), dim3(kThreads), 0, (hipStream_t)a.stream, (const T*)a.table, ids, (T*)a.out, a.rows,
                         (int)a.width, a.table_stride, grid, tiles, (Wide<T>)a.scale);
    };
    auto by_ids = [&](auto* ids) {
      typedef std::remove_const_t<std::remove_pointer_t<decltype(ids)>> I;
      tiles.bits == 10 ? run(lookup_tile_kernel<T, I, 10>, ids) : run(lookup_tile_kernel<T, I, 12>, ids);
    };
    a.ids64 ? by_ids((const int64_t*)a.ids) : by_ids((const int32_t*)a.ids);
  } else {
    constexpr int V = kPack<T>;
    int group = 64;
    while (group > 1 && group / 2 * V >= a.width) group /= 2;
    hipLaunchKernelGGL((lookup_rows_kernel<T, V>), dim3((unsigned)std::min<int64_t>((tokens * group + kThreads - 1) / kThreads, kMaxBlocks)), dim3(kThreads), 0,
                       (hipStream_t)a.stream, (const T*)a.table, (const void*)a.ids, (T*)a.out, a.rows, a.width, a.table_stride, a.n1, a.s0, a.s1,
                       (int)a.ids64, tokens, group,
                       (Wide<T>)a.scale);
  }
  LGA_HIP_CHECK(hipGetLastError());
}

// Up to this many tokens every workgroup looks through all ids for its own rows; above, or for tables of more rows, they are sorted
// (256 tokens, 8192 rows of 512 fp32 values: 11 against 23 us; 512 tokens: 8192 x 512 13 against 23, 131072 x 512 53 against 69,
// 100000 x 3 19 against 20, but 32000 x 4096 148 against 131; 1024 tokens: 131072 x 512 78 against 70, 8192 x 512 16 against 24).
constexpr int64_t kOwnedTokens = 512, kOwnedTable = 131072;
// Sums in a wave's LDS where the table fits and tokens outnumber its rows.  That is a bet on leaf tokens, whose lanes meet seldom:
// against sorting, 13 M of them in 300 trees of 31 leaves 61 against 289 us (fp32), 1 M 31 against 48, 100 trees of 127 leaves 86 against
// 339; but 3 trees, whose lanes are mostly idle, 296 against 199, and ids drawn from the whole table, where lanes meet in most
// groups, 14 M of 3000 rows 164 against 280, of 9300 rows 324 against 296, of 18000 rows 745 against 300.  Wider rows than
// narrow ones are not worth it: 3 M leaf tokens (100 trees of 31 leaves) of 8 fp32 values 122 against 173 us, of 9 values 234 against 169.
constexpr int64_t kPrivateLds = 160 * 1024, kPrivateRatio = 16;

struct GradPlan {
  TokenGrid grid;
  int64_t g0, g1;
  int payload, vec, group, strip = 32;
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
  const TokenTiles tiles = sort_tiles(p.grid);
  p.vec = 1;
  p.group = 64;
  if (a.width <= kNarrow) {
    p.piece_tokens = kNarrowPiece;
  } else {
    p.vec = (int)(16 / size);
    while (p.group > 8 && p.group / 2 * p.vec >= a.width) p.group /= 2;
    // shorter strips where there are few: 901 tokens of 3154 fp16 values 17 us with 16, 25 us with 32; 65537 of 1024 bf16
    // values 51 us with 16, 49 us with 32
    p.strip = tiles.count <= 16384 ? 16 : 32;
    while (p.strip < 256 && tiles.count / p.strip > 32768) p.strip *= 2;
    p.piece_tokens = (int64_t)p.strip * (kRunThreads / p.group);
  }
  p.pieces = (tiles.count + p.piece_tokens - 1) / p.piece_tokens;
  p.sort_bytes = token_sort_workspace(p.grid, p.payload);
  p.parts_bytes = p.pieces * a.width * wide;
  return p;
}

bool owned(const LookupGradArgs& a) { return a.n0 * a.n1 <= kOwnedTokens && a.rows <= kOwnedTable; }

// Few rows and many tokens: sums of a column of the table in a wave's share of LDS.
struct PrivatePlan {
  TokenGrid grid;
  int64_t g0, g1, lines, steps;
  int items_along0, waves = 0, lds = 0;      // waves 0: not this way
  bool whole = false;
};

PrivatePlan plan_private(const LookupGradArgs& a) {
  PrivatePlan p;
  const int64_t wide = a.type == kF64 ? 8 : 4, tokens = a.n0 * a.n1, lds = (a.rows + 1) * (wide + 1);
  if (a.width > kNarrow || lds > kPrivateLds || tokens < kPrivateRatio * a.rows) return p;
  p.grid.ids = (const void*)a.ids;
  p.grid.ids64 = (int)a.ids64;
  p.grid.rows = a.rows;
  p.grid.n0 = a.n0, p.grid.n1 = a.n1, p.grid.s0 = a.s0, p.grid.s1 = a.s1;
  p.g0 = a.g0, p.g1 = a.g1;
  if (a.n1 > 1 && (a.n0 == 1 || a.s1 < a.s0)) {      // lanes along the axis on which ids are neighbours
    std::swap(p.grid.n0, p.grid.n1);
    std::swap(p.grid.s0, p.grid.s1);
    std::swap(p.g0, p.g1);
  }
  p.items_along0 = p.grid.n1 < kPrivateItems;
  p.lines = p.items_along0 ? p.grid.n1 : (p.grid.n1 + kPrivateItems - 1) / kPrivateItems;
  const int64_t side0 = p.items_along0 ? 64 * kPrivateItems : 64;
  p.steps = (p.grid.n0 + side0 - 1) / side0 * p.lines;
  p.whole = !p.items_along0 && a.width == 1 && p.g1 == 1;
  p.lds = (int)((lds + 15) / 16 * 16);
  const int64_t fit = 256 * std::min<int64_t>(8, std::max<int64_t>(1, 163840 / p.lds));
  // as many tokens a wave as the table has rows, so that the waves' sums are no more than the tokens; fewer where that
  // would leave CUs idle (557 k tokens of 3 values, 23478 rows: 69 waves 88 us, 255 waves 56 us)
  const int64_t chunks = std::max(tokens / std::max<int64_t>(1024, a.rows), std::min(256 / a.width, tokens / std::max<int64_t>(1024, a.rows / 4)));
  p.waves = (int)std::max<int64_t>(1, std::min({fit / a.width, p.steps, chunks}));
  return p;
}

template <typename T, typename O, int V> void launch_runs(const LookupGradArgs& a, const GradPlan& p, const Runs& r, Wide<T>* head, Wide<T>* tail) {
  const int64_t zero_blocks = std::min((a.rows + kZeroRows * (kRunThreads / 64) - 1) / (kZeroRows * (kRunThreads / 64)), kMaxBlocks);
  const dim3 grid((unsigned)(zero_blocks + p.pieces), (unsigned)((a.width + p.group * V - 1) / (p.group * V)));
  hipLaunchKernelGGL((lookup_grad_runs_kernel<T, O, V>), grid, dim3(kRunThreads), 0, (hipStream_t)a.stream, r, (const T*)a.grad, (O*)a.out, head, tail,
                     (int)zero_blocks, p.group, p.strip, (Wide<T>)a.scale);
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
  const PrivatePlan few = plan_private(a);
  if (few.waves) {
    W* parts = (W*)a.work;
    const int64_t values = a.rows * a.width;
    int bits = 1;
    while (a.rows >> bits) ++bits;
    auto run = [&](auto kernel) {
      // the limit belongs to the process: always the same one, or a call from another thread could lower it before this launch
      if (few.lds > 65536) LGA_HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kPrivateLds));
      hipLaunchKernelGGL(kernel, dim3(few.waves, (unsigned)a.width), dim3(64), few.lds, s, (const T*)a.grad, few.grid, few.g0, few.g1, (int)a.width, bits,
                         (int)few.lines, (int)few.steps, (int)((few.steps + few.waves - 1) / few.waves), parts);
    };
    auto by_ids = [&](auto id) {
      typedef decltype(id) I;
      if (few.items_along0) run(lookup_grad_private_kernel<T, I, true, false>);
      else if (few.whole) run(lookup_grad_private_kernel<T, I, false, true>);
      else run(lookup_grad_private_kernel<T, I, false, false>);
    };
    a.ids64 ? by_ids((int64_t)0) : by_ids((int32_t)0);
    LGA_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((lookup_grad_total_kernel<W, O>), dim3((unsigned)((values + 63) / 64)), dim3(kTotalThreads), 0, s, parts, (O*)a.out, values, few.waves,
                       (W)a.scale);
    LGA_HIP_CHECK(hipGetLastError());
    return;
  }
  const GradPlan p = plan_grad(a);
  const SortedTokens t = token_sort(p.grid, p.values ? (const void*)a.grad : nullptr, p.g0, p.g1, p.payload, (void*)a.work, s);
  const Runs r{t.keys, t.payload, t.named, t.count, a.rows, a.width, p.grid.n1, p.g0, p.g1};
  W* head = (W*)((char*)a.work + p.sort_bytes);
  W* tail = (W*)((char*)head + p.parts_bytes);
  if (a.width <= kNarrow) {
    const int zero_blocks = (int)((a.rows + kThreads - 1) / kThreads);
    const dim3 grid((unsigned)(zero_blocks + p.pieces));
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, r, (const T*)a.grad, (O*)a.out, head, tail, zero_blocks, (W)a.scale);
    };
    if constexpr (sizeof(T) >= 4) {
      if (p.values) run(lookup_grad_narrow_kernel<T, O, true, 1>);
    }
    if (!p.values) {
      if (a.width == 1) run(lookup_grad_narrow_kernel<T, O, false, 1>);
      else if (a.width == 2) run(lookup_grad_narrow_kernel<T, O, false, 2>);
      else if (a.width == 3) run(lookup_grad_narrow_kernel<T, O, false, 3>);
      else run(lookup_grad_narrow_kernel<T, O, false, 4>);
    }
  } else {
    launch_runs<T, O, kPack<T>>(a, p, r, head, tail);
  }
  LGA_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL((lookup_grad_join_kernel<W, O>), dim3((unsigned)p.pieces, (unsigned)std::min<int64_t>((a.width + 63) / 64, 8)), dim3(kThreads), 0, s, r, (O*)a.out, head, tail, p.piece_tokens, (W)a.scale);
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
  // rows that no id names are zero, which no other factor leaves a sum of nothing
  if (!std::isfinite(a.type == kF64 ? a.scale : (float)a.scale)) throw std::runtime_error("embedding_grad: the scale has to be finite");
  if (owned(a)) return 0;
  const PrivatePlan few = plan_private(a);
  if (few.waves) return few.waves * a.rows * a.width * (a.type == kF64 ? 8 : 4);
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
