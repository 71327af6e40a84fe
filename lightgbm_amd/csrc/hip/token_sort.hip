// Stable radix sort of tokens by id.  A pass counts the digits of every tile (LDS counters), turns the counts into the
// places where a tile's runs begin, and scatters: a wave ranks its keys digit by digit with ballots (lanes of one digit
// find each other in `bits` of them), the tile is put in order in LDS and written out run by run.  Integers only, so the
// order never depends on timing.  Digits of up to 9 bits, so that 18 bits of rows take two passes (12.5 M tokens in 127500 rows,
// the whole gradient: 309 us; before neighbouring tiles went to one XCD 344 us, and 365 us with three passes of 8 bits); a pass over
// them takes 120 us, of which its 200 MB need 41: runs of 8 keys are written out in pieces of 32 bytes.
#include "token_sort.hpp"
#include "device.hpp"
#include <algorithm>

namespace lga {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxBits = 9, kBins = 1 << kMaxBits;

struct Pass {
  TokenGrid grid;
  TokenTiles tiles;
  const uint32_t* keys_in;      // null: first pass, keys come from the grid
  const void* payload_in;
  int64_t v0, v1;               // first pass: payload (i, j) is at i * v0 + j * v1; payload_in null: the token's number
  uint8_t* named;               // set by the last scatter (null in the passes before)
  uint4* clear;                 // its words, where the first kernel of the sort clears them (else null)
  int64_t clear_words;
  int shift, bits;
  bool few;                     // few tiles: no kernel of its own for the offsets
};
// Up to kFewTiles tiles a scatter adds up the counts of its digits itself, above a kernel of its own does (by itself against
// with that kernel: 50000 rows of 1024 bf16 values, 68 tiles, 85 against 88 us; 70000 rows, 6 tiles 29 against 36, 59 tiles 33 against 34,
// 98 tiles 37 against 34, 293 tiles 60 against 39).
// Up to kSmallTiles small tiles they stay small (1 M tokens, 977 small tiles: 56 against 72 us with tiles of 4096; 3 M in two passes 100
// against 90, in three 101 against 106; 6 M 170 against 146 and 159 against 171).
constexpr int64_t kFewTiles = 128, kSmallTiles = 4096;

__device__ __forceinline__ uint32_t grid_key(const TokenGrid& g, int64_t i, int64_t j) {
  if (i >= g.n0 || j >= g.n1) return (uint32_t)g.rows;
  const int64_t at = i * g.s0 + j * g.s1;
  const int64_t id = g.ids64 ? ((const int64_t*)g.ids)[at] : (int64_t)((const int32_t*)g.ids)[at];
  return id >= 0 && id < g.rows ? (uint32_t)id : (uint32_t)g.rows;
}

// Item q of tile b is token (i, j) with j running fastest.
__device__ __forceinline__ void item_place(const Pass& p, int64_t b, int q, int64_t& i, int64_t& j) {
  const int64_t ti = b / p.tiles.across, tj = b - ti * p.tiles.across;
  i = ti * (1 << (p.tiles.bits - p.tiles.shift1)) + (q >> p.tiles.shift1);
  j = (tj << p.tiles.shift1) + (q & ((1 << p.tiles.shift1) - 1));
}
// The same items walked along the axis on which ids are neighbours: returns the item number.
__device__ __forceinline__ int ids_order(const Pass& p, int n) {
  if (p.grid.s1 <= p.grid.s0 || p.tiles.shift1 == p.tiles.bits) return n;
  const int shift0 = p.tiles.bits - p.tiles.shift1;
  return ((n & ((1 << shift0) - 1)) << p.tiles.shift1) | (n >> shift0);
}

template <int kItems>
__global__ __launch_bounds__(kThreads) void sort_count_kernel(Pass p, uint32_t* __restrict__ counts) {
  constexpr int kTile = kItems * kThreads;
  __shared__ uint32_t bin[kBins];
  const int64_t b = blockIdx.x;
  for (int d = threadIdx.x; d < kBins; d += kThreads) bin[d] = 0;
  __syncthreads();
  if (!p.keys_in && p.clear)
    for (int64_t r = b * kThreads + threadIdx.x; r < p.clear_words; r += (int64_t)gridDim.x * kThreads) p.clear[r] = make_uint4(0, 0, 0, 0);
  const uint32_t mask = (1u << p.bits) - 1;
#pragma unroll 4
  for (int k = 0; k < kItems; ++k) {
    const int n = k * kThreads + threadIdx.x;
    uint32_t key;
    if (p.keys_in) {
      key = p.keys_in[b * kTile + n];
    } else {
      int64_t i, j;
      item_place(p, b, ids_order(p, n), i, j);
      key = grid_key(p.grid, i, j);
    }
    atomicAdd(&bin[(key >> p.shift) & mask], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < (1 << p.bits); d += kThreads) counts[(int64_t)d * p.tiles.blocks + b] = bin[d];
}

__global__ __launch_bounds__(kThreads) void clear_kernel(uint4* __restrict__ p, int64_t words) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < words; i += (int64_t)gridDim.x * kThreads) p[i] = make_uint4(0, 0, 0, 0);
}

// Counts of one digit over the tiles -> where each tile's run of that digit begins among all of that digit; their sum.
__global__ __launch_bounds__(kThreads) void sort_offsets_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals, int64_t blocks) {
  __shared__ uint32_t wave_sum[kWaves];
  uint32_t* row = counts + (int64_t)blockIdx.x * blocks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t before = 0;
  for (int64_t base = 0; base < blocks; base += kThreads * 4) {
    uint32_t v[4], sum = 0;
    for (int k = 0; k < 4; ++k) {
      const int64_t at = base + threadIdx.x * 4 + k;
      v[k] = at < blocks ? row[at] : 0;
      sum += v[k];
    }
    uint32_t scan = sum;
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(scan, d);
      if (lane >= d) scan += o;
    }
    if (lane == 63) wave_sum[wave] = scan;
    __syncthreads();
    uint32_t at = before + scan - sum, all = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) at += wave_sum[w];
      all += wave_sum[w];
    }
    for (int k = 0; k < 4; ++k) {
      const int64_t i = base + threadIdx.x * 4 + k;
      if (i < blocks) row[i] = at;
      at += v[k];
    }
    before += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

// P: what is carried with a key (uint32 or uint64 words).  `offsets` are still counts where there are few tiles.
template <typename P, int kItems>
__global__ __launch_bounds__(kThreads) void sort_scatter_kernel(Pass p, const uint32_t* __restrict__ offsets, const uint32_t* __restrict__ totals,
                                                                uint32_t* __restrict__ keys_out, P* __restrict__ payload_out) {
  constexpr int kTile = kItems * kThreads;
  __shared__ uint32_t skey[kTile];
  __shared__ P spay[kTile];
  __shared__ uint32_t count[kWaves][kBins];     // keys of a digit in a wave, then those in the waves before
  __shared__ uint32_t local[kBins], global[kBins], wave_sum[kWaves][2];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  // Workgroups go round the eight XCDs; each XCD takes neighbouring tiles, whose runs of one digit lie next to each other and
  // fill its L2's lines (12.5 M tokens in 127500 rows: 303 against 344 us for the whole gradient).
  const int64_t each = p.tiles.blocks / 8, more = p.tiles.blocks % 8, xcd = blockIdx.x % 8;
  const int64_t b = xcd * each + min(xcd, more) + blockIdx.x / 8;
  const uint32_t mask = (1u << p.bits) - 1;
  uint32_t key[kItems], rank[kItems];
  P pay[kItems];
  for (int d = t; d < kWaves * kBins; d += kThreads) (&count[0][0])[d] = 0;
  if (!p.keys_in) {
    for (int k = 0; k < kItems; ++k) {
      const int q = ids_order(p, k * kThreads + t);
      int64_t i, j;
      item_place(p, b, q, i, j);
      skey[tile_slot(q)] = grid_key(p.grid, i, j);
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int q = wave * (kTile / kWaves) + k * 64 + lane;
    if (p.keys_in) {
      key[k] = p.keys_in[b * kTile + q];
      pay[k] = ((const P*)p.payload_in)[b * kTile + q];
    } else {
      key[k] = skey[tile_slot(q)];
      int64_t i, j;
      item_place(p, b, q, i, j);
      if (!p.payload_in) pay[k] = (P)(i * p.grid.n1 + j);
      else pay[k] = key[k] < (uint32_t)p.grid.rows ? ((const P*)p.payload_in)[i * p.v0 + j * p.v1] : (P)0;
    }
  }
  // ranks among the wave's keys of the same digit
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const uint32_t digit = (key[k] >> p.shift) & mask;
    uint64_t same = ~0ull;
    for (int bit = 0; bit < p.bits; ++bit) {
      const bool one = (digit >> bit) & 1;
      const uint64_t ones = __ballot(one);
      same &= one ? ones : ~ones;
    }
    in_order();                        // other lanes of the wave write the counters between two keys
    const uint32_t before = count[wave][digit];
    in_order();
    const int lower = __popcll(same & ((1ull << lane) - 1));
    rank[k] = before + (uint32_t)lower;
    if (lower == 0) count[wave][digit] = before + (uint32_t)__popcll(same);
  }
  __syncthreads();
  // a lane's digits t and, in passes of 9 bits, t + kThreads: keys of the digit in the waves before, in the tile, in the digits
  // below (of the tile and of all)
  uint32_t below_tile = 0, below_all = 0;
  for (int d = t; d < (1 << p.bits) || d < kThreads; d += kThreads) {
    uint32_t in_tile = 0, total = 0, ahead = 0;
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t c = count[w][d];
      count[w][d] = in_tile;
      in_tile += c;
    }
    if (d < (1 << p.bits)) {
      const uint32_t* row = offsets + (int64_t)d * p.tiles.blocks;
      if (p.few) {
#pragma unroll 8
        for (int q = 0; q < (int)p.tiles.blocks; q += 4) {       // a multiple of 4
          const uint4 c = *(const uint4*)(row + q);
          total += c.x + c.y + c.z + c.w;
          ahead += (q < (int)b ? c.x : 0) + (q + 1 < (int)b ? c.y : 0) + (q + 2 < (int)b ? c.z : 0) + (q + 3 < (int)b ? c.w : 0);
        }
      } else {
        total = totals[d];
        ahead = row[b];
      }
    }
    uint32_t a = in_tile, g = total;
    for (int e = 1; e < 64; e <<= 1) {
      const uint32_t oa = __shfl_up(a, e), og = __shfl_up(g, e);
      if (lane >= e) a += oa, g += og;
    }
    if (lane == 63) wave_sum[wave][0] = a, wave_sum[wave][1] = g;
    __syncthreads();
    a += below_tile - in_tile;
    g += below_all - total;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) a += wave_sum[w][0], g += wave_sum[w][1];
      below_tile += wave_sum[w][0];
      below_all += wave_sum[w][1];
    }
    local[d] = a;
    global[d] = g + ahead;
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const uint32_t digit = (key[k] >> p.shift) & mask;
    const uint32_t at = local[digit] + count[wave][digit] + rank[k];
    skey[at] = key[k];
    spay[at] = pay[k];
  }
  __syncthreads();
#pragma unroll 4
  for (int k = 0; k < kItems; ++k) {
    const uint32_t n = k * kThreads + t, ky = skey[n], digit = (ky >> p.shift) & mask;
    const uint32_t to = global[digit] + n - local[digit];
    keys_out[to] = ky;
    payload_out[to] = spay[n];
    if (p.named && ky < (uint32_t)p.grid.rows) p.named[ky] = 1;
  }
}

static_assert(kBins % kThreads == 0, "every lane has as many digits");

// Up to kSortTile tokens: one workgroup takes all passes in LDS, in place of two launches a pass.
constexpr int kOneThreads = 1024, kOneWaves = kOneThreads / 64, kOneItems = kSortTile / kOneThreads;

template <typename P>
__global__ __launch_bounds__(kOneThreads) void sort_one_kernel(Pass p, int passes, int total_bits, uint32_t* __restrict__ keys_out, P* __restrict__ payload_out) {
  __shared__ uint32_t skey[kSortTile];
  __shared__ P spay[kSortTile];
  __shared__ uint16_t count[kOneWaves][kBins];
  __shared__ uint32_t local[kBins], wave_sum[kBins / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const uint32_t tokens = (uint32_t)(p.grid.n0 * p.grid.n1);
  uint32_t key[kOneItems], rank[kOneItems];
  P pay[kOneItems];
  if (p.clear)
    for (int64_t r = t; r < p.clear_words; r += kOneThreads) p.clear[r] = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int k = 0; k < kOneItems; ++k) {
    const uint32_t q = wave * (kSortTile / kOneWaves) + k * 64 + lane;
    key[k] = (uint32_t)p.grid.rows;
    pay[k] = 0;
    if (q < tokens) {
      const uint32_t i = q / (uint32_t)p.grid.n1, j = q - i * (uint32_t)p.grid.n1;
      key[k] = grid_key(p.grid, i, j);
      pay[k] = p.payload_in ? ((const P*)p.payload_in)[i * p.v0 + j * p.v1] : (P)q;
    }
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * p.bits, bits = min(p.bits, total_bits - shift);
    const uint32_t mask = (1u << bits) - 1;
    for (int d = t; d < kOneWaves * kBins; d += kOneThreads) (&count[0][0])[d] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kOneItems; ++k) {
      const uint32_t digit = (key[k] >> shift) & mask;
      uint64_t same = ~0ull;
      for (int bit = 0; bit < bits; ++bit) {
        const bool one = (digit >> bit) & 1;
        const uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
      }
      in_order();
      const uint32_t before = count[wave][digit];
      in_order();
      const int lower = __popcll(same & ((1ull << lane) - 1));
      rank[k] = before + (uint32_t)lower;
      if (lower == 0) count[wave][digit] = (uint16_t)(before + (uint32_t)__popcll(same));
    }
    __syncthreads();
    uint32_t in_tile = 0, a = 0;
    if (t < kBins) {
      for (int w = 0; w < kOneWaves; ++w) {
        const uint32_t c = count[w][t];
        count[w][t] = (uint16_t)in_tile;
        in_tile += c;
      }
      a = in_tile;
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(a, d);
        if (lane >= d) a += o;
      }
      if (lane == 63) wave_sum[wave] = a;
    }
    __syncthreads();
    if (t < kBins) {
      for (int w = 0; w < wave; ++w) a += wave_sum[w];
      local[t] = a - in_tile;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kOneItems; ++k) {
      const uint32_t digit = (key[k] >> shift) & mask, at = local[digit] + count[wave][digit] + rank[k];
      skey[at] = key[k];
      spay[at] = pay[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kOneItems; ++k) {
      const int q = wave * (kSortTile / kOneWaves) + k * 64 + lane;
      key[k] = skey[q];
      pay[k] = spay[q];
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kOneItems; ++k) {
    const int q = wave * (kSortTile / kOneWaves) + k * 64 + lane;
    keys_out[q] = key[k];
    payload_out[q] = pay[k];
    if (key[k] < (uint32_t)p.grid.rows) p.named[key[k]] = 1;      // behind the barriers of the passes
  }
}

bool one_tile(const TokenGrid& g) { return g.n0 * g.n1 <= kSortTile; }

int bit_length(int64_t v) {
  int n = 0;
  while (v > 0) ++n, v >>= 1;
  return std::max(n, 1);
}

struct Layout {
  int64_t keys[2], payload[2], counts, totals, named, bytes;
};
Layout layout(const TokenTiles& t, int payload, int64_t rows) {
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t n) { const int64_t here = at; at += (n + 255) / 256 * 256; return here; };
  for (int k = 0; k < 2; ++k) {
    l.keys[k] = take(t.count * 4);
    l.payload[k] = take(t.count * payload);
  }
  l.counts = take(t.blocks * kBins * 4);
  l.totals = take(kBins * 4);
  l.named = take(rows);
  l.bytes = at;
  return l;
}

}  // namespace

TokenTiles token_tiles(const TokenGrid& g, int bits) {
  TokenTiles t;
  // sides: as many tokens along axis 0 as there are, up to 64 (256 bytes of int32 ids where they are neighbours), or more where
  // axis 1 does not fill the rest: a tile is more than half full, and 2^31 - 1 tokens have places of 32 bits
  int shift0 = 0, shift1 = 0;
  while (shift0 < 6 && (1LL << shift0) < g.n0) ++shift0;
  while (shift1 < bits - shift0 && (1LL << shift1) < g.n1) ++shift1;
  shift0 = bits - shift1;
  t.bits = bits;
  t.shift1 = shift1;
  t.across = (g.n1 + (1LL << t.shift1) - 1) >> t.shift1;
  t.blocks = ((g.n0 + (1LL << shift0) - 1) >> shift0) * t.across;
  t.count = t.blocks << bits;
  if (t.count > 4294967295LL - kSortTile) throw std::runtime_error("embedding: too many tokens");
  return t;
}

// Small tiles where tiles of 4096 would leave most of the chip idle (500 k tokens in 127500 rows: 122 of them).
TokenTiles sort_tiles(const TokenGrid& g) {
  if (one_tile(g)) {
    TokenTiles t;
    t.shift1 = t.bits;
    t.across = t.blocks = 1;
    t.count = kSortTile;
    return t;
  }
  TokenTiles t = token_tiles(g, 10);
  if (t.blocks > kSmallTiles) return token_tiles(g);
  t.blocks = (t.blocks + 3) / 4 * 4;      // whole multiples of kSortTile
  t.count = t.blocks << 10;
  return t;
}

int64_t token_sort_workspace(const TokenGrid& g, int payload) { return layout(sort_tiles(g), payload, g.rows).bytes; }

SortedTokens token_sort(const TokenGrid& g, const void* values, int64_t v0, int64_t v1, int payload, void* workspace, hipStream_t s) {
  const TokenTiles tiles = sort_tiles(g);
  const Layout l = layout(tiles, payload, g.rows);
  char* w = (char*)workspace;
  const int bits = bit_length(g.rows), passes = (bits + kMaxBits - 1) / kMaxBits, each = (bits + passes - 1) / passes;
  const bool small = tiles.bits == 10;
  const dim3 grid((unsigned)tiles.blocks), block(kThreads);
  uint32_t *counts = (uint32_t*)(w + l.counts), *totals = (uint32_t*)(w + l.totals);
  uint8_t* named = (uint8_t*)(w + l.named);
  // the named rows: cleared on the way where that is a few words a lane, else by a kernel of its own
  const int64_t words = (g.rows + 15) / 16, lanes = one_tile(g) ? kOneThreads : tiles.blocks * kThreads;
  Pass p{g, tiles, nullptr, values, v0, v1, named, words <= 4 * lanes ? (uint4*)named : nullptr, words, 0, each, tiles.blocks <= kFewTiles && small};
  if (!p.clear) {
    hipLaunchKernelGGL(clear_kernel, dim3((unsigned)std::min<int64_t>((words + kThreads - 1) / kThreads, 4096)), block, 0, s, (uint4*)named, words);
    LGA_HIP_CHECK(hipGetLastError());
  }
  if (one_tile(g)) {
    uint32_t* keys = (uint32_t*)(w + l.keys[0]);
    void* pay = w + l.payload[0];
    p.bits = each;
    if (payload == 8) hipLaunchKernelGGL(sort_one_kernel<uint64_t>, dim3(1), dim3(kOneThreads), 0, s, p, passes, bits, keys, (uint64_t*)pay);
    else hipLaunchKernelGGL(sort_one_kernel<uint32_t>, dim3(1), dim3(kOneThreads), 0, s, p, passes, bits, keys, (uint32_t*)pay);
    LGA_HIP_CHECK(hipGetLastError());
    return {keys, pay, named, tiles.count};
  }
  for (int k = 0; k < passes; ++k) {
    p.shift = k * each;
    p.bits = std::min(each, bits - p.shift);
    uint32_t* keys = (uint32_t*)(w + l.keys[k & 1]);
    void* pay = w + l.payload[k & 1];
    if (small) hipLaunchKernelGGL(sort_count_kernel<kSmallTile / kThreads>, grid, block, 0, s, p, counts);
    else hipLaunchKernelGGL(sort_count_kernel<kSortTile / kThreads>, grid, block, 0, s, p, counts);
    LGA_HIP_CHECK(hipGetLastError());
    if (!p.few) {
      hipLaunchKernelGGL(sort_offsets_kernel, dim3(1u << p.bits), block, 0, s, counts, totals, tiles.blocks);
      LGA_HIP_CHECK(hipGetLastError());
    }
    p.named = k + 1 == passes ? named : nullptr;
    auto scatter = [&](auto kernel, auto* to) {
      hipLaunchKernelGGL(kernel, grid, block, 0, s, p, counts, totals, keys, to);
    };
    if (payload == 8) {
      if (small) scatter(sort_scatter_kernel<uint64_t, kSmallTile / kThreads>, (uint64_t*)pay);
      else scatter(sort_scatter_kernel<uint64_t, kSortTile / kThreads>, (uint64_t*)pay);
    } else {
      if (small) scatter(sort_scatter_kernel<uint32_t, kSmallTile / kThreads>, (uint32_t*)pay);
      else scatter(sort_scatter_kernel<uint32_t, kSortTile / kThreads>, (uint32_t*)pay);
    }
    LGA_HIP_CHECK(hipGetLastError());
    p.keys_in = keys;
    p.payload_in = pay;
  }
  return {p.keys_in, p.payload_in, named, tiles.count};
}

}  // namespace lga
