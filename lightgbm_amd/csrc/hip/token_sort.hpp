// Stable sort of tokens by their id (least significant digit first), for sums over the tokens of a table row.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace lga {

// Token (i, j) of an n0 x n1 grid has the id ids[i * s0 + j * s1]; ids outside [0, rows) sort as `rows`, to the end.
struct TokenGrid {
  const void* ids = nullptr;
  int ids64 = 0;
  int64_t n0 = 1, n1 = 0, s0 = 0, s1 = 1;
  int64_t rows = 0;
};

// The grid is read in tiles of 1 << bits tokens, side[0] x side[1]; a tile that reaches over the edge is filled up with
// absent tokens (id `rows`), so `count` of the sorted arrays is a multiple of kSortTile.
constexpr int kSortTile = 4096, kSmallTile = 1024;
struct TokenTiles {
  int64_t across = 0, count = 0, blocks = 0;   // tiles along axis 1, tokens with the absent ones, tiles
  int bits = 12, shift1 = 0;                   // side[1] = 1 << shift1, side[0] = 1 << (bits - shift1)
};
// `bits`: 12, or 10 for small tiles.
TokenTiles token_tiles(const TokenGrid& g, int bits = 12);

// LDS accesses of a wave run in program order; this keeps the compiler from moving or merging them across this point, as
// it could for accesses of one lane.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

// Where item q of a tile stands in LDS: tiles are written along one axis and read along the other, and this way neither
// walk meets a bank twice.
__device__ __forceinline__ int tile_slot(int q) { return (q & ~63) | ((q ^ (q >> 6)) & 63); }

// Bytes of workspace of a sort with `payload` bytes a token.
int64_t token_sort_workspace(const TokenGrid& g, int payload);

// Sorts ids with the payload of every token: its number i * n1 + j (values == nullptr, payload 4), or its value
// values[i * v0 + j * v1] of `payload` bytes (4 or 8).  keys (uint32), payloads and the named rows are in the workspace.
TokenTiles sort_tiles(const TokenGrid& g);      // what a sort of g uses
struct SortedTokens {
  const uint32_t* keys = nullptr;
  const void* payload = nullptr;
  const uint8_t* named = nullptr;      // [rows]: 1 where an id names the row
  int64_t count = 0;
};
SortedTokens token_sort(const TokenGrid& g, const void* values, int64_t v0, int64_t v1, int payload, void* workspace, hipStream_t s);

}  // namespace lga
