// Row lookup in a table (leaf values, embeddings) and its gradient.
#pragma once
#include <cstdint>

namespace lga {

// Plain words only: the binding packs them one after the other.
struct LookupArgs {
  int64_t table, ids, out;      // addresses
  int64_t stream, device;
  int64_t rows, width;          // of the table
  int64_t table_stride;         // elements between rows
  int64_t n0, n1, s0, s1;       // token (i, j) is ids[i * s0 + j * s1]; out is [n0 * n1][width]
  int64_t type, ids64;
  double scale;
};

struct LookupGradArgs {
  int64_t grad, ids, out, work; // work: lookup_grad_workspace() bytes
  int64_t stream, device;
  int64_t rows, width;
  int64_t n0, n1, s0, s1;       // ids, as above
  int64_t g0, g1;               // token (i, j)'s gradient starts at grad[i * g0 + j * g1]
  int64_t type, out_type, ids64;
  double scale;
};

void lookup(const LookupArgs& a);
int64_t lookup_grad_workspace(const LookupGradArgs& a);
void lookup_grad(const LookupGradArgs& a);

}  // namespace lga
