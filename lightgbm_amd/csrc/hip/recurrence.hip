// The gated linear recurrence over the steps of a batch of sequences,
//   h[t] = a[t] h[t-1] + w[t] x[t],   w = 1 or (mixed form) 1 - a,
// and its gradients.  With e[t] = a[t] c[t] the gradient c[t] of h[t] follows the same recurrence backwards:
//   c[t] = dh[t] + e[t+1],  e[t] = a[t] c[t];   dx = w c,  da = c (h[t-1] - (mixed) x),  dstate = e[0].
// Behind a sequence's length the state is kept and nothing is read: whatever stands there cannot reach a result.
//
// A run of steps is an affine map h -> A h + H, and maps compose associatively: (A, H) after (A', H') is
// (A A', A H' + H).  The steps are cut into chunks that one lane holds in registers, up to kMaxSlots chunks make a tile
// (one workgroup, 64 channel packs wide).  A tile folds its chunks through LDS, hands its map to the tiles behind it
// through memory, folds the maps before it, and then walks its chunks again from the exact state before each: every
// value is read once and written once.  All folds run in the order of the steps, so results do not depend on timing.
//
// Bound by HBM where there are enough rows of tiles: 8 x 4096 x 2560 bf16 with fp32 gates, mixed, 141 us forward (4.8 TB/s) and
// 269 us backward (5.0 TB/s) where a copy reaches 4.9; 500 x 45800 fp64 with one gate a step 94 us (3.9 TB/s).  One sequence of
// 65537 x 1024 bf16 takes 115 us (3.5 TB/s): its eight rows of tiles leave a CU one workgroup, which loads, folds and stores in
// turn.  One lane walking a channel through all steps took 1877 us, 61.6 ms, 265 us and 30.7 ms.
#include "recurrence.hpp"
#include "device.hpp"
#include "seq_types.hpp"
#include <algorithm>

namespace lga {

namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 64;          // channel packs of a tile
constexpr int kScanSteps = 16;      // steps a lane holds
constexpr int kMaxSlots = 16;       // chunks of a tile
constexpr uint64_t kEmpty = ~0ull;  // a word nobody has written yet: a NaN that publish() never stores

enum GateKind { kNoGate, kOwnGate, kSharedGate };

// How the slopes of shared gates are summed: by teams of lanes (0: not), whose sums stand as [rows][steps][teams]; `done`: a
// team is a whole gate group, and its sum is the gate's gradient.
struct GateSums {
  int team = 0, done = 0;
  int64_t rows = 1, teams = 1;
};

__device__ __forceinline__ float abs_of(float x) { return __builtin_fabsf(x); }
__device__ __forceinline__ double abs_of(double x) { return __builtin_fabs(x); }
__device__ __forceinline__ float mantissa(float x) { return __builtin_amdgcn_frexp_mantf(x); }
__device__ __forceinline__ double mantissa(double x) { return __builtin_amdgcn_frexp_mant(x); }
__device__ __forceinline__ int exponent(float x) { return __builtin_amdgcn_frexp_expf(x); }
__device__ __forceinline__ int exponent(double x) { return __builtin_amdgcn_frexp_exp(x); }
__device__ __forceinline__ float times_power(float x, int e) { return __builtin_ldexpf(x, e); }
__device__ __forceinline__ double times_power(double x, int e) { return __builtin_ldexp(x, e); }

// The map of a run of steps, x -> (product of its gates) x + h.  The product is m 2^e and is right whatever its size: a hundred
// gates of a half leave the range of fp32, but what they leave of a state of 1e30 does not, a state of zero stays zero
// under gates above one, and an infinite state is no 0 * inf.  No product runs over more steps than lie between two
// checkpoints, so e stays far from its ends.
template <typename W, bool kGates> struct Map { W m; int e; W h; };
template <typename W> struct Map<W, false> { W h; };      // without gates the product is one
template <typename W, bool kGates> __device__ __forceinline__ Map<W, kGates> no_steps() {
  if constexpr (kGates) return {1, 0, 0};
  else return {0};
}

// 1 <= |m| < 2, or infinite, NaN, or zero (and then e too: it may hold large gates around the gate of zero)
template <typename W> __device__ __forceinline__ Map<W, true> normal(const Map<W, true>& f) {
  return {2 * mantissa(f.m), f.m == 0 ? 0 : f.e + exponent(f.m) - 1, f.h};
}
template <typename W> __device__ __forceinline__ Map<W, false> normal(const Map<W, false>& f) { return f; }

// f normal
template <typename W> __device__ __forceinline__ W apply(const Map<W, true>& f, W x) { return fma_wide(times_power(x, f.e), f.m, f.h); }
template <typename W> __device__ __forceinline__ W apply(const Map<W, false>& f, W x) { return x + f.h; }

// `later` (normal) after `first`; a fold of n normal maps has 1 <= |m| < 2^n
template <typename W> __device__ __forceinline__ Map<W, true> after(const Map<W, true>& later, const Map<W, true>& first) {
  return {later.m * first.m, later.e + first.e, apply(later, first.h)};
}
template <typename W> __device__ __forceinline__ Map<W, false> after(const Map<W, false>& later, const Map<W, false>& first) { return {first.h + later.h}; }

// Words that tiles hand to one another.  Each is written once, whole, and read with agent scope until it is there: the
// value itself is the flag.
__device__ __forceinline__ void put_word(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v == kEmpty ? 0x7ff8000000000000ull : v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// N neighbouring words, loaded together, and again until all are there.
template <int N> __device__ __forceinline__ void load_words(const uint64_t* p, uint64_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = __hip_atomic_load(p + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int N> __device__ __forceinline__ bool lacks(const uint64_t (&w)[N]) {
  bool some = false;
  for (uint64_t x : w) some |= x == kEmpty;
  return some;
}
template <int N> __device__ __forceinline__ void wait_words(const uint64_t* p, uint64_t (&w)[N]) {
  while (lacks(w)) {
    __builtin_amdgcn_s_sleep(1);
    load_words(p, w);
  }
}
// The product of a normal map in as many bits as m: the field of m's exponent and two bits of its fraction hold e, up to 2^509
// (2^4093 for fp64), beyond which the product makes zero or infinity of any state of the type.  What the two bits round is four
// roundings of W, where the gates of a tile have at least 128 (a word of its own for e: 145 against 121 us at 1 x 65537 x 1024 bf16).
template <typename W> struct Bits;
template <> struct Bits<float> { typedef uint32_t U; static constexpr int fraction = 23, exponent = 8; };
template <> struct Bits<double> { typedef uint64_t U; static constexpr int fraction = 52, exponent = 11; };

template <typename W> __device__ __forceinline__ typename Bits<W>::U packed(W m, int e) {
  typedef typename Bits<W>::U U;
  constexpr int F = Bits<W>::fraction, X = Bits<W>::exponent, kMiddle = 1 << (X + 1);
  constexpr U kSign = (U)1 << (F + X), kOnes = ((U)4 << X) - 1;     // of e: 0 for zero, all ones for what is not finite
  U bits;
  __builtin_memcpy(&bits, &m, sizeof m);
  const U scale = (U)(min(max(e, 1 - kMiddle), kMiddle - 3) + kMiddle);
  U p = (scale << (F - 2)) + (((bits & (((U)1 << F) - 1)) + 2) >> 2);      // a fraction rounded up to one goes into e
  if (m == 0) p = 0;
  if (!(abs_of(m) < 2)) p = kOnes << (F - 2) | (m != m);
  return p | (bits & kSign);
}
template <typename W> __device__ __forceinline__ void unpack(typename Bits<W>::U p, W& m, int& e) {
  typedef typename Bits<W>::U U;
  constexpr int F = Bits<W>::fraction, X = Bits<W>::exponent, kMiddle = 1 << (X + 1);
  constexpr U kSign = (U)1 << (F + X), kOnes = ((U)4 << X) - 1;
  const U scale = p >> (F - 2) & kOnes;
  e = (int)scale - kMiddle;
  const U field = scale == 0 ? 0 : scale == kOnes ? ((U)1 << X) - 1 : ((U)1 << (X - 1)) - 1;
  const U bits = (p & kSign) | field << F | (p << 2 & (((U)1 << F) - 1));
  __builtin_memcpy(&m, &bits, sizeof m);
}
// fp32: one word; never kEmpty, whose product is none that packed() gives
__device__ __forceinline__ void publish(uint64_t* p, const Map<float, true>& f) { put_word(p, (uint64_t)packed(f.m, f.e) << 32 | __float_as_uint(f.h)); }
__device__ __forceinline__ void read_map(const uint64_t* w, Map<float, true>& f) {
  unpack((uint32_t)(*w >> 32), f.m, f.e);
  f.h = __uint_as_float((uint32_t)*w);
}
// fp64: two words
__device__ __forceinline__ void publish(uint64_t* p, const Map<double, true>& f) {
  put_word(p, packed(f.m, f.e));
  put_word(p + 1, (uint64_t)__double_as_longlong(f.h));
}
__device__ __forceinline__ void read_map(const uint64_t* w, Map<double, true>& f) {
  unpack(w[0], f.m, f.e);
  f.h = __longlong_as_double((int64_t)w[1]);
}
// states, and maps without gates
__device__ __forceinline__ void publish(uint64_t* p, const Map<float, false>& f) { put_word(p, __float_as_uint(f.h)); }
__device__ __forceinline__ void read_map(const uint64_t* w, Map<float, false>& f) { f = {__uint_as_float((uint32_t)*w)}; }
__device__ __forceinline__ void publish(uint64_t* p, const Map<double, false>& f) { put_word(p, (uint64_t)__double_as_longlong(f.h)); }
__device__ __forceinline__ void read_map(const uint64_t* w, Map<double, false>& f) { f = {__longlong_as_double((int64_t)*w)}; }
// after() for maps that were packed: a product whose e may have been cut has made zero or infinity of every state but zero, which
// later gates do not bring back.
template <typename W> __device__ __forceinline__ Map<W, true> behind(const Map<W, true>& later, const Map<W, true>& first) {
  Map<W, true> f = after(later, first);
  if (abs(first.e) >= (2 << Bits<W>::exponent) - 3) f.e = first.e;
  return f;
}
template <typename W> __device__ __forceinline__ Map<W, false> behind(const Map<W, false>& later, const Map<W, false>& first) { return after(later, first); }
template <typename W, bool kGates> constexpr int kMapWords = kGates ? sizeof(W) / 4 : 1;

__global__ __launch_bounds__(kThreads) void fill_words_kernel(uint4* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) p[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

// How the steps are cut, for both directions.  Channels are counted in packs of V over all sequences.
struct Cut {
  int64_t packs;      // batch * width / V
  int64_t pack_rows;  // workgroups side by side: packs / lanes, rounded up
  int64_t tiles;      // workgroups one behind the other
  int lanes, slots;   // of a workgroup
  int checkpoint;     // every so many tiles one hands on the state itself: no tile folds more maps than come behind it
};

// Workspace of a cut into several tiles, in words: [0] tickets, then the tiles' maps, then the checkpoints' states.
template <typename W> inline int64_t work_words(const Cut& k, int v, bool gates) {
  const int64_t channels = k.pack_rows * k.lanes * v, map = gates ? kMapWords<W, true> : kMapWords<W, false>;
  const int64_t n = 8 + k.tiles * channels * map + (k.tiles / k.checkpoint + 1) * channels;
  return k.tiles < 2 ? 0 : (n + 1) / 2 * 2;
}

// Which tile a workgroup is.  Several tiles: by ticket, in the order in which workgroups really start, so that whatever a
// tile waits for belongs to a workgroup that already runs (and waits for earlier ones only).
__device__ __forceinline__ void take_tile(const Cut& k, uint64_t* work, int64_t& tile, int64_t& row) {
  int64_t ticket = blockIdx.x;
  if (k.tiles > 1) {
    __shared__ uint32_t taken;
    if (threadIdx.x == 0) taken = __hip_atomic_fetch_add((uint32_t*)work, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;   // starts at 2^32 - 1
    __syncthreads();
    ticket = taken;
  }
  tile = ticket / k.pack_rows;
  row = ticket - tile * k.pack_rows;
}

// The state before this lane's chunk, given the chunk's own map.  `first`: the state before the first tile.
// Returns it in `carry`.
template <typename W, int V, bool kGates>
__device__ __forceinline__ void carry_in(const Cut& k, uint64_t* work, int64_t tile, int64_t row, int lane, int slot, const Map<W, kGates> (&own)[V],
                                         const W (&first)[V], W (&carry)[V]) {
  typedef Map<W, kGates> M;
  constexpr int kWords = kMapWords<W, kGates>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  M(*maps)[V] = (M(*)[V])lds;                                 // [slots][lanes]
  M(*parts)[V] = maps + k.slots * k.lanes;                    // partial folds of the tiles before this one
  const int at = slot * k.lanes + lane;
  for (int v = 0; v < V; ++v) maps[at][v] = own[v];
  __syncthreads();
  M mine[V];                                                  // the chunks of this tile before this one
  for (int v = 0; v < V; ++v) mine[v] = no_steps<W, kGates>();
  for (int s = 0; s < slot; ++s)
    for (int v = 0; v < V; ++v) mine[v] = after(maps[s * k.lanes + lane][v], mine[v]);
  for (int v = 0; v < V; ++v) carry[v] = first[v];
  const int64_t channels = k.pack_rows * k.lanes * V, channel = (row * k.lanes + lane) * V;
  if (k.tiles > 1) {
    uint64_t* tile_maps = work + 8 + channel * kWords;        // channels * kWords of them a tile
    if (slot == k.slots - 1 && tile + 1 < k.tiles)
      for (int v = 0; v < V; ++v) publish(tile_maps + tile * channels * kWords + v * kWords, normal(after(own[v], mine[v])));
    const int64_t from = tile / k.checkpoint * k.checkpoint;    // first tile behind the last checkpoint
    const int before = (int)(tile - from), share = (before + k.slots - 1) / k.slots;
    const uint64_t* checkpoint = work + 8 + k.tiles * channels * kWords + (from / k.checkpoint - 1) * channels + channel;
    uint64_t words[V * kWords], state[V];
    if (from > 0) load_words(checkpoint, state);              // on its way while the maps are waited for
    M part[V];
    for (int v = 0; v < V; ++v) part[v] = no_steps<W, kGates>();
    for (int p = slot * share; p < min(before, (slot + 1) * share); ++p) {
      const uint64_t* const map = tile_maps + (from + p) * channels * kWords;
      load_words(map, words);
      wait_words(map, words);
      for (int v = 0; v < V; ++v) {
        M m;
        read_map(words + v * kWords, m);
        part[v] = behind(m, part[v]);
      }
    }
    for (int v = 0; v < V; ++v) parts[at][v] = normal(part[v]);
    if (from > 0) {
      wait_words(checkpoint, state);
      for (int v = 0; v < V; ++v) {
        Map<W, false> c;
        read_map(state + v, c);
        carry[v] = c.h;
      }
    }
    __syncthreads();
    if (before)
      for (int s = 0; s * share < before; ++s)
        for (int v = 0; v < V; ++v) carry[v] = apply(parts[s * k.lanes + lane][v], carry[v]);
  }
  for (int v = 0; v < V; ++v) carry[v] = apply(normal(mine[v]), carry[v]);
  if (slot == k.slots - 1 && (tile + 1) % k.checkpoint == 0 && tile + 1 < k.tiles) {
    uint64_t* checkpoint = work + 8 + k.tiles * channels * kWords + tile / k.checkpoint * channels + channel;
    for (int v = 0; v < V; ++v) publish(checkpoint + v, Map<W, false>{apply(maps[at][v], carry[v])});
  }
}

// The channels of a pack: d .. d + V - 1 of sequence b.  The last pack of a width that V does not divide starts earlier; its
// first `again` channels are those of the pack before too.
template <int V> struct Channels {
  int64_t b, d;
  int again;
  __device__ __forceinline__ Channels(int64_t pack, int64_t width) {
    const int64_t row = (width + V - 1) / V;
    b = pack / row;
    const int64_t first = (pack - b * row) * V;
    d = min(first, width - V);
    again = (int)(first - d);
  }
};

// The gates of a lane's channels.  Of a shared gate one load serves the pack, unless a group ends within a pack of the wave;
// where a step has one gate and steps are neighbours, a chunk's gates are loaded as one pack.
template <typename G, GateKind K, int V> struct GateRow {
  const G* base = nullptr;
  int64_t step = 0;
  int64_t group[V];
  bool split = false;
  __device__ __forceinline__ GateRow(int64_t gate, int64_t b, int64_t gate_b, int64_t gate_t, int64_t d, int64_t per) {
    if constexpr (K != kNoGate) {
      base = (const G*)gate + b * gate_b + (K == kOwnGate ? d : 0);
      step = gate_t;
      for (int v = 0; v < V; ++v) group[v] = K == kSharedGate ? (d + v) / per : v;
      if constexpr (K == kSharedGate && V > 1) split = __any(group[0] != group[V - 1]);
    }
  }
  __device__ __forceinline__ Pack<G, V> load(int64_t t) const {
    Pack<G, V> g;
    if constexpr (K == kOwnGate) {
      g = load_pack<G, V>(base + t * step);
    } else if constexpr (K == kSharedGate) {
      for (int v = 0; v < V; ++v) g.v[v] = base[t * step + group[v]];
    }
    return g;
  }
  // steps t, t + Way, ..., all of them there
  template <int Way, int L> __device__ __forceinline__ void load_steps(int64_t t, Pack<G, V> (&gs)[L]) const {
    if constexpr (K == kSharedGate && L > 1) {
      if (step == 1 && !split) {
        const Pack<G, L> line = load_pack<G, L>(base + group[0] + (Way > 0 ? t : t - (L - 1)));
#pragma unroll
        for (int j = 0; j < L; ++j)
          for (int v = 0; v < V; ++v) gs[j].v[v] = line.v[Way > 0 ? j : L - 1 - j];
        return;
      }
    }
    if (K == kSharedGate && V > 1 && !split) {
#pragma unroll
      for (int j = 0; j < L; ++j) gs[j].v[0] = base[(t + Way * j) * step + group[0]];
#pragma unroll
      for (int j = 0; j < L; ++j)
        for (int v = 1; v < V; ++v) gs[j].v[v] = gs[j].v[0];
      return;
    }
#pragma unroll
    for (int j = 0; j < L; ++j) gs[j] = load(t + Way * j);
  }
};

template <typename T, int V> __device__ __forceinline__ Pack<T, V> constant(float x) {
  Pack<T, V> p;
  for (int v = 0; v < V; ++v) p.v[v] = (T)x;
  return p;
}

// Keeps the compiler from carrying the wide values of the first walk over a chunk into the second: the packs as loaded take
// half the registers or less.
template <typename T, int V, int L> __device__ __forceinline__ void as_loaded(Pack<T, V> (&p)[L]) {
  if constexpr (sizeof(T) * V % 4 == 0) {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      uint32_t w[sizeof(T) * V / 4];
      __builtin_memcpy(w, &p[j], sizeof w);
      for (uint32_t& x : w) asm volatile("" : "+v"(x));
      __builtin_memcpy(&p[j], w, sizeof w);
    }
  }
}

__device__ __forceinline__ int64_t length_of(int64_t lengths, int64_t b, int64_t steps) {
  if (!lengths) return steps;
  return max((int64_t)0, min((int64_t)((const int32_t*)lengths)[b], steps));
}

template <typename T, typename G, GateKind K, int V, int L>
__global__ __launch_bounds__(kLanes* kMaxSlots) void scan_kernel(ScanArgs a, Cut k) {
  typedef Wide<T> W;
  int64_t tile, row;
  take_tile(k, (uint64_t*)a.work, tile, row);
  const int lane = threadIdx.x % k.lanes, slot = threadIdx.x / k.lanes;
  const int64_t pack = row * k.lanes + lane;
  const bool live = pack < k.packs;
  const Channels<V> at(live ? pack : 0, a.width);
  const int64_t b = at.b, d = at.d, c = b * a.width + d;
  const int64_t t0 = (tile * k.slots + slot) * L, len = live ? length_of(a.lengths, b, a.steps) : 0;
  const T* x = (const T*)a.x + b * a.x_b + d;
  const GateRow<G, K, V> gate(a.gate, b, a.gate_b, a.gate_t, d, K == kSharedGate ? a.width / a.groups : 1);
  Pack<T, V> xs[L];
  Pack<G, V> gs[L];
  if (__all(t0 + L <= len)) {
#pragma unroll
    for (int j = 0; j < L; ++j) xs[j] = load_pack<T, V>(x + (t0 + j) * a.x_t);
    gate.template load_steps<1>(t0, gs);
  } else {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      xs[j] = constant<T, V>(0);
      gs[j] = constant<G, V>(1);
      if (t0 + j < len) {
        xs[j] = load_pack<T, V>(x + (t0 + j) * a.x_t);
        gs[j] = gate.load(t0 + j);
      }
    }
  }
  W h[V], first[V];
  for (int v = 0; v < V; ++v) first[v] = a.state && live ? ((const W*)a.state)[c + v] : (W)0;
  if (k.tiles > 1 || k.slots > 1) {
    Map<W, K != kNoGate> own[V];
    for (int v = 0; v < V; ++v) own[v] = no_steps<W, K != kNoGate>();
#pragma unroll
    for (int j = 0; j < L; ++j)
      for (int v = 0; v < V; ++v) {
        W in = (W)xs[j].v[v];
        if constexpr (K == kNoGate) {
          own[v].h += in;
        } else {
          const W g = (W)gs[j].v[v];
          if (a.mix) in *= (W)1 - g;
          own[v].h = fma_wide(g, own[v].h, in);
          own[v].m *= mantissa(g);
          own[v].e += exponent(g);
        }
      }
    for (int v = 0; v < V; ++v) own[v] = normal(own[v]);
    as_loaded(xs);
    if constexpr (K != kNoGate) as_loaded(gs);
    carry_in<W, V, K != kNoGate>(k, (uint64_t*)a.work, tile, row, lane, slot, own, first, h);
  } else {
    for (int v = 0; v < V; ++v) h[v] = first[v];
  }
  if (!live) return;
  T* out = (T*)a.states + b * a.steps * a.width + d;
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const int64_t t = t0 + j;
    Pack<T, V> o;
    for (int v = 0; v < V; ++v) {
      W in = (W)xs[j].v[v];
      if constexpr (K == kNoGate) {
        h[v] += in;
      } else {
        const W g = (W)gs[j].v[v];
        if (a.mix) in *= (W)1 - g;
        h[v] = fma_wide(g, h[v], in);
      }
      o.v[v] = t < len ? (T)h[v] : (T)(W)0;
    }
    if (t < a.steps) store_pack<T, V>(out + t * a.width, o);
  }
  if (tile == k.tiles - 1 && slot == k.slots - 1)
    for (int v = 0; v < V; ++v) ((W*)a.last)[c + v] = h[v];
}

// Sums v[j] over the `team` lanes (a power of two) that this lane belongs to, for all N of them (a power of two): lanes
// exchange halves of what they still hold, so that N sums over 64 lanes take N - 1 + log2(64 / N) exchanges.  Afterwards the
// lane holds in v[0] the sum of item `mine`; `holds`: it is the one of its team that holds it.
template <typename W, int N> __device__ __forceinline__ void team_sums(W (&v)[N], int team, int& mine, bool& holds) {
  const int lane = threadIdx.x & (team - 1);
  int bit = 1;
  mine = 0;
#pragma unroll
  for (int n = N; n > 1; n /= 2) {
    if (bit < team) {
      const bool upper = (lane & bit) != 0;
#pragma unroll
      for (int j = 0; j < N / 2; ++j)
        if (j < n / 2) {
          const W give = upper ? v[j] : v[j + n / 2], keep = upper ? v[j + n / 2] : v[j];
          v[j] = keep + __shfl_xor(give, bit);
        }
      mine += upper ? n / 2 : 0;
      bit *= 2;
    }
  }
  holds = lane < bit;
  for (; bit < team; bit *= 2) v[0] += __shfl_xor(v[0], bit);
}

// Backwards: step r of a chunk is step steps - 1 - r of the sequence.
// Where neighbouring channels share a gate, teams of `team` lanes (at least as many as steps) add their slopes up: `slopes`
// then has one value per team and step, [slope_rows][steps][teams a row].
template <typename T, typename G, GateKind K, int V, int L>
__global__ __launch_bounds__(kLanes* kMaxSlots) void scan_grad_kernel(ScanGradArgs a, Cut k, uint64_t* work, int64_t slopes, GateSums sums) {
  typedef Wide<T> W;
  int64_t tile, row;
  take_tile(k, work, tile, row);
  const int lane = threadIdx.x % k.lanes, slot = threadIdx.x / k.lanes;
  const int64_t pack = row * k.lanes + lane;
  const bool live = pack < k.packs;
  const Channels<V> at(live ? pack : 0, a.width);
  const int64_t b = at.b, d = at.d, c = b * a.width + d;
  const int64_t t0 = a.steps - 1 - (tile * k.slots + slot) * L, len = live ? length_of(a.lengths, b, a.steps) : 0;
  const T* dh = (const T*)a.grad_states + b * a.g_b + d;
  const T* hs = (const T*)a.states + b * a.h_b + d;
  const T* x = (const T*)a.x + b * a.x_b + d;
  const GateRow<G, K, V> gate(a.gate, b, a.gate_b, a.gate_t, d, K == kSharedGate ? a.width / a.groups : 1);
  Pack<T, V> gs[L], before[L], xs[L];
  Pack<G, V> as[L];
  if (__all(t0 < len && t0 - L >= 0)) {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      gs[j] = load_pack<T, V>(dh + (t0 - j) * a.g_t);
      if constexpr (K != kNoGate) {
        before[j] = load_pack<T, V>(hs + (t0 - j - 1) * a.h_t);
        if (a.mix) xs[j] = load_pack<T, V>(x + (t0 - j) * a.x_t);
      }
    }
    gate.template load_steps<-1>(t0, as);
  } else {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const int64_t t = t0 - j;
      gs[j] = before[j] = xs[j] = constant<T, V>(0);
      as[j] = constant<G, V>(1);
      if (t >= 0 && t < len) {
        gs[j] = load_pack<T, V>(dh + t * a.g_t);
        as[j] = gate.load(t);
        if constexpr (K != kNoGate) {
          if (t > 0) before[j] = load_pack<T, V>(hs + (t - 1) * a.h_t);
          if (a.mix) xs[j] = load_pack<T, V>(x + t * a.x_t);
        }
      }
    }
  }
  W e[V], first[V];
  for (int v = 0; v < V; ++v) first[v] = a.grad_last && live ? ((const W*)a.grad_last)[c + v] : (W)0;
  if (k.tiles > 1 || k.slots > 1) {
    Map<W, K != kNoGate> own[V];
    for (int v = 0; v < V; ++v) own[v] = no_steps<W, K != kNoGate>();
#pragma unroll
    for (int j = 0; j < L; ++j)
      for (int v = 0; v < V; ++v) {
        own[v].h += (W)gs[j].v[v];
        if constexpr (K != kNoGate) {
          const W g = (W)as[j].v[v];
          own[v].h *= g;
          own[v].m *= mantissa(g);
          own[v].e += exponent(g);
        }
      }
    for (int v = 0; v < V; ++v) own[v] = normal(own[v]);
    as_loaded(gs);
    if constexpr (K != kNoGate) as_loaded(as);
    carry_in<W, V, K != kNoGate>(k, work, tile, row, lane, slot, own, first, e);
  } else {
    for (int v = 0; v < V; ++v) e[v] = first[v];
  }
  if (!live && (K != kSharedGate || !sums.team)) return;
  T* dx = (T*)a.grad_x + b * a.steps * a.width + d;
  G* da = (G*)a.grad_gate + b * a.steps * a.width + d;
  W* slope = (W*)slopes + b * a.steps * a.width + d;
  W total[L];
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const int64_t t = t0 - j;
    Pack<T, V> o;
    Pack<G, V> og;
    Pack<W, V> os;
    for (int v = 0; v < V; ++v) {
      const W cc = (W)gs[j].v[v] + e[v];
      W value = cc;
      if constexpr (K == kNoGate) {
        e[v] = cc;
      } else {
        const W g = (W)as[j].v[v];
        W from = t == 0 ? (a.state ? ((const W*)a.state)[c + v] : (W)0) : (W)before[j].v[v];
        if (a.mix) {
          from -= (W)xs[j].v[v];
          value *= (W)1 - g;
        }
        os.v[v] = t < len ? cc * from : (W)0;
        og.v[v] = (G)os.v[v];
        e[v] = g * cc;
      }
      o.v[v] = t < len ? (T)value : (T)(W)0;
    }
    if (t >= 0 && live) {
      store_pack<T, V>(dx + t * a.width, o);
      if constexpr (K != kNoGate) {
        if (K != kSharedGate || !sums.team) {
          if (slopes) store_pack<W, V>(slope + t * a.width, os);
          else store_pack<G, V>(da + t * a.width, og);
        }
      }
    }
    if constexpr (K == kSharedGate) {
      total[j] = 0;
      for (int v = 0; v < V; ++v) total[j] += live && v >= at.again ? os.v[v] : (W)0;
    }
  }
  if constexpr (K == kSharedGate) {
    if (sums.team) {
      int mine;
      bool holds;
      team_sums<W, L>(total, sums.team, mine, holds);
      const int64_t t = t0 - mine, part = pack / sums.team, r = part / sums.teams;
      if (holds && t >= 0 && r < sums.rows) {
        const int64_t to = (r * a.steps + t) * sums.teams + part - r * sums.teams;
        if (sums.done) ((G*)a.grad_gate)[to] = (G)total[0];
        else ((W*)slopes)[to] = total[0];
      }
    }
    if (!live) return;
  }
  if (tile == k.tiles - 1 && slot == k.slots - 1)
    for (int v = 0; v < V; ++v) ((W*)a.grad_state)[c + v] = e[v];
}

// grad_gate[q][t][g] = sum of the slopes of the sequences and channels that share the gate, in a fixed order: `team` lanes
// (one where a group is one channel, a wave, or the workgroup where more than kWaveTerms share a gate) side by side, then a tree.
constexpr int64_t kWaveTerms = 2048;

template <typename W, typename G, int kTeam>
__global__ __launch_bounds__(kThreads) void gate_sum_kernel(const W* __restrict__ slope, G* __restrict__ out, int64_t batch, int64_t steps,
                                                            int64_t width, int64_t groups, int64_t gate_batch) {
  __shared__ W part[kThreads / 64];
  const int64_t per = width / groups, shared = gate_batch == batch ? 1 : batch, sums = gate_batch * steps * groups;
  const int lane = threadIdx.x % kTeam;
  for (int64_t base = (int64_t)blockIdx.x * (kThreads / kTeam); base < sums; base += (int64_t)gridDim.x * (kThreads / kTeam)) {
    const int64_t o = base + threadIdx.x / kTeam;
    W sum = 0;
    if (o < sums) {
      const int64_t qt = o / groups, g = o - qt * groups, q = qt / steps, t = qt - q * steps;
      for (int64_t b = q; b < q + shared; ++b) {
        const W* row = slope + (b * steps + t) * width + g * per;
#pragma unroll 4
        for (int64_t d = lane; d < per; d += kTeam) sum += row[d];
      }
    }
    if constexpr (kTeam > 1)
      for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    if constexpr (kTeam > 64) {
      if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = sum;
      __syncthreads();
      sum = 0;
      for (int w = 0; w < kThreads / 64; ++w) sum += part[w];
      __syncthreads();
    }
    if (lane == 0 && o < sums) out[o] = (G)sum;
  }
}

// Two channels a lane for the types of up to 32 bits.
template <typename A> bool two_wide(const A& a) { return a.type != kF64 && a.width >= 2; }

Cut cut_steps(int64_t batch, int64_t steps, int64_t width, int v, int per_lane, int max_slots) {
  Cut k;
  k.packs = batch * ((width + v - 1) / v);
  k.lanes = kLanes;
  while (k.lanes > 1 && k.lanes / 2 >= k.packs) k.lanes /= 2;
  const int64_t chunks = std::max<int64_t>(1, (steps + per_lane - 1) / per_lane);
  k.slots = 1;
  while (k.slots < max_slots && k.slots < chunks) k.slots *= 2;
  k.slots = std::min(k.slots, max_slots);
  k.tiles = (chunks + k.slots - 1) / k.slots;
  if (k.tiles == 1 && k.slots == 1) k.lanes = k.packs >= kThreads ? kThreads : k.lanes;
  k.pack_rows = (k.packs + k.lanes - 1) / k.lanes;
  // Close checkpoints leave little to fold, far ones make a short chain of tiles that wait for one another; with many rows
  // of tiles the chain has time.  bf16, every 8 against every 32 tiles, forward and backward: 1 row of 65537 steps 111 / 145 against
  // 47 / 58 us, 8 x 48828 99 / 151 against 86 / 126, 16 x 24414 84 / 124 against 83 / 115, 31 x 12600 82 / 112 against 84 / 111,
  // 64 x 6103 76 / 106 against 79 / 111, 160 x 2441 72 / 106 against 76 / 110.
  k.checkpoint = k.pack_rows >= 32 ? 8 : 32;
  if (k.tiles * k.pack_rows * k.lanes * k.slots > 4294967295LL) throw std::runtime_error("gated_scan: the tensor is too large");
  return k;
}

// Chunks of a tile forwards.  Two workgroups of 8 chunks a CU overlap loads with sums better than one of 16 where there are many
// rows of tiles; few rows rather have fewer maps to fold, unless there are few steps in all (bf16, 8 against 16 chunks: 8 rows of 16384
// steps 44 against 38 us, 32 x 4096 37 against 33, 128 x 1024 34 against 31, 64 x 16384 184 against 192, 160 x 4096 112 against 125,
// 24 x 1024 16.5 against 18.0; with fp32 gates, in fp32 and in fp64 the two change places at the same sizes or, for fp32 gates, at
// 48 rows).  Up to kMaxSlots chunks are one tile, which needs neither a workspace nor tickets.
int scan_slots(const ScanArgs& a, int v) {
  const int64_t rows = (a.batch * ((a.width + v - 1) / v) + kLanes - 1) / kLanes;
  return a.steps > kMaxSlots * kScanSteps && (rows >= 160 || (rows >= 64 && a.steps >= 4096) || rows * a.steps <= 32768) ? 8 : kMaxSlots;
}

// Backwards: values of 16 bits leave room for 16 steps a lane in 128 registers (8 x 4096 x 2560 bf16: 277 us with 16 steps and 8
// chunks, 299 us with 8 and 16); of fp32 (1 x 423 x 26734: 69 against 109 us) and fp64 they do not.
constexpr int grad_steps(int64_t type) { return type == kBf16 || type == kF16 ? 16 : 8; }
constexpr int grad_slots(int64_t type) { return type == kBf16 || type == kF16 ? 8 : kMaxSlots; }

template <typename A> void check_args(const A& a) {
  if (a.batch < 0 || a.steps < 0 || a.width < 0) throw std::runtime_error("gated_scan: a negative size");
  if (a.steps > 2147483647LL) throw std::runtime_error("gated_scan: the tensor is too large");
  if (a.gate && (a.groups <= 0 || a.width % a.groups)) throw std::runtime_error("gated_scan: the width is not a multiple of the gate's groups");
}

// type and gate_type -> template arguments
template <typename F> auto by_types(int64_t type, int64_t gate_type, bool gate, F f) {
  if (!gate) gate_type = type;
  if (type == kBf16 && gate_type == kBf16) return f((__bf16)0, (__bf16)0);
  if (type == kBf16 && gate_type == kF32) return f((__bf16)0, (float)0);
  if (type == kF16 && gate_type == kF16) return f((_Float16)0, (_Float16)0);
  if (type == kF16 && gate_type == kF32) return f((_Float16)0, (float)0);
  if (type == kF32 && gate_type == kF32) return f((float)0, (float)0);
  if (type == kF64 && gate_type == kF64) return f((double)0, (double)0);
  throw std::runtime_error("gated_scan: unknown pair of types");
}

template <int N> struct Const { static constexpr int value = N; };

// f(gate kind, channels a lane, steps a lane)
template <bool Two, int Steps, typename A, typename F> void by_shape(const A& a, F f) {
  auto with_kind = [&](auto kind) {
    if constexpr (Two) {
      if (two_wide(a)) return a.steps <= 1 ? f(kind, Const<2>(), Const<1>()) : f(kind, Const<2>(), Const<Steps>());
    }
    return a.steps <= 1 ? f(kind, Const<1>(), Const<1>()) : f(kind, Const<1>(), Const<Steps>());
  };
  if (!a.gate) with_kind(Const<kNoGate>());
  else if (a.groups == a.width) with_kind(Const<kOwnGate>());
  else with_kind(Const<kSharedGate>());
}

template <typename W> size_t fold_bytes(const Cut& k, int v, bool gates) {
  return k.tiles * k.slots == 1 ? 0 : 2 * k.slots * k.lanes * v * (gates ? sizeof(Map<W, true>) : sizeof(Map<W, false>));
}

template <typename W> void clear_work(const Cut& k, int v, bool gates, uint64_t* work, hipStream_t s) {
  const int64_t n = work_words<W>(k, v, gates);
  if (!n) return;
  hipLaunchKernelGGL(fill_words_kernel, dim3((unsigned)std::min<int64_t>((n / 2 + kThreads - 1) / kThreads, 2048)), dim3(kThreads), 0, s, (uint4*)work, n / 2);
  LGA_HIP_CHECK(hipGetLastError());
}

bool sums_gates(const ScanGradArgs& a) { return a.gate && (a.groups != a.width || a.gate_batch != a.batch); }

// Teams of at least 8 lanes, and as many as a lane holds steps, within a gate group (or, with one gate a step for everything, over all lanes) sum up in the
// backward kernel; a group like 103 channels has none, and its slopes go through memory value by value.
GateSums gate_sums(const ScanGradArgs& a, const Cut& k, int v, int per_lane) {
  GateSums g;
  if (!sums_gates(a) || a.groups == a.width) return g;
  const int64_t per = a.width / a.groups;
  const int most = std::min(k.lanes, 64);
  int team = 0;
  if (a.groups == 1 && a.gate_batch == 1) {
    team = most;
    g.teams = (k.packs + team - 1) / team;
  } else if (per % v == 0) {
    team = 1;
    while (team < most && per / v % (team * 2) == 0) team *= 2;
    g.rows = a.batch;
    g.teams = a.width / v / team;
    g.done = per / v == team && a.gate_batch == a.batch;
  }
  g.team = team >= std::max(8, per_lane) ? team : 0;
  if (!g.team) return GateSums{};
  if (a.groups == 1 && a.gate_batch == 1 && g.teams == 1) g.done = 1;
  return g;
}

int64_t slope_values(const ScanGradArgs& a, const GateSums& g) {
  if (!sums_gates(a) || g.done) return 0;
  return g.team ? g.rows * a.steps * g.teams : a.batch * a.steps * a.width;
}

}  // namespace

int64_t scan_workspace(const ScanArgs& a) {
  check_args(a);
  const int v = two_wide(a) ? 2 : 1;
  const Cut k = cut_steps(a.batch, a.steps, a.width, v, a.steps <= 1 ? 1 : kScanSteps, scan_slots(a, v));
  return 8 * (a.type == kF64 ? work_words<double>(k, v, a.gate != 0) : work_words<float>(k, v, a.gate != 0));
}

void gated_scan(const ScanArgs& a) {
  check_args(a);
  if (a.batch * a.width == 0) return;
  DeviceScope scope(a.device);
  by_types(a.type, a.gate_type, a.gate != 0, [&](auto tt, auto gg) {
    typedef decltype(tt) T;
    typedef decltype(gg) G;
    by_shape<sizeof(T) < 8, kScanSteps>(a, [&](auto kind, auto v, auto l) {
      constexpr int V = decltype(v)::value, L = decltype(l)::value;
      const Cut k = cut_steps(a.batch, a.steps, a.width, V, L, scan_slots(a, V));
      clear_work<Wide<T>>(k, V, a.gate != 0, (uint64_t*)a.work, (hipStream_t)a.stream);
      hipLaunchKernelGGL((scan_kernel<T, G, (GateKind)decltype(kind)::value, V, L>), dim3((unsigned)(k.tiles * k.pack_rows)), dim3(k.lanes * k.slots),
                         fold_bytes<Wide<T>>(k, V, a.gate != 0), (hipStream_t)a.stream, a, k);
      LGA_HIP_CHECK(hipGetLastError());
    });
  });
}

int64_t scan_grad_workspace(const ScanGradArgs& a) {
  check_args(a);
  const int v = two_wide(a) ? 2 : 1;
  const int steps = a.steps <= 1 ? 1 : grad_steps(a.type);
  const Cut k = cut_steps(a.batch, a.steps, a.width, v, steps, grad_slots(a.type));
  return 8 * (a.type == kF64 ? work_words<double>(k, v, a.gate != 0) : work_words<float>(k, v, a.gate != 0)) + slope_values(a, gate_sums(a, k, v, steps)) * (a.type == kF64 ? 8 : 4);
}

void gated_scan_grad(const ScanGradArgs& a) {
  check_args(a);
  if (a.batch * a.width == 0) return;
  DeviceScope scope(a.device);
  by_types(a.type, a.gate_type, a.gate != 0, [&](auto tt, auto gg) {
    typedef decltype(tt) T;
    typedef decltype(gg) G;
    typedef Wide<T> W;
    const hipStream_t s = (hipStream_t)a.stream;
    by_shape<sizeof(T) < 8, sizeof(T) == 2 ? grad_steps(kBf16) : grad_steps(kF32)>(a, [&](auto kind, auto v, auto l) {
      constexpr int V = decltype(v)::value, L = decltype(l)::value;
      const Cut k = cut_steps(a.batch, a.steps, a.width, V, L, grad_slots(a.type));
      uint64_t* work = (uint64_t*)a.work;
      clear_work<W>(k, V, a.gate != 0, work, s);
      const GateSums g = gate_sums(a, k, V, L);
      const int64_t slopes = slope_values(a, g) ? (int64_t)(work + work_words<W>(k, V, a.gate != 0)) : 0;
      hipLaunchKernelGGL((scan_grad_kernel<T, G, (GateKind)decltype(kind)::value, V, L>), dim3((unsigned)(k.tiles * k.pack_rows)), dim3(k.lanes * k.slots),
                         fold_bytes<W>(k, V, a.gate != 0), s, a, k, work, slopes, g);
      LGA_HIP_CHECK(hipGetLastError());
      if (slopes) {
        // the slopes, or the teams' sums of them: [rows][steps][across]
        const int64_t rows = g.team ? g.rows : a.batch, across = g.team ? g.teams : a.width;
        const int64_t sums = a.gate_batch * a.steps * a.groups, terms = across / a.groups * (rows / std::min(rows, a.gate_batch));
        auto run = [&](auto kernel, int64_t team) {
          hipLaunchKernelGGL(kernel, dim3((unsigned)std::min<int64_t>((sums * team + kThreads - 1) / kThreads, 1 << 20)), dim3(kThreads), 0, s,
                             (const W*)slopes, (G*)a.grad_gate, rows, a.steps, across, a.groups, a.gate_batch);
        };
        if (across == a.groups) run(gate_sum_kernel<W, G, 1>, 1);
        else if (terms <= kWaveTerms) run(gate_sum_kernel<W, G, 64>, 64);
        else run(gate_sum_kernel<W, G, kThreads>, kThreads);
        LGA_HIP_CHECK(hipGetLastError());
      }
    });
  });
}

}  // namespace lga
