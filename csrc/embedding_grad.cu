// Scaled embedding lookup, and the gradient of its table by sorted tokens.
//
//   y_t = s E[i_t]          dE[v] = s * sum of dy_t over the tokens t with i_t = v
//
// Memory bound: the lookup reads and writes T rows; the gradient reads dy once
// and writes the whole table, or reads and writes the touched rows when it adds
// to a gradient that is there.
//
// Adding rows of dy with atomics would make the result depend on timing and, in
// bf16, round at every addition.  The tokens are sorted by id instead (ties by
// position), every row's tokens are then a run of the sorted list, and each run
// is added in fp32 in token order and rounded once.
//  * Sort: 1024 tokens at a time, one per thread (bitonic; shuffles within a warp,
//    shared memory across); a token's place in the whole is its place in its own
//    chunk plus the number of smaller ids in every other chunk (a binary search
//    each, the chunks shared out over a block's warps).  Two launches and no
//    counters, for any number of tokens; the searches grow with the square of the
//    tokens (5 us of 32 at 8192, 104 of 180 at 131072, 5.7 of 6.0 ms at a million,
//    each 256 columns wide).
//  * Long runs (one id over thousands of tokens, as padding makes them): aligned
//    groups of 32 equal tokens, and of 32 such groups, are added first, all at
//    once, and a run then adds those sums: at most 62 tokens, 62 groups and its
//    large groups one after the other.
//  * Rows: one kernel for rows of at most one token (most of them), one for rows
//    of several, where runs start.  A warp takes a few rows (or places of the
//    sorted list) and a slab of columns, neighbouring warps neighbouring slabs:
//    blocks write contiguous memory, and the chains of dependent loads that bound
//    a row run beside one another.
//
// Measured on a B200: 8192 tokens x 4096 bf16, table of 151936 rows: lookup 23 us,
// sort and places 14 us, table 193 us (6.5 TB/s), runs and groups 32 us.  24571
// tokens x 1001 fp32 (two fifths one id) into 50001 rows: lookup 39 us, sort 12 us,
// groups 23 us, single rows 23 us, runs 33 us.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <stdexcept>

#include "sm100_common.cuh"
#include "vec_types.cuh"

namespace gb {

namespace {

constexpr int kSortKeys = 1024;       // tokens per sorted chunk, one per thread
constexpr int kGroup = 32;            // tokens of a pre-added group, and groups of a large one
constexpr int kGroupFrom = 128;       // tokens from which groups are worth their launch
constexpr int kLargeFrom = 4096;      // ... and large groups theirs
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTableRows = 8;         // table rows per warp
constexpr int kListRows = 28;         // sorted places per warp at most: a lane each, and one on either side
template <int N>
constexpr int kLookup = N == 1 ? 16 : 8;  // packs per thread of the lookup,
constexpr int kLookupBlocks = 4;          // whose blocks stay on their SM
constexpr unsigned kNoId = 0xffffffffu;  // sorts last: no row takes it
constexpr unsigned kAll = 0xffffffffu;

// Packs per lane of a slab, and rows of it in flight.
template <int N>
constexpr int kSlab = N == 1 ? 4 : 1;
constexpr int kFlight = 8;       // tokens: 32 registers of loads
constexpr int kSumFlight = 4;    // sums of groups, which are fp32 for every type

// y[t] = scale * table[id]; NaN for an id outside the table.  `lanes` threads a row.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, kLookupBlocks) embed_fwd_kernel(const int64_t* __restrict__ ids, long tokens, long V,
                                                             const T* __restrict__ table, long ldt, int H, float scale,
                                                             T* __restrict__ y, int lanes, int* __restrict__ err) {
  constexpr int N = kPackSize<T, WIDE>;
  const int per_block = kThreads / lanes;
  const int lane = threadIdx.x % lanes;
  const int packs = H / N;
  const long step = gridDim.x * static_cast<long>(per_block);
  long t = blockIdx.x * static_cast<long>(per_block) + threadIdx.x / lanes;
  long next = t < tokens ? ids[t] : 0;   // a row's id is there before its turn
  for (; t < tokens; t += step) {
    const long id = next;
    if (t + step < tokens) next = ids[t + step];
    const bool ok = id >= 0 && id < V;
    if (!ok && lane == 0) atomicExch(err + 1, kErrBadToken);
    const T* src = table + (ok ? id : 0) * ldt;
    T* dst = y + t * H;
    for (int p0 = lane; p0 < packs; p0 += kLookup<N> * lanes) {
      Pack<T, N> k[kLookup<N>];
#pragma unroll
      for (int u = 0; u < kLookup<N>; ++u)
        if (p0 + u * lanes < packs) k[u] = load_raw<T, N>(src + static_cast<long>(p0 + u * lanes) * N);
#pragma unroll
      for (int u = 0; u < kLookup<N>; ++u)
        if (p0 + u * lanes < packs) {
          float f[N];
#pragma unroll
          for (int i = 0; i < N; ++i) f[i] = ok ? value(k[u], i) * scale : __int_as_float(0x7fc00000);
          store_pack<T, N>(dst + static_cast<long>(p0 + u * lanes) * N, f);
        }
    }
  }
}

// One step of the bitonic network on a key per thread: with the key `gap` threads
// away, the lower thread of an ascending pair keeps the smaller one.
template <int SPAN, int GAP, typename Key>
__device__ __forceinline__ Key sort_step(Key k, Key (&s)[2][kSortKeys], int& flip) {
  const int t = threadIdx.x;
  Key other;
  if constexpr (GAP >= 32) {
    s[flip][t] = k;
    __syncthreads();
    other = s[flip][t ^ GAP];
    flip ^= 1;  // the next step writes the other buffer: its readers are past this barrier
  } else {
    other = __shfl_xor_sync(kAll, k, GAP);
  }
  const bool keep_small = ((t & SPAN) == 0) == ((t & GAP) == 0);
  k = keep_small ? min(k, other) : max(k, other);
  if constexpr (GAP > 1) k = sort_step<SPAN, GAP / 2>(k, s, flip);
  return k;
}

template <int SPAN, typename Key>
__device__ __forceinline__ Key sort_keys(Key k, Key (&s)[2][kSortKeys], int& flip, int size) {
  k = sort_step<SPAN, SPAN / 2>(k, s, flip);
  if constexpr (SPAN < kSortKeys)
    if (SPAN < size) k = sort_keys<2 * SPAN>(k, s, flip, size);
  return k;
}

// Sorted chunks of (id, place in the chunk).  Padding ids, and ids outside the
// table (reported unless they are `ignore`), become the largest id, kNoId in the
// output.
template <typename Key>
__global__ void __launch_bounds__(kSortKeys) embed_sort_kernel(const int64_t* __restrict__ ids, long tokens, long V,
                                                               long padding, long ignore,
                                                               unsigned* __restrict__ id_out,
                                                               int* __restrict__ token_out, int* __restrict__ err) {
  constexpr int kPlaceBits = 10;
  constexpr Key kNone = ~Key(0) >> kPlaceBits;
  static_assert(1 << kPlaceBits == kSortKeys, "a place fits its bits");
  __shared__ Key s[2][kSortKeys];
  const long base = static_cast<long>(blockIdx.x) * kSortKeys;
  const int n = static_cast<int>(min(tokens - base, static_cast<long>(kSortKeys)));
  const int t = threadIdx.x;
  Key k = ~Key(0);  // past the end: after every token
  if (t < n) {
    const long id = ids[base + t];
    Key u = kNone;
    if (id >= 0 && id < V) {
      if (id != padding) u = static_cast<Key>(id);
    } else if (id != ignore) {
      atomicExch(err + 1, kErrBadToken);
    }
    k = u << kPlaceBits | static_cast<Key>(t);
  }
  int flip = 0;
  k = sort_keys<2>(k, s, flip, n);  // the network of the next power of two
  if (t < n) {
    const Key id = k >> kPlaceBits;
    id_out[base + t] = id == kNone ? kNoId : static_cast<unsigned>(id);
    token_out[base + t] = static_cast<int>(base + static_cast<long>(k & (kSortKeys - 1)));
  }
}

// Place of every token among all chunks: ids of earlier chunks come before equal
// ids, those of later chunks after.  A block takes 32 tokens; its warps share out
// the other chunks, four at a time, so that their loads do not wait for one another.
__global__ void __launch_bounds__(kThreads) embed_merge_kernel(const unsigned* __restrict__ id,
                                                               const int* __restrict__ token, int tokens,
                                                               unsigned* __restrict__ id_out,
                                                               int* __restrict__ token_out) {
  __shared__ int before[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  const bool live = i < tokens;
  const unsigned k = live ? id[i] : 0;
  const int own = blockIdx.x * 32 / kSortKeys;
  const int chunks = (tokens + kSortKeys - 1) / kSortKeys;
  int place = 0;
  for (int c0 = warp; c0 < chunks; c0 += 4 * kWarps) {
    int lo[4], n[4];
    const unsigned* at[4];
    bool equal[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + u * kWarps;
      at[u] = id + static_cast<long>(c) * kSortKeys;
      n[u] = live && c < chunks && c != own ? min(tokens - c * kSortKeys, kSortKeys) : 0;
      equal[u] = c < own;
      lo[u] = 0;
    }
#pragma unroll
    for (int step = kSortKeys; step > 0; step >>= 1) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (lo[u] + step <= n[u]) {
          const unsigned v = at[u][lo[u] + step - 1];
          if (v < k || (equal[u] && v == k)) lo[u] += step;
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) place += lo[u];
  }
  before[warp][lane] = place;
  __syncthreads();
  if (warp == 0 && live) {
    place = i - own * kSortKeys;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) place += before[w][lane];
    id_out[place] = k;
    token_out[place] = token[i];
  }
}

// start[v] = first place of the sorted list whose id is not below v, v = 0 .. V.
__global__ void __launch_bounds__(kThreads) embed_start_kernel(const unsigned* __restrict__ id, int tokens, int V,
                                                               int* __restrict__ start) {
  const int v = blockIdx.x * kThreads + threadIdx.x;
  if (v > V) return;
  int lo = 0, hi = tokens;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (id[mid] < static_cast<unsigned>(v)) lo = mid + 1;
    else hi = mid;
  }
  start[v] = lo;
}

// First place in [lo, hi) whose id is not below `id`; a whole warp calls it.
__device__ __forceinline__ int lower_bound_warp(const unsigned* __restrict__ ids, int lo, int hi, unsigned id) {
  const int lane = threadIdx.x & 31;
  while (hi - lo > 32) {
    const int step = (hi - lo + 32) / 33;
    const int at = lo + (lane + 1) * step - 1;
    const bool below = at < hi && ids[at] < id;
    const int k = __popc(__ballot_sync(kAll, below));
    hi = min(hi, lo + (k + 1) * step - (k < 32 ? 1 : 0));
    lo = lo + k * step;
  }
  const bool below = lo + lane < hi && ids[lo + lane] < id;
  return lo + __popc(__ballot_sync(kAll, below));
}

struct GradRows {
  const void* dy;
  long ld;             // row stride of dy
  const unsigned* id;  // sorted
  const int* token;
  const float* group;  // [tokens / 32][ldg] sums of whole groups, null without them
  const float* large;  // [tokens / 1024][ldg]
  const int* start;    // [V + 1]; the whole table only
  long ldg;
  int tokens, V, H;
  unsigned slabs;      // of columns
  int places;          // sorted places per warp
  float scale;
  void* out;
};

// acc[s] += row(j) at pack p0 + 32 s, j = lo .. hi - 1 in order.  U rows are in
// flight; `row` gives a row's address.
template <typename T, int N, int S, int U, typename Row>
__device__ __forceinline__ void add_rows(float (&acc)[S][N], int lo, int hi, int p0, int packs, Row&& row) {
  int j = lo;
#pragma unroll 1
  for (; j + U <= hi; j += U) {
    Pack<T, N> k[U][S];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* src = row(j + u);
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (p0 + 32 * s < packs) k[u][s] = load_raw<T, N>(src + static_cast<long>(p0 + 32 * s) * N);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (p0 + 32 * s < packs)
#pragma unroll
          for (int i = 0; i < N; ++i) acc[s][i] += value(k[u][s], i);
  }
#pragma unroll 1
  for (; j < hi; ++j) {
    const T* src = row(j);
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (p0 + 32 * s < packs) {
        const Pack<T, N> k = load_raw<T, N>(src + static_cast<long>(p0 + 32 * s) * N);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[s][i] += value(k, i);
      }
  }
}

template <typename T, int U, int N, int S>
__device__ __forceinline__ void add_tokens(float (&acc)[S][N], const GradRows& g, int lo, int hi, int p0, int packs) {
  // 32 tokens' positions at once, one per lane
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int mine = j0 + lane < hi ? g.token[j0 + lane] : 0;
    add_rows<T, N, S, U>(acc, j0, min(hi, j0 + 32), p0, packs, [&](int j) {
      return static_cast<const T*>(g.dy) + __shfl_sync(kAll, mine, j - j0) * g.ld;
    });
  }
}

template <int U, int N, int S>
__device__ __forceinline__ void add_sums(float (&acc)[S][N], const float* sums, long ld, int lo, int hi, int p0,
                                         int packs) {
  add_rows<float, N, S, U>(acc, lo, hi, p0, packs, [&](int j) { return sums + j * ld; });
}

// A row's slab: scaled, added to what is there (ADD), and stored.
template <typename O, bool ADD, int N, int S>
__device__ __forceinline__ void store_row(const float (&acc)[S][N], float scale, O* out, int p0, int packs) {
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (p0 + 32 * s < packs) {
      O* at = out + static_cast<long>(p0 + 32 * s) * N;
      float f[N] = {};
      if constexpr (ADD) load_pack<O, N>(at, f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] += acc[s][i] * scale;
      store_pack<O, N>(at, f);
    }
}

// The same for a row of at most one token, token[a] where there is one.
template <typename T, typename O, bool ADD, int N, int S>
__device__ __forceinline__ void put_row(const GradRows& g, int a, bool some, int p0, int packs, O* out) {
  float acc[S][N] = {};
  if (some) {
    const T* src = static_cast<const T*>(g.dy) + g.token[a] * g.ld;
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (p0 + 32 * s < packs) load_pack<T, N>(src + static_cast<long>(p0 + 32 * s) * N, acc[s]);
  }
  store_row<O, ADD>(acc, g.scale, out, p0, packs);
}

// A warp's work: its item (a group, some rows or places) and its first pack.
// Neighbouring warps take neighbouring slabs of an item.
struct WarpWork {
  long item;
  int pack;
};

template <int S>
__device__ __forceinline__ WarpWork warp_work(const GradRows& g) {
  const long w = blockIdx.x * static_cast<long>(kWarps) + (threadIdx.x >> 5);
  const long item = w / g.slabs;
  return {item, static_cast<int>(w - item * g.slabs) * 32 * S + static_cast<int>(threadIdx.x & 31)};
}

// Sums of the whole groups (LARGE: of the whole groups of groups) of one id.
template <typename T, bool WIDE, bool LARGE>
__global__ void __launch_bounds__(kThreads, 3) embed_group_kernel(const GradRows g, int groups, float* __restrict__ out) {
  constexpr int N = kPackSize<T, WIDE>, S = kSlab<N>;
  const WarpWork w = warp_work<S>(g);
  if (w.item >= groups) return;
  const int group = static_cast<int>(w.item), p0 = w.pack;
  const int lo = group * (LARGE ? kGroup * kGroup : kGroup);
  const unsigned id = g.id[lo];
  if (id == kNoId || id != g.id[lo + (LARGE ? kGroup * kGroup : kGroup) - 1]) return;
  const int packs = g.H / N;
  float acc[S][N] = {};
  if constexpr (LARGE) add_sums<kSumFlight>(acc, g.group, g.ldg, group * kGroup, (group + 1) * kGroup, p0, packs);
  else add_tokens<T, kFlight>(acc, g, lo, lo + kGroup, p0, packs);
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (p0 + 32 * s < packs) store_pack<float, N>(out + group * g.ldg + static_cast<long>(p0 + 32 * s) * N, acc[s]);
}

// The whole table but for rows of several tokens: a warp writes kTableRows rows'
// slabs, zeros where no token is.  (Rows of several tokens in the same kernel
// made it spill, and the spills of mostly empty rows were more traffic than the
// rows.)
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) embed_table_kernel(const GradRows g) {
  constexpr int N = kPackSize<T, WIDE>, S = kSlab<N>;
  const int lane = threadIdx.x & 31;
  const int packs = g.H / N;
  const WarpWork w = warp_work<S>(g);
  const long v0 = w.item * kTableRows;
  if (v0 >= g.V) return;
  const int rows = static_cast<int>(min(static_cast<long>(kTableRows), g.V - v0));
  const int p0 = w.pack;
  const int bound = lane <= rows ? g.start[v0 + lane] : 0;
  for (int r = 0; r < rows; ++r) {
    const int a = __shfl_sync(kAll, bound, r), b = __shfl_sync(kAll, bound, r + 1);
    if (b - a < 2) put_row<T, T, false, N, S>(g, a, a < b, p0, packs, static_cast<T*>(g.out) + (v0 + r) * g.H);
  }
}

// The sorted places that a warp takes: bit l of `starts` where a run starts at
// place j0 - 1 + l, of one token (`single`) or of several.
struct Places {
  unsigned near;   // id of place j0 - 1 + lane
  int j0;
  unsigned single, several;
};

__device__ __forceinline__ Places places_of(const GradRows& g, long item) {
  Places p;
  const int lane = threadIdx.x & 31;
  p.j0 = static_cast<int>(item) * g.places;
  const int at = p.j0 - 1 + lane;
  p.near = at >= 0 && at < g.tokens ? g.id[at] : kNoId;
  const unsigned before = __shfl_up_sync(kAll, p.near, 1), after = __shfl_down_sync(kAll, p.near, 1);
  const bool start = lane >= 1 && lane <= g.places && p.near != kNoId && (at == 0 || before != p.near);
  p.single = __ballot_sync(kAll, start && after != p.near);
  p.several = __ballot_sync(kAll, start && after == p.near);
  return p;
}

// Adds rows of one token to an existing gradient.
template <typename T, typename O, bool WIDE>
__global__ void __launch_bounds__(kThreads) embed_single_kernel(const GradRows g) {
  constexpr int N = kPackSize<T, WIDE>, S = kSlab<N>;
  const WarpWork w = warp_work<S>(g);
  if (w.item * g.places >= g.tokens) return;
  const Places at = places_of(g, w.item);
  for (unsigned todo = at.single; todo != 0; todo &= todo - 1) {
    const int l = __ffs(todo) - 1;
    const unsigned id = __shfl_sync(kAll, at.near, l);
    put_row<T, O, true, N, S>(g, at.j0 - 1 + l, true, w.pack, g.H / N,
                              static_cast<O*>(g.out) + static_cast<long>(id) * g.H);
  }
}

// Rows of several tokens: tokens up to the first whole group, groups up to the
// first large one, large groups, and back.  A warp takes the runs that start in
// its sorted places, the last places first: a padding token is mostly one of the
// last ids, and its run, the longest chain, must not be the last work.
template <typename T, typename O, bool ADD, bool WIDE>
__global__ void __launch_bounds__(kThreads, 2) embed_run_kernel(const GradRows g) {
  constexpr int N = kPackSize<T, WIDE>, S = kSlab<N>;
  const WarpWork w = warp_work<S>(g);
  const int items = (g.tokens + g.places - 1) / g.places;
  if (w.item >= items) return;
  const Places at = places_of(g, items - 1 - w.item);
  const int packs = g.H / N, p0 = w.pack;
#pragma unroll 1
  for (unsigned todo = at.several; todo != 0; todo &= todo - 1) {
    const int l = __ffs(todo) - 1, j = at.j0 - 1 + l;
    const unsigned id = __shfl_sync(kAll, at.near, l);
    // lanes from this place on that hold the id; up to the last lane: search on
    const int lane = threadIdx.x & 31;
    const unsigned same = __ballot_sync(kAll, at.near == id && lane >= l);
    int b = j + __popc(same);
    if (same >> 31) b = lower_bound_warp(g.id, b, g.tokens, id + 1);
    const bool groups = g.group != nullptr && (j + kGroup - 1) / kGroup < b / kGroup;
    const int ga = groups ? (j + kGroup - 1) / kGroup : 0, gb = groups ? b / kGroup : 0;
    const bool larges = groups && g.large != nullptr && (ga + kGroup - 1) / kGroup < gb / kGroup;
    const int la = larges ? (ga + kGroup - 1) / kGroup : 0, lb = larges ? gb / kGroup : 0;
    float acc[S][N] = {};
#pragma unroll 1
    for (int part = 0; part < 5; ++part) {
      if (part == 0 || part == 4) {
        const int lo = part == 0 ? j : gb * kGroup, hi = part == 0 && groups ? ga * kGroup : b;
        add_tokens<T, kFlight>(acc, g, lo, hi, p0, packs);
        if (!groups) break;
      } else {
        const int lo = part == 1 ? ga : part == 2 ? la : larges ? lb * kGroup : gb;
        const int hi = part == 2 ? lb : part == 1 && larges ? la * kGroup : gb;
        add_sums<kSumFlight>(acc, part == 2 ? g.large : g.group, g.ldg, lo, hi, p0, packs);
      }
    }
    store_row<O, ADD>(acc, g.scale, static_cast<O*>(g.out) + static_cast<long>(id) * g.H, p0, packs);
  }
}

// A ValueError in Python, as the CPU form's checks give.
void require(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

torch::Tensor flat_ids(const torch::Tensor& ids, const torch::Tensor& like) {
  require(ids.device() == like.device() && (ids.scalar_type() == torch::kInt64 || ids.scalar_type() == torch::kInt32),
          "ids must be int64 or int32 on the table's device");
  const torch::Tensor wide = ids.scalar_type() == torch::kInt64 ? ids : ids.to(torch::kInt64);
  return wide.contiguous();
}

unsigned blocks_for(long a, long b) {
  const long n = (a + b - 1) / b;
  require(n < (1L << 31), "sizes too large for one launch");
  return static_cast<unsigned>(n);
}

}  // namespace

// ids [0, vocab) sorted, ties by position, `skip` and ids outside (reported unless
// they are `ignore`) last as kNoId.  ints: the ids, the positions, and for more than
// kSortKeys tokens as many of scratch (the sorted chunks before their merge).  One
// launch, or two.
void sort_tokens(const int64_t* ids, int64_t tokens, int64_t vocab, int64_t skip, int64_t ignore, int* ints, int* err,
                 cudaStream_t stream) {
  const bool one = tokens <= kSortKeys;
  unsigned* id = reinterpret_cast<unsigned*>(ints);
  int* token = ints + tokens;
  unsigned* id_chunks = one ? id : reinterpret_cast<unsigned*>(ints + 2 * tokens);
  int* token_chunks = one ? token : ints + 3 * tokens;
  // 32-bit keys hold 10 bits of place and 22 of the id, whose last value is kept
  (vocab < (1L << 22) ? embed_sort_kernel<unsigned> : embed_sort_kernel<unsigned long long>)<<<
      blocks_for(tokens, kSortKeys), kSortKeys, 0, stream>>>(ids, tokens, vocab, skip, ignore, id_chunks,
                                                             token_chunks, err);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (!one) {
    embed_merge_kernel<<<blocks_for(tokens, 32), kThreads, 0, stream>>>(id_chunks, token_chunks,
                                                                        static_cast<int>(tokens), id, token);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

torch::Tensor embed_fwd(torch::Tensor ids, torch::Tensor table, double scale, torch::Tensor err) {
  require(table.is_cuda() && is_storage_type(table) && table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1 &&
              table.size(1) < (1L << 30),
          "table must be a bf16, fp16 or fp32 CUDA matrix");
  const torch::Tensor flat = flat_ids(ids, table);
  const c10::cuda::CUDAGuard guard(table.device());
  const torch::Tensor rows = table.stride(1) == 1 || table.size(1) == 1 ? table : table.contiguous();
  const long tokens = flat.numel();
  const int H = static_cast<int>(table.size(1));
  auto shape = ids.sizes().vec();
  shape.push_back(H);
  torch::Tensor y = torch::empty(shape, table.options());
  if (tokens == 0) return y;
  const bool wide = wide_rows(rows);
  by_type(table.scalar_type(), [&](auto tag) {
    using T = decltype(tag);
    const int packs = wide ? H / kPackSize<T, true> : H;
    const int each = wide ? kLookup<kPackSize<T, true>> : kLookup<1>;
    int lanes = 32;
    while (lanes < kThreads && lanes * each < packs) lanes <<= 1;
    const unsigned blocks = static_cast<unsigned>(std::min<long>(blocks_for(tokens, kThreads / lanes), 148 * kLookupBlocks));
    (wide ? embed_fwd_kernel<T, true> : embed_fwd_kernel<T, false>)<<<blocks, kThreads, 0,
                                                                      at::cuda::getCurrentCUDAStream()>>>(
        flat.data_ptr<int64_t>(), tokens, rows.size(0), reinterpret_cast<const T*>(rows.data_ptr()), rows.stride(0), H,
        static_cast<float>(scale), reinterpret_cast<T*>(y.data_ptr()), lanes, err.data_ptr<int>());
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return y;
}

// The gradient [vocab, H]: a new one of dy's type, or `out` added to.  padding: an
// id without a gradient; one that no token has for none.
torch::Tensor embed_bwd(torch::Tensor dy, torch::Tensor ids, int64_t vocab, c10::optional<torch::Tensor> into,
                        double scale, int64_t padding, torch::Tensor err) {
  require(dy.is_cuda() && is_storage_type(dy) && dy.dim() >= 1 && dy.size(-1) >= 1 && dy.size(-1) < (1L << 30),
          "dy must be a bf16, fp16 or fp32 CUDA tensor [*ids.shape, H]");
  const int64_t H = dy.size(-1), tokens = dy.numel() / H;
  require(dy.sizes().slice(0, dy.dim() - 1) == ids.sizes(), "dy must have one row per id");
  require(vocab >= 1 && vocab < (1L << 31) - kTableRows * kWarps && tokens < (1L << 31) - kSortKeys,
          "the table needs a row, and sizes must fit 31 bits");
  if (into.has_value())
    require(into->device() == dy.device() && is_storage_type(*into) && into->is_contiguous() && into->dim() == 2 &&
                into->size(0) == vocab && into->size(1) == H,
            "out must be a contiguous bf16, fp16 or fp32 [vocab, H] on the device of dy");
  const torch::Tensor flat = flat_ids(ids, dy);
  const c10::cuda::CUDAGuard guard(dy.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  torch::Tensor out = into.has_value() ? *into : torch::empty({vocab, H}, dy.options());
  if (tokens == 0) return into.has_value() ? out : out.zero_();
  torch::Tensor rows = dy.reshape({tokens, H});
  if (rows.stride(1) != 1 && H != 1) rows = rows.contiguous();

  // sorted ids and tokens, the sorted chunks before their merge, and the rows' places
  const bool one = tokens <= kSortKeys, whole = !into.has_value();
  torch::Tensor ints = torch::empty({(one ? 2 : 4) * tokens + (whole ? vocab + 1 : 0)},
                                    dy.options().dtype(torch::kInt32));
  int* at = ints.data_ptr<int>();
  unsigned* id = reinterpret_cast<unsigned*>(at);
  int* token = at + tokens;
  int* start = at + (one ? 2 : 4) * tokens;
  sort_tokens(flat.data_ptr<int64_t>(), tokens, vocab, padding, /*ignore (none)=*/0, at, err.data_ptr<int>(), stream);
  if (whole) {
    embed_start_kernel<<<blocks_for(vocab + 1, kThreads), kThreads, 0, stream>>>(id, static_cast<int>(tokens),
                                                                                 static_cast<int>(vocab), start);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  const bool wide = wide_rows(rows) && aligned16(out.data_ptr()) && H * out.element_size() % 16 == 0;
  GradRows g{};
  g.dy = rows.data_ptr();
  g.ld = rows.stride(0);
  g.id = id;
  g.token = token;
  g.start = start;
  g.tokens = static_cast<int>(tokens), g.V = static_cast<int>(vocab), g.H = static_cast<int>(H);
  g.scale = static_cast<float>(scale);
  g.out = out.data_ptr();
  torch::Tensor sums;
  by_type(dy.scalar_type(), [&](auto tag) {
    using T = decltype(tag);
    const auto run = [&](auto wide_tag) {
      constexpr bool W = decltype(wide_tag)::value;
      constexpr int N = kPackSize<T, W>;
      g.slabs = blocks_for(H / N, 32 * kSlab<N>);
      if (tokens >= kGroupFrom) {
        const long groups = tokens / kGroup, large = tokens >= kLargeFrom ? groups / kGroup : 0;
        g.ldg = (H + 3) / 4 * 4;
        sums = torch::empty({groups + large, g.ldg}, dy.options().dtype(torch::kFloat32));
        float* group_sums = sums.data_ptr<float>();
        embed_group_kernel<T, W, false><<<blocks_for(groups * g.slabs, kWarps), kThreads, 0, stream>>>(
            g, static_cast<int>(groups), group_sums);
        C10_CUDA_KERNEL_LAUNCH_CHECK();
        g.group = group_sums;
        if (large > 0) {
          embed_group_kernel<T, W, true><<<blocks_for(large * g.slabs, kWarps), kThreads, 0, stream>>>(
              g, static_cast<int>(large), group_sums + groups * g.ldg);
          C10_CUDA_KERNEL_LAUNCH_CHECK();
          g.large = group_sums + groups * g.ldg;
        }
      }
      // few places per warp while that fills the GPU, more where starting warps would be the work
      g.places = static_cast<int>(std::clamp<long>(tokens * g.slabs / (148 * 64), 4, kListRows));
      const unsigned list_blocks = blocks_for(blocks_for(tokens, g.places) * static_cast<long>(g.slabs), kWarps);
      if (whole) {
        embed_table_kernel<T, W>
            <<<blocks_for(blocks_for(vocab, kTableRows) * static_cast<long>(g.slabs), kWarps), kThreads, 0, stream>>>(g);
        C10_CUDA_KERNEL_LAUNCH_CHECK();
        if (tokens > 1) embed_run_kernel<T, T, false, W><<<list_blocks, kThreads, 0, stream>>>(g);
      } else {
        by_type(out.scalar_type(), [&](auto otag) {
          using O = decltype(otag);
          embed_single_kernel<T, O, W><<<list_blocks, kThreads, 0, stream>>>(g);
          C10_CUDA_KERNEL_LAUNCH_CHECK();
          if (tokens > 1) embed_run_kernel<T, O, true, W><<<list_blocks, kThreads, 0, stream>>>(g);
        });
      }
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    };
    if (wide) run(std::true_type{});
    else run(std::false_type{});
  });
  return out;
}

}  // namespace gb
