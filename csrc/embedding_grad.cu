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
//  * Sort: keys (id, position), sorted in shared memory 2048 at a time; a key's
//    place in the whole is its place in its own chunk plus the number of smaller
//    keys in every other chunk (a binary search each).  Two launches and no
//    counters, for any number of tokens.
//  * Long runs (one id over thousands of tokens, as padding makes them): whole
//    groups of kGroup equal tokens are added first, all groups at once, and a run
//    then adds those sums.
//  * Rows: blocks take ranges of the table and find their tokens by binary
//    search, so that every row is written once; or they take ranges of the
//    sorted list when only touched rows are wanted.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>

#include "sm100_common.cuh"
#include "vec_types.cuh"

namespace gb {

namespace {

constexpr int kSortKeys = 2048;       // keys per sorted chunk
constexpr int kSortThreads = 1024;
constexpr int kGroup = 32;            // tokens of a pre-added group
constexpr int kRowThreads = 256;
constexpr int kTableRows = 16;        // table rows per block
constexpr int kListRows = 16;         // sorted positions per block
constexpr unsigned kNoId = 0xffffffffu;  // sorts last: no row takes it

using Key = unsigned long long;

// y[t] = scale * table[id]; NaN for an id outside the table.  `lanes` threads a row.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRowThreads) embed_fwd_kernel(const int64_t* __restrict__ ids, long T_, long V,
                                                                const T* __restrict__ table, long ldt, int H,
                                                                float scale, T* __restrict__ y, int lanes,
                                                                int* __restrict__ err) {
  constexpr int N = kPackSize<T, WIDE>;
  const int per_block = kRowThreads / lanes;
  const int lane = threadIdx.x % lanes;
  const int packs = H / N;
  for (long t = blockIdx.x * static_cast<long>(per_block) + threadIdx.x / lanes; t < T_;
       t += gridDim.x * static_cast<long>(per_block)) {
    const long id = ids[t];
    const bool ok = id >= 0 && id < V;
    if (!ok && lane == 0) atomicExch(err + 1, kErrBadToken);
    const Pack<T, N>* src = reinterpret_cast<const Pack<T, N>*>(table + (ok ? id : 0) * ldt);
    T* dst = y + t * H;
#pragma unroll 4
    for (int p = lane; p < packs; p += lanes) {
      Pack<T, N> k;
      if (ok) k = src[p];
      float f[N];
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = ok ? to_f(k.v[i]) * scale : __int_as_float(0x7fc00000);
      store_pack<T, N>(dst + static_cast<long>(p) * N, f);
    }
  }
}

// Sorted chunks of (id, position).  Padding ids, and ids outside the table
// (reported), become kNoId.  With one chunk the result is final.
__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const int64_t* __restrict__ ids, long T, long V,
                                                                  long padding, Key* __restrict__ keys,
                                                                  unsigned* __restrict__ id_out,
                                                                  int* __restrict__ token_out, bool final,
                                                                  int* __restrict__ err) {
  __shared__ Key s[kSortKeys];
  const long base = static_cast<long>(blockIdx.x) * kSortKeys;
  const int n = static_cast<int>(min(T - base, static_cast<long>(kSortKeys)));
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = threadIdx.x; i < size; i += kSortThreads) {
    Key k = ~0ull;
    if (i < n) {
      const long id = ids[base + i];
      unsigned u = static_cast<unsigned>(id);
      if (id < 0 || id >= V) {
        atomicExch(err + 1, kErrBadToken);
        u = kNoId;
      } else if (id == padding) {
        u = kNoId;
      }
      k = static_cast<Key>(u) << 32 | static_cast<Key>(base + i);
    }
    s[i] = k;
  }
  __syncthreads();
  for (int span = 2; span <= size; span <<= 1) {
    for (int gap = span >> 1; gap > 0; gap >>= 1) {
      for (int j = threadIdx.x; j < size >> 1; j += kSortThreads) {
        const int i = (j / gap) * 2 * gap + j % gap;
        const bool up = (i & span) == 0;
        const Key a = s[i], b = s[i + gap];
        if ((a > b) == up) {
          s[i] = b;
          s[i + gap] = a;
        }
      }
      __syncthreads();
    }
  }
  for (int i = threadIdx.x; i < n; i += kSortThreads) {
    if (final) {
      id_out[i] = static_cast<unsigned>(s[i] >> 32);
      token_out[i] = static_cast<int>(s[i]);
    } else {
      keys[base + i] = s[i];
    }
  }
}

// Place of every key among all chunks.  Four chunks are searched side by side:
// their loads do not wait for one another.
__global__ void __launch_bounds__(256) embed_merge_kernel(const Key* __restrict__ keys, long T,
                                                          unsigned* __restrict__ id_out, int* __restrict__ token_out) {
  const long i = blockIdx.x * 256L + threadIdx.x;
  if (i >= T) return;
  const Key k = keys[i];
  const int own = static_cast<int>(i / kSortKeys);
  const int chunks = static_cast<int>((T + kSortKeys - 1) / kSortKeys);
  long place = i - static_cast<long>(own) * kSortKeys;
  for (int c0 = 0; c0 < chunks; c0 += 4) {
    int lo[4], n[4];
    const Key* at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + u;
      at[u] = keys + static_cast<long>(c) * kSortKeys;
      n[u] = c < chunks && c != own ? static_cast<int>(min(T - static_cast<long>(c) * kSortKeys, static_cast<long>(kSortKeys))) : 0;
      lo[u] = 0;
    }
#pragma unroll
    for (int step = kSortKeys; step > 0; step >>= 1) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (lo[u] + step <= n[u] && at[u][lo[u] + step - 1] < k) lo[u] += step;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) place += lo[u];
  }
  id_out[place] = static_cast<unsigned>(k >> 32);
  token_out[place] = static_cast<int>(k);
}

// First position in [lo, hi) whose id is not below `id`; a whole warp calls it.
__device__ __forceinline__ int lower_bound_warp(const unsigned* __restrict__ ids, int lo, int hi, unsigned id) {
  const int lane = threadIdx.x & 31;
  while (hi - lo > 32) {
    const int step = (hi - lo + 32) / 33;
    const int at = lo + (lane + 1) * step - 1;
    const bool below = at < hi && ids[at] < id;
    const int k = __popc(__ballot_sync(0xffffffffu, below));
    hi = min(hi, lo + (k + 1) * step - (k < 32 ? 1 : 0));
    lo = lo + k * step;
  }
  const bool below = lo + lane < hi && ids[lo + lane] < id;
  return lo + __popc(__ballot_sync(0xffffffffu, below));
}

template <int N>
__device__ __forceinline__ void add_to(float (&acc)[N], const float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] += f[i];
}

// acc += dy[token[j]] at one pack, j = lo .. hi - 1 in order, eight loads in flight.
template <typename T, int N>
__device__ __forceinline__ void add_tokens(float (&acc)[N], const T* __restrict__ dy, long ld, int pack,
                                           const int* __restrict__ token, int lo, int hi) {
  int j = lo;
  for (; j + 8 <= hi; j += 8) {
    Pack<T, N> k[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) k[u] = reinterpret_cast<const Pack<T, N>*>(dy + token[j + u] * ld)[pack];
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += to_f(k[u].v[i]);
  }
  for (; j < hi; ++j) {
    float f[N];
    load_pack<T, N>(dy + token[j] * ld + static_cast<long>(pack) * N, f);
    add_to(acc, f);
  }
}

// Sums of the groups of kGroup sorted tokens that are all of one id.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRowThreads) embed_group_kernel(const T* __restrict__ dy, long ld, int H,
                                                                  const unsigned* __restrict__ id,
                                                                  const int* __restrict__ token, int ldg,
                                                                  float* __restrict__ group) {
  constexpr int N = kPackSize<T, WIDE>;
  const int lo = blockIdx.x * kGroup;
  if (id[lo] != id[lo + kGroup - 1] || id[lo] == kNoId) return;
  const int packs = H / N;
  for (int p = blockIdx.y * kRowThreads + threadIdx.x; p < packs; p += gridDim.y * kRowThreads) {
    float acc[N] = {};
    add_tokens<T, N>(acc, dy, ld, p, token, lo, lo + kGroup);
#pragma unroll
    for (int i = 0; i < N; ++i) group[static_cast<long>(blockIdx.x) * ldg + p * N + i] = acc[i];
  }
}

// Sum of the run [a, b) at one pack: single tokens up to the first whole group,
// the groups' sums, and the tokens after the last.
template <typename T, int N>
__device__ __forceinline__ void add_run(float (&acc)[N], const T* __restrict__ dy, long ld, int pack,
                                        const int* __restrict__ token, const float* __restrict__ group, int ldg, int a,
                                        int b) {
  const int g0 = (a + kGroup - 1) / kGroup, g1 = b / kGroup;
  if (g0 >= g1) {
    add_tokens<T, N>(acc, dy, ld, pack, token, a, b);
    return;
  }
  add_tokens<T, N>(acc, dy, ld, pack, token, a, g0 * kGroup);
  for (int g = g0; g < g1; g += 8) {
    float f[8][N];
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i)
        f[u][i] = g + u < g1 ? group[static_cast<long>(g + u) * ldg + pack * N + i] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) add_to(acc, f[u]);
  }
  add_tokens<T, N>(acc, dy, ld, pack, token, g1 * kGroup, b);
}

struct GradRows {
  const void* dy;
  long ld;          // row stride of dy
  const unsigned* id;
  const int* token;
  const float* group;
  int ldg;
  int T, V, H;
  float scale;
  void* out;
};

// The whole table: a block writes kTableRows rows, zeros where no token is.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRowThreads) embed_table_kernel(const GradRows g) {
  constexpr int N = kPackSize<T, WIDE>;
  __shared__ int bound[kTableRows + 1];
  const int v0 = blockIdx.x * kTableRows;
  const int rows = min(kTableRows, g.V - v0);
  const int warp = threadIdx.x >> 5;
  for (int i = warp; i <= rows; i += kRowThreads / 32) {
    const int at = lower_bound_warp(g.id, 0, g.T, static_cast<unsigned>(v0 + i));
    if ((threadIdx.x & 31) == 0) bound[i] = at;
  }
  __syncthreads();
  const int packs = g.H / N;
  for (int r = 0; r < rows; ++r) {
    const int a = bound[r], b = bound[r + 1];
    T* out = static_cast<T*>(g.out) + static_cast<long>(v0 + r) * g.H;
    for (int p = blockIdx.y * kRowThreads + threadIdx.x; p < packs; p += gridDim.y * kRowThreads) {
      float acc[N] = {};
      if (a < b) {
        add_run<T, N>(acc, static_cast<const T*>(g.dy), g.ld, p, g.token, g.group, g.ldg, a, b);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] *= g.scale;
      }
      store_pack<T, N>(out + static_cast<long>(p) * N, acc);
    }
  }
}

// Adds to the touched rows of an existing gradient of type O: a block takes the
// runs that start in its kListRows sorted positions.
template <typename T, typename O, bool WIDE>
__global__ void __launch_bounds__(kRowThreads) embed_list_kernel(const GradRows g) {
  constexpr int N = kPackSize<T, WIDE>;
  const int packs = g.H / N;
  const int j0 = blockIdx.x * kListRows;
  const int j1 = min(g.T, j0 + kListRows);
  for (int j = j0; j < j1; ++j) {
    const unsigned id = g.id[j];
    if (id == kNoId) break;
    if (j > 0 && g.id[j - 1] == id) continue;
    const int end = lower_bound_warp(g.id, j, g.T, id + 1);
    O* out = static_cast<O*>(g.out) + static_cast<long>(id) * g.H;
    for (int p = blockIdx.y * kRowThreads + threadIdx.x; p < packs; p += gridDim.y * kRowThreads) {
      float acc[N] = {}, old[N];
      add_run<T, N>(acc, static_cast<const T*>(g.dy), g.ld, p, g.token, g.group, g.ldg, j, end);
      load_pack<O, N>(out + static_cast<long>(p) * N, old);
#pragma unroll
      for (int i = 0; i < N; ++i) old[i] += acc[i] * g.scale;
      store_pack<O, N>(out + static_cast<long>(p) * N, old);
    }
  }
}

}  // namespace

void embed_fwd(torch::Tensor ids, torch::Tensor table, torch::Tensor y, double scale, torch::Tensor err) {
  TORCH_CHECK(table.is_cuda() && is_storage_type(table) && table.dim() == 2 &&
                  (table.stride(1) == 1 || table.size(1) == 1) && table.size(0) >= 1 && table.size(1) >= 1 &&
                  table.size(1) < (1L << 31),
              "table must be a bf16, fp16 or fp32 CUDA matrix with unit inner stride");
  TORCH_CHECK(ids.device() == table.device() && ids.scalar_type() == torch::kInt64 && ids.is_contiguous(),
              "ids must be contiguous int64 on the table's GPU");
  TORCH_CHECK(y.device() == table.device() && y.scalar_type() == table.scalar_type() && y.is_contiguous() &&
                  y.dim() == 2 && y.size(0) == ids.numel() && y.size(1) == table.size(1), "y must be [tokens, H] like the table");
  const c10::cuda::CUDAGuard guard(table.device());
  const long T = ids.numel();
  if (T == 0) return;
  const int H = static_cast<int>(table.size(1));
  const bool wide = wide_rows(table) && wide_rows(y);
  by_type(table.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    const int packs = wide ? H / kPackSize<E, true> : H;
    int lanes = 32;
    while (lanes < kRowThreads && lanes < packs) lanes <<= 1;
    const long per_block = kRowThreads / lanes;
    const unsigned blocks = static_cast<unsigned>(std::min<long>((T + per_block - 1) / per_block, 1L << 30));
    (wide ? embed_fwd_kernel<E, true> : embed_fwd_kernel<E, false>)<<<blocks, kRowThreads, 0,
                                                                      at::cuda::getCurrentCUDAStream()>>>(
        ids.data_ptr<int64_t>(), T, table.size(0), reinterpret_cast<const E*>(table.data_ptr()), table.stride(0), H,
        static_cast<float>(scale), reinterpret_cast<E*>(y.data_ptr()), lanes, err.data_ptr<int>());
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// dE [V, H]: written whole, or (accumulate) added to.  padding: an id without a gradient; one that no token has for none.
void embed_bwd(torch::Tensor dy, torch::Tensor ids, torch::Tensor out, double scale, int64_t padding, bool accumulate,
               torch::Tensor err) {
  TORCH_CHECK(dy.is_cuda() && is_storage_type(dy) && dy.dim() == 2 && (dy.stride(1) == 1 || dy.size(1) == 1) &&
                  dy.size(1) >= 1,
              "dy must be a bf16, fp16 or fp32 CUDA matrix with unit inner stride");
  TORCH_CHECK(ids.device() == dy.device() && ids.scalar_type() == torch::kInt64 && ids.is_contiguous() &&
                  ids.numel() == dy.size(0), "ids must be contiguous int64, one per row of dy");
  TORCH_CHECK(out.device() == dy.device() && is_storage_type(out) && out.is_contiguous() && out.dim() == 2 &&
                  out.size(1) == dy.size(1) && out.size(0) >= 1, "the gradient must be a contiguous [V, H]");
  TORCH_CHECK(accumulate || out.scalar_type() == dy.scalar_type(), "a gradient that is written whole has dy's type");
  TORCH_CHECK(dy.size(0) < (1L << 31) - kSortKeys && out.size(0) < (1L << 31) - kTableRows && dy.size(1) < (1L << 31),
              "sizes must fit 31 bits");
  const c10::cuda::CUDAGuard guard(dy.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int T = static_cast<int>(dy.size(0)), H = static_cast<int>(dy.size(1)), V = static_cast<int>(out.size(0));
  const int chunks = (T + kSortKeys - 1) / kSortKeys, groups = T / kGroup;
  if (T == 0 && accumulate) return;
  torch::Tensor ints = torch::empty({2, std::max(T, 1)}, dy.options().dtype(torch::kInt32));
  unsigned* id = reinterpret_cast<unsigned*>(ints.data_ptr<int>());
  int* token = ints.data_ptr<int>() + std::max(T, 1);
  torch::Tensor keys, group;
  if (chunks > 1) keys = torch::empty({T}, dy.options().dtype(torch::kInt64));
  Key* k = chunks > 1 ? reinterpret_cast<Key*>(keys.data_ptr<int64_t>()) : nullptr;
  if (T > 0) {
    embed_sort_kernel<<<chunks, kSortThreads, 0, stream>>>(ids.data_ptr<int64_t>(), T, V, padding, k, id, token,
                                                           chunks == 1, err.data_ptr<int>());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  if (chunks > 1) {
    embed_merge_kernel<<<(T + 255) / 256, 256, 0, stream>>>(k, T, id, token);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  const bool wide = wide_rows(dy) && aligned16(out.data_ptr()) && H * out.element_size() % 16 == 0;
  GradRows g{};
  g.dy = dy.data_ptr();
  g.ld = dy.stride(0);
  g.id = id;
  g.token = token;
  g.T = T, g.V = V, g.H = H;
  g.scale = static_cast<float>(scale);
  g.out = out.data_ptr();
  by_type(dy.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    const int packs = wide ? H / kPackSize<E, true> : H;
    const int columns = (packs + kRowThreads - 1) / kRowThreads;
    if (groups > 0) {
      g.ldg = static_cast<int>((H + 3) / 4 * 4);
      group = torch::empty({groups, g.ldg}, dy.options().dtype(torch::kFloat32));
      g.group = group.data_ptr<float>();
      const dim3 grid(groups, std::min(columns, 8));
      (wide ? embed_group_kernel<E, true> : embed_group_kernel<E, false>)<<<grid, kRowThreads, 0, stream>>>(
          static_cast<const E*>(g.dy), g.ld, H, id, token, g.ldg, group.data_ptr<float>());
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
    if (!accumulate) {
      const dim3 grid((V + kTableRows - 1) / kTableRows, 1);
      (wide ? embed_table_kernel<E, true> : embed_table_kernel<E, false>)<<<grid, kRowThreads, 0, stream>>>(g);
    } else {
      const dim3 grid((T + kListRows - 1) / kListRows, std::min(columns, 8));
      by_type(out.scalar_type(), [&](auto otag) {
        using O = decltype(otag);
        (wide ? embed_list_kernel<E, O, true> : embed_list_kernel<E, O, false>)<<<grid, kRowThreads, 0, stream>>>(g);
      });
    }
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
}

}  // namespace gb
