// Global norm of many gradient tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2),  c = min(1, max_norm / (norm + 1e-6)),  out = c g
//
// Memory bound: one read for the norm; with an output one more read (from L2
// where the tensors fit) and a write.  In place and below the limit the second
// kernel returns after reading the norm.
//
// The tensors' addresses and sizes travel in the kernels' parameters, so a call
// with some hundred tensors is two launches and copies no table to the GPU; no
// address outlives the call.  The tensors are cut into chunks of kChunk values,
// which blocks take in turn: the work is even however the sizes differ.  Each
// block writes one double, and every block of the second kernel adds them in
// the same order: the result does not depend on timing, and there is no counter
// to reset.  Sums of squares are fp32 over at most some hundred values of one
// thread, double from there on.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <stdexcept>
#include <vector>

#include "sm100_common.cuh"
#include "vec_types.cuh"

namespace gb {

namespace {

constexpr int kChunk = 16384;        // values per chunk
constexpr int kClipThreads = 256;
constexpr int kClipBlocks = 148 * 4;
constexpr int kPerLaunch = 896;      // tensors per launch: the table stays below the 32 KB of kernel parameters

enum GradType : uint8_t { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct GradEntry {
  const void* in;
  void* out;
  long n;
  int first;       // index of its first chunk
  uint8_t tin, tout;
};

template <int N>
struct GradTable {
  GradEntry e[N];
  int tensors;
  int chunks;      // in all
};

// Entry of chunk c: the last one whose first chunk is not past it.
template <int N>
__device__ __forceinline__ int entry_of(const GradTable<N>& t, int c) {
  int lo = 0, hi = t.tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.e[mid].first <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename F>
__device__ __forceinline__ void by_grad_type(uint8_t type, F&& f) {
  if (type == kF32) f(static_cast<float*>(nullptr));
  else if (type == kBF16) f(static_cast<__nv_bfloat16*>(nullptr));
  else f(static_cast<__half*>(nullptr));
}

// Sum of squares of values [lo, hi) of g: 16-byte loads, four in flight per thread,
// between the values before the first and after the last 16-byte boundary.
template <typename T>
__device__ __forceinline__ float sumsq_range(const T* g, long lo, long hi) {
  constexpr int V = 16 / sizeof(T);
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(g + lo) & 15) / sizeof(T));
  const long a = min(hi, lo + (skew == 0 ? 0 : V - skew));
  const long packs = (hi - a) / V;
  float s[4] = {};
  for (long i = lo + threadIdx.x; i < a; i += kClipThreads) s[0] += to_f(g[i]) * to_f(g[i]);
  for (long i = a + packs * V + threadIdx.x; i < hi; i += kClipThreads) s[1] += to_f(g[i]) * to_f(g[i]);
  const T* body = g + a;
  for (long p = threadIdx.x; p < packs; p += 4 * kClipThreads) {
    Pack<T, V> k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (p + u * kClipThreads < packs) k[u] = reinterpret_cast<const Pack<T, V>*>(body)[p + u * kClipThreads];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (p + u * kClipThreads < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) s[u] += to_f(k[u].v[i]) * to_f(k[u].v[i]);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kClipThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kClipThreads / 32; ++w) v += part[w];
  return v;
}

template <int N>
__global__ void __launch_bounds__(kClipThreads) grad_norm_kernel(const __grid_constant__ GradTable<N> t,
                                                                 double* __restrict__ partial) {
  double total = 0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const GradEntry& e = t.e[entry_of(t, c)];
    const long lo = static_cast<long>(c - e.first) * kChunk;
    const long hi = min(e.n, lo + kChunk);
    by_grad_type(e.tin, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      total += sumsq_range(static_cast<const T*>(e.in), lo, hi);
    });
  }
  total = block_sum(total);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

__device__ __forceinline__ float norm_of(const double* __restrict__ partial, int count) {
  double s = 0;
  for (int i = threadIdx.x; i < count; i += kClipThreads) s += partial[i];
  return static_cast<float>(sqrt(block_sum(s)));
}

__global__ void __launch_bounds__(kClipThreads) grad_norm_finish_kernel(const double* __restrict__ partial, int count,
                                                                        float* __restrict__ norm) {
  const float n = norm_of(partial, count);
  if (threadIdx.x == 0) *norm = n;
}

// out = coef * in over [lo, hi).  16-byte accesses where the input and the output
// reach their boundaries at the same value, single values elsewhere.
template <typename T, typename O>
__device__ __forceinline__ void scale_range(const T* g, O* out, long lo, long hi, float coef) {
  constexpr int V = 8, W = 16 / sizeof(T);
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(g + lo) & 15) / sizeof(T));
  long a = min(hi, lo + (skew == 0 ? 0 : W - skew));
  if ((reinterpret_cast<uintptr_t>(out + a) & 15) != 0) a = hi;
  const long packs = (hi - a) / V;
  for (long i = lo + threadIdx.x; i < a; i += kClipThreads) out[i] = from_f<O>(to_f(g[i]) * coef);
  for (long i = a + packs * V + threadIdx.x; i < hi; i += kClipThreads) out[i] = from_f<O>(to_f(g[i]) * coef);
  for (long p = threadIdx.x; p < packs; p += 2 * kClipThreads) {
    float f[2][V];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (p + u * kClipThreads < packs) load_pack<T, V>(g + a + (p + u * kClipThreads) * V, f[u]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (p + u * kClipThreads < packs) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[u][i] *= coef;
        store_pack<O, V>(out + a + (p + u * kClipThreads) * V, f[u]);
      }
  }
}

// `in_place`: every output is its input, so a coefficient of 1 leaves nothing to do.
template <int N>
__global__ void __launch_bounds__(kClipThreads) grad_scale_kernel(const __grid_constant__ GradTable<N> t,
                                                                  const double* __restrict__ partial, int count,
                                                                  float max_norm, bool in_place,
                                                                  float* __restrict__ norm) {
  const float n = norm_of(partial, count);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  float coef = 1.f;
  if (max_norm > 0.f) {
    const float q = max_norm / (n + 1e-6f);
    coef = q > 1.f ? 1.f : q;  // a NaN norm stays one
  }
  if (in_place && coef == 1.f) return;
  // from the end: the norm's walk read those values last
  for (int c = t.chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
    const GradEntry& e = t.e[entry_of(t, c)];
    const long lo = static_cast<long>(c - e.first) * kChunk;
    const long hi = min(e.n, lo + kChunk);
    by_grad_type(e.tin, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      by_grad_type(e.tout, [&](auto* otag) {
        using O = std::remove_pointer_t<decltype(otag)>;
        scale_range(static_cast<const T*>(e.in), static_cast<O*>(e.out), lo, hi, coef);
      });
    });
  }
}

uint8_t grad_type(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return kF32;
    case torch::kBFloat16: return kBF16;
    case torch::kHalf: return kF16;
    default: throw std::invalid_argument("gradients and outputs must be fp32, bf16 or fp16");
  }
}

// A ValueError in Python, as the other operators' argument checks give.
void require(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

// Entries of the tensors that hold values; chunks counted per launch.
std::vector<GradEntry> entries(const std::vector<torch::Tensor>& in, const std::vector<torch::Tensor>* out,
                               const torch::Tensor& like) {
  std::vector<GradEntry> v;
  v.reserve(in.size());
  for (size_t i = 0; i < in.size(); ++i) {
    const torch::Tensor& t = in[i];
    require(t.device() == like.device() && t.is_contiguous(), "gradients must be contiguous and on one device");
    GradEntry e{};
    e.in = t.data_ptr();
    e.n = t.numel();
    e.tin = e.tout = grad_type(t);
    e.out = t.data_ptr();
    if (out != nullptr) {
      const torch::Tensor& o = (*out)[i];
      require(o.device() == like.device() && o.is_contiguous() && o.sizes() == t.sizes(),
              "outputs must be contiguous, on the gradients' device and of their shapes");
      e.out = o.data_ptr();
      e.tout = grad_type(o);
    }
    if (e.n > 0) v.push_back(e);
  }
  return v;
}

template <typename F>
void for_tables(const std::vector<GradEntry>& v, F&& launch) {
  const auto fill = [&](auto& table, size_t from, size_t count) {
    long chunks = 0;
    for (size_t i = 0; i < count; ++i) {
      table.e[i] = v[from + i];
      table.e[i].first = static_cast<int>(chunks);
      chunks += (v[from + i].n + kChunk - 1) / kChunk;
    }
    require(chunks < (1L << 31) - kClipBlocks, "gradients too large for one call");
    table.tensors = static_cast<int>(count);
    table.chunks = static_cast<int>(chunks);
  };
  for (size_t from = 0; from < v.size(); from += kPerLaunch) {
    const size_t count = std::min<size_t>(kPerLaunch, v.size() - from);
    if (count <= 64) {  // 2 KB of parameters instead of 32
      GradTable<64> table;
      fill(table, from, count);
      launch(table);
    } else {
      GradTable<kPerLaunch> table;
      fill(table, from, count);
      launch(table);
    }
  }
}

int table_blocks(int chunks) { return std::min(chunks, kClipBlocks); }

// Sums of squares of all tensors: one double per block, every launch its own range.
torch::Tensor norm_partials(const std::vector<GradEntry>& v, const torch::Tensor& like, cudaStream_t stream,
                            int* count) {
  const int launches = static_cast<int>((v.size() + kPerLaunch - 1) / kPerLaunch);
  torch::Tensor partial = torch::empty({std::max(launches, 1) * kClipBlocks}, like.options().dtype(torch::kFloat64));
  int at = 0;
  for_tables(v, [&](auto& table) {
    const int blocks = table_blocks(table.chunks);
    grad_norm_kernel<<<blocks, kClipThreads, 0, stream>>>(table, partial.data_ptr<double>() + at);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    at += blocks;
  });
  *count = at;
  return partial;
}

}  // namespace

void grad_norm(std::vector<torch::Tensor> grads, torch::Tensor norm) {
  TORCH_CHECK(norm.is_cuda() && norm.scalar_type() == torch::kFloat32 && norm.numel() == 1, "norm must be one CUDA fp32 value");
  const c10::cuda::CUDAGuard guard(norm.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  int count = 0;
  const torch::Tensor partial = norm_partials(entries(grads, nullptr, norm), norm, stream, &count);
  grad_norm_finish_kernel<<<1, kClipThreads, 0, stream>>>(partial.data_ptr<double>(), count, norm.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// out: empty to scale the gradients in place.
void grad_clip(std::vector<torch::Tensor> grads, std::vector<torch::Tensor> out, double max_norm, torch::Tensor norm) {
  TORCH_CHECK(norm.is_cuda() && norm.scalar_type() == torch::kFloat32 && norm.numel() == 1, "norm must be one CUDA fp32 value");
  require(out.empty() || out.size() == grads.size(), "one output per gradient");
  require(max_norm >= 0, "max_norm must not be negative");
  const c10::cuda::CUDAGuard guard(norm.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool in_place = out.empty();
  const std::vector<GradEntry> v = entries(grads, in_place ? nullptr : &out, norm);
  int count = 0;
  const torch::Tensor partial = norm_partials(v, norm, stream, &count);
  if (v.empty()) {
    grad_norm_finish_kernel<<<1, kClipThreads, 0, stream>>>(partial.data_ptr<double>(), 0, norm.data_ptr<float>());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  for_tables(v, [&](auto& table) {
    grad_scale_kernel<<<table_blocks(table.chunks), kClipThreads, 0, stream>>>(
        table, partial.data_ptr<double>(), count, static_cast<float>(max_norm), in_place, norm.data_ptr<float>());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
}

}  // namespace gb
