// Global norm of many gradient tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2),  c = min(1, max_norm / (norm + 1e-6)),  out = c g
//
// Memory bound: one read for the norm; with an output one more read (from L2
// where the tensors fit) and a write.  In place and below the limit the second
// kernel returns after reading the norm.
//
// The tensors' addresses and sizes travel in the first kernel's parameters, so a
// call with some hundred tensors copies no table to the GPU and is two launches;
// the first kernel leaves the table in memory for the second.  No address
// outlives the call.  The tensors are cut into chunks of kChunk values and every
// block takes an equal stretch of them: the work is even however the sizes
// differ, a block searches the table once, and runs through a large tensor in one
// loop.  Each block writes one double, and
// every block of the second kernel adds them in the same order: the result does
// not depend on timing, and there is no counter to reset.  Sums of squares are
// fp32 over the values that a thread loads at once, double from there on.  fp32
// squares leave the range of fp32 at values of 1e19 and 1e-19; a round whose sum is
// outside [kLeast, largest float] is taken again with squares in double, so that the
// norm is right wherever it is a float itself (400 M fp32 values: 229 us, zeros 234,
// values of 1e-25 256; 228, 233 and 230 without).
//
// Measured on a B200: norm of 504 fp32 tensors, 43.6 M values, 28 us (6.2 TB/s); of 220
// bf16 tensors, 600 M values, 201 us (6.0 TB/s), and 670 us to scale them into fp32
// (5.4 TB/s).  (Chunk by chunk with a search each: 37, 360 and 1145 us.)
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <stdexcept>
#include <vector>

#include "sm100_common.cuh"
#include "vec_types.cuh"

namespace gb {

// The caller's tensors, which it keeps through the call (bindings.cpp): hundreds of
// them, so no handle is copied.
using TensorRefs = std::vector<const torch::Tensor*>;

namespace {

constexpr int kChunk = 4096;         // values; what the stretches are cut at
constexpr int kClipThreads = 256;
constexpr int kClipBlocks = 148 * 6;
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
  int at;          // place of entry 0 in the whole table, and
  int first;       // of chunk 0 among all chunks
};

// Entry of chunk c: the last one whose first chunk is not past it.
__device__ __forceinline__ int entry_of(const GradEntry* e, int tensors, int c) {
  int lo = 0, hi = tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (e[mid].first <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Stretch [begin, end) of `chunks` that a block takes.
__device__ __forceinline__ int2 stretch(int chunks) {
  return make_int2(static_cast<int>(static_cast<long>(chunks) * blockIdx.x / gridDim.x),
                   static_cast<int>(static_cast<long>(chunks) * (blockIdx.x + 1) / gridDim.x));
}

template <typename F>
__device__ __forceinline__ void by_grad_type(uint8_t type, F&& f) {
  if (type == kF32) f(static_cast<float*>(nullptr));
  else if (type == kBF16) f(static_cast<__nv_bfloat16*>(nullptr));
  else f(static_cast<__half*>(nullptr));
}

// The least fp32 sum of up to 32 squares that has lost nothing that counts to the
// small end of the range (2^-150 a square at most).
constexpr float kLeast = 0x1p-100f;

__device__ __forceinline__ bool in_range(float sum) { return sum >= kLeast && sum < INFINITY; }

// Sum of squares in double, over the packs p, p + kClipThreads, ... below `end`.
template <typename T>
__device__ __noinline__ double sumsq_far(const T* __restrict__ body, long p, long end) {
  constexpr int V = 16 / sizeof(T);
  double total = 0;
#pragma unroll 1
  for (; p < end; p += kClipThreads) {
    const Pack<T, V> k = load_raw<T, V>(body + p * V);
#pragma unroll
    for (int i = 0; i < V; ++i) total += static_cast<double>(value(k, i)) * value(k, i);
  }
  return total;
}

// Sum of squares of this thread's values among [lo, hi) of g: 16-byte loads, four
// in flight, between the values before the first and after the last 16-byte
// boundary; fp32 over one round of loads, double across rounds.
template <typename T>
__device__ __noinline__ double sumsq_range(const T* __restrict__ g, long lo, long hi) {
  constexpr int V = 16 / sizeof(T), U = 4;
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(g + lo) & 15) / sizeof(T));
  const long a = min(hi, lo + (skew == 0 ? 0 : V - skew));
  const long packs = (hi - a) / V;
  const T* body = g + a;
  double total = 0;
  long p = threadIdx.x;
  for (; p + (U - 1) * kClipThreads < packs; p += U * kClipThreads) {
    Pack<T, V> k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = load_raw<T, V>(body + (p + u * kClipThreads) * V);
    float s[U] = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) s[u] += value(k[u], i) * value(k[u], i);
    const float round = (s[0] + s[1]) + (s[2] + s[3]);
    if (in_range(round)) {
      total += round;
    } else {
      uint32_t any = 0;   // zeros, the usual case outside the range
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < Pack<T, V>::kWords; ++i) any |= k[u].w[i];
      if (any != 0) total += sumsq_far(body, p, p + U * kClipThreads);
    }
  }
  const long tail = a + packs * V + threadIdx.x;
  const float head = lo + threadIdx.x < a ? to_f(g[lo + threadIdx.x]) : 0.f, last = tail < hi ? to_f(g[tail]) : 0.f;
  float s = 0.f;
  for (long q = p; q < packs; q += kClipThreads) {
    const Pack<T, V> k = load_raw<T, V>(body + q * V);
#pragma unroll
    for (int i = 0; i < V; ++i) s += value(k, i) * value(k, i);
  }
  s += head * head;
  s += last * last;
  if (in_range(s)) return total + s;
  return total + sumsq_far(body, p, packs) + static_cast<double>(head) * head + static_cast<double>(last) * last;
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

// `table`: the whole call's entries for the second kernel, null without one.
template <int N>
__global__ void __launch_bounds__(kClipThreads, 6) grad_norm_kernel(const __grid_constant__ GradTable<N> t,
                                                                 GradEntry* __restrict__ table,
                                                                 double* __restrict__ partial) {
  if (table != nullptr && blockIdx.x == 0) {
    for (int i = threadIdx.x; i < t.tensors; i += kClipThreads) {
      GradEntry e = t.e[i];
      e.first += t.first;
      table[t.at + i] = e;
    }
  }
  double total = 0;
  const int2 own = stretch(t.chunks);
  int i = entry_of(t.e, t.tensors, own.x);
  for (int c = own.x; c < own.y; ++i) {
    const GradEntry& e = t.e[i];
    const int past = i + 1 < t.tensors ? min(own.y, t.e[i + 1].first) : own.y;
    const long lo = static_cast<long>(c - e.first) * kChunk;
    const long hi = min(e.n, static_cast<long>(past - e.first) * kChunk);
    by_grad_type(e.tin, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      total += sumsq_range(static_cast<const T*>(e.in), lo, hi);
    });
    c = past;
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
__device__ __noinline__ void scale_range(const T* g, O* out, long lo, long hi, float coef) {
  // a warp's accesses of the wider type are 512 contiguous bytes
  constexpr int V = 16 / static_cast<int>(sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
  constexpr int A = V * static_cast<int>(sizeof(T)), B = V * static_cast<int>(sizeof(O));
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(g + lo) & (A - 1)) / sizeof(T));
  long a = min(hi, lo + (skew == 0 ? 0 : V - skew));
  if ((reinterpret_cast<uintptr_t>(out + a) & (B - 1)) != 0) a = hi;
  const long packs = (hi - a) / V;
  for (long i = lo + threadIdx.x; i < a; i += kClipThreads) out[i] = from_f<O>(to_f(g[i]) * coef);
  for (long i = a + packs * V + threadIdx.x; i < hi; i += kClipThreads) out[i] = from_f<O>(to_f(g[i]) * coef);
  constexpr int U = 4;
  const long rounds = packs / (U * kClipThreads);
  for (long p = rounds * U * kClipThreads + threadIdx.x; p < packs; p += kClipThreads) {
    float f[V];
    load_pack<T, V>(g + a + p * V, f);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] *= coef;
    store_pack<O, V>(out + a + p * V, f);
  }
  for (long p = (rounds - 1) * U * kClipThreads + threadIdx.x; p >= 0; p -= U * kClipThreads) {
    Pack<T, V> k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = load_raw<T, V>(g + a + (p + u * kClipThreads) * V);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[V];
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = value(k[u], i) * coef;
      store_pack<O, V>(out + a + (p + u * kClipThreads) * V, f);
    }
  }
}

// `in_place`: every output is its input, so a coefficient of 1 leaves nothing to do.
__global__ void __launch_bounds__(kClipThreads, 4) grad_scale_kernel(const GradEntry* __restrict__ table, int tensors,
                                                                  int chunks, const double* __restrict__ partial,
                                                                  int count, float max_norm, bool in_place,
                                                                  float* __restrict__ norm) {
  const float n = norm_of(partial, count);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  float coef = 1.f;
  if (max_norm > 0.f) {
    const float q = max_norm / (n + 1e-6f);
    coef = q > 1.f ? 1.f : q;  // a NaN norm stays one
  }
  if (in_place && coef == 1.f) return;
  // backwards: the norm's walk read the ends of the stretches last, and they may still be in L2
  const int2 own = stretch(chunks);
  int i = entry_of(table, tensors, own.y - 1);
  for (int past = own.y; past > own.x; --i) {
    const GradEntry e = table[i];
    const int c = max(own.x, e.first);
    const long lo = static_cast<long>(c - e.first) * kChunk;
    const long hi = min(e.n, static_cast<long>(past - e.first) * kChunk);
    by_grad_type(e.tin, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      by_grad_type(e.tout, [&](auto* otag) {
        using O = std::remove_pointer_t<decltype(otag)>;
        scale_range(static_cast<const T*>(e.in), static_cast<O*>(e.out), lo, hi, coef);
      });
    });
    past = c;
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

// Entries of the tensors that hold values.
std::vector<GradEntry> entries(const TensorRefs& in, const TensorRefs* out,
                               const torch::Tensor& like) {
  std::vector<GradEntry> v;
  v.reserve(in.size());
  const auto device = like.device();
  for (size_t i = 0; i < in.size(); ++i) {
    const torch::Tensor& t = *in[i];
    require(t.device() == device && t.is_contiguous(), "gradients must be contiguous and on one device");
    GradEntry e{};
    e.in = t.data_ptr();
    e.n = t.numel();
    e.tin = e.tout = grad_type(t);
    e.out = const_cast<void*>(e.in);
    if (out != nullptr) {
      const torch::Tensor& o = *(*out)[i];
      require(o.device() == device && o.is_contiguous() && o.sizes() == t.sizes(),
              "outputs must be contiguous, on the gradients' device and of their shapes");
      e.out = o.data_ptr();
      e.tout = grad_type(o);
    }
    if (e.n > 0) v.push_back(e);
  }
  return v;
}

// The norm's launches: sums of squares of all tensors, one double per block.
struct NormPass {
  torch::Tensor buffer;       // doubles, then the table
  const double* partial;
  int count = 0;              // doubles
  const GradEntry* table;     // filled when asked for
  int tensors, chunks = 0;
};

NormPass norm_pass(const std::vector<GradEntry>& v, bool want_table, const torch::Tensor& like, cudaStream_t stream) {
  NormPass r;
  const size_t launches = std::max<size_t>((v.size() + kPerLaunch - 1) / kPerLaunch, 1);
  const int64_t doubles = static_cast<int64_t>(launches) * kClipBlocks;
  r.buffer = torch::empty({doubles * 8 + static_cast<int64_t>(want_table ? v.size() * sizeof(GradEntry) : 0)},
                          like.options().dtype(torch::kUInt8));
  double* partial = reinterpret_cast<double*>(r.buffer.data_ptr());
  GradEntry* table = want_table ? reinterpret_cast<GradEntry*>(partial + doubles) : nullptr;
  r.partial = partial;
  r.table = table;
  r.tensors = static_cast<int>(v.size());
  long chunks_before = 0;
  const auto run = [&](auto& t, size_t from, size_t count) {
    long chunks = 0;
    for (size_t i = 0; i < count; ++i) {
      t.e[i] = v[from + i];
      t.e[i].first = static_cast<int>(chunks);
      chunks += (v[from + i].n + kChunk - 1) / kChunk;
      require(chunks_before + chunks < (1L << 31) - kClipBlocks, "gradients too large for one call");
    }
    t.tensors = static_cast<int>(count);
    t.chunks = static_cast<int>(chunks);
    t.at = static_cast<int>(from);
    t.first = static_cast<int>(chunks_before);
    const int blocks = static_cast<int>(std::min<long>(chunks, kClipBlocks));
    grad_norm_kernel<<<blocks, kClipThreads, 0, stream>>>(t, table, partial + r.count);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    r.count += blocks;
    chunks_before += chunks;
  };
  for (size_t from = 0; from < v.size(); from += kPerLaunch) {
    const size_t count = std::min<size_t>(kPerLaunch, v.size() - from);
    if (count <= 64) {  // 2 KB of parameters instead of 28
      GradTable<64> t;
      run(t, from, count);
    } else {
      GradTable<kPerLaunch> t;
      run(t, from, count);
    }
  }
  r.chunks = static_cast<int>(chunks_before);
  return r;
}

torch::Tensor norm_on(int64_t device) {
  require(device >= 0, "a CUDA device");
  return torch::empty({}, torch::TensorOptions().dtype(torch::kFloat32).device(torch::kCUDA, static_cast<c10::DeviceIndex>(device)));
}

}  // namespace

// 2-norm of all values; `device` where there are no tensors to tell it.
torch::Tensor grad_norm(const TensorRefs& grads, int64_t device) {
  torch::Tensor norm = norm_on(device);
  const c10::cuda::CUDAGuard guard(norm.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const NormPass r = norm_pass(entries(grads, nullptr, norm), false, norm, stream);
  grad_norm_finish_kernel<<<1, kClipThreads, 0, stream>>>(r.partial, r.count, norm.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return norm;
}

// out: empty to scale the gradients in place.
torch::Tensor grad_clip(const TensorRefs& grads, const TensorRefs& out, double max_norm, int64_t device) {
  require(out.empty() || out.size() == grads.size(), "one output per gradient");
  require(max_norm >= 0, "max_norm must not be negative");
  torch::Tensor norm = norm_on(device);
  const c10::cuda::CUDAGuard guard(norm.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool in_place = out.empty();
  const NormPass r = norm_pass(entries(grads, in_place ? nullptr : &out, norm), true, norm, stream);
  const int blocks = std::max(1, std::min(r.chunks, kClipBlocks));
  if (r.tensors > 0)
    grad_scale_kernel<<<blocks, kClipThreads, 0, stream>>>(r.table, r.tensors, r.chunks, r.partial, r.count,
                                                           static_cast<float>(max_norm), in_place,
                                                           norm.data_ptr<float>());
  else
    grad_norm_finish_kernel<<<1, kClipThreads, 0, stream>>>(r.partial, 0, norm.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return norm;
}

}  // namespace gb
