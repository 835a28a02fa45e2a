// Layer norm over the last dimension, forward and backward, with the
// reductions of the weight's and the bias's gradient.
//
//   n = (x - mean) rstd,  y = n w + b                       mean, rstd per row
//   a = dy w,  dx = rstd (a - mean(a) - n mean(a n))        per row
//   dw = sum_rows dy n,  db = sum_rows dy                   per column
//
// Memory bound: the forward reads x and writes y, the backward reads x and dy
// and writes dx.  A row is read once and kept in registers, where the mean and
// then the centred sum of squares are taken (fp32; no cancellation of
// E[x^2] - mean^2).  A thread meets the same columns in every row that its
// block walks, so it carries its columns' dw and db in registers; the blocks'
// sums are joined by a second, small kernel in a fixed order.
//
// Variants: up to 160 packs of 16 bytes a row (1280 bf16 values) take a warp a
// row, several rows per block and no barrier; longer ones a block a row; rows
// past 2048 packs are read several times (they stay in L1/L2).  Rows that are no
// multiple of 16 bytes are read value by value.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>

#include "sm100_common.cuh"
#include "vec_types.cuh"

namespace gb {

namespace {

constexpr int kWarpRows = 8;   // rows in flight per block of the warp-a-row variants
constexpr int kSMs = 148;

// Sum over the threads that share a row: a warp, or the block.
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  v = warp_sum(v);
  if constexpr (BLOCK) {
    const int warps = blockDim.x >> 5;
    __syncthreads();  // the last sum has been read
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < warps; ++w) v += scratch[w];
  }
  return v;
}

template <bool BLOCK>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* scratch) {
  a = warp_sum(a);
  b = warp_sum(b);
  if constexpr (BLOCK) {
    const int warps = blockDim.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
    for (int w = 0; w < warps; ++w) {
      a += scratch[w].x;
      b += scratch[w].y;
    }
  }
  return make_float2(a, b);
}

// weight / bias values: fp32, or the type of x
template <typename T, int V>
__device__ __forceinline__ void load_param(const void* p, bool fp32, long i, float (&f)[V]) {
  if (fp32) {
    const float* q = static_cast<const float*>(p) + i;
    if constexpr (V % 4 == 0) {
#pragma unroll
      for (int k = 0; k < V; k += 4) {
        const float4 t = *reinterpret_cast<const float4*>(q + k);
        f[k] = t.x, f[k + 1] = t.y, f[k + 2] = t.z, f[k + 3] = t.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = q[k];
    }
  } else {
    load_pack<T, V>(static_cast<const T*>(p) + i, f);
  }
}

struct NormArgs {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  void* out;          // y or dx
  float* mean;
  float* rstd;
  float* part;        // [blocks][2][H] sums of dw and db
  long rows, ldx, ldy;
  int H;
  float eps;
  bool w32, b32;
};

template <typename T, int V, int VPT, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : 32 * kWarpRows) ln_fwd_kernel(const NormArgs a) {
  __shared__ float scratch[32];
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const int width = BLOCK ? blockDim.x : 32;
  const long first = BLOCK ? blockIdx.x : blockIdx.x * static_cast<long>(kWarpRows) + (threadIdx.x >> 5);
  const long step = BLOCK ? gridDim.x : gridDim.x * static_cast<long>(kWarpRows);
  const int packs = a.H / V;
  const float inv_h = 1.f / static_cast<float>(a.H);
  for (long r = first; r < a.rows; r += step) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    Pack<T, V> raw[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * width < packs) raw[k] = reinterpret_cast<const Pack<T, V>*>(x)[lane + k * width];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * width < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) s += to_f(raw[k].v[i]);
    const float mean = row_sum<BLOCK>(s, scratch) * inv_h;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * width < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float c = to_f(raw[k].v[i]) - mean;
          s += c * c;
        }
    const float rstd = 1.f / sqrtf(row_sum<BLOCK>(s, scratch) * inv_h + a.eps);
    T* y = static_cast<T*>(a.out) + r * a.H;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int p = lane + k * width;
      if (p < packs) {
        float w[V], b[V] = {}, o[V];
        load_param<T, V>(a.w, a.w32, static_cast<long>(p) * V, w);
        if (a.b != nullptr) load_param<T, V>(a.b, a.b32, static_cast<long>(p) * V, b);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (to_f(raw[k].v[i]) - mean) * rstd * w[i] + b[i];
        store_pack<T, V>(y + static_cast<long>(p) * V, o);
      }
    }
    if (lane == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
  }
}

// Rows that do not fit the registers: three walks of the row, a block each.
template <typename T>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(const NormArgs a) {
  __shared__ float scratch[32];
  const float inv_h = 1.f / static_cast<float>(a.H);
  for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) s += to_f(x[c]);
    const float mean = row_sum<true>(s, scratch) * inv_h;
    s = 0.f;
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
      const float d = to_f(x[c]) - mean;
      s += d * d;
    }
    const float rstd = 1.f / sqrtf(row_sum<true>(s, scratch) * inv_h + a.eps);
    T* y = static_cast<T*>(a.out) + r * a.H;
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
      float w[1], b[1] = {};
      load_param<T, 1>(a.w, a.w32, c, w);
      if (a.b != nullptr) load_param<T, 1>(a.b, a.b32, c, b);
      y[c] = from_f<T>((to_f(x[c]) - mean) * rstd * w[0] + b[0]);
    }
    if (threadIdx.x == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
  }
}

template <typename T, int V, int VPT, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : 32 * kWarpRows) ln_bwd_kernel(const NormArgs a) {
  extern __shared__ float smem[];  // warp-a-row: the warps' column sums at the end
  __shared__ float2 scratch[32];
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int width = BLOCK ? blockDim.x : 32;
  const long first = BLOCK ? blockIdx.x : blockIdx.x * static_cast<long>(kWarpRows) + warp;
  const long step = BLOCK ? gridDim.x : gridDim.x * static_cast<long>(kWarpRows);
  const int packs = a.H / V;
  const float inv_h = 1.f / static_cast<float>(a.H);
  float dw[VPT * V], db[VPT * V];
#pragma unroll
  for (int i = 0; i < VPT * V; ++i) dw[i] = db[i] = 0.f;
  for (long r = first; r < a.rows; r += step) {
    const Pack<T, V>* x = reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.x) + r * a.ldx);
    const Pack<T, V>* dy = reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.dy) + r * a.ldy);
    Pack<T, V> rx[VPT], rd[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * width < packs) {
        rx[k] = x[lane + k * width];
        rd[k] = dy[lane + k * width];
      }
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sa = 0.f, san = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int p = lane + k * width;
      if (p < packs) {
        float w[V];
        load_param<T, V>(a.w, a.w32, static_cast<long>(p) * V, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float g = to_f(rd[k].v[i]);
          const float n = (to_f(rx[k].v[i]) - mean) * rstd;
          dw[k * V + i] += g * n;
          db[k * V + i] += g;
          sa += g * w[i];
          san += g * w[i] * n;
        }
      }
    }
    const float2 sums = row_sum2<BLOCK>(sa, san, scratch);
    const float ma = sums.x * inv_h, man = sums.y * inv_h;
    T* dx = static_cast<T*>(a.out) + r * a.H;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int p = lane + k * width;
      if (p < packs) {
        float w[V], o[V];
        load_param<T, V>(a.w, a.w32, static_cast<long>(p) * V, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float n = (to_f(rx[k].v[i]) - mean) * rstd;
          o[i] = rstd * (to_f(rd[k].v[i]) * w[i] - ma - n * man);
        }
        store_pack<T, V>(dx + static_cast<long>(p) * V, o);
      }
    }
  }
  float* part = a.part + static_cast<long>(blockIdx.x) * 2 * a.H;
  if constexpr (BLOCK) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int p = lane + k * width;
      if (p < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          part[p * V + i] = dw[k * V + i];
          part[a.H + p * V + i] = db[k * V + i];
        }
    }
  } else {
    // one warp after the other adds its sums: a fixed order
    for (int w = 0; w < kWarpRows; ++w) {
      if (warp == w) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          const int p = lane + k * width;
          if (p < packs)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float* at = smem + p * V + i;
              at[0] = (w == 0 ? 0.f : at[0]) + dw[k * V + i];
              at[a.H] = (w == 0 ? 0.f : at[a.H]) + db[k * V + i];
            }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * a.H; c += blockDim.x) part[c] = smem[c];
  }
}

// dx of rows that do not fit the registers; their dw and db come from ln_cols_long.
template <typename T>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(const NormArgs a) {
  __shared__ float2 scratch[32];
  const float inv_h = 1.f / static_cast<float>(a.H);
  for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + r * a.ldy;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sa = 0.f, san = 0.f;
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
      float w[1];
      load_param<T, 1>(a.w, a.w32, c, w);
      const float g = to_f(dy[c]) * w[0];
      sa += g;
      san += g * ((to_f(x[c]) - mean) * rstd);
    }
    const float2 sums = row_sum2<true>(sa, san, scratch);
    const float ma = sums.x * inv_h, man = sums.y * inv_h;
    T* dx = static_cast<T*>(a.out) + r * a.H;
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
      float w[1];
      load_param<T, 1>(a.w, a.w32, c, w);
      const float n = (to_f(x[c]) - mean) * rstd;
      dx[c] = from_f<T>(rstd * (to_f(dy[c]) * w[0] - ma - n * man));
    }
  }
}

// Column sums of dy n and dy over every gridDim.y-th row, a thread per column.
template <typename T>
__global__ void __launch_bounds__(256) ln_cols_long_kernel(const NormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.H) return;
  float dw = 0.f, db = 0.f;
  for (long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const float g = to_f(static_cast<const T*>(a.dy)[r * a.ldy + c]);
    dw += g * ((to_f(static_cast<const T*>(a.x)[r * a.ldx + c]) - a.mean[r]) * a.rstd[r]);
    db += g;
  }
  float* part = a.part + static_cast<long>(blockIdx.y) * 2 * a.H;
  part[c] = dw;
  part[a.H + c] = db;
}

// out[c] = sum over the blocks' partial sums, in a fixed order; columns [0, H)
// are dw, [H, 2H) db.  32 columns per block, 32 threads down each.
template <typename T>
__global__ void __launch_bounds__(1024) ln_join_kernel(const float* __restrict__ part, int blocks, int H, void* dw,
                                                       void* db, bool w32, bool b32) {
  __shared__ float sum[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < 2 * H)
    for (int p = threadIdx.y; p < blocks; p += 32) s += part[static_cast<long>(p) * 2 * H + c];
  sum[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  const float v = warp_sum(sum[threadIdx.x][threadIdx.y]);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < 2 * H) {
    const bool is_w = col < H;
    void* out = is_w ? dw : db;
    const int i = is_w ? col : col - H;
    if (out != nullptr) {
      if (is_w ? w32 : b32) static_cast<float*>(out)[i] = v;
      else static_cast<T*>(out)[i] = from_f<T>(v);
    }
  }
}

using NormKernel = void (*)(NormArgs);

// The kernel for rows of H values, its threads per block and rows per block.
struct NormPlan {
  NormKernel kernel;   // null: the long variant
  int threads;
  int rows;
};

template <typename T, int V, bool FWD, int VPT, bool BLOCK>
NormKernel pick() {
  if constexpr (FWD) return &ln_fwd_kernel<T, V, VPT, BLOCK>;
  else return &ln_bwd_kernel<T, V, VPT, BLOCK>;
}

template <typename T, int V, bool FWD>
NormPlan norm_plan(int packs) {
  if (packs <= 32) return {pick<T, V, FWD, 1, false>(), 32 * kWarpRows, kWarpRows};
  if (packs <= 64) return {pick<T, V, FWD, 2, false>(), 32 * kWarpRows, kWarpRows};
  if (packs <= 96) return {pick<T, V, FWD, 3, false>(), 32 * kWarpRows, kWarpRows};
  if (packs <= 128) return {pick<T, V, FWD, 4, false>(), 32 * kWarpRows, kWarpRows};
  if (packs <= 160) return {pick<T, V, FWD, 5, false>(), 32 * kWarpRows, kWarpRows};
  const auto threads = [&](int per) { return (packs + 32 * per - 1) / (32 * per) * 32; };
  if (packs <= 1024) return {pick<T, V, FWD, 2, true>(), threads(2), 1};
  if (packs <= 2048) return {pick<T, V, FWD, 4, true>(), threads(4), 1};
  if (V == 1 && packs <= 4096) return {pick<T, V, FWD, 8, true>(), threads(8), 1};
  return {nullptr, 1024, 1};
}

template <typename T, bool FWD>
NormPlan norm_plan_of(int H, bool wide) {
  constexpr int W = kPackSize<T, true>;
  return wide ? norm_plan<T, W, FWD>(H / W) : norm_plan<T, 1, FWD>(H);
}

void check_rows(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.dim() == 2 &&
                  t.sizes() == like.sizes() && (t.stride(1) == 1 || t.size(1) == 1),
              name, " must be [rows, H] of x's type and device with unit inner stride");
}

void check_param(const torch::Tensor& p, const char* name, const torch::Tensor& x) {
  TORCH_CHECK(p.device() == x.device() && p.dim() == 1 && p.size(0) == x.size(1) && p.is_contiguous() &&
                  (p.scalar_type() == x.scalar_type() || p.scalar_type() == torch::kFloat32),
              name, " must be a contiguous [H] of x's type or fp32");
}

}  // namespace

void layer_norm_fwd(torch::Tensor x, torch::Tensor w, c10::optional<torch::Tensor> b, torch::Tensor y,
                    torch::Tensor mean, torch::Tensor rstd, double eps) {
  TORCH_CHECK(is_storage_type(x), "x must be bf16, fp16 or fp32");
  check_rows(x, "x", x);
  check_rows(y, "y", x);
  check_param(w, "weight", x);
  if (b.has_value()) check_param(*b, "bias", x);
  TORCH_CHECK(y.is_contiguous() && x.size(1) >= 1, "y must be contiguous and H at least 1");
  TORCH_CHECK(mean.scalar_type() == torch::kFloat32 && rstd.scalar_type() == torch::kFloat32 &&
                  mean.is_contiguous() && rstd.is_contiguous() && mean.numel() == x.size(0) &&
                  rstd.numel() == x.size(0), "mean and rstd must be fp32 [rows]");
  const c10::cuda::CUDAGuard guard(x.device());
  if (x.size(0) == 0) return;
  NormArgs a{};
  a.x = x.data_ptr();
  a.w = w.data_ptr();
  a.b = b.has_value() ? b->data_ptr() : nullptr;
  a.out = y.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.rows = x.size(0);
  a.ldx = x.stride(0);
  a.H = static_cast<int>(x.size(1));
  a.eps = static_cast<float>(eps);
  a.w32 = w.scalar_type() == torch::kFloat32;
  a.b32 = b.has_value() && b->scalar_type() == torch::kFloat32;
  const bool wide = wide_rows(x) && wide_rows(y) && aligned16(a.w) && aligned16(a.b);
  auto stream = at::cuda::getCurrentCUDAStream();
  by_type(x.scalar_type(), [&](auto tag) {
    using T = decltype(tag);
    const NormPlan p = norm_plan_of<T, true>(a.H, wide);
    const long blocks = (a.rows + p.rows - 1) / p.rows;
    if (p.kernel != nullptr) p.kernel<<<static_cast<unsigned>(std::min<long>(blocks, 1L << 30)), p.threads, 0, stream>>>(a);
    else ln_fwd_long_kernel<T><<<static_cast<unsigned>(std::min<long>(blocks, 1L << 30)), 1024, 0, stream>>>(a);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void layer_norm_bwd(torch::Tensor dy, torch::Tensor x, torch::Tensor w, torch::Tensor mean, torch::Tensor rstd,
                    torch::Tensor dx, torch::Tensor dw, c10::optional<torch::Tensor> db) {
  TORCH_CHECK(is_storage_type(x), "x must be bf16, fp16 or fp32");
  check_rows(x, "x", x);
  check_rows(dy, "dy", x);
  check_rows(dx, "dx", x);
  check_param(w, "weight", x);
  check_param(dw, "dw", x);
  if (db.has_value()) check_param(*db, "db", x);
  TORCH_CHECK(dx.is_contiguous() && x.size(1) >= 1, "dx must be contiguous and H at least 1");
  TORCH_CHECK(mean.scalar_type() == torch::kFloat32 && rstd.scalar_type() == torch::kFloat32 &&
                  mean.is_contiguous() && rstd.is_contiguous() && mean.numel() == x.size(0) &&
                  rstd.numel() == x.size(0), "mean and rstd must be fp32 [rows]");
  const c10::cuda::CUDAGuard guard(x.device());
  NormArgs a{};
  a.x = x.data_ptr();
  a.dy = dy.data_ptr();
  a.w = w.data_ptr();
  a.out = dx.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.rows = x.size(0);
  a.ldx = x.stride(0);
  a.ldy = dy.stride(0);
  a.H = static_cast<int>(x.size(1));
  a.w32 = w.scalar_type() == torch::kFloat32;
  const bool wide = wide_rows(x) && wide_rows(dy) && wide_rows(dx) && aligned16(a.w);
  auto stream = at::cuda::getCurrentCUDAStream();
  by_type(x.scalar_type(), [&](auto tag) {
    using T = decltype(tag);
    const NormPlan p = norm_plan_of<T, false>(a.H, wide);
    // as many blocks as run at once: each carries its column sums through its rows
    const long per_sm = p.kernel == nullptr ? 1 : std::max(1, 512 / p.threads);
    const int blocks = static_cast<int>(std::max<long>(1, std::min<long>((a.rows + p.rows - 1) / p.rows, kSMs * per_sm)));
    torch::Tensor part = torch::empty({blocks, 2, a.H}, x.options().dtype(torch::kFloat32));
    a.part = part.data_ptr<float>();
    if (p.kernel != nullptr) {
      const int smem = p.rows > 1 ? 2 * a.H * 4 : 0;
      p.kernel<<<blocks, p.threads, smem, stream>>>(a);
    } else {
      if (a.rows > 0) {
        ln_bwd_long_kernel<T><<<static_cast<unsigned>(std::min<long>(a.rows, kSMs * 2)), 1024, 0, stream>>>(a);
        C10_CUDA_KERNEL_LAUNCH_CHECK();
      }
      ln_cols_long_kernel<T><<<dim3((a.H + 255) / 256, blocks), 256, 0, stream>>>(a);
    }
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    ln_join_kernel<T><<<(2 * a.H + 31) / 32, dim3(32, 32), 0, stream>>>(
        a.part, blocks, a.H, dw.data_ptr(), db.has_value() ? db->data_ptr() : nullptr,
        dw.scalar_type() == torch::kFloat32, db.has_value() && db->scalar_type() == torch::kFloat32);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
}

}  // namespace gb
