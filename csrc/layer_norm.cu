// Layer norm over the last dimension, forward and backward, with the
// reductions of the weight's and the bias's gradient.
//
//   n = (x - mean) rstd,  y = n w + b                       mean, rstd per row
//   a = dy w,  dx = rstd (a - mean(a) - n mean(a n))        per row
//   dw = sum_rows dy n,  db = sum_rows dy                   per column
//
// Memory bound: the forward reads x and writes y, the backward reads x and dy
// and writes dx.
//
// Forward: a row is read once and kept in registers, where the mean and then the
// centred sum of squares are taken (fp32; no cancellation of E[x^2] - mean^2).
// Up to 1280 bf16 values a warp takes a row: no barrier, many rows in flight.
//
// Backward: besides a row's two sums there are two sums per column.  A thread
// owns a few columns for all rows of its block, so that those stay in registers,
// and takes R rows at a time: their loads are in flight together and their 2 R
// row sums share a barrier.  (A warp a row needs 80 registers of column sums
// a thread at 1152 columns and left one block of 256 threads per SM.)  Rows of
// up to 64 packs keep the warp-a-row form.  The blocks' column sums are joined
// by a second, small kernel in a fixed order.
//
// Rows that are no multiple of 16 bytes are read value by value; rows past the
// variants below are walked several times (they stay in L1/L2).
//
// Measured on a B200, 65536 x 1152 bf16: forward 47 us (6.4 TB/s), backward 107 us
// (4.2 TB/s; 150 us with the rows in registers), 5003 x 1001 fp32 20 and 20 us.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <stdexcept>

#include "sm100_common.cuh"
#include "vec_types.cuh"

namespace gb {

namespace {

constexpr int kWarpRows = 8;   // rows in flight per block of the warp-a-row variants,
constexpr int kFewRows = 4;    // and of the forward where rows are few: even shares of the SMs
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

// Sums of N values over the warp (N a power of two, at most 32): each step
// exchanges half of the values, so that N - 1 + 5 - log2 N shuffles do it rather
// than 5 N.  Lane l gets the sum of value l >> (5 - log2 N).
template <int N>
__device__ __forceinline__ float warp_sum_many(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int bit = 16;
#pragma unroll
  for (int half = N / 2; half > 0; half >>= 1) {
    const bool up = (lane & bit) != 0;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float give = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
    }
    bit >>= 1;
  }
  for (; bit > 0; bit >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit);
  return v[0];
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
  int* err;           // ring kernel: set when a row's copy never arrives
};

template <typename T, int V, int VPT, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : 32 * kFewRows, BLOCK ? 2 : 8) ln_fwd_kernel(const NormArgs a) {
  __shared__ float scratch[32];
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const int width = BLOCK ? blockDim.x : 32;
  const long first = BLOCK ? blockIdx.x : blockIdx.x * static_cast<long>(kFewRows) + (threadIdx.x >> 5);
  const long step = BLOCK ? gridDim.x : gridDim.x * static_cast<long>(kFewRows);
  const int packs = a.H / V;
  const float inv_h = 1.f / static_cast<float>(a.H);
  for (long r = first; r < a.rows; r += step) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    Pack<T, V> raw[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * width < packs) raw[k] = load_raw<T, V>(x + static_cast<long>(lane + k * width) * V);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * width < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) s += value(raw[k], i);
    const float mean = row_sum<BLOCK>(s, scratch) * inv_h;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * width < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float c = value(raw[k], i) - mean;
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
        for (int i = 0; i < V; ++i) o[i] = (value(raw[k], i) - mean) * rstd * w[i] + b[i];
        store_pack<T, V>(y + static_cast<long>(p) * V, o);
      }
    }
    if (lane == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
  }
}

// The warp-a-row forward for many rows: blocks stay, weight and bias wait in
// shared memory as fp32 (unpacking them for every row was a quarter of the
// instructions), and a warp's next row is on its way while it works on one.
template <typename T, int V, int VPT>
__global__ void __launch_bounds__(32 * kWarpRows, 3) ln_fwd_many_kernel(const NormArgs a) {
  static_assert(V % 4 == 0, "whole float4");
  __shared__ float4 param[2][VPT * (V / 4)][32];  // [weight, bias][pack and quarter][lane]
  const int lane = threadIdx.x & 31;
  const int packs = a.H / V;
  const float inv_h = 1.f / static_cast<float>(a.H);
  for (int p = threadIdx.x; p < packs; p += blockDim.x) {
    float w[V], b[V] = {};
    load_param<T, V>(a.w, a.w32, static_cast<long>(p) * V, w);
    if (a.b != nullptr) load_param<T, V>(a.b, a.b32, static_cast<long>(p) * V, b);
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      param[0][(p >> 5) * (V / 4) + q][p & 31] = make_float4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
      param[1][(p >> 5) * (V / 4) + q][p & 31] = make_float4(b[4 * q], b[4 * q + 1], b[4 * q + 2], b[4 * q + 3]);
    }
  }
  __syncthreads();
  const long step = gridDim.x * static_cast<long>(kWarpRows);
  long r = blockIdx.x * static_cast<long>(kWarpRows) + (threadIdx.x >> 5);
  Pack<T, V> next[VPT];
  const auto fetch = [&](long row) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * 32 < packs) next[k] = load_raw<T, V>(x + (lane + k * 32) * V);
  };
  if (r < a.rows) fetch(r);
  for (; r < a.rows; r += step) {
    Pack<T, V> raw[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) raw[k] = next[k];
    if (r + step < a.rows) fetch(r + step);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * 32 < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) s += value(raw[k], i);
    const float mean = warp_sum(s) * inv_h;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * 32 < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float c = value(raw[k], i) - mean;
          s += c * c;
        }
    const float rstd = 1.f / sqrtf(warp_sum(s) * inv_h + a.eps);
    T* y = static_cast<T*>(a.out) + r * a.H;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (lane + k * 32 < packs) {
        float o[V];
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
          const float4 w = param[0][k * (V / 4) + q][lane], b = param[1][k * (V / 4) + q][lane];
          o[4 * q] = (value(raw[k], 4 * q) - mean) * rstd * w.x + b.x;
          o[4 * q + 1] = (value(raw[k], 4 * q + 1) - mean) * rstd * w.y + b.y;
          o[4 * q + 2] = (value(raw[k], 4 * q + 2) - mean) * rstd * w.z + b.z;
          o[4 * q + 3] = (value(raw[k], 4 * q + 3) - mean) * rstd * w.w + b.w;
        }
        store_pack<T, V>(y + (lane + k * 32) * V, o);
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

// Backward of narrow rows, a warp each (packs <= 32 VPT).
template <typename T, int V, int VPT>
__global__ void __launch_bounds__(32 * kWarpRows) ln_bwd_warp_kernel(const NormArgs a) {
  __shared__ float sum[kWarpRows / 2][2 * 32 * VPT * V];  // half of the warps' column sums
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int packs = a.H / V;
  const float inv_h = 1.f / static_cast<float>(a.H);
  float dw[VPT * V], db[VPT * V];
#pragma unroll
  for (int i = 0; i < VPT * V; ++i) dw[i] = db[i] = 0.f;
  for (long r = blockIdx.x * static_cast<long>(kWarpRows) + warp; r < a.rows;
       r += gridDim.x * static_cast<long>(kWarpRows)) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + r * a.ldy;
    Pack<T, V> rx[VPT], rd[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (lane + k * 32 < packs) {
        rx[k] = load_raw<T, V>(x + (lane + k * 32) * V);
        rd[k] = load_raw<T, V>(dy + (lane + k * 32) * V);
      }
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sa = 0.f, san = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int p = lane + k * 32;
      if (p < packs) {
        float w[V];
        load_param<T, V>(a.w, a.w32, static_cast<long>(p) * V, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float g = value(rd[k], i);
          const float n = (value(rx[k], i) - mean) * rstd;
          dw[k * V + i] += g * n;
          db[k * V + i] += g;
          sa += g * w[i];
          san += g * w[i] * n;
        }
      }
    }
    const float ma = warp_sum(sa) * inv_h, man = warp_sum(san) * inv_h;
    T* dx = static_cast<T*>(a.out) + r * a.H;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int p = lane + k * 32;
      if (p < packs) {
        float w[V], o[V];
        load_param<T, V>(a.w, a.w32, static_cast<long>(p) * V, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float n = (value(rx[k], i) - mean) * rstd;
          o[i] = rstd * (value(rd[k], i) * w[i] - ma - n * man);
        }
        store_pack<T, V>(dx + static_cast<long>(p) * V, o);
      }
    }
  }
  // the upper half of the warps hands its sums to the lower half until one has them all;
  // value-major, so that a warp's accesses fall into different banks
  for (int half = kWarpRows / 2; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) {
#pragma unroll
      for (int i = 0; i < VPT * V; ++i) {
        sum[warp - half][i * 32 + lane] = dw[i];
        sum[warp - half][(VPT * V + i) * 32 + lane] = db[i];
      }
    }
    __syncthreads();
    if (warp < half) {
#pragma unroll
      for (int i = 0; i < VPT * V; ++i) {
        dw[i] += sum[warp][i * 32 + lane];
        db[i] += sum[warp][(VPT * V + i) * 32 + lane];
      }
    }
    __syncthreads();
  }
  float* part = a.part + static_cast<long>(blockIdx.x) * 2 * a.H;
  if (warp == 0) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int p = lane + k * 32;
      if (p < packs)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          part[p * V + i] = dw[k * V + i];
          part[a.H + p * V + i] = db[k * V + i];
        }
    }
  }
}

// Two fp32 values in a 64-bit register: one instruction for both.
struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// Backward of wider rows: thread t owns the packs t + k blockDim.x of every row
// of its block and takes R rows at a time; the next R are on their way while it
// waits for their sums.  Values past the row or past the last row are zeros, so
// that only loads and stores ask.  Bound by instructions before the arithmetic
// went in pairs (45 a value, 148 us at 65536 x 1152).
template <typename T, int V, int VPT, int R>
__global__ void __maxnreg__(V * VPT * R <= 16 ? 104 : 128) ln_bwd_kernel(const NormArgs a) {
  constexpr int E = V * VPT;            // values per thread and row
  static_assert(E % 2 == 0, "pairs");
  __shared__ float part_s[2][2 * R][17];   // [turn][row sum][warp]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int packs = a.H / V;
  const float inv_h = 1.f / static_cast<float>(a.H);
  const long per = (a.rows + gridDim.x - 1) / gridDim.x;
  const long begin = min(a.rows, blockIdx.x * per), end = min(a.rows, begin + per);
  Two w[E / 2], dw[E / 2], db[E / 2];
  {
    float f[E] = {};
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int p = threadIdx.x + k * blockDim.x;
      float q[V];
      if (p < packs) {
        load_param<T, V>(a.w, a.w32, static_cast<long>(p) * V, q);
#pragma unroll
        for (int i = 0; i < V; ++i) f[k * V + i] = q[i];
      }
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      w[i] = two(f[2 * i], f[2 * i + 1]);
      dw[i] = db[i] = two(0.f, 0.f);
    }
  }
  Pack<T, V> rx[R][VPT], rd[R][VPT];
  float mean[R], rstd[R];
  const auto fetch = [&](long r0) {
    const T* x = static_cast<const T*>(a.x) + r0 * a.ldx + threadIdx.x * V;
    const T* dy = static_cast<const T*>(a.dy) + r0 * a.ldy + threadIdx.x * V;
#pragma unroll
    for (int j = 0; j < R; ++j, x += a.ldx, dy += a.ldy) {
      const bool row = r0 + j < end;
      mean[j] = row ? a.mean[r0 + j] : 0.f;
      rstd[j] = row ? a.rstd[r0 + j] : 0.f;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        rx[j][k] = rd[j][k] = Pack<T, V>{};
        if (row && threadIdx.x + k * blockDim.x < packs) {
          rx[j][k] = load_raw<T, V>(x + k * blockDim.x * V);
          rd[j][k] = load_raw<T, V>(dy + k * blockDim.x * V);
        }
      }
    }
  };
  int turn = 0;
  fetch(begin);
  for (long r0 = begin; r0 < end; r0 += R) {
    Two n[R][E / 2], gw[R][E / 2];   // normalised values, dy w
    float s[2 * R], scale[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const Two shift = two(-mean[j], -mean[j]), mul = two(rstd[j], rstd[j]);
      scale[j] = rstd[j];
      Two sa = two(0.f, 0.f), san = two(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const int k0 = 2 * i / V, i0 = 2 * i % V, k1 = (2 * i + 1) / V, i1 = (2 * i + 1) % V;
        const Two g = two(value(rd[j][k0], i0), value(rd[j][k1], i1));
        n[j][i] = mul2(add2(two(value(rx[j][k0], i0), value(rx[j][k1], i1)), shift), mul);
        gw[j][i] = mul2(g, w[i]);
        dw[i] = fma2(g, n[j][i], dw[i]);
        db[i] = add2(db[i], g);
        sa = add2(sa, gw[j][i]);
        san = fma2(gw[j][i], n[j][i], san);
      }
      const float2 p = both(sa), q = both(san);
      s[j] = p.x + p.y;
      s[R + j] = q.x + q.y;
    }
    fetch(r0 + R);
    const float mine = warp_sum_many<2 * R>(s);
    constexpr int kSpread = 32 / (2 * R);  // lanes that hold the same sum
    if (lane % kSpread == 0) part_s[turn][lane / kSpread][warp] = mine;
    __syncthreads();
    // every warp adds the warps' parts itself: one barrier, and the other buffer next
    float total = 0.f;
#pragma unroll 4
    for (int v = 0; v < warps; ++v) total += part_s[turn][lane % (2 * R)][v];
    total *= inv_h;
    turn ^= 1;
    T* dx = static_cast<T*>(a.out) + r0 * a.H + threadIdx.x * V;
#pragma unroll
    for (int j = 0; j < R; ++j, dx += a.H) {
      const float ma = -__shfl_sync(0xffffffffu, total, j), man = -__shfl_sync(0xffffffffu, total, R + j);
      const Two ma2 = two(ma, ma), man2 = two(man, man), mul = two(scale[j], scale[j]);
      float o[E];
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 q = both(mul2(add2(fma2(n[j][i], man2, gw[j][i]), ma2), mul));
        o[2 * i] = q.x;
        o[2 * i + 1] = q.y;
      }
      if (r0 + j < end) {
#pragma unroll
        for (int k = 0; k < VPT; ++k)
          if (threadIdx.x + k * blockDim.x < packs) {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = o[k * V + i];
            store_pack<T, V>(dx + k * blockDim.x * V, f);
          }
      }
    }
  }
  float* part = a.part + static_cast<long>(blockIdx.x) * 2 * a.H;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int p = threadIdx.x + k * blockDim.x;
    if (p < packs)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 x = both(dw[(k * V + i) / 2]), y = both(db[(k * V + i) / 2]);
        part[p * V + i] = (k * V + i) % 2 ? x.y : x.x;
        part[a.H + p * V + i] = (k * V + i) % 2 ? y.y : y.x;
      }
  }
}

// The same for many rows of up to 2048 values: rows come by bulk copies into a
// ring of shared-memory stages (R rows of x and dy each) instead of registers.
// The register form kept 9 warps of 104 registers on an SM, whose loads in flight
// reached 2.9 TB/s; the ring holds some 100 KB of loads whatever the registers do.
// A stage is read before its rows' barrier and refilled after it by one thread, so
// it needs no second barrier.  4 values per thread and row.  Where a wait gives up,
// that barrier tells the whole block, which fills no stage again and ends there; the
// copies under way are waited for, whatever the error word says, since the next
// block on the SM gets this one's shared memory.  (Through shared memory: 103 -> 107 us; a
// barrier with a vote, or leaving the loop, made the kernel spill, 187 us.)
constexpr int kRing = 3;

template <typename T, int R>
__global__ void __maxnreg__(80) ln_bwd_ring_kernel(const NormArgs a) {
  constexpr int V = 4;
  extern __shared__ __align__(128) uint8_t ring[];   // [stage][x, dy][row][H]
  __shared__ __align__(8) uint64_t full[kRing];
  __shared__ int late[2];                  // [turn] whether a wait gave up
  __shared__ float part_s[2][2 * R][17];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const bool mine_in = static_cast<int>(threadIdx.x) * V < a.H;
  const float inv_h = 1.f / static_cast<float>(a.H);
  const uint32_t row_bytes = a.H * sizeof(T);
  const uint32_t stage_bytes = 2 * R * row_bytes;
  const long per = (a.rows + gridDim.x - 1) / gridDim.x;
  const long begin = min(a.rows, blockIdx.x * per);
  long end = min(a.rows, begin + per);
  const auto fill = [&](long r0, int stage) {   // one thread
    if (r0 >= end) return;
    const int rows = static_cast<int>(min(static_cast<long>(R), end - r0));
    mbar_arrive_expect_tx(&full[stage], 2 * rows * row_bytes);
    uint8_t* at = ring + stage * stage_bytes;
    for (int j = 0; j < rows; ++j) {
      bulk_copy_g2s(at + j * row_bytes, static_cast<const T*>(a.x) + (r0 + j) * a.ldx, row_bytes, &full[stage]);
      bulk_copy_g2s(at + (R + j) * row_bytes, static_cast<const T*>(a.dy) + (r0 + j) * a.ldy, row_bytes, &full[stage]);
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) mbar_init(&full[s], 1);
    late[0] = late[1] = 0;
    fence_mbar_init();
    for (int s = 0; s < kRing; ++s) fill(begin + s * R, s);
  }
  Two w[2], dw[2], db[2];
  {
    float f[V] = {};
    if (mine_in) load_param<T, V>(a.w, a.w32, static_cast<long>(threadIdx.x) * V, f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = two(f[2 * i], f[2 * i + 1]);
      dw[i] = db[i] = two(0.f, 0.f);
    }
  }
  float mean[R], rstd[R];
  const auto stats = [&](long r0) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      mean[j] = r0 + j < end ? a.mean[r0 + j] : 0.f;
      rstd[j] = r0 + j < end ? a.rstd[r0 + j] : 0.f;
    }
  };
  stats(begin);
  __syncthreads();
  int turn = 0, stage = 0;
  uint32_t phase = 0;
  for (long r0 = begin; r0 < end; r0 += R) {
    if (!mbar_wait(&full[stage], phase, a.err, kErrTmaFullTimeout)) late[turn] = 1;
    Two n[R][2], gw[R][2];
    float s[2 * R], scale[R];
    const T* at = reinterpret_cast<const T*>(ring + stage * stage_bytes) + threadIdx.x * V;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      Pack<T, V> rx{}, rd{};
      if (mine_in && r0 + j < end) {
        rx = load_raw<T, V>(at + j * a.H);
        rd = load_raw<T, V>(at + (R + j) * a.H);
      }
      const Two shift = two(-mean[j], -mean[j]), mul = two(rstd[j], rstd[j]);
      scale[j] = rstd[j];
      Two sa = two(0.f, 0.f), san = two(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Two g = two(value(rd, 2 * i), value(rd, 2 * i + 1));
        n[j][i] = mul2(add2(two(value(rx, 2 * i), value(rx, 2 * i + 1)), shift), mul);
        gw[j][i] = mul2(g, w[i]);
        dw[i] = fma2(g, n[j][i], dw[i]);
        db[i] = add2(db[i], g);
        sa = add2(sa, gw[j][i]);
        san = fma2(gw[j][i], n[j][i], san);
      }
      const float2 p = both(sa), q = both(san);
      s[j] = p.x + p.y;
      s[R + j] = q.x + q.y;
    }
    stats(r0 + R);
    const float mine = warp_sum_many<2 * R>(s);
    constexpr int kSpread = 32 / (2 * R);
    if (lane % kSpread == 0) part_s[turn][lane / kSpread][warp] = mine;
    __syncthreads();
    if (late[turn] != 0) end = r0;
    if (threadIdx.x == 0) fill(r0 + kRing * R, stage);  // everyone has read this stage
    if (++stage == kRing) {
      stage = 0;
      phase ^= 1u;
    }
    float total = 0.f;
#pragma unroll 4
    for (int v = 0; v < warps; ++v) total += part_s[turn][lane % (2 * R)][v];
    total *= inv_h;
    turn ^= 1;
    T* dx = static_cast<T*>(a.out) + r0 * a.H + threadIdx.x * V;
#pragma unroll
    for (int j = 0; j < R; ++j, dx += a.H) {
      const float ma = -__shfl_sync(0xffffffffu, total, j), man = -__shfl_sync(0xffffffffu, total, R + j);
      const Two ma2 = two(ma, ma), man2 = two(man, man), mul = two(scale[j], scale[j]);
      const float2 p = both(mul2(add2(fma2(n[j][0], man2, gw[j][0]), ma2), mul));
      const float2 q = both(mul2(add2(fma2(n[j][1], man2, gw[j][1]), ma2), mul));
      const float o[V] = {p.x, p.y, q.x, q.y};
      if (mine_in && r0 + j < end) store_pack<T, V>(dx, o);
    }
  }
  if (threadIdx.x == 0)   // what was filled and not read
    for (long r0 = end; r0 < min(min(a.rows, begin + per), end + kRing * R); r0 += R) {
      const long i = (r0 - begin) / R;
      mbar_wait(&full[i % kRing], static_cast<uint32_t>(i / kRing) & 1u, nullptr, kErrTmaFullTimeout);
    }
  if (mine_in) {
    float* part = a.part + static_cast<long>(blockIdx.x) * 2 * a.H + threadIdx.x * V;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 x = both(dw[i]), y = both(db[i]);
      part[2 * i] = x.x, part[2 * i + 1] = x.y;
      part[a.H + 2 * i] = y.x, part[a.H + 2 * i + 1] = y.y;
    }
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

// The kernel for rows of H values (null: the one for long rows), its threads per
// block, and the rows that a block takes at least (0: as many blocks as stay resident).
struct NormPlan {
  NormKernel kernel;
  int threads;
  int rows;
};

int threads_for(int packs, int per) { return (packs + 32 * per - 1) / (32 * per) * 32; }

// many: rows for several rounds of the resident warps
template <typename T, bool WIDE>
NormPlan fwd_plan(int H, bool many) {
  constexpr int V = kPackSize<T, WIDE>;
  const int packs = H / V;
  constexpr int T1 = 32 * kWarpRows;
  if constexpr (WIDE) {
    if (many && packs <= 160) {
      if (packs <= 32) return {&ln_fwd_many_kernel<T, V, 1>, T1, 0};
      if (packs <= 64) return {&ln_fwd_many_kernel<T, V, 2>, T1, 0};
      if (packs <= 96) return {&ln_fwd_many_kernel<T, V, 3>, T1, 0};
      if (packs <= 128) return {&ln_fwd_many_kernel<T, V, 4>, T1, 0};
      return {&ln_fwd_many_kernel<T, V, 5>, T1, 0};
    }
  }
  if (packs <= 32) return {&ln_fwd_kernel<T, V, 1, false>, 32 * kFewRows, kFewRows};
  if (packs <= 64) return {&ln_fwd_kernel<T, V, 2, false>, 32 * kFewRows, kFewRows};
  if constexpr (WIDE) {
    if (packs <= 96) return {&ln_fwd_kernel<T, V, 3, false>, 32 * kFewRows, kFewRows};
    if (packs <= 128) return {&ln_fwd_kernel<T, V, 4, false>, 32 * kFewRows, kFewRows};
    if (packs <= 160) return {&ln_fwd_kernel<T, V, 5, false>, 32 * kFewRows, kFewRows};
    if (packs <= 1024) return {&ln_fwd_kernel<T, V, 2, true>, threads_for(packs, 2), 1};
    if (packs <= 2048) return {&ln_fwd_kernel<T, V, 4, true>, threads_for(packs, 4), 1};
  } else {
    if (packs <= 128) return {&ln_fwd_kernel<T, V, 4, false>, 32 * kFewRows, kFewRows};
    if (packs <= 256) return {&ln_fwd_kernel<T, V, 8, false>, 32 * kFewRows, kFewRows};
    if (packs <= 512) return {&ln_fwd_kernel<T, V, 16, false>, 32 * kFewRows, kFewRows};
    if (packs <= 1024) return {&ln_fwd_kernel<T, V, 32, false>, 32 * kFewRows, kFewRows};
    if (packs <= 8192) return {&ln_fwd_kernel<T, V, 16, true>, threads_for(packs, 16), 1};
  }
  return {nullptr, 1024, 1};
}

template <typename T, bool WIDE>
NormPlan bwd_plan(int H) {
  constexpr int V = kPackSize<T, WIDE>;
  const int packs = H / V;
  if (packs <= 32) return {&ln_bwd_warp_kernel<T, V, 1>, 32 * kWarpRows, kWarpRows};
  if (packs <= 64) return {&ln_bwd_warp_kernel<T, V, 2>, 32 * kWarpRows, kWarpRows};
  if constexpr (WIDE) {
    // half packs up to 2048 columns: twice the threads, twice the rows in flight
    if (sizeof(T) == 2 && H <= 2048) return {&ln_bwd_kernel<T, 4, 1, 4>, threads_for(H / 4, 1), 2};
    if (packs <= 512) return {&ln_bwd_kernel<T, V, 1, 16 / V>, threads_for(packs, 1), 1};
    if (packs <= 1024) return {&ln_bwd_kernel<T, V, 2, 2>, threads_for(packs, 2), 1};
    if constexpr (sizeof(T) == 4)
      if (packs <= 2048) return {&ln_bwd_kernel<T, V, 4, 1>, threads_for(packs, 4), 1};
  } else {
    if (packs <= 1024) return {&ln_bwd_kernel<T, V, 4, 4>, threads_for(packs, 4), 2};
    if (packs <= 4096) return {&ln_bwd_kernel<T, V, 8, 2>, threads_for(packs, 8), 1};
    if (packs <= 8192) return {&ln_bwd_kernel<T, V, 16, 1>, threads_for(packs, 16), 1};
  }
  return {nullptr, 1024, 1};
}

// A ValueError in Python, as the CPU form's checks give.
void require(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

void check_param(const torch::Tensor& p, const torch::Tensor& x, const char* what) {
  require(p.device() == x.device() && p.dim() == 1 && p.size(0) == x.size(-1) &&
              (p.scalar_type() == x.scalar_type() || p.scalar_type() == torch::kFloat32), what);
}

// [rows, H] with unit inner stride
torch::Tensor as_rows(const torch::Tensor& t) {
  if (t.dim() == 2 && t.stride(1) == 1) return t;
  torch::Tensor r = t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

void check_x(const torch::Tensor& x) {
  // (the column sums' 2 H indexes, rounded up to blocks of 32, are ints)
  require(x.is_cuda() && is_storage_type(x) && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= (1L << 30) - 16,
          "x must be a bf16, fp16 or fp32 CUDA tensor with a last dimension to normalise");
}

constexpr unsigned kMaxBlocks = 1u << 30;

}  // namespace

// (y, mean, rstd)
std::vector<torch::Tensor> layer_norm_fwd(torch::Tensor x, torch::Tensor w, c10::optional<torch::Tensor> b,
                                          double eps) {
  check_x(x);
  check_param(w, x, "weight must be [H] of x's type or fp32 on its device");
  if (b.has_value()) check_param(*b, x, "bias must be [H] of x's type or fp32 on its device");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t H = x.size(-1);
  const torch::Tensor rows = x.numel() > 0 ? as_rows(x) : x;
  const int64_t n = x.numel() / H;
  torch::Tensor y = torch::empty(x.sizes(), x.options());
  const auto f32 = x.options().dtype(torch::kFloat32);
  torch::Tensor mean = torch::empty({n}, f32), rstd = torch::empty({n}, f32);
  if (n == 0) return {y, mean, rstd};
  const torch::Tensor wc = w.contiguous(), bc = b.has_value() ? b->contiguous() : torch::Tensor();
  NormArgs a{};
  a.x = rows.data_ptr();
  a.w = wc.data_ptr();
  a.b = b.has_value() ? bc.data_ptr() : nullptr;
  a.out = y.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.rows = n;
  a.ldx = rows.stride(0);
  a.H = static_cast<int>(H);
  a.eps = static_cast<float>(eps);
  a.w32 = w.scalar_type() == torch::kFloat32;
  a.b32 = b.has_value() && b->scalar_type() == torch::kFloat32;
  const bool wide = wide_rows(rows) && aligned16(a.w) && aligned16(a.b);
  auto stream = at::cuda::getCurrentCUDAStream();
  by_type(x.scalar_type(), [&](auto tag) {
    using T = decltype(tag);
    const bool many = a.rows >= kSMs * 3 * kWarpRows * 4;
    const NormPlan p = wide ? fwd_plan<T, true>(a.H, many) : fwd_plan<T, false>(a.H, many);
    const long blocks = p.rows == 0 ? kSMs * 3 : (a.rows + p.rows - 1) / p.rows;
    const unsigned grid = static_cast<unsigned>(std::min<long>(blocks, kMaxBlocks));
    if (p.kernel != nullptr) p.kernel<<<grid, p.threads, 0, stream>>>(a);
    else ln_fwd_long_kernel<T><<<grid, 1024, 0, stream>>>(a);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {y, mean, rstd};
}

// (dx, dw, db); db is fp32 or of x's type
std::vector<torch::Tensor> layer_norm_bwd(torch::Tensor dy, torch::Tensor x, torch::Tensor w, torch::Tensor mean,
                                          torch::Tensor rstd, bool bias32, torch::Tensor err) {
  check_x(x);
  check_param(w, x, "weight must be [H] of x's type or fp32 on its device");
  require(dy.device() == x.device() && dy.scalar_type() == x.scalar_type() && dy.sizes() == x.sizes(),
          "dy must be like x");
  const int64_t H = x.size(-1), n = x.numel() / H;
  for (const torch::Tensor& t : {mean, rstd})
    require(t.device() == x.device() && t.scalar_type() == torch::kFloat32 && t.is_contiguous() && t.dim() == 1 &&
                t.size(0) == n, "mean and rstd must hold one fp32 value per row of x");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto f32 = x.options().dtype(torch::kFloat32);
  torch::Tensor dx = torch::empty(x.sizes(), x.options());
  torch::Tensor dw = torch::empty({H}, w.options()), db = torch::empty({H}, bias32 ? f32 : x.options());
  if (n == 0) {
    dw.zero_();
    db.zero_();
    return {dx, dw, db};
  }
  const torch::Tensor rows = as_rows(x), g = as_rows(dy), wc = w.contiguous();
  NormArgs a{};
  a.x = rows.data_ptr();
  a.dy = g.data_ptr();
  a.w = wc.data_ptr();
  a.out = dx.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.rows = n;
  a.ldx = rows.stride(0);
  a.ldy = g.stride(0);
  a.err = err.data_ptr<int>();
  a.H = static_cast<int>(H);
  a.w32 = w.scalar_type() == torch::kFloat32;
  const bool wide = wide_rows(rows) && wide_rows(g) && aligned16(a.w);
  auto stream = at::cuda::getCurrentCUDAStream();
  by_type(x.scalar_type(), [&](auto tag) {
    using T = decltype(tag);
    NormPlan p = wide ? bwd_plan<T, true>(a.H) : bwd_plan<T, false>(a.H);
    constexpr int kRingRows = 4;
    const int ring_bytes = kRing * 2 * kRingRows * a.H * static_cast<int>(sizeof(T));
    // several rounds of the ring per block, rows wide enough for some warps, and two blocks' rings on an SM
    const bool ring = wide && a.rows >= kSMs * 2 * kRingRows * 4 && a.H >= 512 && a.H <= 2048 && ring_bytes <= 100 * 1024;
    if (ring) p = {&ln_bwd_ring_kernel<T, kRingRows>, threads_for(a.H / 4, 1), 1};
    // as many blocks as run at once: each carries its column sums through its rows
    const long per_sm = p.kernel == nullptr ? 1 : std::max(1, 600 / p.threads);
    const int blocks = static_cast<int>(std::min<long>((a.rows + p.rows - 1) / p.rows, kSMs * per_sm));
    torch::Tensor part = torch::empty({blocks, 2, H}, f32);
    a.part = part.data_ptr<float>();
    if (ring) {
      C10_CUDA_CHECK(cudaFuncSetAttribute(p.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_bytes));
      p.kernel<<<blocks, p.threads, ring_bytes, stream>>>(a);
    } else if (p.kernel != nullptr) {
      p.kernel<<<blocks, p.threads, 0, stream>>>(a);
    } else {
      ln_bwd_long_kernel<T><<<static_cast<unsigned>(std::min<long>(a.rows, kSMs * 2)), 1024, 0, stream>>>(a);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      ln_cols_long_kernel<T><<<dim3((a.H + 255) / 256, blocks), 256, 0, stream>>>(a);
    }
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    ln_join_kernel<T><<<(2 * a.H + 31) / 32, dim3(32, 32), 0, stream>>>(a.part, blocks, a.H, dw.data_ptr(),
                                                                       db.data_ptr(), a.w32, bias32);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  return {dx, dw, db};
}

}  // namespace gb
