// Cross entropy of hidden states against a vocabulary projection, without
// keeping the logits, and its gradients for both.
//
//   l_tv = h_t . W_v     lse_t = log sum_v exp l_tv     loss_t = lse_t - l_{t,y_t}
//   d_tv = s_t (exp(l_tv - lse_t) - [v = y_t])     dh = d W     dW = d^T h
//
// s_t is the upstream gradient of token t's loss (over the number of trained
// tokens for the mean).  Tokens whose target is `ignore_index` take no part:
// their rows are left out before the products (`ce_scan`, `ce_gather`), so
// neither their time is spent nor can what they hold (NaN, infinities) reach
// a sum.  How many remain is known to the device only; the products read that
// count (GemmArgs::live).
//
// The vocabulary is walked in pieces of columns.  Per piece one product remakes
// the logits and its epilogue writes d in bf16 (tokens x piece), a second adds
// d W to fp32 sums of dh, a third contracts d with h over the tokens into the
// piece's rows of dW, which are complete then.  Pieces of columns rather than
// of tokens, because dh (tokens x hidden) is the smaller sum to carry.
//
// d is rounded to bf16: the tensor cores take bf16 operands, and the rounding
// of each entry is independent, so that it averages out in both contractions.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>

#include "gemm_tc.cuh"
#include "vec_types.cuh"

namespace gb {

namespace {

constexpr int kScanThreads = 1024;
constexpr int kScanPer = 8;     // tokens per thread and tile
constexpr int kRowPad = BM;     // rows of the compacted buffers come in whole GEMM tiles
constexpr int kCeBN = 256;      // vocabulary columns per tile; pieces are whole tiles

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// Places of the trained tokens: place[t] = position of token t among them (-1
// for an ignored one), token[m] and target[m] of the m-th.  A target outside
// the vocabulary that is not ignore_index is reported in err[1] and gets a NaN
// loss and a zero gradient.  One block: a token costs 24 bytes here and the
// products some 10 ns.
__global__ void __launch_bounds__(kScanThreads) ce_scan_kernel(const int64_t* __restrict__ targets, long T, long V,
                                                               long ignore, int* __restrict__ token,
                                                               int* __restrict__ place, int64_t* __restrict__ target,
                                                               float* __restrict__ loss, int* __restrict__ count,
                                                               int* __restrict__ err) {
  __shared__ int warp_sum_s[kScanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (long t0 = 0; t0 < T; t0 += kScanThreads * kScanPer) {
    const long first = t0 + static_cast<long>(threadIdx.x) * kScanPer;
    int64_t y[kScanPer];
    unsigned keep = 0;
#pragma unroll
    for (int i = 0; i < kScanPer; ++i) {
      y[i] = first + i < T ? targets[first + i] : ignore;
      if (first + i < T) {
        const bool in = y[i] >= 0 && y[i] < V;
        const bool live = in && y[i] != ignore;
        if (live) keep |= 1u << i;
        else {
          const bool bad = y[i] != ignore;
          if (bad) atomicExch(err + 1, kErrBadToken);
          place[first + i] = -1;
          loss[first + i] = bad ? __int_as_float(0x7fc00000) : 0.f;
        }
      }
    }
    int incl = __popc(keep);
    const int own = incl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sum_s[warp] = incl;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kScanThreads / 32; ++w) {
      const int s = warp_sum_s[w];
      if (w < warp) before += s;
      total += s;
    }
    int m = base + before + incl - own;
#pragma unroll
    for (int i = 0; i < kScanPer; ++i) {
      if (keep >> i & 1u) {
        token[m] = static_cast<int>(first + i);
        target[m] = y[i];
        place[first + i] = m;
        ++m;
      }
    }
    base += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}

// out[m] = in[token[m]] (in[m] without a token list) for m < count, zeros in
// the rows that fill the last tile and in the columns [H, ldo).
template <bool WIDE>
__global__ void __launch_bounds__(256) ce_gather_kernel(const __nv_bfloat16* __restrict__ in, long ldi, int H,
                                                        const int* __restrict__ token, const int* __restrict__ count,
                                                        long rows, __nv_bfloat16* __restrict__ out, int ldo) {
  constexpr int V = WIDE ? 8 : 1;
  const long n = count != nullptr ? *count : rows;
  const long end = count != nullptr ? min(rows, (n + kRowPad - 1) / kRowPad * kRowPad) : rows;
  for (long m = blockIdx.x; m < end; m += gridDim.x) {
    const bool live = m < n;
    const long src = !live ? 0 : token != nullptr ? token[m] : m;
    for (int c = threadIdx.x * V; c < ldo; c += blockDim.x * V) {
      Pack<__nv_bfloat16, V> p = {};
      if (live && c < H) p = load_raw<__nv_bfloat16, V>(in + src * ldi + c);
      store_raw<__nv_bfloat16, V>(out + m * ldo + c, p);
    }
  }
}

// The weight of a token's loss in the result: the upstream gradient, over the
// number of trained tokens for the mean.
__device__ __forceinline__ float ce_weight(const float* g, int per_token, int mean, int t, int n) {
  const float s = g == nullptr ? 1.f : per_token ? g[t] : g[0];
  return mean ? s / static_cast<float>(n) : s;
}

// lse and loss of every trained token from its blocks' (max, sum exp), one warp each.
__global__ void __launch_bounds__(256) ce_finish_kernel(const float2* __restrict__ part, int nblk,
                                                        const float* __restrict__ tgt_logit,
                                                        const int* __restrict__ token, const int* __restrict__ count,
                                                        const float* __restrict__ g, int per_token, int mean,
                                                        float* __restrict__ lse, float* __restrict__ loss,
                                                        float* __restrict__ scale) {
  const int n = *count;
  const int lane = threadIdx.x & 31;
  for (long m = blockIdx.x * 8L + (threadIdx.x >> 5); m < n; m += gridDim.x * 8L) {
    const float2* row = part + m * nblk;
    float mx = -INFINITY, sum = 0.f;
    for (int b = lane; b < nblk; b += 32) {
      const float2 p = row[b];
      const float top = fmaxf(mx, p.x);
      if (top > -INFINITY) sum = sum * __expf(mx - top) + p.y * __expf(p.x - top);
      else sum += p.y;  // a block of NaN only has a NaN sum and no maximum
      mx = top;
    }
    const float top = warp_max(mx);
    sum = warp_sum(top > -INFINITY ? sum * __expf(mx - top) : sum);
    if (lane == 0) {
      const int t = token[m];
      const float l = top + logf(sum);
      lse[m] = l;
      loss[t] = l - tgt_logit[m];
      if (scale != nullptr) scale[m] = ce_weight(g, per_token, mean, t, n);
    }
  }
}

__global__ void __launch_bounds__(256) ce_scale_kernel(const int* __restrict__ token, const int* __restrict__ count,
                                                       const float* __restrict__ g, int per_token, int mean,
                                                       float* __restrict__ scale) {
  const int n = *count;
  for (long m = blockIdx.x * 256L + threadIdx.x; m < n; m += gridDim.x * 256L)
    scale[m] = ce_weight(g, per_token, mean, token[m], n);
}

// Sum of the tokens' losses in a fixed order, over the trained tokens for the
// mean (no trained token: 0).
__global__ void __launch_bounds__(1024) ce_total_kernel(const float* __restrict__ loss, long T,
                                                        const int* __restrict__ count, int mean,
                                                        float* __restrict__ out) {
  __shared__ double part[32];
  double s = 0;
  for (long t = threadIdx.x; t < T; t += 1024) s += loss[t];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = part[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) *out = static_cast<float>(mean ? s / max(1, *count) : s);
  }
}

// dh[t] = sum of the slices' row place[t], rounded once; zero for an ignored token.
template <bool WIDE>
__global__ void __launch_bounds__(256) ce_scatter_kernel(const float* __restrict__ acc, int lda, long slice, int splits,
                                                         const int* __restrict__ place, long T, int H,
                                                         __nv_bfloat16* __restrict__ dh) {
  constexpr int V = WIDE ? 8 : 1;
  for (long t = blockIdx.x; t < T; t += gridDim.x) {
    const int m = place[t];
    for (int c = threadIdx.x * V; c < H; c += 256 * V) {
      float s[V] = {};
      if (m >= 0) {
        const float* src = acc + static_cast<long>(m) * lda + c;
        for (int k = 0; k < splits; ++k, src += slice) {
          if constexpr (WIDE) {
            const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
            s[0] += a.x, s[1] += a.y, s[2] += a.z, s[3] += a.w;
            s[4] += b.x, s[5] += b.y, s[6] += b.z, s[7] += b.w;
          } else {
            s[0] += *src;
          }
        }
      }
      store_pack<__nv_bfloat16, V>(dh + t * H + c, s);
    }
  }
}

template <typename T>
T* ptr(const torch::Tensor& t) {
  return reinterpret_cast<T*>(t.data_ptr());
}

// TMA reads rows of 16-byte multiples from a 16-byte boundary; W in another
// layout is copied into one (the columns past H are zero).
torch::Tensor tma_rows(const torch::Tensor& W, cudaStream_t stream) {
  const int64_t V = W.size(0), H = W.size(1);
  if (W.stride(1) == 1 && W.stride(0) % 8 == 0 && W.stride(0) >= H && aligned16(W.data_ptr())) return W;
  const torch::Tensor src = W.stride(1) == 1 ? W : W.contiguous();
  torch::Tensor out = torch::empty({V, round_up(H, 8)}, W.options());
  ce_gather_kernel<false><<<static_cast<int>(std::min<int64_t>(V, 148 * 16)), 256, 0, stream>>>(
      ptr<__nv_bfloat16>(src), src.stride(0), static_cast<int>(H), nullptr, nullptr, V, ptr<__nv_bfloat16>(out),
      static_cast<int>(out.size(1)));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

void launch_ce(GemmLauncher fn, const CUtensorMap& a, const CUtensorMap& b, GemmArgs args, cudaStream_t stream,
               int device) {
  fn(a, b, a, b, args, 0, stream, device);
}

}  // namespace

GemmLauncher gemm_launcher_ce(int epi) {
  switch (epi) {
    case kCeLse: return &launch_gemm<kCeBN, kCeLse, false, 0>;
    case kCeGrad: return &launch_gemm<kCeBN, kCeGrad, false, 0>;
    case kCeDh: return &launch_gemm<kCeBN, kCeDh, false, 1>;
    case kCeDw: return &launch_gemm<kCeBN, kCeDw, false, 3>;
    default: return nullptr;
  }
}

// Forward.  reduction: 0 none, 1 sum, 2 mean.  Returns (loss, compacted h,
// token, place, target, count, lse, scale); scale is filled when `grad`
// (upstream gradient, fp32: one value, or one per token without a reduction)
// says that the backward follows with it, or with_scale asks for that of 1.
std::vector<torch::Tensor> ce_forward(torch::Tensor h, torch::Tensor W, torch::Tensor targets, int64_t ignore_index,
                                      int64_t reduction, c10::optional<torch::Tensor> grad, bool with_scale,
                                      torch::Tensor err) {
  TORCH_CHECK(h.is_cuda() && h.scalar_type() == torch::kBFloat16 && h.dim() == 2, "h must be a 2-D CUDA bf16 tensor");
  TORCH_CHECK(W.device() == h.device() && W.scalar_type() == torch::kBFloat16 && W.dim() == 2 &&
                  W.size(1) == h.size(1) && W.size(0) >= 1 && W.size(1) >= 1,
              "weight must be a bf16 matrix [V, H] on the device of h");
  TORCH_CHECK(targets.device() == h.device() && targets.scalar_type() == torch::kInt64 && targets.dim() == 1 &&
                  targets.is_contiguous() && targets.size(0) == h.size(0),
              "targets must be a contiguous int64 vector with one entry per row of h");
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "reduction must be 0, 1 or 2");
  TORCH_CHECK(h.size(0) < (1LL << 31) - kRowPad && W.size(0) < (1LL << 31) - kCeBN && W.size(1) < (1LL << 31) - kCeBN,
              "sizes must fit 31 bits");
  const c10::cuda::CUDAGuard guard(h.device());
  const int device = h.get_device();
  auto stream = at::cuda::getCurrentCUDAStream();
  const int64_t T = h.size(0), H = h.size(1), V = W.size(0);
  const int64_t cap = std::max<int64_t>(round_up(T, kRowPad), kRowPad), Hp = round_up(H, 8);
  const int nblk = static_cast<int>((V + kCeBN - 1) / kCeBN);
  const auto f32 = h.options().dtype(torch::kFloat32);
  const auto i32 = h.options().dtype(torch::kInt32);
  torch::Tensor ints = torch::empty({cap + T + 1}, i32);
  torch::Tensor token = ints.narrow(0, 0, cap), place = ints.narrow(0, cap, T), count = ints.narrow(0, cap + T, 1);
  torch::Tensor target = torch::empty({cap}, targets.options());
  torch::Tensor floats = torch::empty({3, cap}, f32);
  torch::Tensor tgt_logit = floats[0], lse = floats[1], scale = floats[2];
  torch::Tensor loss = torch::empty({T}, f32);
  torch::Tensor hc = torch::empty({cap, Hp}, h.options());
  torch::Tensor part = torch::empty({cap, nblk, 2}, f32);

  ce_scan_kernel<<<1, kScanThreads, 0, stream>>>(targets.data_ptr<int64_t>(), T, V, ignore_index, token.data_ptr<int>(),
                                                 place.data_ptr<int>(), target.data_ptr<int64_t>(),
                                                 loss.data_ptr<float>(), count.data_ptr<int>(), err.data_ptr<int>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  const torch::Tensor hs = H == 1 || h.stride(1) == 1 ? h : h.contiguous();
  const bool wide = H % 8 == 0 && hs.stride(0) % 8 == 0 && aligned16(hs.data_ptr());
  const int rows = static_cast<int>(std::min<int64_t>(cap, 148 * 16));
  (wide ? ce_gather_kernel<true> : ce_gather_kernel<false>)<<<rows, 256, 0, stream>>>(
      ptr<__nv_bfloat16>(hs), hs.stride(0), static_cast<int>(H), token.data_ptr<int>(), count.data_ptr<int>(), cap,
      ptr<__nv_bfloat16>(hc), static_cast<int>(Hp));
  C10_CUDA_KERNEL_LAUNCH_CHECK();

  const torch::Tensor Wt = tma_rows(W, stream);
  GemmArgs args{};
  args.M = static_cast<int>(cap);
  args.N = static_cast<int>(V);
  args.kb_main = static_cast<int>((H + BK - 1) / BK);
  args.splits = args.nonempty_splits = 1;
  args.aux = part.data_ptr();
  args.ldaux = nblk;
  args.targets = target.data_ptr<int64_t>();
  args.tgt_logit = tgt_logit.data_ptr<float>();
  args.err = err.data_ptr<int>();
  args.live = count.data_ptr<int>();
  launch_ce(gemm_launcher_ce(kCeLse), make_tmap_bf16(hc.data_ptr(), cap, Hp, Hp, BM),
            make_tmap_bf16(Wt.data_ptr(), V, H, Wt.stride(0), kCeBN), args, stream, device);

  const bool per_token = grad.has_value() && grad->numel() != 1;
  if (grad.has_value())
    TORCH_CHECK(grad->device() == h.device() && grad->scalar_type() == torch::kFloat32 && grad->is_contiguous() &&
                    grad->numel() == (reduction == 0 ? T : 1),
                "grad must be fp32: one value per token without a reduction, else one value");
  ce_finish_kernel<<<static_cast<int>(std::min<int64_t>((cap + 7) / 8, 148 * 8)), 256, 0, stream>>>(
      reinterpret_cast<const float2*>(part.data_ptr()), nblk, tgt_logit.data_ptr<float>(), token.data_ptr<int>(),
      count.data_ptr<int>(), grad.has_value() ? grad->data_ptr<float>() : nullptr, per_token, reduction == 2,
      lse.data_ptr<float>(), loss.data_ptr<float>(),
      grad.has_value() || with_scale ? scale.data_ptr<float>() : nullptr);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  torch::Tensor result = loss;
  if (reduction != 0) {
    result = torch::empty({}, f32);
    ce_total_kernel<<<1, 1024, 0, stream>>>(loss.data_ptr<float>(), T, count.data_ptr<int>(), reduction == 2,
                                            result.data_ptr<float>());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {result, hc, token, place, target, count, lse, scale};
}

// scale[m] of the backward from an upstream gradient that came after the forward.
void ce_scale(torch::Tensor token, torch::Tensor count, torch::Tensor grad, int64_t reduction, torch::Tensor scale) {
  const c10::cuda::CUDAGuard guard(scale.device());
  TORCH_CHECK(grad.is_cuda() && grad.scalar_type() == torch::kFloat32 && grad.is_contiguous(),
              "grad must be a contiguous CUDA fp32 tensor");
  ce_scale_kernel<<<static_cast<int>(std::min<int64_t>((scale.numel() + 255) / 256, 592)), 256, 0,
                    at::cuda::getCurrentCUDAStream()>>>(token.data_ptr<int>(), count.data_ptr<int>(),
                                                        grad.data_ptr<float>(), reduction == 0, reduction == 2,
                                                        scale.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Backward from the forward's compacted state.  dh [T, H] and dW [V, H] (either
// may be absent) are written whole.  piece: vocabulary columns per piece, 0 for
// the default.
void ce_backward(torch::Tensor hc, torch::Tensor W, torch::Tensor place, torch::Tensor target, torch::Tensor count,
                 torch::Tensor lse, torch::Tensor scale, c10::optional<torch::Tensor> dh,
                 c10::optional<torch::Tensor> dW, int64_t piece, torch::Tensor err) {
  const c10::cuda::CUDAGuard guard(hc.device());
  const int device = hc.get_device();
  auto stream = at::cuda::getCurrentCUDAStream();
  const int64_t cap = hc.size(0), Hp = hc.size(1), T = place.size(0), V = W.size(0), H = W.size(1);
  TORCH_CHECK(piece >= 0 && piece % kCeBN == 0, "piece must be a multiple of 256");
  TORCH_CHECK(round_up(H, 8) == Hp && cap >= T && lse.numel() >= T && scale.numel() >= T, "state of another call");
  if (dh.has_value())
    TORCH_CHECK(dh->scalar_type() == torch::kBFloat16 && dh->is_contiguous() && dh->dim() == 2 && dh->size(0) == T &&
                    dh->size(1) == H && (H % 8 != 0 || aligned16(dh->data_ptr())),
                "dh must be a contiguous bf16 [T, H]");
  if (dW.has_value())
    TORCH_CHECK(dW->scalar_type() == torch::kBFloat16 && dW->is_contiguous() && dW->dim() == 2 && dW->size(0) == V &&
                    dW->size(1) == H && (H % 8 != 0 || aligned16(dW->data_ptr())),
                "dW must be a contiguous bf16 [V, H]");
  if (!dh.has_value() && !dW.has_value()) return;
  const torch::Tensor Wt = tma_rows(W, stream);
  // A piece of d is at most 256 MiB: large enough that the three products of a
  // piece run for many waves of tiles, small against the logits.
  if (piece == 0) piece = std::max<int64_t>((256LL << 20) / (cap * 2) / kCeBN * kCeBN, kCeBN);
  piece = std::min(piece, round_up(V, kCeBN));
  torch::Tensor d = torch::empty({cap, piece}, hc.options());
  // Few tokens: the contraction over the vocabulary is split until the tiles fill the SMs.
  const int64_t tiles = cap / BM * ((H + kCeBN - 1) / kCeBN);
  const int64_t kb_piece = (std::min(piece, V) + BK - 1) / BK;
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>(num_sms(device) / tiles, kb_piece / 4));
  const int64_t per = (kb_piece + splits - 1) / splits;
  splits = (kb_piece + per - 1) / per;  // none of them empty
  torch::Tensor acc;
  if (dh.has_value()) acc = torch::empty({splits, cap, Hp}, hc.options().dtype(torch::kFloat32));

  const CUtensorMap map_h = make_tmap_bf16(hc.data_ptr(), cap, Hp, Hp, BM);
  const CUtensorMap map_h_mn = make_tmap_bf16(hc.data_ptr(), cap, Hp, Hp, 64);
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t nv = std::min(piece, V - v0);
    const __nv_bfloat16* Wv = ptr<__nv_bfloat16>(Wt) + v0 * Wt.stride(0);
    GemmArgs args{};
    args.splits = args.nonempty_splits = 1;
    args.err = err.data_ptr<int>();
    args.live = count.data_ptr<int>();
    args.M = static_cast<int>(cap);
    args.N = static_cast<int>(nv);
    args.kb_main = static_cast<int>((H + BK - 1) / BK);
    args.C = d.data_ptr();
    args.ldc = piece;
    args.targets = target.data_ptr<int64_t>();
    args.row_lse = lse.data_ptr<float>();
    args.row_scale = scale.data_ptr<float>();
    args.n_first = static_cast<int>(v0);
    launch_ce(gemm_launcher_ce(kCeGrad), map_h, make_tmap_bf16(Wv, nv, H, Wt.stride(0), kCeBN), args, stream, device);
    if (dh.has_value()) {
      GemmArgs a = args;
      a.N = static_cast<int>(H);
      a.kb_main = static_cast<int>((nv + BK - 1) / BK);
      a.splits = static_cast<int>(std::min<int64_t>(splits, a.kb_main));
      a.C = acc.data_ptr();
      a.ldc = Hp;
      a.slice = cap * Hp;
      a.add = v0 > 0;
      launch_ce(gemm_launcher_ce(kCeDh), make_tmap_bf16(d.data_ptr(), cap, nv, piece, BM),
                make_tmap_bf16(Wv, nv, H, Wt.stride(0), 64), a, stream, device);
    }
    if (dW.has_value()) {
      GemmArgs a = args;
      a.M = static_cast<int>(nv);
      a.N = static_cast<int>(H);
      a.kb_main = static_cast<int>(cap / BK);
      a.C = ptr<__nv_bfloat16>(*dW) + v0 * H;
      a.ldc = H;
      launch_ce(gemm_launcher_ce(kCeDw), make_tmap_bf16(d.data_ptr(), cap, nv, piece, 64), map_h_mn, a, stream, device);
    }
  }
  if (dh.has_value() && T > 0) {
    const int rows = static_cast<int>(std::min<int64_t>(T, 148 * 16));
    (H % 8 == 0 ? ce_scatter_kernel<true> : ce_scatter_kernel<false>)<<<rows, 256, 0, stream>>>(
        acc.data_ptr<float>(), static_cast<int>(Hp), cap * Hp, static_cast<int>(splits), place.data_ptr<int>(), T,
        static_cast<int>(H), ptr<__nv_bfloat16>(*dh));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

}  // namespace gb
