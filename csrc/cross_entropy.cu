// Cross entropy of hidden states against a vocabulary projection, without
// keeping the logits, and its gradients for both.
//
//   l_tv = h_t . W_v     lse_t = log sum_v exp l_tv     loss_t = lse_t - l_{t,y_t}
//   d_tv = s_t (exp(l_tv - lse_t) - [v = y_t])     dh = d W     dW = d^T h
//
// s_t is the upstream gradient of token t's loss (over the number of trained
// tokens for the mean).  Tokens whose target is `ignore_index` take no part:
// their rows are left out before the products (`ce_compact`), so neither their
// time is spent nor can what they hold (NaN, infinities) reach a sum.  How many
// remain is known to the device only; the products read that count.
//
// The vocabulary is walked in pieces of columns.  Per piece one product remakes
// the logits and its epilogue writes d in bf16 (tokens x piece), a second adds
// d W to fp32 sums of dh, a third contracts d with h over the tokens into the
// piece's rows of dW, which are complete then.  Pieces of columns rather than
// of tokens, because dh (tokens x hidden) is the smaller sum to carry.
//
// d is rounded to bf16: the tensor cores take bf16 operands, and the rounding of
// each entry is independent, so that it averages out in both contractions.  That
// holds only without a factor that is common to all tokens: 1 / n times (p - 1)
// would round the same way in every row that matters.  So s_t = unit * r_t, with
// the largest |s_t| as the unit; d carries r_t (1 for a mean or a sum), and the
// unit multiplies the fp32 sums.  Nor does r_t (p - 1) average out, in dh_t and in a
// row of dW that is the target of a token or a few: what its rounding leaves out is
// added to the fp32 sums: to dh_t where its row is put together (ce_scatter), to the
// rows of dW in the product's epilogue, from sums by target (ce_rest).  Without it the gradients were 2.4e-3 of
// their norm off with a weight per token at 466 x 1000 x 50001, where rounding the
// exact ones is 1.7e-3.
// The order of the targets, the sums and their addition cost 9 us at 61 x 512 x 4096,
// 14 at 466 x 1000 x 50001 (whatever the targets: all in one row, or none twice) and
// 0.1 ms at 6144 x 4096 x 151936.
//
// Bound by the tensor cores where there are many tokens.  Measured on a B200, loss
// and both gradients: 6144 trained tokens x 4096 x 151936 25.6 to 26.5 ms (four
// products at 1180 TFLOP/s under the power cap), 466 x 1000 x 50001 0.30 ms, 61 x 512 x
// 4096 49 us.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>

#include "ce_gemm.cuh"
#include "vec_types.cuh"

namespace gb {

// embedding_grad.cu: ids [0, vocab) sorted, ties by position, the others last; ints:
// the ids, the positions, and as many of scratch.  Two launches (over 1024 tokens).
void sort_tokens(const int64_t* ids, int64_t tokens, int64_t vocab, int64_t skip, int64_t ignore, int* ints, int* err,
                 cudaStream_t stream);

namespace {

constexpr int kRowPad = BM;     // rows of the compacted buffers come in whole GEMM tiles,
constexpr int kColumnPad = 64;  // and start on 128-byte lines
constexpr int kBlock = 256;
constexpr int kTokens = 32;     // tokens per block of ce_compact
// Tokens up to which ce_finish ranks the targets by counting, the square of the tokens
// (3 us of 9 at 2048 tokens, 40 of 44 at 8192); beyond, they are sorted, in three more
// launches (14 us at 2049, 17 at 8192).
constexpr int64_t kRankTokens = 2048;
// Tokens from which a row's rests are joined in a launch of their own; up to it dW's
// epilogue adds at most kJoinTokens / kGroup + 1 of them.
constexpr int64_t kJoinTokens = 256;
constexpr int kRestThreads = 128, kRestColumns = kRestThreads * 8;

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// What the forward leaves for the backward, in one int32 tensor.  `unit` and `ratio`
// (and `rest`) are those of an upstream gradient of 1; a backward of its own replaces
// them.
struct State {
  int* count;           // number of trained tokens
  float* unit;          // what the tokens' weights are multiples of
  int64_t* target;      // of the m-th trained token
  int* token;           // its position
  int* place;           // position -> m, -1 for an ignored token
  float* lse;
  float* ratio;         // its weight over the unit
  float* target_logit;
  float* hot;           // p - 1 of its target
  int* order;           // the trained tokens by target, equal ones in their order,
  unsigned* sorted;     // and their targets,
  float* rest;          // and what rounding their entry of d leaves out (over the unit)
  int* start;           // [V / 32 + 1] where each 32 vocabulary rows' tokens start among them
  static int64_t words(int64_t cap, int64_t V) { return 4 + 11 * cap + ce::row_blocks(V) + 1; }
  State(const torch::Tensor& t, int64_t cap) {
    int* p = t.data_ptr<int>();
    count = p;
    unit = reinterpret_cast<float*>(p + 1);
    target = reinterpret_cast<int64_t*>(p + 4);
    token = p + 4 + 2 * cap;
    place = token + cap;
    lse = reinterpret_cast<float*>(place + cap);
    ratio = lse + cap;
    target_logit = ratio + cap;
    hot = target_logit + cap;
    order = reinterpret_cast<int*>(hot + cap);
    sorted = reinterpret_cast<unsigned*>(order + cap);
    rest = reinterpret_cast<float*>(sorted + cap);
    start = reinterpret_cast<int*>(rest + cap);
  }
};

int64_t capacity(int64_t T) { return std::max<int64_t>(round_up(T, kRowPad), kRowPad); }

__device__ __forceinline__ bool is_live(int64_t y, long V, long ignore) { return y >= 0 && y < V && y != ignore; }

__device__ __forceinline__ int block_sum(int v) {
  __shared__ int part[kBlock / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kBlock / 32; ++w) v += part[w];
  __syncthreads();
  return v;
}

// Row of `in` to row of `out`, zeros in the columns [H, ldo); zeros without `in`.
// Rows of `out` are whole 128-byte lines; those of `in` that are not on 16-byte
// boundaries are read value by value, eight in flight.
template <bool WIDE>
__device__ __forceinline__ void copy_row(const __nv_bfloat16* in, int H, __nv_bfloat16* out, int ldo) {
  const int lane = threadIdx.x & 31;
  if constexpr (WIDE) {
#pragma unroll 4
    for (int c = lane * 8; c < ldo; c += 256) {
      Pack<__nv_bfloat16, 8> p = {};
      if (in != nullptr && c < H) p = load_raw<__nv_bfloat16, 8>(in + c);
      store_raw<__nv_bfloat16, 8>(out + c, p);
    }
  } else {
    const uint16_t* src = reinterpret_cast<const uint16_t*>(in);
    for (int c0 = 0; c0 < ldo; c0 += 256) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + i * 64 + lane * 2;
        const uint32_t lo = in != nullptr && c < H ? src[c] : 0u, hi = in != nullptr && c + 1 < H ? src[c + 1] : 0u;
        w[i] = hi << 16 | lo;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c0 + i * 64 + lane * 2 < ldo) *reinterpret_cast<uint32_t*>(out + c0 + i * 64 + lane * 2) = w[i];
    }
  }
}

// The trained tokens' rows of h, one after the other, and their places.  A block
// counts the trained tokens before its own 32 itself, so that there is no second
// pass.  That is T / 8 bytes a token from L2 and grows with the square of the
// tokens: 7 us of 156 at 8192 tokens x 256 x 4096, 141 us of 4.3 ms at 131072, 6.8 of
// 112 ms at a million.  The last block knows the count and zeroes the rows that fill
// the last K-block of dW (what the rest of the last tile holds stays in its own
// rows).  A target outside the vocabulary that is not ignore_index is reported in
// err[1] and gets a NaN loss and a zero gradient.
template <bool WIDE>
__global__ void __launch_bounds__(kBlock) ce_compact_kernel(const int64_t* __restrict__ targets, long T, long V,
                                                              long ignore, const __nv_bfloat16* __restrict__ h, long ldh,
                                                              int H, State st, float* __restrict__ loss,
                                                              __nv_bfloat16* __restrict__ out, int ldo,
                                                              int* __restrict__ err) {
  pdl_trigger();
  __shared__ int own[kTokens];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long first = static_cast<long>(blockIdx.x) * kTokens;
  int before = 0;
#pragma unroll 8
  for (long t = threadIdx.x; t < first; t += kBlock) before += is_live(targets[t], V, ignore);
  before = block_sum(before);
  const long t = first + lane;
  const int64_t y = t < T ? targets[t] : ignore;
  const bool live = t < T && is_live(y, V, ignore);
  const unsigned mask = __ballot_sync(0xffffffffu, live);
  const int count = __popc(mask);
  if (warp == 0 && t < T) {
    const int k = __popc(mask & ((1u << lane) - 1u));
    if (live) {
      own[k] = lane;
      st.token[before + k] = static_cast<int>(t);
      st.target[before + k] = y;
    } else {
      if (y != ignore) atomicExch(err + 1, kErrBadToken);
      loss[t] = y != ignore ? __int_as_float(0x7fc00000) : 0.f;
    }
    st.place[t] = live ? before + k : -1;
  }
  __syncthreads();
  for (int k = warp; k < count; k += kBlock / 32)
    copy_row<WIDE>(h + (first + own[k]) * ldh, H, out + static_cast<long>(before + k) * ldo, ldo);
  if (blockIdx.x == gridDim.x - 1) {
    const int total = before + count;
    if (threadIdx.x == 0) *st.count = total;
    for (long m = total + warp; m < (total + BK - 1) / BK * BK; m += kBlock / 32)
      copy_row<WIDE>(nullptr, H, out + m * ldo, ldo);
  }
}

// Rows of W with zeros in the columns [H, ldo).
template <bool WIDE>
__global__ void __launch_bounds__(kBlock) ce_pad_kernel(const __nv_bfloat16* __restrict__ in, long ldi, int H,
                                                          long rows, __nv_bfloat16* __restrict__ out, int ldo) {
  pdl_trigger();
  pdl_wait();
  for (long r = blockIdx.x * (kBlock / 32L) + (threadIdx.x >> 5); r < rows; r += gridDim.x * (kBlock / 32L))
    copy_row<WIDE>(in + r * ldi, H, out + r * ldo, ldo);
}

// The upstream gradient of a reduced loss as every token's weight.
__device__ __forceinline__ float common_weight(const float* g, bool mean, int n) {
  return (g == nullptr ? 1.f : *g) / (mean ? static_cast<float>(max(n, 1)) : 1.f);
}

// lse and loss of every trained token from its target's logit t and the others'
// (max, sum exp) per half tile, one warp each; ratios of 1, and the unit of a
// reduced loss.  With z = log sum exp(others) - t the loss is log(1 + e^z): exact
// relative to itself however small it is.  (lse - t, both rounded first, has steps
// of the largest logit's last place, 2e-6 at 20 and 3e-5 at 300, where a confident
// token's loss is 1e-6.)  p - 1 = expm1(-loss) likewise: exp(l - lse) - 1 from the
// remade logit was off by 2.5e-5, a quarter of it at a loss of 1e-4.
// Also the tokens by target (`rank`; else ce_list_kernel makes the list): a token's
// place is the number of smaller targets, and of equal ones before it, which its warp
// counts; a further warp counts for each start of 32 vocabulary rows.
__global__ void __launch_bounds__(kBlock) ce_finish_kernel(const float2* part, int parts, State st,
                                                             const float* __restrict__ g, bool mean, bool rank,
                                                             int row_blocks, float* __restrict__ loss) {
  pdl_trigger();
  pdl_wait();
  const int n = *st.count;
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x == 0) *st.unit = common_weight(g, mean, n);
  const long items = n + (rank ? row_blocks + 1 : 0);
  for (long m = blockIdx.x * (kBlock / 32L) + (threadIdx.x >> 5); m < items; m += gridDim.x * (kBlock / 32L)) {
    float hot = 0.f;
    if (m < n) {
      const float2* row = part + m * parts;
      float mx = -INFINITY, sum = 0.f;
#pragma unroll 4
      for (int b = lane; b < parts; b += 32) {
        const float2 p = row[b];
        const float top = fmaxf(mx, p.x);
        if (top > -INFINITY) sum = sum * __expf(mx - top) + p.y * __expf(p.x - top);
        else sum += p.y;  // a half tile of NaN only has a NaN sum and no maximum
        mx = top;
      }
      const float top = warp_max(mx);
      sum = warp_sum(top > -INFINITY ? sum * __expf(mx - top) : sum);
      const float t = st.target_logit[m], others = logf(sum);
      const float z = (top - t) + others;
      const float q = log1pf(expf(-fabsf(z)));
      // an infinite logit of the target leaves no loss, as inf - inf; -inf gives inf, NaN stays NaN
      const bool lost = t == INFINITY;
      const float l = lost ? __int_as_float(0x7fc00000) : fmaxf(z, 0.f) + q;
      hot = expm1f(-l);
      if (lane == 0) {
        st.lse[m] = lost ? l : z > 0.f ? (top + others) + q : t + q;
        st.ratio[m] = 1.f;
        st.hot[m] = hot;
        loss[st.token[m]] = l;
      }
    }
    if (!rank) continue;
    const int64_t y = m < n ? st.target[m] : (m - n) * 32;
    int place = 0;
#pragma unroll 8
    for (int k = lane; k < n; k += 32) {
      const int64_t z = st.target[k];
      place += z < y || (z == y && k < m && m < n);
    }
    place = __reduce_add_sync(0xffffffffu, place);
    if (lane == 0) {
      if (m < n) {
        st.order[place] = static_cast<int>(m);
        st.sorted[place] = static_cast<unsigned>(y);
        st.rest[place] = ce::rounded_off(hot);
      } else {
        st.start[m - n] = place;
      }
    }
  }
}

// The tokens by target from the sorted targets and their positions, whose first n are
// the trained ones.
__global__ void __launch_bounds__(kBlock) ce_list_kernel(const unsigned* __restrict__ by_id,
                                                           const int* __restrict__ token_by_id, State st,
                                                           int row_blocks) {
  pdl_trigger();
  const int n = *st.count;
  const int first = blockIdx.x * kBlock + threadIdx.x, step = gridDim.x * kBlock;
  for (int k = first; k < n; k += step) {
    const int m = st.place[token_by_id[k]];
    st.order[k] = m;
    st.sorted[k] = by_id[k];
    st.rest[k] = ce::rounded_off(st.hot[m]);
  }
  for (int b = first; b <= row_blocks; b += step) {
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (by_id[mid] < 32u * static_cast<unsigned>(b)) lo = mid + 1;
      else hi = mid;
    }
    st.start[b] = lo;
  }
}

// What rows of dW lack: sums of rest_t h_t over the tokens of a target, at its first
// place in the order of the targets.  A block takes kGroup places and kRestColumns
// columns, and leaves a sum at the first place of every target among them: a target
// of many tokens has one per group (joined below), and no chain is longer than that.
__global__ void __launch_bounds__(kRestThreads) ce_rest_kernel(const __nv_bfloat16* hc, int Hp, int slabs, State st,
                                                               float* out) {
  pdl_trigger();
  pdl_wait();
  constexpr int G = ce::kGroup, U = 8;
  __shared__ int token[G];
  __shared__ unsigned target[G];
  __shared__ float rest[G];
  const int n = *st.count;
  const long first = static_cast<long>(blockIdx.x / slabs) * G;
  if (first >= n) return;
  const int count = static_cast<int>(min(static_cast<long>(G), n - first));
  const int t = threadIdx.x;
  if (t < count) {
    token[t] = st.order[first + t];
    target[t] = st.sorted[first + t];
    rest[t] = st.rest[first + t];
  }
  __syncthreads();
  const int column = static_cast<int>(blockIdx.x % slabs) * kRestColumns + t * 8;
  if (column >= Hp) return;
  float sum[8] = {};
  int head = 0;
  const auto flush = [&] {
    store_pack<float, 8>(out + (first + head) * Hp + column, sum);
  };
#pragma unroll 1
  for (int j0 = 0; j0 < count; j0 += U) {
    Pack<__nv_bfloat16, 8> p[U];
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (j0 + j < count) p[j] = load_raw<__nv_bfloat16, 8>(hc + static_cast<long>(token[j0 + j]) * Hp + column);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (j0 + j >= count) break;
      if (target[j0 + j] != target[head]) {
        flush();
        head = j0 + j;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = 0.f;
      }
      const float e = rest[j0 + j];
      if (e != 0.f)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = fmaf(e, value(p[j], i), sum[i]);
    }
  }
  flush();
}

// Joins the sums of targets that go on past a group, onto the first of them; the block
// of the first group that a target goes on into does it.
__global__ void __launch_bounds__(kRestThreads) ce_join_kernel(int Hp, int slabs, State st, float* sums) {
  pdl_trigger();
  pdl_wait();
  constexpr int G = ce::kGroup, U = 8;
  const int n = *st.count;
  const long first = static_cast<long>(blockIdx.x / slabs) * G;
  if (first == 0 || first >= n) return;
  const unsigned target = st.sorted[first];
  if (st.sorted[first - 1] != target || (first > G && st.sorted[first - G - 1] == target)) return;
  const int column = static_cast<int>(blockIdx.x % slabs) * kRestColumns + static_cast<int>(threadIdx.x) * 8;
  if (column >= Hp) return;
  long head = first - 1;   // the target's first place
  while (head > first - G && st.sorted[head - 1] == target) --head;
  float sum[8];
  load_pack<float, 8>(sums + head * Hp + column, sum);
  for (long k0 = first; k0 < n && st.sorted[k0] == target; k0 += U * G) {
    Pack<float, 8> p[U];
    bool some[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      some[j] = k0 + j * G < n && st.sorted[k0 + j * G] == target;
      if (some[j]) p[j] = load_raw<float, 8>(sums + (k0 + j * G) * Hp + column);
    }
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (some[j])
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += value(p[j], i);
  }
  store_pack<float, 8>(sums + head * Hp + column, sum);
}

// Unit and ratios from an upstream gradient per token (the unit is the largest
// finite size, 1 where there is none), or the unit of a reduced loss.
__global__ void __launch_bounds__(1024) ce_weight_kernel(const float* __restrict__ g, bool per_token, bool mean, bool ordered,
                                                         State st) {
  pdl_trigger();
  pdl_wait();
  __shared__ float part[32];
  const int n = *st.count;
  if (!per_token) {
    if (threadIdx.x == 0) *st.unit = common_weight(g, mean, n);
    return;
  }
  float top = 0.f;
  for (int m = threadIdx.x; m < n; m += 1024) {
    const float s = fabsf(g[st.token[m]]);
    if (s < INFINITY) top = fmaxf(top, s);
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
  top = warp_max(part[threadIdx.x & 31]);
  const float unit = top > 0.f ? top : 1.f;
  if (threadIdx.x == 0) *st.unit = unit;
  for (int m = threadIdx.x; m < n; m += 1024) st.ratio[m] = g[st.token[m]] / unit;
  for (int k = threadIdx.x; ordered && k < n; k += 1024) {
    const int m = st.order[k];
    st.rest[k] = ce::rounded_off(g[st.token[m]] / unit * st.hot[m]);
  }
}

// Sum of the tokens' losses in a fixed order, over the trained tokens for the
// mean (no trained token: 0).  One block.
__device__ void total_loss(const float* loss, long T, int n, bool mean, float* __restrict__ out) {
  __shared__ double part[kBlock / 32];
  double s = 0;
#pragma unroll 8
  for (long t = threadIdx.x; t < T; t += kBlock) s += loss[t];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0;
    for (int w = 0; w < kBlock / 32; ++w) s += part[w];
    *out = static_cast<float>(mean ? s / max(1, n) : s);
  }
}

__global__ void __launch_bounds__(kBlock) ce_total_kernel(const float* loss, long T, State st, bool mean,
                                                            float* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  total_loss(loss, T, *st.count, mean, out);
}

// dh[t] = unit * (sum of the slices' row place[t], and what the rounding of d left out
// of the target's entry times its row of W), rounded once; zero for an ignored token.  A last block adds the losses up where `total` wants them.
template <bool WIDE>
__global__ void __launch_bounds__(kBlock) ce_scatter_kernel(const float* acc, int lda, State st, long T,
                                                              int H, int kb_first, int sms,
                                                              const __nv_bfloat16* W, long ldw,
                                                              __nv_bfloat16* __restrict__ dh,
                                                              const float* loss, bool mean,
                                                              float* __restrict__ total) {
  pdl_trigger();
  pdl_wait();
  constexpr int V = WIDE ? 8 : 1;
  const int n = *st.count;
  const int row_blocks = gridDim.x - (total != nullptr ? 1 : 0);
  if (static_cast<int>(blockIdx.x) == row_blocks) {
    total_loss(loss, T, n, mean, total);
    return;
  }
  const float unit = *st.unit;
  const int slices = ce::dh_slices(n, H, kb_first, sms);
  const long slice = ce::dh_slice_elements(n, lda);
  const int per_row = (H + kBlock * V - 1) / (kBlock * V);  // blocks' columns
  for (long i = blockIdx.x; i < T * per_row; i += row_blocks) {
    const long t = i / per_row;
    const int c = static_cast<int>(i - t * per_row) * kBlock * V + threadIdx.x * V;
    const int m = st.place[t];
    if (c >= H) continue;
    float s[V] = {};
    if (m >= 0) {
      const float* src = acc + static_cast<long>(m) * lda + c;
#pragma unroll 8
      for (int k = 0; k < slices; ++k) {
        float f[V];
        load_pack<float, V>(src + k * slice, f);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] += f[j];
      }
      const float rest = ce::rounded_off(st.ratio[m] * st.hot[m]);
      float row[V];
      load_pack<__nv_bfloat16, V>(W + st.target[m] * ldw + c, row);
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = (rest != 0.f ? fmaf(rest, row[j], s[j]) : s[j]) * unit;
    }
    store_pack<__nv_bfloat16, V>(dh + t * H + c, s);
  }
}

template <typename T>
T* ptr(const torch::Tensor& t) {
  return reinterpret_cast<T*>(t.data_ptr());
}

// W as TMA reads it: rows of 16-byte multiples from a 16-byte boundary.  Rows that
// are no multiple of 32 bytes apart cross one more sector each, which every one of
// the products that read W pays (65 against 48 us at 466 tokens x 50001 x 1000).  Both
// the copy and what it saves grow with V H, the latter with the tokens too; loss and
// gradients as W is / with a copy, at 1000 x 50001, 4088 x 20001, 520 x 150001 and
// 2056 x 151936: 256 tokens 175 / 192, 287 / 309, 294 / 330, 885 / 950 us; 512 tokens
// 265 / 263, 417 / 419, 495 / 507, 1551 / 1509; 1024 tokens 469 / 431, 735 / 653,
// 931 / 898, 2832 / 2530.
constexpr int64_t kCopyTokens = 512;

torch::Tensor tma_rows(const torch::Tensor& W, int64_t tokens, cudaStream_t stream) {
  const int64_t V = W.size(0), H = W.size(1);
  const bool readable = W.stride(1) == 1 && W.stride(0) % 8 == 0 && W.stride(0) >= H && aligned16(W.data_ptr());
  if (readable && (W.stride(0) % 16 == 0 || tokens < kCopyTokens)) return W;
  const torch::Tensor src = W.stride(1) == 1 ? W : W.contiguous();
  torch::Tensor out = torch::empty({V, round_up(H, kColumnPad)}, W.options());
  const bool wide = H % 8 == 0 && src.stride(0) % 8 == 0 && aligned16(src.data_ptr());
  (wide ? ce_pad_kernel<true> : ce_pad_kernel<false>)<<<static_cast<int>(std::min<int64_t>((V + 7) / 8, 148 * 32)),
                                                        kBlock, 0, stream>>>(
      ptr<__nv_bfloat16>(src), src.stride(0), static_cast<int>(H), V, ptr<__nv_bfloat16>(out),
      static_cast<int>(out.size(1)));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

// A ValueError in Python, as the CPU form's checks give.
void require(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

enum Reduction : int64_t { kNone = 0, kSum = 1, kMean = 2 };

bool launches_early(int64_t cap, int64_t V, int64_t H) {
  return static_cast<double>(cap) * static_cast<double>(V) * static_cast<double>(H) < ce::kEarlyWork;
}

struct Forward {
  torch::Tensor loss, hc, state, W;   // loss per token; W as TMA reads it
  int64_t T, H, V, cap, Hp;
  int64_t launches;
};

Forward forward(const torch::Tensor& h, const torch::Tensor& W, const torch::Tensor& targets, int64_t ignore_index,
                const float* grad, int64_t reduction, bool want_w, int* err, cudaStream_t stream) {
  Forward f;
  const int device = h.get_device();
  f.T = targets.numel(), f.H = W.size(1), f.V = W.size(0);
  f.cap = capacity(f.T), f.Hp = round_up(f.H, kColumnPad);
  const int num_n = static_cast<int>((f.V + ce::BN - 1) / ce::BN);
  const auto f32 = h.options().dtype(torch::kFloat32);
  f.loss = torch::empty({f.T}, f32);
  f.state = torch::empty({State::words(f.cap, f.V)}, h.options().dtype(torch::kInt32));
  f.hc = torch::empty({f.cap, f.Hp}, h.options());
  torch::Tensor part = torch::empty({f.cap, 2 * num_n, 2}, f32);
  const State st(f.state, f.cap);
  torch::Tensor rows = h.reshape({f.T, f.H});
  if (rows.stride(1) != 1 && f.H != 1) rows = rows.contiguous();
  const bool wide = f.H % 8 == 0 && rows.stride(0) % 8 == 0 && aligned16(rows.data_ptr());
  const int blocks = static_cast<int>(std::max<int64_t>((f.T + kTokens - 1) / kTokens, 1));
  (wide ? ce_compact_kernel<true> : ce_compact_kernel<false>)<<<blocks, kBlock, 0, stream>>>(
      targets.data_ptr<int64_t>(), f.T, f.V, ignore_index, ptr<__nv_bfloat16>(rows), rows.stride(0),
      static_cast<int>(f.H), st, f.loss.data_ptr<float>(), ptr<__nv_bfloat16>(f.hc), static_cast<int>(f.Hp), err);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  f.W = tma_rows(W, f.T, stream);
  ce::Args args{};
  args.early = launches_early(f.cap, f.V, f.H);
  args.M = static_cast<int>(f.cap);
  args.N = static_cast<int>(f.V);
  args.kb = static_cast<int>((f.H + BK - 1) / BK);
  args.live = st.count;
  args.err = err;
  args.target = st.target;
  args.part = reinterpret_cast<float2*>(part.data_ptr());
  args.target_logit = st.target_logit;
  ce::launch<ce::kLse, 0>(make_tmap_bf16(f.hc.data_ptr(), f.cap, f.Hp, f.Hp, BM),
                          make_tmap_bf16(f.W.data_ptr(), f.V, f.H, f.W.stride(0), ce::BN), args, stream, device);
  // the tokens by target, for dW
  const bool rank = want_w && f.T <= kRankTokens, sort = want_w && !rank;
  const int row_blocks = static_cast<int>(ce::row_blocks(f.V));
  ce::launch_chained(args.early, ce_finish_kernel,
                     static_cast<unsigned>(std::min<int64_t>((f.cap + row_blocks + 8) / 8, 148 * 8)), kBlock, 0, stream,
                     static_cast<const float2*>(args.part), 2 * num_n, st, grad, reduction == kMean, rank, row_blocks,
                     f.loss.data_ptr<float>());
  if (sort) {
    torch::Tensor sorted = torch::empty({4 * f.T}, f.state.options());
    int* ints = sorted.data_ptr<int>();
    sort_tokens(targets.data_ptr<int64_t>(), f.T, f.V, ignore_index, ignore_index, ints, err, stream);
    ce_list_kernel<<<148 * 4, kBlock, 0, stream>>>(reinterpret_cast<const unsigned*>(ints), ints + f.T, st, row_blocks);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  f.launches = 3 + !f.W.is_same(W) + (sort ? 3 : 0);
  return f;
}

// dh [T, H] with the loss's total (where `total` is given), and dW [V, H].  The
// number of kernels launched.
int64_t backward(const torch::Tensor& hc, const State& st, const torch::Tensor& W, int64_t T, int64_t V, int64_t H,
              int64_t piece, torch::Tensor* dh, torch::Tensor* dW, const torch::Tensor& loss, bool mean,
              torch::Tensor* total, int* err, cudaStream_t stream) {
  const int device = hc.get_device();
  const int64_t cap = hc.size(0), Hp = hc.size(1);
  const bool early = launches_early(cap, V, H);
  // A piece of d is at most 256 MiB: large enough that the three products of a
  // piece run for many waves of tiles, small against the logits.  256 columns are the
  // least, which are more than that from 524289 tokens on (512 bytes a token); dW then
  // has as few tiles as ceil(H / 256) x 2 a piece, and a call should be split.
  if (piece == 0) piece = std::max<int64_t>((256LL << 20) / (cap * 2) / ce::BN * ce::BN, ce::BN);
  piece = std::min(piece, round_up(V, ce::BN));
  torch::Tensor d = torch::empty({cap, piece}, hc.options());
  const int64_t num_n = (H + ce::BN - 1) / ce::BN;
  const int sms = num_sms(device);
  const int kb_first = static_cast<int>((std::min(piece, V) + BK - 1) / BK);
  // room for dh's slices of any number of trained tokens (dh_slices), then what rows of dW lack
  const int64_t acc_rows = dh != nullptr ? std::max<int64_t>(sms / num_n, 2 * cap / BM) * BM : 0;
  const torch::Tensor sums =
      torch::empty({acc_rows + (dW != nullptr ? cap : 0), Hp}, hc.options().dtype(torch::kFloat32));
  float* acc = sums.data_ptr<float>();
  float* rests = acc + acc_rows * Hp;
  const bool join = T > kJoinTokens;
  if (dW != nullptr) {
    const unsigned slabs = static_cast<unsigned>((Hp + kRestColumns - 1) / kRestColumns);
    ce::launch_chained(early, ce_rest_kernel, static_cast<unsigned>(cap / ce::kGroup) * slabs, kRestThreads, 0, stream,
                       static_cast<const __nv_bfloat16*>(ptr<__nv_bfloat16>(hc)), static_cast<int>(Hp),
                       static_cast<int>(slabs), st, rests);
    if (join)
      ce::launch_chained(early, ce_join_kernel, static_cast<unsigned>(cap / ce::kGroup) * slabs, kRestThreads, 0, stream,
                         static_cast<int>(Hp), static_cast<int>(slabs), st, rests);
  }
  const CUtensorMap map_h = make_tmap_bf16(hc.data_ptr(), cap, Hp, Hp, BM);
  const CUtensorMap map_h_mn = make_tmap_bf16(hc.data_ptr(), cap, Hp, Hp, 64);
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t nv = std::min(piece, V - v0);
    const __nv_bfloat16* Wv = ptr<__nv_bfloat16>(W) + v0 * W.stride(0);
    ce::Args args{};
    args.early = early;
    args.M = static_cast<int>(cap);
    args.N = static_cast<int>(nv);
    args.kb = static_cast<int>((H + BK - 1) / BK);
    args.live = st.count;
    args.err = err;
    args.target = st.target;
    args.lse = st.lse;
    args.hot = st.hot;
    args.ratio = st.ratio;
    args.n_first = static_cast<int>(v0);
    args.C = d.data_ptr();
    args.ldc = piece;
    ce::launch<ce::kGrad, 0>(map_h, make_tmap_bf16(Wv, nv, H, W.stride(0), ce::BN), args, stream, device);
    if (dh != nullptr) {
      ce::Args a = args;
      a.N = static_cast<int>(H);
      a.kb = static_cast<int>((nv + BK - 1) / BK);
      a.kb_first = kb_first;
      a.C = acc;
      a.ldc = Hp;
      a.add = v0 > 0;
      ce::launch<ce::kDh, 1>(make_tmap_bf16(d.data_ptr(), cap, nv, piece, BM),
                             make_tmap_bf16(Wv, nv, H, W.stride(0), 64), a, stream, device);
    }
    if (dW != nullptr) {
      ce::Args a = args;
      a.M = static_cast<int>(nv);
      a.N = static_cast<int>(H);
      a.kb = static_cast<int>(cap / BK);
      a.C = ptr<__nv_bfloat16>(*dW) + v0 * H;
      a.ldc = H;
      a.unit = st.unit;
      a.sorted = st.sorted;
      a.start = st.start;
      a.rest = rests;
      a.ldr = Hp;
      a.joined = join;
      a.row_blocks = static_cast<int>(ce::row_blocks(V));
      ce::launch<ce::kDw, 3>(make_tmap_bf16(d.data_ptr(), cap, nv, piece, 64), map_h_mn, a, stream, device);
    }
  }
  if (dh != nullptr) {
    const int64_t per_row = (H + kBlock * (H % 8 == 0 ? 8 : 1) - 1) / (kBlock * (H % 8 == 0 ? 8 : 1));
    const int rows = static_cast<int>(std::max<int64_t>(std::min<int64_t>(T * per_row, 148 * 16), 1));
    ce::launch_chained(early, H % 8 == 0 ? ce_scatter_kernel<true> : ce_scatter_kernel<false>,
                       rows + (total != nullptr ? 1 : 0), kBlock, 0, stream,
                       static_cast<const float*>(acc), static_cast<int>(Hp), st, static_cast<long>(T),
                       static_cast<int>(H), kb_first, sms, static_cast<const __nv_bfloat16*>(ptr<__nv_bfloat16>(W)),
                       static_cast<long>(W.stride(0)), ptr<__nv_bfloat16>(*dh),
                       static_cast<const float*>(loss.defined() ? loss.data_ptr<float>() : nullptr), mean,
                       total != nullptr ? total->data_ptr<float>() : nullptr);
  }
  const int64_t pieces = (V + piece - 1) / piece, each = 1 + (dh != nullptr) + (dW != nullptr);
  return pieces * each + (dh != nullptr) + (dW != nullptr ? 1 + join : 0);
}

void check_inputs(const torch::Tensor& h, const torch::Tensor& W, const torch::Tensor& targets, int64_t reduction) {
  require(h.is_cuda() && h.scalar_type() == torch::kBFloat16 && W.scalar_type() == torch::kBFloat16,
          "h and weight must be bf16 on the GPU");
  require(W.dim() == 2 && h.dim() >= 1 && W.size(0) >= 1 && W.size(1) >= 1 && h.size(-1) == W.size(1),
          "h [..., H] and weight [V, H] do not match");
  require(h.sizes().slice(0, h.dim() - 1) == targets.sizes(), "targets must have one entry per row of h");
  require(targets.scalar_type() == torch::kInt64 || targets.scalar_type() == torch::kInt32,
          "targets must be int64 or int32");
  require(W.device() == h.device() && targets.device() == h.device(), "h, weight and targets must be on one device");
  require(reduction >= kNone && reduction <= kMean, "reduction must be none, sum or mean");
  require(targets.numel() < (1LL << 31) - kRowPad && W.size(0) < (1LL << 31) - ce::BN &&
              W.size(1) < (1LL << 31) - ce::BN, "sizes must fit 31 bits");
}

const float* check_grad(const c10::optional<torch::Tensor>& grad, const torch::Tensor& h, int64_t reduction, int64_t T) {
  if (!grad.has_value()) return nullptr;
  require(grad->device() == h.device() && grad->scalar_type() == torch::kFloat32 && grad->is_contiguous() &&
              grad->numel() == (reduction == kNone ? T : 1),
          "grad must be fp32: one value, or one per token for reduction none, on the device of h");
  return grad->data_ptr<float>();
}

void check_piece(int64_t piece) { require(piece >= 0 && piece % ce::BN == 0, "piece must be a multiple of 256"); }

torch::Tensor flat_targets(const torch::Tensor& t) {
  return (t.scalar_type() == torch::kInt64 ? t : t.to(torch::kInt64)).contiguous();
}

}  // namespace

// Each with the number of kernels launched.
using Launched = std::pair<std::vector<torch::Tensor>, int64_t>;

// (loss, compacted h, state): what ce_backward needs; `want_w`: whether for dW too.
Launched ce_forward(torch::Tensor h, torch::Tensor W, torch::Tensor targets, int64_t ignore_index, int64_t reduction,
                    bool want_w, torch::Tensor err) {
  check_inputs(h, W, targets, reduction);
  const c10::cuda::CUDAGuard guard(h.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const Forward f = forward(h, W, flat_targets(targets), ignore_index, nullptr, reduction, want_w,
                            err.data_ptr<int>(), stream);
  if (reduction == kNone) return {{f.loss.view(targets.sizes()), f.hc, f.state}, f.launches};
  torch::Tensor total = torch::empty({}, f.loss.options());
  ce_total_kernel<<<1, kBlock, 0, stream>>>(f.loss.data_ptr<float>(), f.T, State(f.state, f.cap), reduction == kMean,
                                              total.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {{total, f.hc, f.state}, f.launches + 1};
}

// (dh [tokens, H], dW); what is not wanted is None.  grad: fp32, one value, or one
// per token for reduction none.
Launched ce_backward(torch::Tensor hc, torch::Tensor state, torch::Tensor W, int64_t tokens, torch::Tensor grad,
                     int64_t reduction, bool want_h, bool want_w, int64_t piece, torch::Tensor err) {
  const int64_t H = W.size(1), V = W.size(0), cap = capacity(tokens);
  require(hc.is_cuda() && hc.size(0) == cap && hc.size(1) == round_up(H, kColumnPad) && state.numel() == State::words(cap, V),
          "state of another call");
  check_piece(piece);
  const float* g = check_grad(grad, hc, reduction, tokens);
  const c10::cuda::CUDAGuard guard(hc.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  torch::Tensor dh, dW;
  if (!want_h && !want_w) return {{dh, dW}, 0};
  // two backward passes of one graph may run at once: the weights are this call's own
  State st(state, cap);
  torch::Tensor weights = torch::empty({4 + (reduction == kNone ? 2 * cap : 0)}, hc.options().dtype(torch::kFloat32));
  st.unit = weights.data_ptr<float>();
  if (reduction == kNone) {
    st.ratio = st.unit + 4;
    st.rest = st.ratio + cap;
  }
  ce_weight_kernel<<<1, 1024, 0, stream>>>(g, reduction == kNone, reduction == kMean, want_w, st);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (want_h) dh = torch::empty({tokens, H}, hc.options());
  if (want_w) dW = torch::empty({V, H}, hc.options());
  const torch::Tensor Wt = tma_rows(W, tokens, stream);
  const int64_t n = backward(hc, st, Wt, tokens, V, H, piece, want_h ? &dh : nullptr, want_w ? &dW : nullptr,
                             torch::Tensor(), false, nullptr, err.data_ptr<int>(), stream);
  return {{dh, dW}, 1 + !Wt.is_same(W) + n};
}

// (loss, dh, dW) in one call; dW is None where it is not wanted.
Launched ce_grads(torch::Tensor h, torch::Tensor W, torch::Tensor targets, c10::optional<torch::Tensor> grad,
                  int64_t ignore_index, int64_t reduction, bool want_w, int64_t piece, torch::Tensor err) {
  check_inputs(h, W, targets, reduction);
  check_piece(piece);
  const float* g = check_grad(grad, h, reduction, targets.numel());
  const c10::cuda::CUDAGuard guard(h.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  int* e = err.data_ptr<int>();
  const Forward f = forward(h, W, flat_targets(targets), ignore_index, reduction == kNone ? nullptr : g, reduction, want_w,
                            e, stream);
  const State st(f.state, f.cap);
  const bool weighted = reduction == kNone && g != nullptr;
  if (weighted) {
    ce::launch_chained(launches_early(f.cap, f.V, f.H), ce_weight_kernel, 1, 1024, 0, stream, g, true, false, want_w,
                       st);
  }
  torch::Tensor dh = torch::empty(h.sizes(), h.options()), dW, total;
  if (want_w) dW = torch::empty({f.V, f.H}, h.options());
  if (reduction != kNone) total = torch::empty({}, f.loss.options());
  const int64_t n = backward(f.hc, st, f.W, f.T, f.V, f.H, piece, &dh, want_w ? &dW : nullptr, f.loss,
                             reduction == kMean, reduction != kNone ? &total : nullptr, e, stream);
  return {{reduction == kNone ? f.loss.view(targets.sizes()) : total, dh, dW}, f.launches + weighted + n};
}

}  // namespace gb
