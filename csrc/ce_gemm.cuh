#pragma once
// The products of the cross entropy over a vocabulary projection
// (cross_entropy.cu): a persistent tcgen05 GEMM, C[M, N] = A[M, K] B[N, K]^T,
// fp32 accumulation, 128 x 256 tiles, whose extent in tokens is read on the
// device (the number of trained tokens) and whose epilogues are the loss's.
//
//   kCeLse    rows tokens, columns vocabulary.  Per row and half tile of 128
//             columns (max, sum of exp) without the row's target; the target's
//             logit by itself.
//   kCeGrad   the same product; d = r exp(l - lse) in bf16, and r (p - 1) from the
//             forward's loss in the target's column.
//   kCeDh     rows tokens, columns hidden, K a vocabulary piece: fp32 sums of
//             dh, K split into slices where there are few tiles.
//   kCeDw     rows vocabulary, columns hidden, K the tokens: dW in bf16, with what
//             the rounding of d took from the targets' entries.
//
// One CTA per SM, 10 warps: TMA producer, MMA issuer, eight epilogue warps (two
// per 32-lane quarter of the accumulator, 128 columns each).  Four epilogue warps
// were not enough: at H = 1000 a tile's main loop is 8192 cycles, and the
// exponentials of 128 x 256 logits took longer with one warp per scheduler (88 us
// at 466 tokens x 50001).
//
// The tensor cores truncate the running sum at every step of 16 products, which
// shrinks a logit by some 1e-9 of itself per product: 4e-6 at H = 4096, seen as
// 2.5e-5 in every loss.  kCeLse therefore takes the reduction in segments of
// kSegment K-blocks and adds those in registers, round to nearest.  kCeGrad does
// without: an error of a logit is one relative to exp(l - lse), which is rounded to
// bf16.  Only p - 1 cancels, and that is not made from the remade logit: it is
// expm1(-loss), relatively as exact as the loss.  In the sums of kCeDh and kCeDw
// the truncation is far below the bf16 of their operands.
#include "gemm_tc.cuh"

namespace gb {

CUtensorMap make_tmap_bf16(const void* ptr, long rows, long cols, long ld, int box_rows);  // gemm_tc.cu

namespace ce {

enum Mode : int { kLse, kGrad, kDh, kDw };

constexpr int BN = 256;
constexpr int kThreads = 320;
constexpr int kEpilogue = 256;        // threads
constexpr int kSegment = 16;          // K-blocks of 64 per fp32 partial sum of a logit
using TileCfg = Cfg<BN>;

struct Args {
  int M, N;               // rows and columns; tokens at most, where they are counted on the device
  int kb;                 // K-blocks (kDw: at most)
  const int* live;        // number of trained tokens
  int* err;
  // kLse, kGrad
  const int64_t* target;
  float2* part;           // [M][2 blocks]
  float* target_logit;
  const float* lse;
  const float* hot;       // p - 1 of each token's target
  const float* ratio;     // r of each token
  int n_first;            // vocabulary index of column 0
  // results
  void* C;
  long ldc;
  int kb_first;           // kDh: K-blocks of the first piece, which fix the slices
  bool add;               // kDh: a later piece
  const float* unit;      // kDw: what the ratios are multiples of
  const unsigned* sorted; // kDw: the tokens' targets in order,
  const int* start;       //   where each 32 vocabulary rows start among them,
  int row_blocks;         //   for so many of 32,
  const float* rest;      //   and what a row lacks, at its first token and, not `joined`,
  long ldr;               //   at every kGroup-th place of the order that is its too
  bool joined;
  bool early;             // host: how the kernel is launched
};

constexpr int kGroup = 32;   // tokens, in the order of their targets, whose rests are added at once

__host__ __device__ __forceinline__ long row_blocks(long V) { return (V + 31) / 32; }

// What rounding the target's entry of d to bf16 leaves out.
__device__ __forceinline__ float rounded_off(float d) {
  const float rest = d - __bfloat162float(__float2bfloat16(d));
  return fabsf(rest) < INFINITY ? rest : 0.f;   // an entry that is not finite stays what it is
}

// Slices that the reduction of dh is split into, none of them empty: as many as
// fill the SMs, with at least four K-blocks each; with more tiles than SMs two
// where they fill the last round better (768 tiles on 148 SMs are 6 rounds, 1536
// halves 11).
__host__ __device__ __forceinline__ int dh_slices(int live, int hidden, int kb_first, int sms) {
  const int tiles = max(1, (live + BM - 1) / BM) * ((hidden + BN - 1) / BN);
  int want = max(1, min(sms / tiles, kb_first / 4));
  if (tiles >= sms && kb_first >= 64 && ((2 * tiles + sms - 1) / sms) * 100 < ((tiles + sms - 1) / sms) * 2 * 96) want = 2;
  const int per = (kb_first + want - 1) / want;
  return (kb_first + per - 1) / per;
}

// Elements between the slices, whose rows are those of whole tiles.
__host__ __device__ __forceinline__ long dh_slice_elements(int live, long ld) {
  return static_cast<long>((live + BM - 1) / BM) * BM * ld;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 columns of a thread's TMEM lane (the 128 sums of kCeLse leave no room for 32)
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// 32 bytes in one store
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 32 values of an output row; `align`: bytes that the row's chunks are multiples of.
__device__ __forceinline__ void store_chunk(__nv_bfloat16* C, const float (&v)[32], int count, int align) {
  if (count >= 32 && align >= 16) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
    if (align >= 32) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t o[8] = {w[8 * q], w[8 * q + 1], w[8 * q + 2], w[8 * q + 3],
                               w[8 * q + 4], w[8 * q + 5], w[8 * q + 6], w[8 * q + 7]};
        store32(C + 16 * q, o);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        reinterpret_cast<uint4*>(C)[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < count) C[j] = __float2bfloat16(v[j]);
  }
}

// The warp's 32 rows x 32 values, row per lane, to 32 rows of C (the lane's first
// value at C, rows ldc apart) through 2 KB of shared memory, so that an access
// covers 8 rows of 64 bytes instead of 32 of 16: with a row per lane the stores
// of dW took as many cycles in L1 as 8 K-blocks of products.  Rows that start off a
// 16-byte boundary (`wide` false), and the last columns, are written a row at a time,
// a value per lane.
__device__ __forceinline__ void store_rows(uint8_t* stage, __nv_bfloat16* C, long ldc, const float (&v)[32], int rows,
                                           int count, bool wide) {
  const int lane = threadIdx.x & 31;
  uint4* s = reinterpret_cast<uint4*>(stage);
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q)
    s[lane * 4 + (q ^ ((lane >> 1) & 3))] =
        make_uint4(bf16_pair(v[8 * q], v[8 * q + 1]), bf16_pair(v[8 * q + 2], v[8 * q + 3]),
                   bf16_pair(v[8 * q + 4], v[8 * q + 5]), bf16_pair(v[8 * q + 6], v[8 * q + 7]));
  __syncwarp();
  if (wide && count >= 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2), q = lane & 3;
      const uint4 x = s[r * 4 + (q ^ ((r >> 1) & 3))];
      if (r < rows) reinterpret_cast<uint4*>(C + r * ldc)[q] = x;
    }
  } else {
    const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(stage);
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows && lane < count) C[r * ldc + lane] = h[r * 32 + ((lane >> 3) ^ ((r >> 1) & 3)) * 8 + (lane & 7)];
  }
}

template <int MODE, int LAYOUT>
__global__ void __launch_bounds__(kThreads, 1)
    ce_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Args args) {
  constexpr int STAGES = TileCfg::STAGES;
  constexpr bool A_MN = (LAYOUT & 2) != 0, B_MN = (LAYOUT & 1) != 0;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);  // 128-byte swizzle atoms
  uint8_t* smA = smem;
  uint8_t* smB = smem + STAGES * TileCfg::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * TileCfg::STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* done = tempty + 2;   // every product issued has ended
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], kEpilogue);
    }
    mbar_init(done, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) tmem_alloc(tmem_slot, TileCfg::TMEM_COLS);
  pdl_trigger();
  pdl_wait();
  const int live = __ldcg(args.live);
  const int M = MODE == kDw ? args.M : min(args.M, live);
  const int kb_total = MODE == kDw ? min(args.kb, (live + BK - 1) / BK) : args.kb;
  const int splits = MODE == kDh ? min(dh_slices(live, args.N, args.kb_first, gridDim.x), kb_total) : 1;
  const int num_m = (M + BM - 1) / BM, num_n = (args.N + BN - 1) / BN;
  const int units = num_m * num_n * splits;
  constexpr int kSeg = MODE == kLse ? kSegment : 1 << 30;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const Unit w = decode_unit(u, num_m, num_n, splits, kb_total);
        for (int kb = w.kb_begin; kb < w.kb_end; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, args.err, kErrSmemEmptyTimeout)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[stage], TileCfg::STAGE_BYTES);
          uint8_t* a_dst = smA + stage * TileCfg::A_BYTES;
          uint8_t* b_dst = smB + stage * TileCfg::B_BYTES;
          if constexpr (A_MN) {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j)
              tma_load_2d(a_dst + j * kMnAtomBytes, &tmA, &full[stage], w.m_block * BM + j * 64, kb * BK);
          } else {
            tma_load_2d(a_dst, &tmA, &full[stage], kb * BK, w.m_block * BM);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j)
              tma_load_2d(b_dst + j * kMnAtomBytes, &tmB, &full[stage], w.n_block * BN + j * 64, kb * BK);
          } else {
            tma_load_2d(b_dst, &tmB, &full[stage], kb * BK, w.n_block * BN);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // No copy into this CTA's shared memory may be in flight at its exit, after a wait
      // that gave up either: the last fill of every stage is waited for, whatever the
      // error word says (a stage never filled counts as complete).
      for (int s = 0; s < STAGES; ++s) {
        mbar_wait(&full[stage], phase ^ 1u, nullptr, kErrTmaFullTimeout);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc_bf16(BM, BN, A_MN, B_MN);
      constexpr uint64_t a_step = A_MN ? (2048 >> 4) : 2, b_step = B_MN ? (2048 >> 4) : 2;
      int stage = 0, acc_iter = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const Unit w = decode_unit(u, num_m, num_n, splits, kb_total);
        for (int kb0 = w.kb_begin; kb0 < w.kb_end && ok; kb0 += kSeg) {
          const int kb1 = w.kb_end - kb0 > kSeg ? kb0 + kSeg : w.kb_end;
          const int acc = acc_iter & 1;
          if (!mbar_wait(&tempty[acc], ((acc_iter >> 1) & 1) ^ 1u, args.err, kErrTmemEmptyTimeout)) {
            ok = false;
            break;
          }
          tc_fence_after();
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&full[stage], phase, args.err, kErrTmaFullTimeout)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a_addr = smem_addr(smA + stage * TileCfg::A_BYTES);
            const uint32_t b_addr = smem_addr(smB + stage * TileCfg::B_BYTES);
            const uint64_t a_desc = A_MN ? umma_desc_mn_sw128(a_addr, kMnAtomBytes, 1024) : umma_desc_k_sw128(a_addr);
            const uint64_t b_desc = B_MN ? umma_desc_mn_sw128(b_addr, kMnAtomBytes, 1024) : umma_desc_k_sw128(b_addr);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              umma_bf16(tmem_base + acc * BN, a_desc + a_step * k, b_desc + b_step * k, idesc,
                        (kb > kb0 || k > 0) ? 1u : 0u);
            umma_commit(&empty[stage]);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          umma_commit(&tfull[acc]);
          ++acc_iter;
        }
      }
      // nor any product, whose accumulators are given back below
      umma_commit(done);
      mbar_wait(done, 0, nullptr, kErrTmemFullTimeout);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;            // TMEM lanes this warp may access
    const int half = (warp - 2) >> 2;        // which 128 columns of the tile
    const uint32_t t_col = static_cast<uint32_t>(half * 128) + (static_cast<uint32_t>(quarter * 32) << 16);
    const int align = (args.ldc & 15) == 0 ? 32 : (args.ldc & 7) == 0 ? 16 : 2;
    constexpr float kLog2e = 1.4426950408889634f;
    const float unit = MODE == kDw ? __ldcg(args.unit) : 1.f;
    int acc_iter = 0;
    // kDw: the first token of this lane's row in the order of the targets, -1 without one;
    // found, and its rests fetched, during the unit before
    int next_at = -1;
    const auto look_up = [&](int u) {
      const Unit w = decode_unit(u, num_m, num_n, 1, kb_total);
      const unsigned row = static_cast<unsigned>(args.n_first + w.m_block * BM + quarter * 32 + lane);
      const int block = min(static_cast<int>(row / 32), args.row_blocks);
      int lo = args.start[block], hi = args.start[min(block + 1, args.row_blocks)];
      const int past = hi;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (args.sorted[mid] < row) lo = mid + 1;
        else hi = mid;
      }
      next_at = lo < past && args.sorted[lo] == row ? lo : -1;
      if (next_at >= 0) {
        const float* rest = args.rest + next_at * args.ldr + w.n_block * BN + half * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (w.n_block * BN + half * 128 + i * 32 < args.ldr)
            asm volatile("prefetch.global.L1 [%0];" ::"l"(rest + i * 32));
      }
    };
    if constexpr (MODE == kDw)
      if (static_cast<int>(blockIdx.x) < units) look_up(blockIdx.x);
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const Unit w = decode_unit(u, num_m, num_n, splits, kb_total);
      const int m = w.m_block * BM + quarter * 32 + lane;
      const int n0 = w.n_block * BN + half * 128;
      if constexpr (MODE == kDw) {
        if (kb_total == 0) {  // no trained token: the gradient is zero
          const float z[32] = {};
          for (int c = 0; c < 4; ++c)
            if (m < M) store_chunk(static_cast<__nv_bfloat16*>(args.C) + m * args.ldc + n0 + c * 32, z,
                                   args.N - n0 - c * 32, align);
          continue;
        }
      }
      if (w.kb_end <= w.kb_begin) continue;
      long target = 0;
      float lse2 = 0.f, ratio = 0.f, hot_d = 0.f;
      if (m < M) {
        if constexpr (MODE == kLse || MODE == kGrad) target = args.target[m] - args.n_first - n0;
        if constexpr (MODE == kGrad) {
          lse2 = args.lse[m] * kLog2e;
          ratio = args.ratio[m];
          hot_d = ratio * args.hot[m];
        }
      }
      if constexpr (MODE == kLse) {
        float logit[128];
#pragma unroll
        for (int j = 0; j < 128; ++j) logit[j] = 0.f;
#pragma unroll 1
        for (int kb0 = w.kb_begin; kb0 < w.kb_end; kb0 += kSeg, ++acc_iter) {
          const int acc = acc_iter & 1;
          mbar_wait(&tfull[acc], (acc_iter >> 1) & 1, args.err, kErrTmemFullTimeout);
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float v[16];
            tmem_ld16(tmem_base + acc * BN + t_col + c * 16, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) logit[c * 16 + j] += v[j];
          }
          tc_fence_before();
          mbar_arrive(&tempty[acc]);
        }
        const int count = args.N - n0;  // columns that exist
        if (m < M && target >= 0 && target < 128) {  // the target is not among the others
#pragma unroll
          for (int j = 0; j < 128; ++j)
            if (target == j) {
              args.target_logit[m] = logit[j];
              logit[j] = -INFINITY;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 128; ++j) {
          if (j >= count) logit[j] = -INFINITY;
          top = fmaxf(top, logit[j]);
        }
        // (nothing but -inf or NaN: exp(-inf) = 0 and NaN stay what they are)
        const float base = top > -INFINITY ? top * kLog2e : 0.f;
        float s[4] = {};
#pragma unroll
        for (int j = 0; j < 128; ++j) s[j & 3] += ex2(fmaf(logit[j], kLog2e, -base));
        if (m < M)
          args.part[static_cast<long>(m) * (2 * num_n) + 2 * w.n_block + half] =
              make_float2(top, (s[0] + s[1]) + (s[2] + s[3]));
      } else {
        const int acc = acc_iter & 1;
        const int token_at = next_at;
        if constexpr (MODE == kDw)
          if (u + static_cast<int>(gridDim.x) < units) look_up(u + gridDim.x);
        const bool have = mbar_wait(&tfull[acc], (acc_iter >> 1) & 1, args.err, kErrTmemFullTimeout);
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < (have ? 4 : 0); ++c) {
          float v[32];
          tmem_ld32(tmem_base + acc * BN + t_col + c * 32, v);
          const int nc = n0 + c * 32, count = args.N - nc;
          if constexpr (MODE == kGrad) {
            __nv_bfloat16* C = static_cast<__nv_bfloat16*>(args.C) + m * args.ldc + nc;
            if (m < M) {
              const int hot = static_cast<int>(target) - c * 32;
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = j == hot ? hot_d : ratio * ex2(fmaf(v[j], kLog2e, -lse2));
              store_chunk(C, v, count, align);
            } else if (m < (M + BK - 1) / BK * BK) {
              // dW contracts over whole blocks of BK tokens: the rows that fill the last one are zero
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = 0.f;
              store_chunk(C, v, count, align);
            }
          } else if constexpr (MODE == kDh) {
            if (m < M) {
              float* C = static_cast<float*>(args.C) + w.split * dh_slice_elements(live, args.ldc) + m * args.ldc + nc;
              if (count >= 32) {  // ldc is a multiple of 8
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  if (args.add) {
                    const float4 x = reinterpret_cast<const float4*>(C)[2 * q], y = reinterpret_cast<const float4*>(C)[2 * q + 1];
                    v[8 * q] += x.x, v[8 * q + 1] += x.y, v[8 * q + 2] += x.z, v[8 * q + 3] += x.w;
                    v[8 * q + 4] += y.x, v[8 * q + 5] += y.y, v[8 * q + 6] += y.z, v[8 * q + 7] += y.w;
                  }
                  uint32_t o[8];
#pragma unroll
                  for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(v[8 * q + i]);
                  store32(C + 8 * q, o);
                }
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (j < count) C[j] = (args.add ? C[j] : 0.f) + v[j];
              }
            }
          } else if constexpr (MODE == kDw) {
            if (token_at >= 0 && count > 0) {   // `rest` has whole lines
              const unsigned row = static_cast<unsigned>(args.n_first + m);
              int at = token_at;
              do {
                const float4* src = reinterpret_cast<const float4*>(args.rest + at * args.ldr + nc);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                  const float4 x = src[q];
                  v[4 * q] += x.x, v[4 * q + 1] += x.y, v[4 * q + 2] += x.z, v[4 * q + 3] += x.w;
                }
                at = (at / kGroup + 1) * kGroup;
              } while (!args.joined && at < live && args.sorted[at] == row);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= unit;
            __nv_bfloat16* C = static_cast<__nv_bfloat16*>(args.C) + nc;
            // the 16 KB past the stages and barriers belong to the epilogue's warps
            store_rows(smem + STAGES * TileCfg::STAGE_BYTES + 256 + (warp - 2) * 2048, C + (m - lane) * args.ldc,
                       args.ldc, v, M - (m - lane), count, align >= 16);
          }
        }
        tc_fence_before();
        mbar_arrive(&tempty[acc]);
        ++acc_iter;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TileCfg::TMEM_COLS);
  }
}

// Launches a kernel of the loss's chain.  `early`: it may start while its
// predecessor runs; it comes up beside it and waits in pdl_wait().  Every kernel of
// the chain calls pdl_wait() before it touches memory, in every thread, so that the
// end of one implies the end of all before it.  What the chain writes is read by
// plain or L2 loads, never through `const __restrict__` or __ldg: those are for
// memory that is constant while a kernel lives, and an early one lives before it is
// written.  Between kernels of some 8 us the gaps were a fifth of the time: without /
// with early launches 61 x 512 x 4096 (work 1.3e8) 52 / 43 us, 512 x 1024 x 4096 (2e9)
// 64 / 52, 1024 x 1024 x 16384 (1.7e10) 150 / 140, 128 x 2048 x 151936 (4e10) 552 / 548,
// 1024 x 2048 x 32000 (7e10) 444 / 443; at 6144 x 4096 x 151936 (3.8e12) the waiting
// blocks take up room that the running kernel's last tiles share (25.9 / 28.4 ms).
// kEarlyWork keeps to calls that are certain to gain; some up to 2e10 would too.
constexpr double kEarlyWork = 4e9;   // tokens x vocabulary x hidden

template <typename... KArgs, typename... A>
void launch_chained(bool early, void (*kernel)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...));
}

template <int MODE, int LAYOUT>
void launch(const CUtensorMap& a, const CUtensorMap& b, const Args& args, cudaStream_t stream, int device) {
  auto kern = ce_gemm_kernel<MODE, LAYOUT>;
  // MN-major operands: every address that a stage's descriptor can reach stays inside,
  // and kDw's warps stage their rows there, past the 256 bytes of barriers
  constexpr int smem = TileCfg::SMEM_BYTES + (LAYOUT != 0 ? 16384 : 0);
  static_assert(smem <= 227 * 1024, "shared memory budget");
  static bool configured[64] = {false};
  if (!configured[device]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    configured[device] = true;
  }
  // kDh splits by the grid's size: always one CTA per SM.  The others need no more than their tiles.
  const long tiles = static_cast<long>((args.M + BM - 1) / BM) * ((args.N + BN - 1) / BN);
  const int grid = MODE == kDh ? num_sms(device) : static_cast<int>(std::min<long>(tiles, num_sms(device)));
  launch_chained(args.early, kern, grid, kThreads, smem, stream, a, b, args);
}

}  // namespace ce
}  // namespace gb
