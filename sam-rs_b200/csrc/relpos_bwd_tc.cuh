// relpos_bwd_tc.cuh - tcgen05 kernels of the attention's backward pass: f16 / bf16, head_dim a multiple of 16 up to
// 128, grids up to 64 x 64. The mathematics and the reason for walking the scores twice are in relpos_bwd_simt.cuh.
//
// Both kernels recompute a 128 x 64 block of scores per step. The side that stays (128 queries in bwd_dq_tc, 128 keys in
// bwd_dkv_tc) is the A operand of its products and sits in TMEM; the side that passes by comes through shared memory by
// TMA. A block's S and dP are accumulators in TMEM; warps turn them into P and dS, a thread per row and 32 columns, and
// write those back as 16-bit pairs over the columns they came from, where they are the A operand of the products that
// follow. So no score, probability or gradient of one touches shared memory, and each operand tile that is read from it
// feeds 128 rows. Sixteen scoring warps in two groups take alternate steps: while one waits for its products the other
// computes.
//
//   bwd_dq_tc   S = Q K^T, dP = dO V^T, then dQ += dS K. A step's keys are 4 grid rows x 16 grid columns, all grid rows of
//               one band of 16 columns before the next band: a thread keeps the 16 rw of its row and band in registers
//               and reads 2 rh per step.
//               The bias: U = Q table^T once per tile (a product of the tile with the whole table) gives rh and rw by
//               shifted reads; they stay in shared memory and go to the workspace for the other kernel.
//               The bias gradients dRh, dRw are sums of dS over grid columns and rows: a thread's step sums are its share
//               of dRh (added in shared memory, each by its own thread), and a product of dS with a constant 0/1 matrix
//               E[kw][key] adds up dRw beside dQ.
//               Then G[r][t] = dRh[r, i+h-1-t] | dRw[r, j+w-1-t'] (zero where there is no such key) turns both remaining
//               products into plain ones: dQ += G table, dtable += G^T Q. G goes in as two 16-bit terms, so that dRh and
//               dRw are not rounded once more: side by side where shared memory holds both (windows), else the
//               second over the first (every global layer, head dim 128). 16 heads of 64 x 64 x 80 bf16: dtable's
//               error 2.1e-3 and dQ's 2.3e-3, 2.7e-3 and 2.6e-3 with one term, for 17 us.
//   bwd_dkv_tc  S^T = K Q^T, dP^T = V dO^T, then dV += P^T dO, dK += dS^T Q. The 128 keys are 8 x 16 (or 16 x 8) of the
//               grid: a step then needs 8 rows of rh (with lse subtracted) and 16 of rw instead of the 66 of two grid
//               rows. (rw as further columns of the S^T product, in two 16-bit terms against 0/1 columns of K, measured
//               slower: it saves the scoring warps a shared-memory read per four scores, but the issuer is the busier.)
//               A CTA per SM takes one key tile after the other, so that a tile's first copies run under the tile before.
//
// Bound by the tensor core in that it hardly ever waits for memory, and short of it by the hand-overs: a step's products
// take 650 to 750 cycles of it, a step about 2000 with its share of a tile's beginning and end, of which each wait and each
// commit on the way from products to scores and back costs about 50. 400 heads of 14 x 14 x 80 (196 rows in two tiles of
// 128): 89 + 57 us, 16 heads of 64 x 64 x 80: 278 + 271 us, 390 TFLOP/s of the five products that the gradients need.
//
// f16: P and dS of long rows fall below f16's normal range. P is kept as 2^12 P, and dS times a power of two per head
// that brings the largest possible |dS| near 2^13 (relpos_bwd.cuh); both are taken out again in f32. bf16 needs neither.
// P and dS are rounded to 16 bits as operands, once (dRw adds the rounded dS, dRh the unrounded); D is taken from the
// rounded out, as the forward pass left it.
//
// Warps (640 threads): 0 TMA producer, 1 MMA issuer, 2 TMEM allocator, 4-19 the scores. In bwd_dq_tc warp 3 issues the
// products that follow the scores, and warp 2 writes the bias out for the other kernel; in bwd_dkv_tc one issuer does
// better than two. Every wait is bounded (sm100::mbar_wait); the scoring warps meet on an mbarrier too, so that a timeout
// leaves nobody waiting.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "relpos_bwd_simt.cuh"
#include "sm100.cuh"

namespace samrs {
namespace bwd {

constexpr int kTcThreads = 640;
constexpr int kScoreWarps = 16;
constexpr int kStep = 64;       // keys (bwd_dq_tc) or queries (bwd_dkv_tc) per step
constexpr int kBandH = 4, kBandW = 16;  // a step's keys in bwd_dq_tc
constexpr int kMaxStages = 6;
constexpr int kEBytes = kBandW * 128;   // E [16][64 keys]
constexpr float kPShift = 12.f; // f16: P is kept as 2^12 P

__host__ __device__ constexpr int round_up(int x, int m) { return (x + m - 1) / m * m; }
// Bands of 16 grid columns, and blocks of 4 grid rows: an even number where there are several bands, so that a block
// falls to the same group of scoring warps in every band (its threads alone add to its dRh).
__host__ __device__ constexpr int bands(int w) { return (w + kBandW - 1) / kBandW; }
__host__ __device__ constexpr int blocks_h(int h, int w) {
  return bands(w) > 1 ? round_up((h + kBandH - 1) / kBandH, 2) : (h + kBandH - 1) / kBandH;
}

struct TcArgs {
  Args a;                    // a.rel: rh [bh][hq][np] f32, hq = h rounded up to 16
  float* rw;                 // rw [bh][wq][np] f32, wq = w rounded up to 16
  const float* amax;         // f16: [bh][norm_blocks][2], squared row norms of dout and v (row_norms); else null
  int norm_blocks;
  float gain;                // f16: what the largest possible |dS| is brought near, else 0
  int nbuf, nstages, stage_bytes;
  // bwd_dq_tc
  int halves, split;         // 128-row halves of the table; both terms of G fit at once
  int off_drh, off_e, off_tab, off_q, off_stage, off_bar;
  // bwd_dkv_tc
  int th, tw, tiles_h, tiles_w;
};

struct TcBars {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t s_full[2], dp_full[2], ds_full[2];
  uint64_t tab_full, q_full, ops, u_done, rel_done, ws_done, acc_done, g_done, fin, out_done, meet, final_mma;
  uint32_t tmem_base;
  int abort_flag;
};

// The power of two that dS of a head is multiplied by (1 for bf16).
__device__ __forceinline__ float ds_factor(const TcArgs& p, long bh) {
  if (!p.amax) return 1.f;
  float a = 0.f, b = 0.f;
  for (int k = 0; k < p.norm_blocks; ++k) {
    const float2 x = reinterpret_cast<const float2*>(p.amax)[bh * p.norm_blocks + k];
    a = fmaxf(a, x.x);
    b = fmaxf(b, x.y);
  }
  const float bound = 2.f * sqrtf(a) * sqrtf(b);
  if (!(bound > 0.f) || !(bound < INFINITY)) return 1.f;
  const int e = (int)fminf(fmaxf(floorf(log2f(p.gain / bound)), -24.f), 60.f);
  return __int_as_float((127 + e) << 23);
}

// 16 consecutive 16-bit elements as 8 words, zeros if not ok.
__device__ __forceinline__ void load_row16(const void* src, bool ok, uint32_t (&r)[8]) {
  uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
  if (ok) {
    a = __ldg(static_cast<const uint4*>(src));
    b = __ldg(static_cast<const uint4*>(src) + 1);
  }
  r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w, r[4] = b.x, r[5] = b.y, r[6] = b.z, r[7] = b.w;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint16_t to16(float x) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}
template <bool BF16>
__device__ __forceinline__ float from16(uint16_t x) {
  if constexpr (BF16) return __uint_as_float((uint32_t)x << 16);
  return __half2float(__ushort_as_half(x));
}

// The score block's columns of one 16-key (16-query) k-step as an A operand: a thread of half hf has packed its 32
// columns into the first 16 of them.
__device__ __forceinline__ constexpr int kstep_col(int k) { return 32 * (k >> 1) + 8 * (k & 1); }

// ------------------------------------------------------------------------------------------------ dQ
template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    bwd_dq_tc(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
              const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
              const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmT,
              const __grid_constant__ TcArgs p) {
  using namespace sm100;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int HC = HD / 16;
  constexpr int kKChunk = HD * 32, kKBytes = 4 * kKChunk;  // K of a step: [4 grid rows][HD][16 keys], 32-byte swizzle
  extern __shared__ uint8_t smem_raw[];
  if (__syncthreads_or(threadIdx.x == 0 && device_faulted())) return;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars* bars = reinterpret_cast<TcBars*>(smem + p.off_bar);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = p.a.h, w = p.a.w, n = h * w, hd = p.a.hd;
  const int nhb = blocks_h(h, w), nwb = bands(w), steps = nhb * nwb;
  const int hp = nhb * kBandH, wp = nwb * kBandW;
  const int qtiles = (n + 127) / 128, tr = table_rows(h, w);
  const long tiles = p.a.bh * qtiles;
  const int n_tiles = (int)((tiles - blockIdx.x + gridDim.x - 1) / gridDim.x);  // 0 if blockIdx.x >= tiles
  const int nbuf = p.nbuf, nst = p.nstages;  // nbuf is 1 or 2
  // TMEM columns; U and, at the end, dtable's two halves take over columns that are free then
  const int T_ACC = 0, T_E = HD, T_QA = HD + wp, T_OA = T_QA + HD / 2, T_S = T_OA + HD / 2;
  const int T_U1 = T_S + 256 <= 512 ? T_S + 128 : T_ACC;
  const int buf1 = nbuf == 2 ? 128 : 0;  // where the second buffer of S and dP begins

  if (threadIdx.x == 0) {
    for (int s = 0; s < nst; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->s_full[b], 1);
      mbar_init(&bars->dp_full[b], 1);
      mbar_init(&bars->ds_full[b], kScoreWarps / 2);
    }
    mbar_init(&bars->tab_full, 1);
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->u_done, 1);
    mbar_init(&bars->acc_done, 1);
    mbar_init(&bars->fin, 1);
    mbar_init(&bars->ws_done, 1);
    mbar_init(&bars->final_mma, 2);
    mbar_init(&bars->ops, kScoreWarps);
    mbar_init(&bars->rel_done, kScoreWarps);
    mbar_init(&bars->g_done, kScoreWarps);
    mbar_init(&bars->out_done, kScoreWarps);
    mbar_init(&bars->meet, kScoreWarps);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  // E: 1 where key 16 kh + kw of a step has kw = row (K-major, 128-byte swizzle)
  for (int idx = threadIdx.x; idx < kBandW * 64; idx += kTcThreads) {
    const int row = idx >> 6, key = idx & 63;
    *reinterpret_cast<uint16_t*>(smem + p.off_e + row * 128 + ((((key >> 3) ^ (row & 7)) << 4) | ((key & 7) * 2))) =
        (key & 15) == row ? to16<kBf16>(1.f) : (uint16_t)0;
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_previous_launch();  // bwd_prepare's
  constexpr uint32_t tmem = 0;  // (an allocation of all 512 columns; as a constant it spares the issuers registers)

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0 && n_tiles > 0) {
      const int tab_bytes = 128 * HD * 2;
      mbar_arrive_expect_tx(&bars->tab_full, p.halves * tab_bytes);
      for (int b = 0; b < p.halves; ++b)
        tma_load_3d(smem + p.off_tab + b * tab_bytes, &tmT, &bars->tab_full, 0, 128 * b, 0);
      Armed rows, ring;  // on q_full, and on full[]
      // test hook: CTA 0 never loads this step of its own (-1: none), so the issuers' waits for it run out
      const int withhold = blockIdx.x == 0 ? *reinterpret_cast<volatile int*>(&g_withhold_key_tile) : -1;
      int st = 0;
      uint32_t ph = 1;
      bool okk = true;
      for (int tl = 0; tl < n_tiles && okk; ++tl) {
        const long tile = blockIdx.x + (long)tl * gridDim.x;
        const int bh = (int)((unsigned)tile / (unsigned)qtiles), r0 = (int)(tile - (long)bh * qtiles) * 128;
        // Q, dO and O rows, once the previous tile's results have left the memory they go to
        if (tl > 0 && !mbar_wait_hot(&bars->out_done, (tl - 1) & 1, abort_flag)) break;
        mbar_arrive_expect_tx(&bars->q_full, 3 * 128 * HD * 2);
        ++rows.n;
        tma_load_4d(smem + p.off_q, &tmQ, &bars->q_full, 0, r0, 0, bh);
        tma_load_4d(smem, &tmDO, &bars->q_full, 0, r0, 0, bh);
        tma_load_4d(smem + 128 * HD * 2, &tmO, &bars->q_full, 0, r0, 0, bh);
        for (int pb = 0; pb < nwb && okk; ++pb)
          for (int s = 0; s < nhb; ++s, ++ring.n) {
            if (ring.n >= nst && !mbar_wait_hot(&bars->empty[st], ph, abort_flag)) {
              okk = false;
              break;
            }
            uint8_t* dst = smem + p.off_stage + st * p.stage_bytes;
            if (ring.n != withhold) {
              mbar_arrive_expect_tx(&bars->full[st], kKBytes + kStep * HD * 2);
              tma_load_4d(dst, &tmK, &bars->full[st], pb * kBandW, 0, s * kBandH, bh);
              tma_load_5d(dst + kKBytes, &tmV, &bars->full[st], 0, pb * kBandW, s * kBandH, 0, bh);
            }
            if (++st == nst) st = 0, ph ^= 1;
          }
      }
      mbar_drain(&bars->tab_full, 0);
      rows.pending(1, [&](int, uint32_t parity) { mbar_drain(&bars->q_full, parity); });
      ring.pending(nst, [&](int k, uint32_t parity) { mbar_drain(&bars->full[k], parity); });
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer of U, S and dP
    constexpr uint32_t idS = idesc_f16(kBf16, 128, kStep, false, true);     // S = Q K^T, K MN-major
    constexpr uint32_t idP = idesc_f16(kBf16, 128, kStep, false, false);    // dP = dO V^T
    constexpr uint32_t idU = idesc_f16(kBf16, 128, 128, false, false);      // U = Q table^T
    const uint32_t sb = smem_u32(smem);
    const uint64_t dK = smem_desc(sb + p.off_stage, kKChunk, 256, kLayoutSw32);
    const uint64_t dV = smem_desc(sb + p.off_stage + kKBytes, 16, 256, kLayoutSw32);
    const uint64_t dTabK = smem_desc(sb + p.off_tab, 16, 256, kLayoutSw32);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_hot(bar, parity, abort_flag)); };
    bool okk = true;
    int is = 0;             // steps issued,
    int st = 0, est = 0;    // their stage, and that of the step whose buffer is taken next,
    uint32_t ph = 0, eph = 0;
    for (int tl = 0; tl < n_tiles && okk; ++tl) {
      const uint32_t tp = tl & 1;
      okk = wait(&bars->ops, tp) && (tl > 0 || wait(&bars->tab_full, 0));
      if (!okk) break;
      tc_fence_after();
      for (int b = 0; b < p.halves; ++b)
#pragma unroll
        for (int c = 0; c < HC; ++c)
          mma_ts_w(tmem + (b ? T_U1 : T_S), tmem + T_QA + 8 * c, desc_add(dTabK, b * 128 * HD * 2 + c * 4096), idU, c > 0);
      mma_commit_w(&bars->u_done);
      if (!(okk = wait(&bars->rel_done, tp))) break;
      for (int s = 0; s < steps; ++s, ++is) {
        if (!(okk = wait(&bars->full[st], ph))) break;
        // the buffer's last step has gone into dQ (its stage is free then)
        if (is >= nbuf) {
          if (!(okk = wait(&bars->empty[est], eph))) break;
          if (++est == nst) est = 0, eph ^= 1;
        }
        tc_fence_after();
        const uint32_t tS = tmem + T_S + (is & 1) * buf1;
        const uint64_t kd = desc_add(dK, st * p.stage_bytes), vd = desc_add(dV, st * p.stage_bytes);
#pragma unroll
        for (int c = 0; c < HC; ++c) mma_ts_w(tS, tmem + T_QA + 8 * c, desc_add(kd, c * 512), idS, c > 0);
        mma_commit_w(&bars->s_full[is & 1]);
#pragma unroll
        for (int c = 0; c < HC; ++c) mma_ts_w(tS + 64, tmem + T_OA + 8 * c, desc_add(vd, c * 2048), idP, c > 0);
        mma_commit_w(&bars->dp_full[is & 1]);
        if (++st == nst) st = 0, ph ^= 1;
      }
    }
    // every MMA issued by this warp has completed before the CTA tears down TMEM
    mma_commit_w(&bars->final_mma);
    mbar_drain(&bars->final_mma, 0);
  } else if (warp == 3) {
    // ---------------------------------------------------------------- MMA issuer of dQ, dRw and dtable
    // (An issuer's wait costs the tensor core about 200 cycles, since it queues behind the issuer's own products: with
    // two issuers one's waits pass while the other's products run.)
    constexpr uint32_t idQ = idesc_f16(kBf16, 128, HD, false, false);       // dQ += dS K
    constexpr uint32_t idE = idesc_f16(kBf16, 128, kBandW, false, false);   // dRw += dS E
    constexpr uint32_t idG = idesc_f16(kBf16, 128, HD, false, true);        // dQ += G table
    constexpr uint32_t idT = idesc_f16(kBf16, 128, HD, true, true);         // dtable = G^T Q
    const uint32_t sb = smem_u32(smem);
    const uint64_t dKk = smem_desc(sb + p.off_stage, 16, 256, kLayoutSw32);
    const uint64_t dE = smem_desc(sb + p.off_e, 16, 1024, kLayoutSw128);
    const uint64_t dTabN = smem_desc(sb + p.off_tab, 4096, 256, kLayoutSw32);
    const uint64_t dQn = smem_desc(sb + p.off_q, 4096, 256, kLayoutSw32);
    const uint64_t dGk = smem_desc(sb, 16, 1024, kLayoutSw128);
    const uint64_t dGm = smem_desc(sb, 16384, 1024, kLayoutSw128);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_hot(bar, parity, abort_flag)); };
    bool okk = true;
    int id = 0, st = 0;  // steps issued, their stage
    for (int tl = 0; tl < n_tiles && okk; ++tl) {
      for (int pb = 0; pb < nwb && okk; ++pb)
        for (int s = 0; s < nhb; ++s, ++id) {
          const int b = id & 1;
          if (!(okk = wait(&bars->ds_full[b], (id >> 1) & 1))) break;
          tc_fence_after();
          const uint64_t kd = desc_add(dKk, st * p.stage_bytes);
          const uint32_t tS = tmem + T_S + b * buf1;
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
            mma_ts_w(tmem + T_ACC, tS + kstep_col(k), desc_add(kd, kKChunk * k), idQ, (pb > 0 || s > 0 || k > 0) ? 1u : 0u);
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
            mma_ts_w(tmem + T_E + kBandW * pb, tS + kstep_col(k), desc_add(dE, 32 * k), idE, (s > 0 || k > 0) ? 1u : 0u);
          mma_commit_w(&bars->empty[st]);
          if (++st == nst) st = 0;
        }
      if (!okk) break;
      mma_commit_w(&bars->acc_done);
      for (int v = 0; v < 2; ++v) {  // G's two terms: side by side, or the second over the first once that has been read
        if (v == 0 || !p.split) {
          okk = wait(&bars->g_done, p.split ? tl & 1 : v) && (tl > 0 || wait(&bars->tab_full, 0));
          if (!okk) break;
          tc_fence_after();
        }
        const int at = v * p.split * p.halves * 32768;
        const uint64_t gk = desc_add(dGk, at), gm = desc_add(dGm, at);
        for (int k = 0; k < (tr + 15) / 16; ++k)  // 16 table rows each
          mma_ss_w(tmem + T_ACC, desc_add(gk, (k >> 2) * 16384 + 32 * (k & 3)),
                   desc_add(dTabN, (k >> 3) * 128 * HD * 2 + 512 * (k & 7)), idG, 1u);
        for (int b = 0; b < p.halves; ++b)
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 query rows each
            mma_ss_w(tmem + (b ? T_QA : T_S), desc_add(gm, b * 32768 + 2048 * k), desc_add(dQn, 512 * k), idT,
                     (v > 0 || k > 0) ? 1u : 0u);
        if (v > 0 || !p.split) mma_commit_w(&bars->fin);
      }
    }
    mma_commit_w(&bars->final_mma);
    mbar_drain(&bars->final_mma, 0);
  } else if (warp == 2) {
    // ---------------------------------------------------------------- the bias for the other kernel
    // Beside the steps: rh and rw as they are, zeros past the grid.
    const float* relh = reinterpret_cast<const float*>(smem);
    const float* relw = relh + hp * 128;
    const int hq = round_up(h, 16), wq16 = round_up(w, 16);
    for (int tl = 0; tl < n_tiles; ++tl) {
      const long tile = blockIdx.x + (long)tl * gridDim.x;
      const long bh = tile / qtiles;
      const int r0 = (int)(tile - bh * qtiles) * 128;
      if (!__all_sync(0xffffffffu, mbar_wait_hot(&bars->rel_done, tl & 1, abort_flag))) break;
      auto copy = [&](float* dst, const float* src, int rows, int padded) {
#pragma unroll 4
        for (int k = 0; k < padded; ++k)
          reinterpret_cast<float4*>(dst + (long)k * p.a.np)[lane] =
              k < rows ? reinterpret_cast<const float4*>(src + k * 128)[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      copy(p.a.rel + bh * hq * p.a.np + r0, relh, h, hq);
      copy(p.rw + bh * wq16 * p.a.np + r0, relw, w, wq16);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->ws_done);
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- scores
    const int cg = (warp - 4) >> 2, wq = warp & 3;  // (outside the steps: a quarter of the columns each)
    const int grp = cg >> 1, hf = cg & 1;           // step parity, half of a step's columns
    const int r = 32 * wq + lane;                   // TMEM lane = query row of the tile
    const uint32_t tl0 = tmem + ((uint32_t)(32 * wq) << 16);
    float* relh = reinterpret_cast<float*>(smem);             // [hp][128]; later G
    float* relw = relh + hp * 128;                            // [wp][128]
    float* drh = reinterpret_cast<float*>(smem + p.off_drh);  // [hp][128]
    float* dpart = drh;                                       // [4][128], before the steps
    const float c_log2 = p.a.scale * kLog2e;
    const float2 c2 = make_float2(c_log2, c_log2);
    uint32_t meets = 0;
    bool okk = true;
    auto arrive = [&](uint64_t* bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return okk = okk && __all_sync(0xffffffffu, mbar_wait_hot(bar, parity, abort_flag));
    };
    auto meet = [&]() {
      arrive(&bars->meet);
      return wait(&bars->meet, meets++ & 1);
    };
    int gs = 0;  // steps before this tile
    int first = p.a.first;
    float* part = p.a.partial + (long)blockIdx.x * tr * hd;
    for (int tl = 0; tl < n_tiles && okk; ++tl, gs += steps) {
      const uint32_t tp = tl & 1;
      const unsigned tile = blockIdx.x + tl * gridDim.x, ubh = tile / (unsigned)qtiles;
      const long bh = ubh;
      const int r0 = (int)(tile - ubh * qtiles) * 128, row = r0 + r;
      const bool valid = row < n;
      const int i = row / w, j = row - i * w;
      const float fac2 = ds_factor(p, bh);                      // dS is kept as dS fac2,
      const float fac = kBf16 ? fac2 : fac2 * exp2f(-kPShift);  // P as P 2^shift: dS fac2 = (P 2^shift) (dP - D) fac
      const float lse2 = valid ? p.a.lse[bh * n + row] * kLog2e : 0.f;
      // Q and dO rows to TMEM, D from dO and O. The rows come through shared memory: a row to a lane straight from global
      // memory costs the load unit a line per lane, 7000 cycles a tile.
      {
        if (!wait(&bars->q_full, tp)) break;
        const uint8_t* sq = smem + p.off_q + r * 32;
        const uint8_t* sd = smem + r * 32;
        const uint8_t* so = sd + 128 * HD * 2;
        const int sw = ((r >> 2) & 1) * 16;  // 32-byte swizzle
        float d = 0.f;
        auto load = [&](const uint8_t* at, uint32_t (&x)[8]) {
          const uint4 lo = *reinterpret_cast<const uint4*>(at + sw), hi = *reinterpret_cast<const uint4*>(at + (sw ^ 16));
          x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
        };
        for (int c = cg; c < HC; c += 4) {
          uint32_t a[8], g[8], o[8];
          load(sq + c * 4096, a);
          load(sd + c * 4096, g);
          load(so + c * 4096, o);
          tmem_st8(tl0 + T_QA + 8 * c, a);
          tmem_st8(tl0 + T_OA + 8 * c, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 x = unpack2<kBf16>(g[e]), y = unpack2<kBf16>(o[e]);
            d = fmaf(x.x, y.x, d);
            d = fmaf(x.y, y.y, d);
          }
        }
        dpart[cg * 128 + r] = d;
        tmem_wait_st();
        tc_fence_before();
        arrive(&bars->ops);
      }
      if (!meet()) break;  // (dO and O have been read: rel may go over them)
      const float dsum = ((dpart[r] + dpart[128 + r]) + (dpart[256 + r] + dpart[384 + r])) * fac;
      if (cg == 0) p.a.dsum[bh * p.a.np + row] = -dsum;
      if (!wait(&bars->u_done, tp)) break;
      tc_fence_after();
      {
        // rh[kh] = U[i + h - 1 - kh] - lse and rw[kw] = U[2h - 1 + j + w - 1 - kw]: column t of U is row kh = th - t of
        // relh, or row kw = tw - t of relw
        const float top = (kBf16 ? 0.f : kPShift) - lse2;
        const int th = valid ? i + h - 1 : -4096, tw = valid ? j + w - 1 + 2 * h - 1 : -4096;  // (no row: nothing is in range)
        for (int c = cg; c < 8 * p.halves; c += 4) {
          uint32_t u[16];
          tmem_ld16(tl0 + (c < 8 ? T_S + 16 * c : T_U1 + 16 * (c - 8)), u);
          tmem_wait_ld_regs(u);
          if (16 * c < 2 * h - 1) {
            float* dst = relh + (th - 16 * c) * 128 + r;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (16 * c + e < 2 * h - 1 && (unsigned)(th - 16 * c - e) < (unsigned)h)
                dst[-e * 128] = fmaf(__uint_as_float(u[e]), kLog2e, top);
          }
          if (16 * c + 15 >= 2 * h - 1) {
            float* dst = relw + (tw - 16 * c) * 128 + r;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (16 * c + e >= 2 * h - 1 && (unsigned)(tw - 16 * c - e) < (unsigned)w)
                dst[-e * 128] = __uint_as_float(u[e]) * kLog2e;
          }
        }
        // no such key: P = 0; no such query: any finite bias does, its rows of Q, dO and O are zeros
        for (int k = (valid ? h : 0) + cg; k < hp; k += 4) relh[k * 128 + r] = k < h ? 0.f : -INFINITY;
        for (int k = (valid ? w : 0) + cg; k < wp; k += 4) relw[k * 128 + r] = k < w ? 0.f : -INFINITY;
      }
      tc_fence_before();
      arrive(&bars->rel_done);  // U has been read
      if (!meet()) break;       // all of relh and relw is written
      if (cg < 3) {
        // the next tile's rows into L2
        const unsigned nt = tile + gridDim.x, nbh = nt / (unsigned)qtiles;
        const int nrow = (int)(nt - nbh * qtiles) * 128 + r;
        if (nt < tiles && nrow < n) {
          const void* base = cg == 0 ? p.a.q : cg == 1 ? p.a.dout : p.a.out;
          const char* at = reinterpret_cast<const char*>(static_cast<const T*>(base) + ((long)nbh * n + nrow) * hd);
          for (int k = 0; k < hd * 2; k += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + k));
        }
      }
      const float2 f2 = make_float2(fac, fac), nd2 = make_float2(-dsum, -dsum);
      // this group's steps: step s of the tile has number gs + s, and the group takes those of its parity
      int s = (gs + grp) & 1;  // first step of the tile with (gs + s) & 1 == grp
      int pb = 0, sb = s;
      while (sb >= nhb) sb -= nhb, ++pb;
      int have = -1;  // the band whose rw are in registers
      float2 rw[8];
      for (; s < steps; s += 2) {
        const int g = gs + s;
        if (pb != have) {
          have = pb;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            rw[e] = make_float2(relw[(kBandW * pb + 2 * e) * 128 + r], relw[(kBandW * pb + 2 * e + 1) * 128 + r]);
        }
        const uint32_t tS = tl0 + T_S + grp * buf1 + 32 * hf;
        const int kh = kBandH * sb + 2 * hf;
        const float rh[2] = {relh[kh * 128 + r], relh[(kh + 1) * 128 + r]};
        float sums[2];
        if (!wait(&bars->s_full[grp], (g >> 1) & 1)) break;
        tc_fence_after();
        uint32_t sv[2][16], dv[16], pk[8];
        tmem_ld16(tS, sv[0]);
        tmem_ld16(tS + 16, sv[1]);
        tmem_wait_ld_regs(sv[0]);
        tmem_wait_ld_regs(sv[1]);
        // P of both grid rows while dP is still being computed
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float2 rh2 = make_float2(rh[q], rh[q]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float2 y = fma2(make_float2(__uint_as_float(sv[q][2 * e]), __uint_as_float(sv[q][2 * e + 1])), c2, add2(rw[e], rh2));
            y = make_float2(ex2(y.x), ex2(y.y));
            sv[q][2 * e] = __float_as_uint(y.x);
            sv[q][2 * e + 1] = __float_as_uint(y.y);
          }
        }
        if (!wait(&bars->dp_full[grp], (g >> 1) & 1)) break;
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          tmem_ld16(tS + 64 + 16 * q, dv);
          tmem_wait_ld_regs(dv);
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 gd = fma2(make_float2(__uint_as_float(dv[2 * e]), __uint_as_float(dv[2 * e + 1])), f2, nd2);
            const float2 y = mul2(make_float2(__uint_as_float(sv[q][2 * e]), __uint_as_float(sv[q][2 * e + 1])), gd);
            pk[e] = pack2(y.x, y.y, kBf16);
            sum = add2(sum, y);
          }
          tmem_st8(tS + 8 * q, pk);
          sums[q] = sum.x + sum.y;
        }
        tmem_wait_st();
        tc_fence_before();
        arrive(&bars->ds_full[grp]);
        // dRh of these two grid rows over this band (this thread alone adds to them)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float* d = drh + (kh + q) * 128 + r;
          *d = pb > 0 ? *d + sums[q] : sums[q];
        }
        sb += 2;
        while (sb >= nhb) sb -= nhb, ++pb;
      }
      if (!okk || !wait(&bars->acc_done, tp)) break;
      tc_fence_after();
      if (!wait(&bars->ws_done, tp) || !meet()) break;  // drh is complete, relh and relw have been read
      // G (16-bit, 128-byte swizzle, 64 table rows per atom) goes over relh and relw: zeros, then dRh and dRw where they
      // belong. G takes 1 / scale along, so that dQ and dtable are scaled once at the end.
      {
        uint8_t* G = smem;
        for (int v = threadIdx.x - 128; v < 2048 * p.halves * (p.split + 1); v += 32 * kScoreWarps)
          reinterpret_cast<uint4*>(G)[v] = make_uint4(0u, 0u, 0u, 0u);
        if (!meet()) break;
        const float inv = 1.f / p.a.scale;
        const int th = i + h - 1, tw = j + w - 1 + 2 * h - 1, lo = p.halves * 32768;
        auto put = [&](int t, float x, bool rest) {
          uint8_t* at = G + (t >> 6) * 16384 + r * 128 + (((((t >> 3) & 7) ^ (r & 7)) << 4) | ((t & 7) * 2));
          const uint16_t hi = to16<kBf16>(x);
          *reinterpret_cast<uint16_t*>(at) = rest ? to16<kBf16>(x - from16<kBf16>(hi)) : hi;
          if (!rest && p.split) *reinterpret_cast<uint16_t*>(at + lo) = to16<kBf16>(x - from16<kBf16>(hi));
        };
        auto put_all = [&](bool rest) {
          if (valid) {
#pragma unroll 4
            for (int k = cg; k < h; k += 4) put(th - k, drh[k * 128 + r] * inv, rest);
          }
          // (dRw's columns go out in the same quarters: 4 of each band)
          for (int c = 0; c < nwb; ++c) {
            uint32_t u[4];
            tmem_ld4(tl0 + T_E + 16 * c + 4 * cg, u);
            tmem_wait_ld_regs(u);
            if (valid) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (16 * c + 4 * cg + e < w) put(tw - 16 * c - 4 * cg - e, __uint_as_float(u[e]) * inv, rest);
            }
          }
          fence_proxy_async_smem();
          tc_fence_before();
          arrive(&bars->g_done);
        };
        put_all(false);
        if (!p.split) {  // the second term, once the first one's products have read it
          if (!wait(&bars->fin, 0)) break;
          tc_fence_after();
          put_all(true);
        }
      }
      if (!wait(&bars->fin, p.split ? tp : 1)) break;
      tc_fence_after();
      // dQ, and this CTA's share of dtable, by rows through shared memory (over Q, and over G and drh: their products
      // have completed): 16 columns at a time, dealt out among the four column quarters.
      const float outf = p.a.scale / fac2;
      const int items = (1 + p.halves) * HC;
      constexpr int kTabRow = HD * 4 + 16;  // (conflict-free 16-byte stores)
      for (int it = cg; it < items; it += 4) {
        const int of = it / HC, c = it - of * HC;
        uint32_t u[16];
        tmem_ld16(tl0 + (of == 0 ? T_ACC : of == 1 ? T_S : T_QA) + 16 * c, u);
        tmem_wait_ld_regs(u);
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(u[e]) * outf;
        if (of == 0) {
          uint32_t g[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = pack2(f[2 * e], f[2 * e + 1], kBf16);
          uint4* dst = reinterpret_cast<uint4*>(smem + p.off_q + r * (HD * 2) + 32 * c);
          dst[0] = make_uint4(g[0], g[1], g[2], g[3]);
          dst[1] = make_uint4(g[4], g[5], g[6], g[7]);
        } else if (r + 128 * (of - 1) < tr) {
          float4* dst = reinterpret_cast<float4*>(smem + (r + 128 * (of - 1)) * kTabRow + 64 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[e] = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      if (!meet()) break;
      // A row to a lane. An element of dtable is always added by the same thread, one tile after the other: the sum does
      // not depend on scheduling.
      if (cg == 0) {
        if (valid) bulk_store(static_cast<T*>(p.a.dq) + (bh * n + row) * hd, smem + p.off_q + r * (HD * 2), hd * 2);
      } else if (cg <= p.halves) {
        const int t = r + 128 * (cg - 1);
        if (t < tr) {
          bulk_wait();  // the previous tile's addition
          if (first)
            bulk_store(part + (long)t * hd, smem + t * kTabRow, hd * 4);
          else
            bulk_add_f32(part + (long)t * hd, smem + t * kTabRow, hd * 4);
        }
      }
      bulk_commit();
      bulk_wait_read();
      arrive(&bars->out_done);
      first = 0;
    }
    bulk_wait();
    __syncwarp();
    tmem_wait_st();  // (a wait may have run out between a store and its wait)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// --------------------------------------------------------------------------------------------- dK, dV
// Shared memory of a stage: Q and dO [HD / 16][64][32 B], rh [th <= 16][64] f32, rw of 32 queries [tw <= 16][32] f32 twice
// (128-byte swizzle), D [64] f32.
__host__ __device__ constexpr int dkv_stage_bytes(int hd) { return 2 * kStep * hd * 2 + 16 * 256 + 32 * 128 + 1024; }

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    bwd_dkv_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmO,
               const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW,
               const __grid_constant__ TcArgs p) {
  using namespace sm100;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int HC = HD / 16, kTile = kStep * HD * 2, kStage = dkv_stage_bytes(HD);
  constexpr int off_w = 2 * kTile, off_h = off_w + 32 * 128, off_d = off_h + 16 * 256;
  constexpr int T_DK = 0, T_DV = HD, T_KA = 2 * HD, T_VA = T_KA + HD / 2, T_S = 3 * HD;  // TMEM columns
  constexpr int buf1 = T_S + 256 <= 512 ? 128 : 0;  // where the second buffer of S^T and dP^T begins
  constexpr int nbuf = buf1 ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  if (__syncthreads_or(threadIdx.x == 0 && device_faulted())) return;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars* bars = reinterpret_cast<TcBars*>(smem + p.off_bar);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = p.a.h, w = p.a.w, n = h * w, hd = p.a.hd;
  const int steps = (n + kStep - 1) / kStep, nst = p.nstages;
  const unsigned per_head = p.tiles_h * p.tiles_w, tiles = (unsigned)p.a.bh * per_head;
  const int n_tiles = (int)((tiles - blockIdx.x + gridDim.x - 1) / gridDim.x);  // (the grid has at most `tiles` CTAs)
  // head, first grid row and column of this CTA's tile tl
  auto place = [&](int tl, int& bh, int& kh0, int& kw0) {
    const unsigned t = blockIdx.x + (unsigned)tl * gridDim.x;
    bh = (int)(t / per_head);
    const int kt = (int)(t - (unsigned)bh * per_head), y = kt / p.tiles_w;
    kh0 = y * p.th;
    kw0 = (kt - y * p.tiles_w) * p.tw;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < nst; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->s_full[b], 1);
      mbar_init(&bars->dp_full[b], 1);
      mbar_init(&bars->ds_full[b], kScoreWarps / 2);
    }
    mbar_init(&bars->ops, kScoreWarps);
    mbar_init(&bars->acc_done, 1);
    mbar_init(&bars->final_mma, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_previous_launch();  // bwd_dq_tc's rh, rw and D
  constexpr uint32_t tmem = 0;  // (an allocation of all 512 columns; as a constant it spares the issuers registers)

  if (warp == 0) {
    if (lane == 0) {
      const int hq = round_up(h, 16), wq16 = round_up(w, 16);
      // test hook, as in bwd_dq_tc: 1000 + the step
      const int withhold = blockIdx.x == 0 ? *reinterpret_cast<volatile int*>(&g_withhold_key_tile) - 1000 : -1;
      Armed ring;
      int st = 0;
      uint32_t ph = 1;
      bool okk = true;
      for (int tl = 0; tl < n_tiles && okk; ++tl) {
        int bh, kh0, kw0;
        place(tl, bh, kh0, kw0);
        for (int s = 0; s < steps; ++s, ++ring.n) {
          if (ring.n >= nst && !mbar_wait_hot(&bars->empty[st], ph, abort_flag)) {
            okk = false;
            break;
          }
          uint8_t* dst = smem + st * kStage;
          if (ring.n != withhold) {
            mbar_arrive_expect_tx(&bars->full[st], 2 * kTile + p.th * 256 + 2 * p.tw * 128 + kStep * 4);
            tma_load_4d(dst, &tmQ, &bars->full[st], 0, s * kStep, 0, bh);
            tma_load_4d(dst + kTile, &tmO, &bars->full[st], 0, s * kStep, 0, bh);
            for (int b = 0; b < 2; ++b)
              tma_load_2d(dst + off_w + b * 2048, &tmW, &bars->full[st], s * kStep + 32 * b, bh * wq16 + kw0);
            tma_load_2d(dst + off_h, &tmH, &bars->full[st], s * kStep, bh * hq + kh0);
            bulk_load(dst + off_d, p.a.dsum + (long)bh * p.a.np + s * kStep, kStep * 4, &bars->full[st]);
          }
          if (++st == nst) st = 0, ph ^= 1;
        }
      }
      ring.pending(nst, [&](int k, uint32_t parity) { mbar_drain(&bars->full[k], parity); });
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t idS = idesc_f16(kBf16, 128, kStep, false, false);  // S^T = K Q^T, dP^T = V dO^T
    constexpr uint32_t idA = idesc_f16(kBf16, 128, HD, false, true);      // dV += P^T dO, dK += dS^T Q
    const uint32_t sb = smem_u32(smem);
    const uint64_t dQk = smem_desc(sb, 16, 256, kLayoutSw32), dOk = smem_desc(sb + kTile, 16, 256, kLayoutSw32);
    const uint64_t dQn = smem_desc(sb, 2048, 256, kLayoutSw32), dOn = smem_desc(sb + kTile, 2048, 256, kLayoutSw32);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_hot(bar, parity, abort_flag)); };
    bool okk = true;
    int is = 0, id = 0, sst = 0, dst = 0;
    uint32_t sph = 0;
    auto issue_s = [&]() {
      if (!(okk = wait(&bars->full[sst], sph))) return;
      tc_fence_after();
      const uint32_t tS = tmem + T_S + (is & 1) * buf1;
      const uint64_t qd = desc_add(dQk, sst * kStage), od = desc_add(dOk, sst * kStage);
#pragma unroll
      for (int c = 0; c < HC; ++c) mma_ts_w(tS, tmem + T_KA + 8 * c, desc_add(qd, c * 2048), idS, c > 0);
      mma_commit_w(&bars->s_full[is & 1]);
#pragma unroll
      for (int c = 0; c < HC; ++c) mma_ts_w(tS + 64, tmem + T_VA + 8 * c, desc_add(od, c * 2048), idS, c > 0);
      mma_commit_w(&bars->dp_full[is & 1]);
      ++is;
      if (++sst == nst) sst = 0, sph ^= 1;
    };
    for (int tl = 0; tl < n_tiles && okk; ++tl) {
      // (the scoring warps have read the previous tile's dK and dV by then)
      if (!(okk = wait(&bars->ops, tl & 1))) break;
      tc_fence_after();
      for (int s = 0; s < nbuf && s < steps && okk; ++s) issue_s();
      for (int s = 0; s < steps && okk; ++s, ++id) {
        const int b = id & 1;
        if (!(okk = wait(&bars->ds_full[b], (id >> 1) & 1))) break;
        tc_fence_after();
        const uint32_t tS = tmem + T_S + b * buf1;
        const uint64_t qd = desc_add(dQn, dst * kStage), od = desc_add(dOn, dst * kStage);
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          mma_ts_w(tmem + T_DV, tS + kstep_col(k), desc_add(od, 512 * k), idA, (s > 0 || k > 0) ? 1u : 0u);
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          mma_ts_w(tmem + T_DK, tS + 64 + kstep_col(k), desc_add(qd, 512 * k), idA, (s > 0 || k > 0) ? 1u : 0u);
        mma_commit_w(&bars->empty[dst]);
        if (++dst == nst) dst = 0;
        if (s + nbuf < steps) issue_s();  // (in order behind the products that read the buffer)
      }
      if (okk) mma_commit_w(&bars->acc_done);
    }
    mma_commit_w(&bars->final_mma);
    mbar_drain(&bars->final_mma, 0);
  } else if (warp >= 4) {
    const int cg = (warp - 4) >> 2, wq = warp & 3;
    const int grp = cg >> 1, hf = cg & 1;
    const int r = 32 * wq + lane;  // TMEM lane = key of the tile
    const int dh = r / p.tw, dw = r - dh * p.tw;
    const uint32_t tl0 = tmem + ((uint32_t)(32 * wq) << 16);
    const float c_log2 = p.a.scale * kLog2e;
    const float2 c2 = make_float2(c_log2, c_log2);
    bool okk = true;
    int gs = 0;  // steps before this tile
    for (int tl = 0; tl < n_tiles && okk; ++tl, gs += steps) {
      int bh, kh0, kw0;
      place(tl, bh, kh0, kw0);
      const int kh = kh0 + dh, kw = kw0 + dw;
      const bool valid = kh < h && kw < w;
      const int key = valid ? kh * w + kw : 0;
      const float fac = ds_factor(p, bh);
      const float fb = kBf16 ? fac : fac * exp2f(-kPShift);
      const float2 f2 = make_float2(fb, fb);
      {
        const T* kc = static_cast<const T*>(p.a.kt) + (long)bh * hd * n + key;
        const T* vr = static_cast<const T*>(p.a.v) + ((long)bh * n + key) * hd;
        for (int c = cg; c < HC; c += 4) {
          const bool ok = valid && 16 * c < hd;
          uint32_t a[8], g[8];
          uint16_t e[16];
#pragma unroll
          for (int d = 0; d < 16; ++d) e[d] = ok ? __ldg(reinterpret_cast<const uint16_t*>(kc + (long)(16 * c + d) * n)) : 0;
          load_row16(vr + 16 * c, ok, g);
#pragma unroll
          for (int d = 0; d < 8; ++d) a[d] = (uint32_t)e[2 * d] | ((uint32_t)e[2 * d + 1] << 16);
          tmem_st8(tl0 + T_KA + 8 * c, a);
          tmem_st8(tl0 + T_VA + 8 * c, g);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ops);
      }
      const int s0 = (gs + grp) & 1;  // the group's first step of this tile
      int st = (gs + s0) % nst;
      uint32_t ph = ((gs + s0) / nst) & 1;
      if (tl + 1 < n_tiles && cg < 2) {
        // the next tile's K and V into L2 (kt: the thread's key in 16-row strides; v: its row)
        int nb, nh0, nw0;
        place(tl + 1, nb, nh0, nw0);
        const int nk = (nh0 + dh) * w + nw0 + dw;
        if (nh0 + dh < h && nw0 + dw < w) {
          if (cg == 0) {
            const char* at = reinterpret_cast<const char*>(static_cast<const T*>(p.a.v) + ((long)nb * n + nk) * hd);
            for (int k = 0; k < hd * 2; k += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + k));
          } else if (dw == 0) {
            const T* at = static_cast<const T*>(p.a.kt) + (long)nb * hd * n + nk;
            for (int d = 0; d < hd; ++d) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + (long)d * n));
          }
        }
      }
      for (int s = s0; s < steps; s += 2) {
        const int g = gs + s;
        const uint32_t tS = tl0 + T_S + grp * buf1 + 32 * hf;
        // the stage's rh and D (the S products waited for the same copies)
        okk = __all_sync(0xffffffffu, mbar_wait_hot(&bars->full[st], ph, abort_flag) &&
                                          mbar_wait_hot(&bars->s_full[grp], (g >> 1) & 1, abort_flag));
        if (!okk) break;
        tc_fence_after();
        uint32_t sv[2][16], dv[16], pk[8];
        tmem_ld16(tS, sv[0]);
        tmem_ld16(tS + 16, sv[1]);
        const float4* hs = reinterpret_cast<const float4*>(smem + st * kStage + off_h + dh * 256) + 8 * hf;
        const uint8_t* ws = smem + st * kStage + off_w + 2048 * hf + dw * 128;
        const float4* ds = reinterpret_cast<const float4*>(smem + st * kStage + off_d) + 8 * hf;
        tmem_wait_ld_regs(sv[0]);
        tmem_wait_ld_regs(sv[1]);
        // P while dP is still being computed
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const float4 a4 = hs[4 * q + f];
            const float4 b4 = *reinterpret_cast<const float4*>(ws + (((4 * q + f) ^ (dw & 7)) << 4));
#pragma unroll
            for (int e = 2 * f; e < 2 * f + 2; ++e) {
              const float2 x = e & 1 ? add2(make_float2(a4.z, a4.w), make_float2(b4.z, b4.w))
                                     : add2(make_float2(a4.x, a4.y), make_float2(b4.x, b4.y));
              float2 y = fma2(make_float2(__uint_as_float(sv[q][2 * e]), __uint_as_float(sv[q][2 * e + 1])), c2, x);
              y = make_float2(ex2(y.x), ex2(y.y));
              sv[q][2 * e] = __float_as_uint(y.x);
              sv[q][2 * e + 1] = __float_as_uint(y.y);
              pk[e] = pack2(y.x, y.y, kBf16);
            }
          }
          tmem_st8(tS + 8 * q, pk);
        }
        okk = __all_sync(0xffffffffu, mbar_wait_hot(&bars->dp_full[grp], (g >> 1) & 1, abort_flag));
        if (!okk) break;
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          tmem_ld16(tS + 64 + 16 * q, dv);
          tmem_wait_ld_regs(dv);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 d4 = ds[4 * q + (e >> 1)];
            const float2 nd = e & 1 ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y);  // -D
            const float2 gd = fma2(make_float2(__uint_as_float(dv[2 * e]), __uint_as_float(dv[2 * e + 1])), f2, nd);
            const float2 y = mul2(make_float2(__uint_as_float(sv[q][2 * e]), __uint_as_float(sv[q][2 * e + 1])), gd);
            pk[e] = pack2(y.x, y.y, kBf16);
          }
          tmem_st8(tS + 64 + 8 * q, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ds_full[grp]);
        for (int k = 0; k < 2; ++k)
          if (++st == nst) st = 0, ph ^= 1;
      }
      okk = okk && __all_sync(0xffffffffu, mbar_wait_hot(&bars->acc_done, tl & 1, abort_flag));
      if (okk) {
        tc_fence_after();
        const float fk = p.a.scale / fac, fv = kBf16 ? 1.f : exp2f(-kPShift);
        T* dkc = static_cast<T*>(p.a.dkt) + (long)bh * hd * n + key;
        T* dvr = static_cast<T*>(p.a.dv) + ((long)bh * n + key) * hd;
        for (int c = cg; c < HC; c += 4) {
          uint32_t u[16], x[16], g[8];
          tmem_ld16(tl0 + T_DK + 16 * c, u);
          tmem_ld16(tl0 + T_DV + 16 * c, x);
          tmem_wait_ld_regs(u);
          tmem_wait_ld_regs(x);
          if (valid && 16 * c < hd) {
#pragma unroll
            for (int d = 0; d < 16; ++d) dkc[(long)(16 * c + d) * n] = from_f<T>(__uint_as_float(u[d]) * fk);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = pack2(__uint_as_float(x[2 * e]) * fv, __uint_as_float(x[2 * e + 1]) * fv, kBf16);
            reinterpret_cast<uint4*>(dvr + 16 * c)[0] = make_uint4(g[0], g[1], g[2], g[3]);
            reinterpret_cast<uint4*>(dvr + 16 * c)[1] = make_uint4(g[4], g[5], g[6], g[7]);
          }
        }
      }
      tc_fence_before();
    }
    __syncwarp();
    tmem_wait_st();  // (a wait may have run out between a store and its wait)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -------------------------------------------------------------------------------------- preparations
// One launch for both, the first `pad_blocks` blocks for kt. Bound by memory and, small as it is, by its launch: 6 us for
// kt of 400 heads of 14 x 14 x 80 (26 MB, 4.4 TB/s), 3 us for 24 heads.
//
// kt's rows of w elements to rows of wp (a multiple of 8, for the TMA's strides): 16 bytes to a thread, four at a time.
// At most kGroupBytes go out, so 32 bits index them.
template <typename Word>
__device__ __forceinline__ void pad_rows(const uint16_t* __restrict__ src, uint4* __restrict__ dst, unsigned rows, unsigned w,
                                         unsigned wp, unsigned blocks) {
  constexpr int kPer = sizeof(Word) / 2, kWords = 8 / kPer;
  const unsigned per = wp / 8, total = rows * per;
  for (unsigned idx0 = blockIdx.x * 1024u + threadIdx.x; idx0 < total; idx0 += blocks * 1024u) {
    Word x[4][kWords];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned idx = idx0 + 256u * j, r = idx / per, c = (idx - r * per) * 8;
      const Word* at = reinterpret_cast<const Word*>(src + (size_t)r * w + c);
#pragma unroll
      for (int k = 0; k < kWords; ++k) x[j][k] = idx < total && c + kPer * k < w ? __ldg(at + k) : Word(0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        y[k] = kPer == 2 ? (uint32_t)x[j][k]
                         : (uint32_t)x[j][2 * k % kWords] | ((uint32_t)x[j][(2 * k + 1) % kWords] << 16);
      if (idx0 + 256u * j < total) dst[idx0 + 256u * j] = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

// f16: the largest squared row norms of dout and v among a block's rows of a head, to amax[bh][block][2] (ds_factor takes
// the largest of them). A row to 2, 4, 8 or 16 lanes, 16 bytes each.
__device__ __forceinline__ void row_norms(const __half* __restrict__ dout, const __half* __restrict__ v,
                                          float* __restrict__ amax, int n, int hd, int block, int blocks) {
  __shared__ float red[2][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lg = hd <= 16 ? 1 : hd <= 32 ? 2 : hd <= 64 ? 3 : 4;  // lanes to a row, as a power of two
  const int sub = lane & ((1 << lg) - 1), per = 256 >> lg;        // rows in work
  const bool on = sub * 8 < hd;
  float m[2] = {0.f, 0.f};
  for (int r0 = block * per; r0 < n; r0 += 2 * blocks * per) {
    uint4 x[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = r0 + j * blocks * per + (threadIdx.x >> lg);
      const bool ok = on && row < n;
      x[j][0] = ok ? __ldg(reinterpret_cast<const uint4*>(dout + (size_t)row * hd) + sub) : make_uint4(0u, 0u, 0u, 0u);
      x[j][1] = ok ? __ldg(reinterpret_cast<const uint4*>(v + (size_t)row * hd) + sub) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t u[4] = {x[j][k].x, x[j][k].y, x[j][k].z, x[j][k].w};
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2<false>(u[e]);
          s = fmaf(f.x, f.x, s);
          s = fmaf(f.y, f.y, s);
        }
        for (int o = 1; o < 1 << lg; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        // a NaN row makes the bound useless, and the factor 1 (ds_factor): inf stands for it
        m[k] = fmaxf(m[k], s == s ? s : INFINITY);
      }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m[k] = fmaxf(m[k], __shfl_xor_sync(0xffffffffu, m[k], o));
    if (lane == 0) red[k][warp] = m[k];
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    float t = red[threadIdx.x][0];
    for (int k = 1; k < 8; ++k) t = fmaxf(t, red[threadIdx.x][k]);
    amax[2 * block + threadIdx.x] = t;
  }
}

struct PrepArgs {
  const void *kt, *dout, *v;
  void* ktp;
  float* amax;
  unsigned rows;           // of kt
  int w, ktw, n, hd;
  int pad_blocks, norm_blocks;  // norm_blocks to a head
};
__global__ void __launch_bounds__(256) bwd_prepare(PrepArgs p) {
  if ((int)blockIdx.x < p.pad_blocks) {
    const uint16_t* src = static_cast<const uint16_t*>(p.kt);
    if (p.w % 2 == 0)
      pad_rows<uint32_t>(src, static_cast<uint4*>(p.ktp), p.rows, p.w, p.ktw, p.pad_blocks);
    else
      pad_rows<uint16_t>(src, static_cast<uint4*>(p.ktp), p.rows, p.w, p.ktw, p.pad_blocks);
  } else {
    const int at = (int)blockIdx.x - p.pad_blocks, bh = at / p.norm_blocks;
    const size_t head = (size_t)bh * p.n * p.hd;
    row_norms(static_cast<const __half*>(p.dout) + head, static_cast<const __half*>(p.v) + head,
              p.amax + (size_t)bh * 2 * p.norm_blocks, p.n, p.hd, at - bh * p.norm_blocks, p.norm_blocks);
  }
}

}  // namespace bwd
}  // namespace samrs
