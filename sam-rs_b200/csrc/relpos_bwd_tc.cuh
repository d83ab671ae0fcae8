// relpos_bwd_tc.cuh - tcgen05 kernels of the attention's backward pass: f16 / bf16, head_dim a multiple of 16 up to
// 128, grids up to 64 x 64. The mathematics and the reason for walking the scores twice are in relpos_bwd_simt.cuh.
//
// Both kernels recompute a 128 x 64 block of scores at a time. The side that stays (128 queries in bwd_dq_tc, 128 keys
// in bwd_dkv_tc) is the A operand of its products and sits in TMEM; the side that passes by comes through shared
// memory by TMA. A block's S and dP are accumulators in TMEM; sixteen warps turn them into P and dS, a thread per row
// and 16 columns, and write those back as 16-bit pairs over the columns they came from, where they are the A operand
// of the products that follow. So no score, probability or gradient of one touches shared memory, and each operand
// tile that is read from it feeds 128 rows.
//
//   bwd_dq_tc   S = Q K^T, dP = dO V^T, then dQ += dS K.
//               The bias: U = Q table^T once per tile (a product of the tile with the whole table) gives rh and rw by
//               shifted reads, kept in shared memory and written to the workspace for the other kernel.
//               The bias gradients dRh, dRw are sums of dS over grid columns and rows. Grids of 64 columns (W64): a
//               64-key step is one grid row and a thread's 16 columns are the same 16 kw in every step, so that rw and
//               the sums dRw stay in its registers, and a step's sum is its share of dRh. Other grids: dS times a 0/1
//               matrix E [kh | kw][key] gives both, as further columns of the dQ product.
//               Then G[r][t] = dRh[r, i+h-1-t] | dRw[r, j+w-1-t'] (zero where there is no such key) turns both remaining
//               products into plain ones: dQ += G table, dtable += G^T Q.
//   bwd_dkv_tc  S^T = K Q^T, dP^T = V dO^T, then dV += P^T dO, dK += dS^T Q. The 128 keys are a block of the grid (8 x 16
//               where the grid allows): its bias rows are then 8 of rh and 16 of rw instead of the 66 of two grid
//               rows, and they come with every step.
//
// f16: P and dS of long rows fall below f16's normal range. P is kept as 2^12 P in bwd_dkv_tc, and dS times a power of two
// per head that brings the largest possible |dS| near 2^13 (relpos_bwd.cuh); both are taken out again in f32. bf16
// needs neither.
//
// Warps (640 threads): 0 TMA producer, 1 MMA issuer, 2 TMEM allocator, 4-19 the scores. Every wait is bounded
// (sm100::mbar_wait); the scoring warps meet on an mbarrier too, so that a timeout leaves nobody waiting.
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
constexpr int kMaxStages = 6;
constexpr float kPShift = 12.f; // f16: P is kept as 2^12 P

struct TcArgs {
  Args a;
  const unsigned int* amax;  // f16: [bh][2], the largest squared row norms of dout and v, as f32 bits; else null
  float gain;                // f16: what the largest possible |dS| is brought near, else 0
  int nbuf, nstages, stage_bytes;
  // bwd_dq_tc
  int e_rows, halves;        // columns of E (0 in W64 kernels), 128-row halves of the table
  int off_tab, off_q, off_stage, off_bar;
  // bwd_dkv_tc
  int th, tw, tiles_h, tiles_w;
};

struct TcBars {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t s_full[2], ds_full[2];
  uint64_t tab_full, q_full, ops, u_done, rel_done, acc_done, g_done, fin, meet, final_mma;
  uint32_t tmem_base;
  int abort_flag;
};

// The power of two that dS of a head is multiplied by (1 for bf16).
__device__ __forceinline__ float ds_factor(const TcArgs& p, long bh) {
  if (!p.amax) return 1.f;
  const float bound = 2.f * sqrtf(__uint_as_float(p.amax[2 * bh])) * sqrtf(__uint_as_float(p.amax[2 * bh + 1]));
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

// ------------------------------------------------------------------------------------------------ dQ
template <typename T, int HD, bool W64>
__global__ void __launch_bounds__(kTcThreads, 1)
    bwd_dq_tc(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
              const __grid_constant__ CUtensorMap tmE, const __grid_constant__ CUtensorMap tmQ,
              const __grid_constant__ CUtensorMap tmT, const __grid_constant__ TcArgs p) {
  using namespace sm100;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int HC = HD / 16;
  constexpr int kKBytes = HD * 128;  // [HD][64 keys], 128-byte swizzle; E's rows follow
  extern __shared__ uint8_t smem_raw[];
  if (__syncthreads_or(threadIdx.x == 0 && device_faulted())) return;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars* bars = reinterpret_cast<TcBars*>(smem + p.off_bar);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = p.a.h, w = p.a.w, n = h * w, hw = h + w, hd = p.a.hd;
  const int qtiles = (n + 127) / 128, steps = (n + kStep - 1) / kStep, tr = table_rows(h, w);
  const long tiles = p.a.bh * qtiles;
  const int n_tiles = (int)((tiles - blockIdx.x + gridDim.x - 1) / gridDim.x);  // 0 if blockIdx.x >= tiles
  const int E = W64 ? 0 : p.e_rows;
  const int nbuf = p.nbuf, nst = p.nstages;  // nbuf is 1 or 2
  // TMEM columns; U and, at the end, dtable's two halves take over columns that are free then
  const int T_ACC = 0, T_QA = HD + E, T_OA = T_QA + HD / 2, T_S = T_OA + HD / 2;
  const int T_U1 = nbuf == 2 ? T_S + 128 : T_ACC;

  if (threadIdx.x == 0) {
    for (int s = 0; s < nst; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->s_full[b], 1);
      mbar_init(&bars->ds_full[b], kScoreWarps);
    }
    mbar_init(&bars->tab_full, 1);
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->u_done, 1);
    mbar_init(&bars->acc_done, 1);
    mbar_init(&bars->fin, 1);
    mbar_init(&bars->final_mma, 1);
    mbar_init(&bars->ops, kScoreWarps);
    mbar_init(&bars->rel_done, kScoreWarps);
    mbar_init(&bars->g_done, kScoreWarps);
    mbar_init(&bars->meet, kScoreWarps);
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
  const uint32_t tmem = bars->tmem_base;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0 && n_tiles > 0) {
      const int tab_bytes = 128 * HD * 2;
      mbar_arrive_expect_tx(&bars->tab_full, p.halves * tab_bytes);
      for (int b = 0; b < p.halves; ++b)
        tma_load_3d(smem + p.off_tab + b * tab_bytes, &tmT, &bars->tab_full, 0, 128 * b, 0);
      int it = 0, tl = 0;
      bool okk = true;
      for (; tl < n_tiles && okk; ++tl) {
        const long tile = blockIdx.x + (long)tl * gridDim.x;
        const int bh = (int)(tile / qtiles), r0 = (int)(tile - (long)bh * qtiles) * 128;
        // the previous tile's last products have read Q and G (G lies over the stages)
        if (tl > 0 && !mbar_wait_hot(&bars->fin, (tl - 1) & 1, abort_flag)) break;
        mbar_arrive_expect_tx(&bars->q_full, 128 * HD * 2);
        tma_load_4d(smem + p.off_q, &tmQ, &bars->q_full, 0, r0, 0, bh);
        for (int s = 0; s < steps; ++s, ++it) {
          const int st = it % nst;
          if (it >= nst && !mbar_wait_hot(&bars->empty[st], ((it / nst) - 1) & 1, abort_flag)) {
            okk = false;
            break;
          }
          uint8_t* dst = smem + p.off_stage + st * p.stage_bytes;
          mbar_arrive_expect_tx(&bars->full[st], kKBytes + E * 128 + kStep * HD * 2);
          tma_load_3d(dst, &tmK, &bars->full[st], s * kStep, 0, bh);
          if constexpr (!W64) tma_load_3d(dst + kKBytes, &tmE, &bars->full[st], s * kStep, 0, 0);
          tma_load_4d(dst + kKBytes + E * 128, &tmV, &bars->full[st], 0, s * kStep, 0, bh);
        }
      }
      if (*abort_flag) {
        // drain the copies in flight before the CTA can exit
        mbar_drain(&bars->tab_full, 0);
        if (tl > 0 || it > 0) mbar_drain(&bars->q_full, (tl < n_tiles ? tl : n_tiles - 1) & 1);
        for (int j = it > nst ? it - nst : 0; j < it; ++j) mbar_drain(&bars->full[j % nst], (j / nst) & 1);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t idS = idesc_f16(kBf16, 128, kStep, false, true);    // S = Q K^T, K MN-major
    constexpr uint32_t idP = idesc_f16(kBf16, 128, kStep, false, false);   // dP = dO V^T
    constexpr uint32_t idU = idesc_f16(kBf16, 128, 128, false, false);     // U = Q table^T
    constexpr uint32_t idG = idesc_f16(kBf16, 128, HD, false, true);       // dQ += G table
    constexpr uint32_t idT = idesc_f16(kBf16, 128, HD, true, true);        // dtable = G^T Q
    const uint32_t idQ = idesc_f16(kBf16, 128, HD + E, false, false);      // dQ | dR += dS [K | E]
    const uint32_t sb = smem_u32(smem);
    const uint64_t dK = smem_desc(sb + p.off_stage, kKBytes, 1024, kLayoutSw128);
    const uint64_t dKE = smem_desc(sb + p.off_stage, 16, 1024, kLayoutSw128);
    const uint64_t dV = smem_desc(sb + p.off_stage + kKBytes + E * 128, 16, 256, kLayoutSw32);
    const uint64_t dTabK = smem_desc(sb + p.off_tab, 16, 256, kLayoutSw32);
    const uint64_t dTabN = smem_desc(sb + p.off_tab, 4096, 256, kLayoutSw32);
    const uint64_t dQn = smem_desc(sb + p.off_q, 4096, 256, kLayoutSw32);
    const uint64_t dGk = smem_desc(sb + p.off_stage, 16, 1024, kLayoutSw128);
    const uint64_t dGm = smem_desc(sb + p.off_stage, 16384, 1024, kLayoutSw128);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_hot(bar, parity, abort_flag)); };
    bool okk = true;
    int is = 0, id = 0;    // steps whose S and dP, and whose dQ, have been issued,
    int sst = 0, dst = 0;  // their stages,
    uint32_t sph = 0;      // and the phase of the former's barrier
    auto issue_s = [&]() {
      const int b = is & (nbuf - 1);
      if (!(okk = wait(&bars->full[sst], sph))) return;
      tc_fence_after();
      const uint32_t tS = tmem + T_S + 128 * b;
      const uint64_t kd = desc_add(dK, sst * p.stage_bytes), vd = desc_add(dV, sst * p.stage_bytes);
#pragma unroll
      for (int c = 0; c < HC; ++c) mma_ts_w(tS, tmem + T_QA + 8 * c, desc_add(kd, c * 2048), idS, c > 0);
#pragma unroll
      for (int c = 0; c < HC; ++c) mma_ts_w(tS + 64, tmem + T_OA + 8 * c, desc_add(vd, c * 2048), idP, c > 0);
      mma_commit_w(&bars->s_full[b]);
      ++is;
      if (++sst == nst) sst = 0, sph ^= 1;
    };
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
      tc_fence_after();
      for (int s = 0; s < nbuf && s < steps && okk; ++s) issue_s();
      for (int s = 0; s < steps && okk; ++s, ++id) {
        const int b = id & (nbuf - 1);
        if (!(okk = wait(&bars->ds_full[b], (id >> (nbuf - 1)) & 1))) break;
        tc_fence_after();
        const uint64_t kd = desc_add(dKE, dst * p.stage_bytes);
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          mma_ts_w(tmem + T_ACC, tmem + T_S + 128 * b + 16 * k, desc_add(kd, 32 * k), idQ, (s > 0 || k > 0) ? 1u : 0u);
        mma_commit_w(&bars->empty[dst]);
        if (++dst == nst) dst = 0;
        if (s + nbuf < steps) issue_s();
      }
      if (!okk) break;
      mma_commit_w(&bars->acc_done);
      okk = wait(&bars->g_done, tp) && wait(&bars->q_full, tp);
      if (!okk) break;
      tc_fence_after();
      for (int k = 0; k < 8 * p.halves; ++k)  // 16 table rows each
        mma_ss_w(tmem + T_ACC, desc_add(dGk, (k >> 2) * 16384 + 32 * (k & 3)),
                 desc_add(dTabN, (k >> 3) * 128 * HD * 2 + 512 * (k & 7)), idG, 1u);
      for (int b = 0; b < p.halves; ++b)
#pragma unroll
        for (int k = 0; k < 8; ++k)  // 16 query rows each
          mma_ss_w(tmem + (b ? T_QA : T_S), desc_add(dGm, b * 32768 + 2048 * k), desc_add(dQn, 512 * k), idT, k > 0);
      mma_commit_w(&bars->fin);
    }
    // every MMA issued by this warp has completed before the CTA tears down TMEM
    mma_commit_w(&bars->final_mma);
    mbar_drain(&bars->final_mma, 0);
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- scores
    const int cg = (warp - 4) >> 2, wq = warp & 3;
    const int r = 32 * wq + lane;  // TMEM lane = query row of the tile
    const uint32_t tl0 = tmem + ((uint32_t)(32 * wq) << 16);
    float* rel = reinterpret_cast<float*>(smem);  // [h + w][128], later dR
    float* dpart = rel;                           // [4][128], before rel is written
    float* ring = rel + (size_t)h * 128;          // W64: [4 steps][4 column groups][128], over rw once it is in registers
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
    int gs = 0;
    int first = p.a.first;
    float* part = p.a.partial + (long)blockIdx.x * tr * hd;
    for (int tl = 0; tl < n_tiles && okk; ++tl) {
      const uint32_t tp = tl & 1;
      const long tile = blockIdx.x + (long)tl * gridDim.x;
      const long bh = tile / qtiles;
      const int r0 = (int)(tile - bh * qtiles) * 128, row = r0 + r;
      const bool valid = row < n;
      const int i = row / w, j = row - i * w;
      const float fac2 = ds_factor(p, bh);             // dS is kept as dS fac2,
      const float fac = kBf16 ? fac2 : fac2 * exp2f(-kPShift);  // P as P 2^shift: dS fac2 = (P 2^shift) (dP - D) fac
      // Q and dO rows to TMEM, D from dO and O
      {
        const long off = (bh * n + (valid ? row : 0)) * hd;
        const T* qr = static_cast<const T*>(p.a.q) + off;
        const T* dr = static_cast<const T*>(p.a.dout) + off;
        const T* orow = static_cast<const T*>(p.a.out) + off;
        float d = 0.f;
        for (int c = cg; c < HC; c += 4) {
          const bool ok = valid && 16 * c < hd;
          uint32_t a[8], g[8], o[8];
          load_row16(qr + 16 * c, ok, a);
          load_row16(dr + 16 * c, ok, g);
          load_row16(orow + 16 * c, ok, o);
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
      if (!meet()) break;
      const float lse2 = valid ? p.a.lse[bh * n + row] * kLog2e : 0.f;
      const float dsum = ((dpart[r] + dpart[128 + r]) + (dpart[256 + r] + dpart[384 + r])) * fac;
      if (cg == 0) p.a.dsum[bh * p.a.np + row] = -dsum;
      if (!meet()) break;  // dpart has been read
      if (!wait(&bars->u_done, tp)) break;
      tc_fence_after();
      {
        const float top = (kBf16 ? 0.f : kPShift) - lse2;
        for (int c = cg; c < 8 * p.halves; c += 4) {
          uint32_t u[16];
          tmem_ld16(tl0 + (c < 8 ? T_S + 16 * c : T_U1 + 16 * (c - 8)), u);
          tmem_wait_ld_regs(u);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int t = 16 * c + e;
            const float x = __uint_as_float(u[e]) * kLog2e;
            if (t < 2 * h - 1) {
              const int kh = i + h - 1 - t;
              if ((unsigned)kh < (unsigned)h) rel[kh * 128 + r] = x + top;
            } else if (t < tr) {
              const int kw = j + w - 1 - (t - (2 * h - 1));
              if ((unsigned)kw < (unsigned)w) rel[(h + kw) * 128 + r] = x;
            }
          }
        }
        if (!valid) {  // (i >= h: no kh was in range) such rows have P = 0 everywhere
          for (int c = cg; c < hw; c += 4) {
            rel[c * 128 + r] = c < h ? -INFINITY : 0.f;
          }
        }
      }
      tc_fence_before();
      arrive(&bars->rel_done);  // U has been read
      if (!meet()) break;       // all of rel is written
      {
        float* out = p.a.rel + bh * hw * p.a.np + r0;
        for (int c = warp - 4; c < hw; c += kScoreWarps)
          reinterpret_cast<float4*>(out + (long)c * p.a.np)[lane] = reinterpret_cast<const float4*>(rel + c * 128)[lane];
      }
      float2 rw[8], dw[8];
      if constexpr (W64) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          rw[e] = make_float2(rel[(h + 16 * cg + 2 * e) * 128 + r], rel[(h + 16 * cg + 2 * e + 1) * 128 + r]);
          dw[e] = make_float2(0.f, 0.f);
        }
        if (!meet()) break;  // the ring may be written
      }
      const float2 f2 = make_float2(fac, fac), nd2 = make_float2(-dsum, -dsum);
      for (int s = 0; s < steps; ++s, ++gs) {
        const int b = gs & (nbuf - 1);
        const uint32_t tS = tl0 + T_S + 128 * b + 16 * cg;
        if (!wait(&bars->s_full[b], (gs >> (nbuf - 1)) & 1)) break;
        tc_fence_after();
        uint32_t sv[16], dv[16], pk[8];
        tmem_ld16(tS, sv);
        tmem_ld16(tS + 64, dv);
        float2 x[8];
        if constexpr (W64) {
          const float rh = rel[s * 128 + r];
          const float2 rh2 = make_float2(rh, rh);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = add2(rw[e], rh2);
          // the four column groups' sums of step s - nbuf, once all of them are in
          if (s >= nbuf && cg == (s & 3)) {
            if (!wait(&bars->ds_full[b], ((gs - nbuf) >> (nbuf - 1)) & 1)) break;
            const float* q4 = ring + ((gs - nbuf) & 3) * 512 + r;
            rel[(s - nbuf) * 128 + r] = (q4[0] + q4[128]) + (q4[256] + q4[384]);
          }
        } else {
          const int k0 = s * kStep + 16 * cg;
          int kh = k0 / w, kw = k0 - kh * w;
          float rh = kh < h ? rel[kh * 128 + r] : -INFINITY;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float v = kh < h ? rel[(h + kw) * 128 + r] + rh : -INFINITY;
            if (e & 1)
              x[e >> 1].y = v;
            else
              x[e >> 1].x = v;
            if (++kw == w) {
              kw = 0;
              ++kh;
              if (kh < h) rh = rel[kh * 128 + r];
            }
          }
        }
        tmem_wait_ld_regs(sv);
        tmem_wait_ld_regs(dv);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float2 y = fma2(make_float2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), c2, x[e]);
          y = make_float2(ex2(y.x), ex2(y.y));
          const float2 g = fma2(make_float2(__uint_as_float(dv[2 * e]), __uint_as_float(dv[2 * e + 1])), f2, nd2);
          y = mul2(y, g);
          pk[e] = pack2(y.x, y.y, kBf16);
          if constexpr (W64) {
            dw[e] = add2(dw[e], y);
            sum = add2(sum, y);
          }
        }
        tmem_st8(tS, pk);
        if constexpr (W64) ring[(gs & 3) * 512 + cg * 128 + r] = sum.x + sum.y;
        tmem_wait_st();
        tc_fence_before();
        arrive(&bars->ds_full[b]);
      }
      if (!okk || !wait(&bars->acc_done, tp)) break;
      tc_fence_after();
      // dRh and dRw to shared memory, [h + w][128]
      if constexpr (W64) {
        for (int s = steps > nbuf ? steps - nbuf : 0; s < steps; ++s) {
          const int g = gs - steps + s;
          if (!wait(&bars->ds_full[g & (nbuf - 1)], (g >> (nbuf - 1)) & 1)) break;
          if (cg == (s & 3)) {
            const float* q4 = ring + (g & 3) * 512 + r;
            rel[s * 128 + r] = (q4[0] + q4[128]) + (q4[256] + q4[384]);
          }
        }
        if (!meet()) break;  // the ring has been read
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          rel[(h + 16 * cg + 2 * e) * 128 + r] = dw[e].x;
          rel[(h + 16 * cg + 2 * e + 1) * 128 + r] = dw[e].y;
        }
      } else {
        for (int c = cg; c < E / 16; c += 4) {
          uint32_t u[16];
          tmem_ld16(tl0 + T_ACC + HD + 16 * c, u);
          tmem_wait_ld_regs(u);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (16 * c + e < hw) rel[(16 * c + e) * 128 + r] = __uint_as_float(u[e]);
        }
      }
      if (!meet()) break;
      // G (16-bit, 128-byte swizzle, 64 table rows per atom), over the stages: their products have completed. G takes
      // 1 / scale along, so that dQ and dtable are scaled once at the end.
      {
        const float inv = 1.f / p.a.scale;
        uint8_t* G = smem + p.off_stage;
        for (int v = cg; v < 16 * p.halves; v += 4) {
          uint32_t g[4];
#pragma unroll
          for (int e2 = 0; e2 < 4; ++e2) {
            float f[2];
#pragma unroll
            for (int e1 = 0; e1 < 2; ++e1) {
              const int t = 8 * v + 2 * e2 + e1;
              f[e1] = 0.f;
              if (t < 2 * h - 1) {
                const int kh = i + h - 1 - t;
                if ((unsigned)kh < (unsigned)h) f[e1] = rel[kh * 128 + r] * inv;
              } else if (t < tr) {
                const int kw = j + w - 1 - (t - (2 * h - 1));
                if ((unsigned)kw < (unsigned)w) f[e1] = rel[(h + kw) * 128 + r] * inv;
              }
            }
            g[e2] = pack2(f[0], f[1], kBf16);
          }
          *reinterpret_cast<uint4*>(G + (v >> 3) * 16384 + r * 128 + (((v & 7) ^ (r & 7)) << 4)) =
              make_uint4(g[0], g[1], g[2], g[3]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        arrive(&bars->g_done);
      }
      if (!wait(&bars->fin, tp)) break;
      tc_fence_after();
      const float outf = p.a.scale / fac2;
      T* dqr = static_cast<T*>(p.a.dq) + (bh * n + (valid ? row : 0)) * hd;
      for (int c = cg; c < HC; c += 4) {
        uint32_t u[16], g[8];
        tmem_ld16(tl0 + T_ACC + 16 * c, u);
        tmem_wait_ld_regs(u);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = pack2(__uint_as_float(u[2 * e]) * outf, __uint_as_float(u[2 * e + 1]) * outf, kBf16);
        if (valid && 16 * c < hd) {
          reinterpret_cast<uint4*>(dqr + 16 * c)[0] = make_uint4(g[0], g[1], g[2], g[3]);
          reinterpret_cast<uint4*>(dqr + 16 * c)[1] = make_uint4(g[4], g[5], g[6], g[7]);
        }
      }
      for (int b = 0; b < p.halves; ++b) {
        const int t = 128 * b + r;
        for (int c = cg; c < HC; c += 4) {
          uint32_t u[16];
          tmem_ld16(tl0 + (b ? T_QA : T_S) + 16 * c, u);
          tmem_wait_ld_regs(u);
          if (t < tr && 16 * c < hd) {
            float4* dst = reinterpret_cast<float4*>(part + (long)t * hd + 16 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float4 x = make_float4(__uint_as_float(u[4 * e]) * outf, __uint_as_float(u[4 * e + 1]) * outf,
                                     __uint_as_float(u[4 * e + 2]) * outf, __uint_as_float(u[4 * e + 3]) * outf);
              if (!first) {
                const float4 y = dst[e];
                x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
              }
              dst[e] = x;
            }
          }
        }
      }
      tc_fence_before();
      first = 0;
      if (!meet()) break;  // every warp has read its columns before the next tile's operands go over them
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// --------------------------------------------------------------------------------------------- dK, dV
// Shared memory of a stage: Q and dO [HD / 16][64][32 B], twice the bias rows of 32 queries (rh rows, then rw rows, 128 B
// each, both blocks rounded to the swizzle's 8 rows), D [64].
__host__ __device__ constexpr int round8(int x) { return (x + 7) / 8 * 8; }
__host__ __device__ constexpr int dkv_stage_bytes(int hd, int th, int tw) {
  return 2 * kStep * hd * 2 + 2 * (round8(th) + round8(tw)) * 128 + 1024;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    bwd_dkv_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmO,
               const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW,
               const __grid_constant__ TcArgs p) {
  using namespace sm100;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int HC = HD / 16, kTile = kStep * HD * 2;
  constexpr int T_DK = 0, T_DV = HD, T_KA = 2 * HD, T_VA = T_KA + HD / 2, T_S = 3 * HD;
  constexpr int nbuf = T_S + 256 <= 512 ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  if (__syncthreads_or(threadIdx.x == 0 && device_faulted())) return;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars* bars = reinterpret_cast<TcBars*>(smem + p.off_bar);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = p.a.h, w = p.a.w, n = h * w, hd = p.a.hd;
  const int steps = (n + kStep - 1) / kStep, nst = p.nstages;
  const int per_head = p.tiles_h * p.tiles_w;
  const int bh = blockIdx.x / per_head, kt = blockIdx.x - bh * per_head;
  const int kh0 = (kt / p.tiles_w) * p.th, kw0 = (kt % p.tiles_w) * p.tw;
  const int off_rel = 2 * kTile, rel_bytes = (round8(p.th) + round8(p.tw)) * 128, off_d = off_rel + 2 * rel_bytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < nst; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->s_full[b], 1);
      mbar_init(&bars->ds_full[b], kScoreWarps);
    }
    mbar_init(&bars->ops, kScoreWarps);
    mbar_init(&bars->acc_done, 1);
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
  const uint32_t tmem = bars->tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (; it < steps; ++it) {
        const int st = it % nst;
        if (it >= nst && !mbar_wait_hot(&bars->empty[st], ((it / nst) - 1) & 1, abort_flag)) break;
        uint8_t* dst = smem + st * p.stage_bytes;
        mbar_arrive_expect_tx(&bars->full[st], 2 * kTile + 2 * (p.th + p.tw) * 128 + kStep * 4);
        tma_load_4d(dst, &tmQ, &bars->full[st], 0, it * kStep, 0, bh);
        tma_load_4d(dst + kTile, &tmO, &bars->full[st], 0, it * kStep, 0, bh);
        for (int b = 0; b < 2; ++b) {
          tma_load_3d(dst + off_rel + b * rel_bytes, &tmH, &bars->full[st], it * kStep + 32 * b, kh0, bh);
          tma_load_3d(dst + off_rel + b * rel_bytes + round8(p.th) * 128, &tmW, &bars->full[st], it * kStep + 32 * b, h + kw0, bh);
        }
        bulk_load(dst + off_d, p.a.dsum + (long)bh * p.a.np + it * kStep, kStep * 4, &bars->full[st]);
      }
      if (*abort_flag)
        for (int j = it > nst ? it - nst : 0; j < it; ++j) mbar_drain(&bars->full[j % nst], (j / nst) & 1);
    }
  } else if (warp == 1) {
    constexpr uint32_t idS = idesc_f16(kBf16, 128, kStep, false, false);  // S^T = K Q^T, dP^T = V dO^T
    constexpr uint32_t idA = idesc_f16(kBf16, 128, HD, false, true);      // dV += P^T dO, dK += dS^T Q
    const uint32_t sb = smem_u32(smem);
    const uint64_t dQk = smem_desc(sb, 16, 256, kLayoutSw32), dOk = smem_desc(sb + kTile, 16, 256, kLayoutSw32);
    const uint64_t dQn = smem_desc(sb, 2048, 256, kLayoutSw32), dOn = smem_desc(sb + kTile, 2048, 256, kLayoutSw32);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_hot(bar, parity, abort_flag)); };
    bool okk = wait(&bars->ops, 0);
    tc_fence_after();
    int is = 0, sst = 0, dst = 0;
    uint32_t sph = 0;
    auto issue_s = [&]() {
      const int b = is % nbuf;
      if (!(okk = wait(&bars->full[sst], sph))) return;
      tc_fence_after();
      const uint32_t tS = tmem + T_S + 128 * b;
      const uint64_t qd = desc_add(dQk, sst * p.stage_bytes), od = desc_add(dOk, sst * p.stage_bytes);
#pragma unroll
      for (int c = 0; c < HC; ++c) mma_ts_w(tS, tmem + T_KA + 8 * c, desc_add(qd, c * 2048), idS, c > 0);
#pragma unroll
      for (int c = 0; c < HC; ++c) mma_ts_w(tS + 64, tmem + T_VA + 8 * c, desc_add(od, c * 2048), idS, c > 0);
      mma_commit_w(&bars->s_full[b]);
      ++is;
      if (++sst == nst) sst = 0, sph ^= 1;
    };
    for (int s = 0; s < nbuf && s < steps && okk; ++s) issue_s();
    for (int s = 0; s < steps && okk; ++s) {
      const int b = s % nbuf;
      if (!(okk = wait(&bars->ds_full[b], (s / nbuf) & 1))) break;
      tc_fence_after();
      const uint64_t qd = desc_add(dQn, dst * p.stage_bytes), od = desc_add(dOn, dst * p.stage_bytes);
#pragma unroll
      for (int k = 0; k < kStep / 16; ++k)
        mma_ts_w(tmem + T_DV, tmem + T_S + 128 * b + 16 * k, desc_add(od, 512 * k), idA, (s > 0 || k > 0) ? 1u : 0u);
#pragma unroll
      for (int k = 0; k < kStep / 16; ++k)
        mma_ts_w(tmem + T_DK, tmem + T_S + 128 * b + 64 + 16 * k, desc_add(qd, 512 * k), idA, (s > 0 || k > 0) ? 1u : 0u);
      mma_commit_w(&bars->empty[dst]);
      if (++dst == nst) dst = 0;
      if (s + nbuf < steps) issue_s();
    }
    mma_commit_w(&bars->acc_done);
    mbar_drain(&bars->acc_done, 0);
  } else if (warp >= 4) {
    const int cg = (warp - 4) >> 2, wq = warp & 3;
    const int r = 32 * wq + lane;  // TMEM lane = key of the tile
    const int dh = r / p.tw, dw = r - dh * p.tw;
    const int kh = kh0 + dh, kw = kw0 + dw;
    const bool valid = kh < h && kw < w;
    const int key = valid ? kh * w + kw : 0;
    const uint32_t tl0 = tmem + ((uint32_t)(32 * wq) << 16);
    const float c_log2 = p.a.scale * kLog2e;
    const float2 c2 = make_float2(c_log2, c_log2);
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
    const int rho_h = dh, rho_w = round8(p.th) + dw;  // this thread's rows of the bias
    const uint8_t* base = smem + off_rel + (cg >> 1) * rel_bytes;
    bool okk = true;
    int st = 0;
    uint32_t ph = 0;
    for (int s = 0; s < steps; ++s) {
      const int b = s % nbuf;
      const uint32_t tS = tl0 + T_S + 128 * b + 16 * cg;
      // the stage's bias rows and D (the S products waited for the same copies)
      okk = __all_sync(0xffffffffu, mbar_wait_hot(&bars->full[st], ph, abort_flag) &&
                                        mbar_wait_hot(&bars->s_full[b], (s / nbuf) & 1, abort_flag));
      if (!okk) break;
      tc_fence_after();
      uint32_t sv[16], dv[16], pp[8], pd[8];
      tmem_ld16(tS, sv);
      tmem_ld16(tS + 64, dv);
      const uint8_t* sp = base + st * p.stage_bytes;
      const float* ds = reinterpret_cast<const float*>(smem + st * p.stage_bytes + off_d) + 16 * cg;
      float4 bias[4], dd[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int ch = 4 * (cg & 1) + c;
        const float4 a = *reinterpret_cast<const float4*>(sp + rho_h * 128 + ((ch ^ (rho_h & 7)) << 4));
        const float4 g = *reinterpret_cast<const float4*>(sp + rho_w * 128 + ((ch ^ (rho_w & 7)) << 4));
        const float2 lo = add2(make_float2(a.x, a.y), make_float2(g.x, g.y));
        const float2 hi = add2(make_float2(a.z, a.w), make_float2(g.z, g.w));
        bias[c] = make_float4(lo.x, lo.y, hi.x, hi.y);
        dd[c] = *reinterpret_cast<const float4*>(ds + 4 * c);
      }
      tmem_wait_ld_regs(sv);
      tmem_wait_ld_regs(dv);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float4 bb = bias[e >> 1], d4 = dd[e >> 1];
        const float2 x = e & 1 ? make_float2(bb.z, bb.w) : make_float2(bb.x, bb.y);
        const float2 nd = e & 1 ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y);  // -D
        float2 y = fma2(make_float2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), c2, x);
        y = make_float2(ex2(y.x), ex2(y.y));
        const float2 g = fma2(make_float2(__uint_as_float(dv[2 * e]), __uint_as_float(dv[2 * e + 1])), f2, nd);
        pp[e] = pack2(y.x, y.y, kBf16);
        y = mul2(y, g);
        pd[e] = pack2(y.x, y.y, kBf16);
      }
      tmem_st8(tS, pp);
      tmem_st8(tS + 64, pd);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->ds_full[b]);
      if (++st == nst) st = 0, ph ^= 1;
    }
    okk = okk && __all_sync(0xffffffffu, mbar_wait_hot(&bars->acc_done, 0, abort_flag));
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
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -------------------------------------------------------------------------------------- preparations
// E [rows][cols]: 1 where key `col` of the grid has kh = row, or kw = row - h.
__global__ void bwd_indicator(uint16_t* __restrict__ e, int rows, int cols, int h, int w, uint16_t one) {
  for (int idx = blockIdx.x * blockDim.x + threadIdx.x; idx < rows * cols; idx += gridDim.x * blockDim.x) {
    const int c = idx / cols, k = idx - c * cols;
    const int kh = k / w, kw = k - kh * w;
    e[idx] = kh < h && (c < h ? kh == c : kw == c - h) ? one : (uint16_t)0;
  }
}

// kt rows of n elements to rows of np (a multiple of 8, for the TMA's strides).
__global__ void bwd_pad_rows(const uint16_t* __restrict__ src, uint16_t* __restrict__ dst, long rows, int n, int np) {
  const long total = rows * np;
  for (long idx = blockIdx.x * (long)blockDim.x + threadIdx.x; idx < total; idx += (long)gridDim.x * blockDim.x) {
    const long r = idx / np;
    const int c = (int)(idx - r * np);
    dst[idx] = c < n ? src[r * n + c] : (uint16_t)0;
  }
}

// f16: the largest squared row norms of dout and v per head (a maximum does not depend on the order).
__global__ void __launch_bounds__(256) bwd_row_norms(const __half* __restrict__ dout, const __half* __restrict__ v,
                                                    unsigned int* __restrict__ amax, int n, int hd) {
  const long bh = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m[2] = {0.f, 0.f};
  for (int row = blockIdx.y * 8 + warp; row < n; row += gridDim.y * 8) {
    float s[2] = {0.f, 0.f};
    for (int d = lane; d < hd; d += 32) {
      const float a = to_f(dout[(bh * n + row) * hd + d]), b = to_f(v[(bh * n + row) * hd + d]);
      s[0] = fmaf(a, a, s[0]);
      s[1] = fmaf(b, b, s[1]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
      // a NaN row makes the bound useless, and the factor 1 (ds_factor): inf stands for it
      m[k] = fmaxf(m[k], s[k] == s[k] ? s[k] : INFINITY);
    }
  }
  if (lane == 0) {
    atomicMax(&amax[2 * bh], __float_as_uint(m[0]));
    atomicMax(&amax[2 * bh + 1], __float_as_uint(m[1]));
  }
}

}  // namespace bwd
}  // namespace samrs
