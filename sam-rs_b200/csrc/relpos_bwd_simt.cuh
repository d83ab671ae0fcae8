// relpos_bwd_simt.cuh - CUDA-core backward pass of the rel-pos attention, any (h, w, hd <= 128), any dtype:
// the f32 path, and the path of 16-bit shapes the tensor-core kernels (relpos_bwd_tc.cuh) do not cover.
//
// Math, with r = (i, j) a query, k = (kh, kw) a key and lse_r the forward pass's log of the softmax sum:
//   x[r,k] = scale q_r.k_k + rh[r,kh] + rw[r,kw],  rh[r,kh] = q_r.Th[i-kh+h-1],  rw[r,kw] = q_r.Tw[j-kw+w-1]
//   P = e^(x - lse),  D_r = dO_r.O_r,  dS = P (dO V^T - D)
//   dV = P^T dO,  dK = scale dS^T Q,  dRh[r,kh] = sum_kw dS,  dRw[r,kw] = sum_kh dS
//   dQ_r = scale dS_r K + sum_kh dRh[r,kh] Th[i-kh+h-1] + sum_kw dRw[r,kw] Tw[j-kw+w-1]
//   dTh[t] = sum over (r, kh) with i-kh+h-1 = t of dRh[r,kh] q_r, and dTw alike.
// No N x N tensor is stored: the probabilities are recomputed from lse, once by query tiles (dQ, the bias
// gradients) and once by key tiles (dK, dV). The second walk costs two of the seven products, and saves
// adding dQ over the key tiles in memory, whose order would change results.
//
// Launch 1 (bwd_dq_simt) walks query tiles, leaves in the workspace what launch 2 reads per query - the bias
// rows rel (log2 units, lse already subtracted from the rh rows) and D - and one partial sum of dtable per
// CTA; launch 2 (bwd_dkv_simt) walks key tiles; launch 3 (bwd_table_reduce) adds the partial sums in CTA
// order. All arithmetic is f32 (exp2f of log2-scaled logits), rounded once to the I/O dtype.
#pragma once
#include "common.cuh"
#include "relpos_simt.cuh"
#include "sm100.cuh"

namespace samrs {
namespace bwd {

// Rows of the side that stays (queries in bwd_dq_simt, keys in bwd_dkv_simt), and of the one that passes, per step of a
// group of 4 warps. A CTA has 1, 2 or 4 groups, which share the side that stays and take the steps in turn.
constexpr int kBR = 32, kGroup = 128, kKeys = 64, kQueries = 32;
// Floats between the rows of tiles 32 and 64 wide: 16-byte reads, and 8 rows hit 32 banks.
constexpr int kS32 = 36, kS64 = 68;
constexpr float kLog2e = 1.4426950408889634f;

// Queries are padded to a multiple of 128 in the workspace arrays (the tensor-core tiles).
__host__ __device__ inline int padded_rows(int n) { return (n + 127) / 128 * 128; }
__host__ __device__ inline int table_rows(int h, int w) { return 2 * h - 1 + 2 * w - 1; }

// What the launches of one call share. rel: [bh][h + w][np], dsum: [bh][np], partial: [ctas][table_rows][hd].
struct Args {
  const void *q, *kt, *v, *table, *out, *dout;
  const float* lse;
  void *dq, *dkt, *dv, *dtable;
  float *rel, *dsum, *partial;
  long bh;      // heads of this launch (q, kt, ... already point at the first)
  int first;    // the CTA's partial sums start here (0: they continue those of an earlier launch)
  int h, w, hd, np;
  float scale;
};

// Dynamic shared memory of the two kernels, in floats, with `g` groups. (Tiles have a multiple of 16 rows of the head:
// mul_tile reads them.)
__host__ __device__ inline int64_t dq_smem_floats(int g, int h, int w, int hd) {
  const int64_t hp = (hd + 15) / 16 * 16;
  return 2 * hp * kS32 + (1 + g) * (int64_t)kBR * (h + w) + kBR + g * (hp * kS64 + (int64_t)kBR * kS64);
}
__host__ __device__ inline int64_t dkv_smem_floats(int g, int hd) {
  const int64_t hp = (hd + 15) / 16 * 16;
  return 2 * hp * kS32 + g * (2 * hp * kS32 + (int64_t)2 * kBR * kS32);
}

// A barrier of this thread's group.
__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory"); }

// By one group: rows r0 .. r0 + ROWS - 1 of src [n][hd], transposed into dst[d][r] (row stride `stride`); rows past n are 0. A warp takes
// 4 rows x 8 columns at a time (whole sectors of f32; the stores hit 32 banks), a batch of loads in flight.
template <typename T, int ROWS>
__device__ __forceinline__ void load_transposed(float* dst, int stride, const T* src, int r0, int n, int hd) {
  constexpr int kWarps = kGroup / 32, kGroups = ROWS / 4, B = kGroups / kWarps, DB = B < 8 ? 16 / B : 2;
  static_assert(kGroups % kWarps == 0, "whole batches");
  const int lane = threadIdx.x & 31, warp = (threadIdx.x % kGroup) >> 5, r = 4 * warp + (lane >> 3);
  for (int d0 = lane & 7; d0 < hd; d0 += 8 * DB) {
    float v[DB][B];
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int k = 0; k < B; ++k) {
        const int row = r0 + r + 4 * kWarps * k, d = d0 + 8 * e;
        v[e][k] = row < n && d < hd ? to_f(src[(long)row * hd + d]) : 0.f;
      }
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int k = 0; k < B; ++k)
        if (d0 + 8 * e < hd) dst[(d0 + 8 * e) * stride + r + 4 * kWarps * k] = v[e][k];
  }
}
// By one group: columns k0 .. k0 + COLS - 1 of src [hd][n] into dst[d][k]; columns past n are 0.
template <typename T, int COLS>
__device__ __forceinline__ void load_columns(float* dst, int stride, const T* src, int k0, int n, int hd) {
  const int k = threadIdx.x % COLS;
  constexpr int kRows = kGroup / COLS, B = 8;
  for (int d0 = threadIdx.x % kGroup / COLS; d0 < hd; d0 += kRows * B) {
    float v[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int d = d0 + kRows * j;
      v[j] = d < hd && k0 + k < n ? to_f(src[(long)d * n + k0 + k]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (d0 + kRows * j < hd) dst[(d0 + kRows * j) * stride + k] = v[j];
  }
}

// out[a][b] = sum_d A[d][ra + a] B[d][cb + b], for 4 rows and NB columns; A has rows of kS32 floats, B of SB
template <int NB, int SB>
__device__ __forceinline__ void dot_tile(float (&out)[4][NB], const float* A, int ra, const float* B, int cb, int hd) {
  float2 acc[4][NB / 2];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < NB / 2; ++b) acc[a][b] = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int d = 0; d < hd; ++d) {
    const float4 av = *reinterpret_cast<const float4*>(&A[d * kS32 + ra]);
    const float m[4] = {av.x, av.y, av.z, av.w};
    float2 bv[NB / 2];
    if constexpr (NB == 4) {
      const float4 t = *reinterpret_cast<const float4*>(&B[d * SB + cb]);
      bv[0] = make_float2(t.x, t.y);
      bv[1] = make_float2(t.z, t.w);
    } else {
      bv[0] = *reinterpret_cast<const float2*>(&B[d * SB + cb]);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < NB / 2; ++b) acc[a][b] = sm100::fma2(make_float2(m[a], m[a]), bv[b], acc[a][b]);
  }
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < NB / 2; ++b) {
      out[a][2 * b] = acc[a][b].x;
      out[a][2 * b + 1] = acc[a][b].y;
    }
}

// acc[a][c] += sum over the X columns x of M[ra + a][x] B[tx + 16c][x], for c < nc; rows of S floats
template <int X, int S>
__device__ __forceinline__ void mul_tile(float (&acc)[4][8], const float* M, int ra, const float* B, int tx, int nc) {
#pragma unroll 2
  for (int x = 0; x < X; x += 4) {
    float4 m[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) m[a] = *reinterpret_cast<const float4*>(&M[(ra + a) * S + x]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (c < nc) {
        const float4 b = *reinterpret_cast<const float4*>(&B[(tx + 16 * c) * S + x]);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          acc[a][c] = fmaf(m[a].x, b.x, acc[a][c]);
          acc[a][c] = fmaf(m[a].y, b.y, acc[a][c]);
          acc[a][c] = fmaf(m[a].z, b.z, acc[a][c]);
          acc[a][c] = fmaf(m[a].w, b.w, acc[a][c]);
        }
      }
    }
  }
}

// The groups' 4 x 8 sums to a thread, by way of shared memory (each group's own `mine`, kGroup x 4 nc floats): the thread
// keeps the total of rows a with a / (4 / G) == group, added in the groups' order. `stride`: floats from one group's `mine`
// to the next one's.
template <int G>
__device__ __forceinline__ void join_groups(float (&acc)[4][8], float* mine, int stride, int group, int nc) {
  if constexpr (G > 1) {
    const int t = threadIdx.x % kGroup;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < nc) mine[(a * nc + c) * kGroup + t] = acc[a][c];
    __syncthreads();
    const float* all = mine - (long)group * stride;
#pragma unroll
    for (int a = 0; a < 4; ++a)
      if (a / (4 / G) == group)
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c < nc) {
            float v = all[(a * nc + c) * kGroup + t];
            for (int q = 1; q < G; ++q) v += all[q * stride + (a * nc + c) * kGroup + t];
            acc[a][c] = v;
          }
  }
}

// dQ, the bias gradients and what the key walk reads. A CTA takes query tiles blockIdx.x, + gridDim.x, ...
// of 32 rows; thread (ty, tx) of a group owns rows 4 ty .. + 3 and keys 4 tx .. + 3 of every key tile of the group. The
// table's products are tiles like the keys': U = Q table^T before them (rh and rw are shifted reads of it), and after them
// G table and G^T Q, where G[r][t] is dRh[r, i+h-1-t] or dRw[r, j+w-1-t'], zero where there is no such key.
template <typename T, int G>
__global__ void __launch_bounds__(kGroup* G, 4 / G) bwd_dq_simt(Args p) {
  constexpr int BQ = kBR, NT = kGroup * G;
  extern __shared__ float4 smem_f4[];
  const int h = p.h, w = p.w, hd = p.hd, n = h * w, hw = h + w, hp = (hd + 15) / 16 * 16, nc = hp / 16;
  const int tid = threadIdx.x, group = tid / kGroup, ty = (tid >> 4) & 7, tx = tid & 15;
  const int own = hp * kS64 + BQ * kS64 + hw * BQ;  // floats of a group
  float* Qs = reinterpret_cast<float*>(smem_f4);    // [hp][kS32]
  float* Os = Qs + hp * kS32;                       // dO [hp][kS32]
  float* rel = Os + hp * kS32;                      // [h + w][BQ]
  float* dsum = rel + hw * BQ;                      // [BQ]
  float* Ks = dsum + BQ + group * own;              // the group's V, then K; the table [hp][kS64]
  float* Ds = Ks + hp * kS64;                       // its dS, at the end G [BQ][kS64]
  float* drel = Ds + BQ * kS64;                     // its share of dRh, dRw [h + w][BQ]
  float* drel0 = drel - group * own;
  const int qtiles = (n + BQ - 1) / BQ, tr = table_rows(h, w);
  const T* table = static_cast<const T*>(p.table);
  float* part = p.partial + (long)blockIdx.x * tr * hd;
  const float c2 = p.scale * kLog2e;
  int first = p.first;
  if (first && (long)blockIdx.x >= p.bh * qtiles)
    for (int idx = tid; idx < tr * hd; idx += NT) part[idx] = 0.f;

  for (long tile = blockIdx.x; tile < p.bh * qtiles; tile += gridDim.x) {
    const long bh = tile / qtiles;
    const int r0 = (int)(tile - bh * qtiles) * BQ;
    const T* qb = static_cast<const T*>(p.q) + bh * n * hd;
    const T* ob = static_cast<const T*>(p.out) + bh * n * hd;
    const T* dob = static_cast<const T*>(p.dout) + bh * n * hd;
    const T* ktb = static_cast<const T*>(p.kt) + bh * (long)hd * n;
    const T* vb = static_cast<const T*>(p.v) + bh * n * hd;
    __syncthreads();  // the previous tile's shared memory has been read
    if (group == 0) load_transposed<T, BQ>(Qs, kS32, qb, r0, n, hd);
    if (group == (G > 1)) load_transposed<T, BQ>(Os, kS32, dob, r0, n, hd);
    if (kKeys * group < tr) load_transposed<T, kKeys>(Ks, kS64, table, kKeys * group, tr, hd);
    {
      const int lane = tid & 31;
#pragma unroll 4
      for (int r = tid >> 5; r < BQ; r += NT / 32) {
        float s = 0.f;
        if (r0 + r < n)
          for (int d = lane; d < hd; d += 32)
            s = fmaf(to_f(ob[(long)(r0 + r) * hd + d]), to_f(dob[(long)(r0 + r) * hd + d]), s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) {
          dsum[r] = s;
          if (r0 + r < n) p.dsum[bh * p.np + r0 + r] = s;
        }
      }
    }
    for (int idx = tid % kGroup; idx < hw * BQ; idx += kGroup) drel[idx] = 0.f;
    {
      int ri[4], rj[4];  // this thread's rows on the grid
      float lse2[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int row = r0 + ty * 4 + a;
        ri[a] = row / w;
        rj[a] = row - ri[a] * w;
        lse2[a] = row < n ? p.lse[bh * n + row] * kLog2e : 0.f;
      }
      __syncthreads();
      for (int t0 = kKeys * group; t0 < tr; t0 += kKeys * G) {
        if (t0 >= kKeys * G) {
          group_sync(group);
          load_transposed<T, kKeys>(Ks, kS64, table, t0, tr, hd);
          group_sync(group);
        }
        float u[4][4];
        dot_tile<4, kS64>(u, Qs, ty * 4, Ks, tx * 4, hd);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int t = t0 + tx * 4 + b;
          const bool is_h = t < 2 * h - 1;
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const int c = is_h ? ri[a] + h - 1 - t : rj[a] + w - 1 - (t - (2 * h - 1));
            if (t < tr && c >= 0 && c < (is_h ? h : w))
              rel[(is_h ? c : h + c) * BQ + ty * 4 + a] = is_h ? fmaf(u[a][b], kLog2e, -lse2[a]) : u[a][b] * kLog2e;
          }
        }
      }
    }
    float acc[4][8];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[a][c] = 0.f;
    __syncthreads();  // rel is whole
    for (int idx = tid; idx < hw * BQ; idx += NT) {
      const int r = idx % BQ, c = idx / BQ;
      if (r0 + r < n) p.rel[(bh * hw + c) * p.np + r0 + r] = rel[idx];
    }

    for (int k0 = kKeys * group; k0 < n; k0 += kKeys * G) {
      group_sync(group);  // the previous key tile's Ks and dS have been read
      load_transposed<T, kKeys>(Ks, kS64, vb, k0, n, hd);
      group_sync(group);
      float s[4][4], dp[4][4];
      dot_tile<4, kS64>(dp, Os, ty * 4, Ks, tx * 4, hd);
      group_sync(group);
      load_columns<T, kKeys>(Ks, kS64, ktb, k0, n, hd);
      group_sync(group);
      dot_tile<4, kS64>(s, Qs, ty * 4, Ks, tx * 4, hd);
      const float4 d4 = *reinterpret_cast<const float4*>(&dsum[ty * 4]);
      const float dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int key = k0 + tx * 4 + b, kh = key < n ? key / w : 0, kw = key < n ? key - kh * w : 0;
        const float4 rh = *reinterpret_cast<const float4*>(&rel[kh * BQ + ty * 4]);
        const float4 rw = *reinterpret_cast<const float4*>(&rel[(h + kw) * BQ + ty * 4]);
        const float bias[4] = {rh.x + rw.x, rh.y + rw.y, rh.z + rw.z, rh.w + rw.w};
#pragma unroll
        for (int a = 0; a < 4; ++a)
          s[a][b] = key < n && r0 + ty * 4 + a < n ? exp2f(fmaf(s[a][b], c2, bias[a])) * (dp[a][b] - dd[a]) : 0.f;
      }
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<float4*>(&Ds[(ty * 4 + a) * kS64 + tx * 4]) = make_float4(s[a][0], s[a][1], s[a][2], s[a][3]);
      group_sync(group);
      // the bias gradients: every (row, kh) and (row, kw) adds its keys of this tile
      const int kend = min(k0 + kKeys, n), kh0 = k0 / w, kh1 = (kend - 1) / w;
      for (int idx = tid % kGroup; idx < (kh1 - kh0 + 1 + w) * BQ; idx += kGroup) {
        const int r = idx % BQ, c = idx / BQ;
        const bool is_h = c <= kh1 - kh0;
        int k = is_h ? (kh0 + c) * w : kh0 * w + c - (kh1 - kh0 + 1);
        const int step = is_h ? 1 : w, end = is_h ? min(kend, k + w) : kend;
        if (k < k0) k = is_h ? k0 : k + w;
        float s2 = 0.f;
#pragma unroll 4
        for (; k < end; k += step) s2 += Ds[r * kS64 + k - k0];
        drel[(is_h ? kh0 + c : h + c - (kh1 - kh0 + 1)) * BQ + r] += s2;
      }
      mul_tile<kKeys, kS64>(acc, Ds, ty * 4, Ks, tx, nc);
    }
    __syncthreads();
    if constexpr (G > 1) {
      for (int idx = tid; idx < hw * BQ; idx += NT) {
        float v = drel0[idx];
        for (int q = 1; q < G; ++q) v += drel0[q * own + idx];
        drel0[idx] = v;
      }
      __syncthreads();
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[a][c] *= p.scale;
    for (int t0 = kKeys * group; t0 < tr; t0 += kKeys * G) {
      if (t0 >= kKeys * G) group_sync(group);  // G and Ks have been read
      load_transposed<T, kKeys>(Ks, kS64, table, t0, tr, hd);
      for (int idx = tid % kGroup; idx < BQ * kS64; idx += kGroup) Ds[idx] = 0.f;
      group_sync(group);
      for (int idx = tid % kGroup; idx < hw * BQ; idx += kGroup) {
        const int r = idx % BQ, c = idx / BQ, i = (r0 + r) / w, j = r0 + r - i * w;
        const int t = (c < h ? i + h - 1 - c : 2 * h - 1 + j + w - 1 - (c - h)) - t0;
        if (r0 + r < n && t >= 0 && t < kKeys) Ds[r * kS64 + t] = drel0[idx];
      }
      group_sync(group);
      mul_tile<kKeys, kS64>(acc, Ds, ty * 4, Ks, tx, nc);
      // this CTA's share of dtable: 32 of the tile's table rows at a time
      for (int q = 0; q < kKeys; q += BQ) {
        float g[4][8];
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
          for (int c = 0; c < 8; ++c) g[a][c] = 0.f;
#pragma unroll 2
        for (int r = 0; r < BQ; r += 4) {
          float4 m[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) m[e] = *reinterpret_cast<const float4*>(&Ds[(r + e) * kS64 + q + ty * 4]);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if (c < nc) {
              const float4 b4 = *reinterpret_cast<const float4*>(&Qs[(tx + 16 * c) * kS32 + r]);
              const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                g[0][c] = fmaf(m[e].x, b[e], g[0][c]);
                g[1][c] = fmaf(m[e].y, b[e], g[1][c]);
                g[2][c] = fmaf(m[e].z, b[e], g[2][c]);
                g[3][c] = fmaf(m[e].w, b[e], g[3][c]);
              }
            }
          }
        }
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int t = t0 + q + ty * 4 + a;
          if (t < tr) {
            float* at = part + (long)t * hd + tx;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              if (tx + 16 * c < hd) at[16 * c] = first ? g[a][c] : at[16 * c] + g[a][c];
          }
        }
      }
    }
    first = 0;
    group_sync(group);
    join_groups<G>(acc, Ks, own, group, nc);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int row = r0 + ty * 4 + a;
      if (a / (4 / G) == group && row < n) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (tx + 16 * c < hd) static_cast<T*>(p.dq)[(bh * n + row) * hd + tx + 16 * c] = from_f<T>(acc[a][c]);
      }
    }
  }
}

// dK and dV: one CTA per head and 32 keys, its groups walking the query tiles; thread (ty, tx) of a group owns keys
// 4 ty .. + 3 and queries 2 tx, 2 tx + 1 of every query tile of the group.
template <typename T, int G>
__global__ void __launch_bounds__(kGroup* G, 4 / G) bwd_dkv_simt(Args p) {
  constexpr int BK = kBR;
  extern __shared__ float4 smem_f4[];
  const int h = p.h, w = p.w, hd = p.hd, n = h * w, hw = h + w, hp = (hd + 15) / 16 * 16, nc = hp / 16;
  const int tid = threadIdx.x, group = tid / kGroup, ty = (tid >> 4) & 7, tx = tid & 15;
  const int own = 2 * hp * kS32 + 2 * BK * kS32;  // floats of a group
  float* Ks = reinterpret_cast<float*>(smem_f4);  // [hp][kS32]
  float* Vs = Ks + hp * kS32;
  float* Qs = Vs + hp * kS32 + group * own;       // the group's queries [hp][kS32]
  float* Os = Qs + hp * kS32;
  float* Ps = Os + hp * kS32;                     // P^T [key][query]
  float* Ds = Ps + BK * kS32;                     // dS^T [key][query]
  const int ktiles = (n + BK - 1) / BK;
  const long bh = blockIdx.x / ktiles;
  const int k0 = (int)(blockIdx.x - bh * ktiles) * BK;
  const T* qb = static_cast<const T*>(p.q) + bh * n * hd;
  const T* dob = static_cast<const T*>(p.dout) + bh * n * hd;
  const float c2 = p.scale * kLog2e;
  if (group == 0) load_columns<T, BK>(Ks, kS32, static_cast<const T*>(p.kt) + bh * (long)hd * n, k0, n, hd);
  if (group == (G > 1)) load_transposed<T, BK>(Vs, kS32, static_cast<const T*>(p.v) + bh * n * hd, k0, n, hd);
  float dk[4][8], dv[4][8];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < 8; ++c) dk[a][c] = dv[a][c] = 0.f;
  __syncthreads();
  for (int r0 = kQueries * group; r0 < n; r0 += kQueries * G) {
    // (the workspace rows are padded: the vectors stay inside them; what is read past n is not used)
    const float2 d2 = __ldg(reinterpret_cast<const float2*>(p.dsum + bh * p.np + r0) + tx);
    const float dsum[2] = {d2.x, d2.y};
    float bias[4][2];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int key = min(k0 + ty * 4 + a, n - 1), kh = key / w, kw = key - kh * w;
      const float2 rh = __ldg(reinterpret_cast<const float2*>(p.rel + (bh * hw + kh) * p.np + r0) + tx);
      const float2 rw = __ldg(reinterpret_cast<const float2*>(p.rel + (bh * hw + h + kw) * p.np + r0) + tx);
      bias[a][0] = rh.x + rw.x;
      bias[a][1] = rh.y + rw.y;
    }
    group_sync(group);
    load_transposed<T, kQueries>(Qs, kS32, qb, r0, n, hd);
    load_transposed<T, kQueries>(Os, kS32, dob, r0, n, hd);
    group_sync(group);
    float s[4][2], dp[4][2];
    dot_tile<2, kS32>(s, Ks, ty * 4, Qs, tx * 2, hd);
    dot_tile<2, kS32>(dp, Vs, ty * 4, Os, tx * 2, hd);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const bool ok = k0 + ty * 4 + a < n;
      float pr[2], g[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const bool in = ok && r0 + tx * 2 + b < n;
        pr[b] = in ? exp2f(fmaf(s[a][b], c2, bias[a][b])) : 0.f;
        g[b] = in ? pr[b] * (dp[a][b] - dsum[b]) : 0.f;
      }
      *reinterpret_cast<float2*>(&Ps[(ty * 4 + a) * kS32 + tx * 2]) = make_float2(pr[0], pr[1]);
      *reinterpret_cast<float2*>(&Ds[(ty * 4 + a) * kS32 + tx * 2]) = make_float2(g[0], g[1]);
    }
    group_sync(group);
    mul_tile<kQueries, kS32>(dv, Ps, ty * 4, Os, tx, nc);
    mul_tile<kQueries, kS32>(dk, Ds, ty * 4, Qs, tx, nc);
  }
  group_sync(group);
  join_groups<G>(dv, Qs, own, group, nc);
  join_groups<G>(dk, Qs + 4 * nc * kGroup, own, group, nc);
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const int key = k0 + ty * 4 + a;
    if (a / (4 / G) == group && key < n) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int d = tx + 16 * c;
        if (d < hd) {
          static_cast<T*>(p.dv)[(bh * n + key) * hd + d] = from_f<T>(dv[a][c]);
          static_cast<T*>(p.dkt)[(bh * hd + d) * n + key] = from_f<T>(dk[a][c] * p.scale);
        }
      }
    }
  }
}

// dtable[e] = the CTAs' partial sums added in a fixed order. A block takes 32 elements; its warps share the slots (16 warps:
// 3.8 us for 148 slots of 54 x 80 elements and 6.9 for 254 x 80; 8 warps 4.8 and 6.3, 32 warps 4.6 and 12).
template <typename T>
__global__ void __launch_bounds__(1024) bwd_table_reduce(const float* __restrict__ partial, T* __restrict__ dtable,
                                                        int slots, int elems) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  sm100::wait_previous_launch();
  float s = 0.f;
  if (e < elems)
#pragma unroll 8
    for (int k = warp; k < slots; k += warps) s += partial[(long)k * elems + e];
  red[warp][lane] = s;
  __syncthreads();
  for (int f = warp; f < 32; f += warps) {
    s = lane < warps ? red[lane][f] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int at = blockIdx.x * 32 + f;
    if (lane == 0 && at < elems) dtable[at] = from_f<T>(s);
  }
}

}  // namespace bwd
}  // namespace samrs
