// relpos_bwd_simt.cuh - backward pass of the rel-pos attention for any (h, w, hd <= 128), any dtype: the f32 path, and
// the path of 16-bit shapes the tcgen05 kernels (relpos_bwd_tc.cuh) do not cover.
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
// order. All sums are f32 (exp2f of log2-scaled logits), rounded once to the I/O dtype.
//
// Bound by the instructions issued: products of operands in shared memory, in tiles of 32 rows. On the f32 pipe a product
// costs an instruction for every 2 multiplications of a lane and as many cycles of shared memory as of arithmetic; through
// mma.sync's TF32, three times for 21 bits, a third of the instructions and a sixth of the reads. That path truncates, a
// bias of about 2e-7, which matters where dP - D cancels: so bwd_dq_simt forms S and dP on the f32 pipe and the rest on
// TF32, bwd_dkv_simt everything on TF32. What a CTA cannot hide itself, 16 resident warps per SM hide.
// 75 heads of 14 x 14 x 64, f32: 91 + 72 us, 11 TFLOP/s of the five products that the gradients need. One head of
// 64 x 64 x 64: 284 + 297 us, 18 TFLOP/s; all of it on the f32 pipe took 1.4 times as long. 16 heads of 64 x 64 x 80: 4.7 +
// 4.9 ms, 22 TFLOP/s. Weakest on few heads of large grids and wide heads: 2 heads of 60 x 60 x 128 take 2.0 ms, where
// library products that store the scores take 1.5.
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
  return 2 * hp * kS32 + (kS32 + g * kBR) * (int64_t)(h + w) + kBR + g * (hp * kS64 + (int64_t)kBR * kS64);
}
__host__ __device__ inline int64_t dkv_smem_floats(int g, int hd) {
  const int64_t hp = (hd + 15) / 16 * 16;
  return 2 * hp * kS32 + g * (2 * hp * kS32 + (int64_t)2 * kBR * kS32);
}

// A barrier of this thread's group.
__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory"); }

// By one group: rows r0 .. r0 + ROWS - 1 of src [n][hd], transposed into dst[d][r] (row stride `stride`); rows past n and
// columns past hd, up to a multiple of 16, are 0. A warp takes 4 rows x 8 columns at a time (whole sectors of f32; the
// stores hit 32 banks), a batch of loads in flight.
template <typename T, int ROWS>
__device__ __forceinline__ void load_transposed(float* dst, int stride, const T* src, int r0, int n, int hd) {
  constexpr int kWarps = kGroup / 32, kGroups = ROWS / 4, B = kGroups / kWarps, DB = B < 8 ? 16 / B : 2;
  static_assert(kGroups % kWarps == 0, "whole batches");
  const int lane = threadIdx.x & 31, warp = (threadIdx.x % kGroup) >> 5, r = 4 * warp + (lane >> 3);
  const int hp = (hd + 15) / 16 * 16;
  for (int d0 = lane & 7; d0 < hp; d0 += 8 * DB) {
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
        if (d0 + 8 * e < hp) dst[(d0 + 8 * e) * stride + r + 4 * kWarps * k] = v[e][k];
  }
}
// By one group: columns k0 .. k0 + COLS - 1 of src [hd][n] into dst[d][k]; columns past n are 0.
template <typename T, int COLS>
__device__ __forceinline__ void load_columns(float* dst, int stride, const T* src, int k0, int n, int hd) {
  const int k = threadIdx.x % COLS;
  constexpr int kRows = kGroup / COLS, B = 8;
  const int hp = (hd + 15) / 16 * 16;
  for (int d0 = threadIdx.x % kGroup / COLS; d0 < hp; d0 += kRows * B) {
    float v[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int d = d0 + kRows * j;
      v[j] = d < hd && k0 + k < n ? to_f(src[(long)d * n + k0 + k]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (d0 + kRows * j < hp) dst[(d0 + kRows * j) * stride + k] = v[j];
  }
}

// out[a][b] = sum_d A[d][ra + a] B[d][cb + b], 4 x 4, on the f32 pipe
__device__ __forceinline__ void fma_dot_tile(float (&out)[4][4], const float* A, int ra, const float* B, int cb, int hd) {
  float2 acc[4][2];
#pragma unroll
  for (int a = 0; a < 4; ++a) acc[a][0] = acc[a][1] = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int d = 0; d < hd; ++d) {
    const float4 av = *reinterpret_cast<const float4*>(&A[d * kS32 + ra]);
    const float4 bv = *reinterpret_cast<const float4*>(&B[d * kS64 + cb]);
    const float m[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      acc[a][0] = sm100::fma2(make_float2(m[a], m[a]), make_float2(bv.x, bv.y), acc[a][0]);
      acc[a][1] = sm100::fma2(make_float2(m[a], m[a]), make_float2(bv.z, bv.w), acc[a][1]);
    }
  }
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    out[a][0] = acc[a][0].x;
    out[a][1] = acc[a][0].y;
    out[a][2] = acc[a][1].x;
    out[a][3] = acc[a][1].y;
  }
}

// f32 products on the tensor cores' TF32 path: x = hi + lo with hi of 11 bits (rounded) and lo the next 11 of the
// rest; x y is hi hi + hi lo + lo hi. What is left out is 2^-21 of x at most, with either sign. (An infinite x
// has no rest: its products are NaN.)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xFFFFE000u;
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
struct FragA {
  uint32_t hi[4], lo[4];
  __device__ __forceinline__ void set(float a0, float a1, float a2, float a3) {
    split_tf32(a0, hi[0], lo[0]);
    split_tf32(a1, hi[1], lo[1]);
    split_tf32(a2, hi[2], lo[2]);
    split_tf32(a3, hi[3], lo[3]);
  }
};
// acc += the sum of K fragments' products. The core truncates the sums that it adds to, which biases them towards zero: so
// a fragment's products go to a sum of their own, the small terms first, and the fragments are added up outside.
template <int K>
__device__ __forceinline__ void mma_3x(float (&acc)[4], const FragA (&a)[K], const float2 (&b)[K]) {
  float c[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    uint32_t hi[2], lo[2];
    split_tf32(b[k].x, hi[0], lo[0]);
    split_tf32(b[k].y, hi[1], lo[1]);
    c[k][0] = c[k][1] = c[k][2] = c[k][3] = 0.f;
    mma_tf32(c[k], a[k].lo, hi);
    mma_tf32(c[k], a[k].hi, lo);
    mma_tf32(c[k], a[k].hi, hi);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float t = c[0][e];
#pragma unroll
    for (int k = 1; k < K; ++k) t += c[k][e];
    acc[e] += t;
  }
}
// A warp's tiles: element e of a 16 x 8 result is row lane / 4 + 8 (e / 2), column 2 (lane % 4) + e % 2. An inner index
// may be dealt out to the fragments in any order that both operands share: pairs 2 t, 2 t + 1 of each 8 for lane t of 4, so
// that operands of either orientation are read without bank conflicts. 

// out[j] = sum_d A[d][ra ..] B[d][cb + 8j ..]: 16 x 8 NT
template <int NT, int SB>
__device__ __forceinline__ void dot_tile(float (&out)[NT][4], const float* A, int ra, const float* B, int cb, int hp) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
  A += 2 * t * kS32 + ra + g;
  B += 2 * t * SB + cb + g;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) out[j][e] = 0.f;
  for (int d0 = 0; d0 < hp; d0 += 16) {
    FragA f[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float* a = A + (d0 + 8 * k) * kS32;
      f[k].set(a[0], a[8], a[kS32], a[kS32 + 8]);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float2 b[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) b[k] = make_float2(B[(d0 + 8 * k) * SB + 8 * j], B[(d0 + 8 * k + 1) * SB + 8 * j]);
      mma_3x(out[j], f, b);
    }
  }
}

// A's fragments of 16 rows and 32 columns: M[ra ..][x], or with kTrans M[x][ra ..]; rows of S floats
template <bool kTrans, int S>
__device__ __forceinline__ void load_a(FragA (&f)[4], const float* M, int ra) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (kTrans) {
      const float* a = M + (8 * k + 2 * t) * S + ra + g;
      f[k].set(a[0], a[8], a[S], a[S + 8]);
    } else {
      const float2 u = *reinterpret_cast<const float2*>(M + (ra + g) * S + 8 * k + 2 * t);
      const float2 v = *reinterpret_cast<const float2*>(M + (ra + g + 8) * S + 8 * k + 2 * t);
      f[k].set(u.x, v.x, u.y, v.y);
    }
  }
}
// acc[j] += sum over 32 x of A[..][x] B[cb + 8j ..][x], for j < nt; rows of S floats
template <int S>
__device__ __forceinline__ void mul_tile(float (&acc)[8][4], const FragA (&f)[4], const float* B, int cb, int nt) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
  B += (cb + g) * S + 2 * t;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < nt) {
      float2 b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) b[k] = *reinterpret_cast<const float2*>(B + 8 * j * S + 8 * k);
      mma_3x(acc[j], f, b);
    }
  }
}

// The groups' nt x 4 sums to a thread, by way of shared memory (each group's own `mine`, kGroup x 4 nt floats): the thread
// keeps the total of elements e with e / (4 / G) == group, added in the groups' order. `stride`: floats from one group's
// `mine` to the next one's.
template <int G>
__device__ __forceinline__ void join_groups(float (&acc)[8][4], float* mine, int stride, int group, int nt) {
  if constexpr (G > 1) {
    const int t = threadIdx.x % kGroup;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j < nt) mine[(4 * j + e) * kGroup + t] = acc[j][e];
    __syncthreads();
    const float* all = mine - (long)group * stride;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j < nt && e / (4 / G) == group) {
          float v = all[(4 * j + e) * kGroup + t];
          for (int q = 1; q < G; ++q) v += all[q * stride + (4 * j + e) * kGroup + t];
          acc[j][e] = v;
        }
  }
}

// dQ, the bias gradients and what the key walk reads. A CTA takes query tiles blockIdx.x, + gridDim.x, ... of 32 rows, its
// groups the key tiles in turn. On the f32 pipe thread (ty, tx) of a group has rows 4 ty .. + 3 and keys 4 tx .. + 3 of a
// tile; of the TF32 products a warp has 16 rows and half of the columns. The table's products are tiles like the keys':
// U = Q table^T before them (rh and rw are shifted reads of it), and after them G table and G^T Q, where G[r][t] is
// dRh[r, i+h-1-t] or dRw[r, j+w-1-t'], zero where there is no such key.
template <typename T, int G>
__global__ void __launch_bounds__(kGroup* G, 4 / G) bwd_dq_simt(Args p) {
  constexpr int BQ = kBR, NT = kGroup * G;
  extern __shared__ float4 smem_f4[];
  const int h = p.h, w = p.w, hd = p.hd, n = h * w, hw = h + w, hp = (hd + 15) / 16 * 16, nt = hp / 16;
  const int tid = threadIdx.x, group = tid / kGroup, warp = (tid % kGroup) >> 5, lane = tid & 31;
  const int ty = (tid >> 4) & 7, tx = tid & 15;
  const int ra = 16 * (warp & 1), half = warp >> 1, cg = lane & 3;  // rows, and half of the columns, of this warp's products
  const int rows[2] = {ra + (lane >> 2), ra + (lane >> 2) + 8};      // this thread's rows of them
  const unsigned wdiv = 0xFFFFFFFFu / (unsigned)w + 1;  // k / w is the high word of k wdiv, for w > 1 and k < 2^14
  const int own = hp * kS64 + BQ * kS64 + hw * BQ;  // floats of a group
  float* Qs = reinterpret_cast<float*>(smem_f4);    // [hp][kS32]
  float* Os = Qs + hp * kS32;                       // dO [hp][kS32]
  float* rel = Os + hp * kS32;                      // [h + w][kS32]
  float* dsum = rel + hw * kS32;                     // [BQ]
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
        fma_dot_tile(u, Qs, ty * 4, Ks, tx * 4, hd);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int t = t0 + tx * 4 + b;
          const bool is_h = t < 2 * h - 1;
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const int c = is_h ? ri[a] + h - 1 - t : rj[a] + w - 1 - (t - (2 * h - 1));
            if (t < tr && c >= 0 && c < (is_h ? h : w))
              rel[(is_h ? c : h + c) * kS32 + ty * 4 + a] = is_h ? fmaf(u[a][b], kLog2e, -lse2[a]) : u[a][b] * kLog2e;
          }
        }
      }
    }
    float acc[8][4];  // dQ: columns 8 (half nt + j) ..
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    __syncthreads();  // rel is whole
    for (int idx = tid; idx < hw * BQ; idx += NT) {
      const int r = idx % BQ, c = idx / BQ;
      if (r0 + r < n) p.rel[(bh * hw + c) * p.np + r0 + r] = rel[c * kS32 + r];
    }

    for (int k0 = kKeys * group; k0 < n; k0 += kKeys * G) {
      group_sync(group);  // the previous key tile's Ks and dS have been read
      load_transposed<T, kKeys>(Ks, kS64, vb, k0, n, hd);
      group_sync(group);
      float s[4][4], dp[4][4];
      fma_dot_tile(dp, Os, ty * 4, Ks, tx * 4, hd);
      group_sync(group);
      load_columns<T, kKeys>(Ks, kS64, ktb, k0, n, hd);
      group_sync(group);
      fma_dot_tile(s, Qs, ty * 4, Ks, tx * 4, hd);
      const float4 d4 = *reinterpret_cast<const float4*>(&dsum[ty * 4]);
      const float dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int key = k0 + tx * 4 + b, kh = key >= n ? 0 : w > 1 ? (int)__umulhi((unsigned)key, wdiv) : key,
                  kw = key >= n ? 0 : key - kh * w;
        const float4 rh = *reinterpret_cast<const float4*>(&rel[kh * kS32 + ty * 4]);
        const float4 rw = *reinterpret_cast<const float4*>(&rel[(h + kw) * kS32 + ty * 4]);
        const float bias[4] = {rh.x + rw.x, rh.y + rw.y, rh.z + rw.z, rh.w + rw.w};
#pragma unroll
        for (int a = 0; a < 4; ++a)
          s[a][b] = key < n && r0 + ty * 4 + a < n ? exp2f(fmaf(s[a][b], c2, bias[a])) * (dp[a][b] - dd[a]) : 0.f;
      }
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<float4*>(&Ds[(ty * 4 + a) * kS64 + tx * 4]) = make_float4(s[a][0], s[a][1], s[a][2], s[a][3]);
      group_sync(group);
      // the bias gradients: 8 rows of a warp add their keys of this tile, four lanes to a row: the four quarters of a grid
      // row's keys, or four grid columns
      {
        const int r = 8 * warp + (lane & 7), q = lane >> 3;
        const int kend = min(k0 + kKeys, n), kh0 = k0 / w, kh1 = (kend - 1) / w;
        const float* d = Ds + r * kS64 - k0;
        for (int kh = kh0; kh <= kh1; ++kh) {
          const int end = min(kend, (kh + 1) * w);
          float s2 = 0.f;
#pragma unroll 4
          for (int k = max(k0, kh * w) + q; k < end; k += 4) s2 += d[k];
          s2 += __shfl_xor_sync(0xffffffffu, s2, 8);
          s2 += __shfl_xor_sync(0xffffffffu, s2, 16);
          if (q == 0) drel[kh * BQ + r] += s2;
        }
#pragma unroll 2
        for (int kw = q; kw < w; kw += 4) {
          int k = kh0 * w + kw;
          if (k < k0) k += w;
          float s2 = 0.f;
          for (; k < kend; k += w) s2 += d[k];
          drel[(h + kw) * BQ + r] += s2;
        }
      }
#pragma unroll
      for (int x = 0; x < kKeys; x += 32) {
        FragA f[4];
        load_a<false, kS64>(f, Ds + x, ra);
        mul_tile<kS64>(acc, f, Ks + x, 8 * half * nt, nt);
      }
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
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] *= p.scale;
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
#pragma unroll
      for (int x = 0; x < kKeys; x += 32) {
        FragA f[4];
        load_a<false, kS64>(f, Ds + x, ra);
        mul_tile<kS64>(acc, f, Ks + x, 8 * half * nt, nt);
      }
      // this CTA's share of dtable: G^T Q, 32 table rows to a warp
#pragma unroll
      for (int q = 0; q < 32; q += 16) {
        float g[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) g[j][e] = 0.f;
        FragA f[4];
        load_a<true, kS64>(f, Ds, 2 * ra + q);
        mul_tile<kS32>(g, f, Qs, 8 * half * nt, nt);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = t0 + 2 * ra + q + (lane >> 2) + 8 * (e >> 1);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int d = 8 * (half * nt + j) + 2 * cg + (e & 1);
            if (j < nt && t < tr && d < hd) {
              float* at = part + (long)t * hd + d;
              *at = first ? g[j][e] : *at + g[j][e];
            }
          }
        }
      }
    }
    first = 0;
    group_sync(group);
    join_groups<G>(acc, Ks, own, group, nt);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = r0 + rows[e >> 1];
      if (e / (4 / G) == group && row < n) {
        T* dq = static_cast<T*>(p.dq) + (bh * n + row) * hd;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = 8 * (half * nt + j) + 2 * cg + (e & 1);
          if (j < nt && d < hd) dq[d] = from_f<T>(acc[j][e]);
        }
      }
    }
  }
}

// dK and dV: one CTA per head and 32 keys, its groups walking the query tiles; the four warps of a group take 16 keys and
// 16 queries each of a query tile of the group.
template <typename T, int G>
__global__ void __launch_bounds__(kGroup* G, 4 / G) bwd_dkv_simt(Args p) {
  constexpr int BK = kBR;
  extern __shared__ float4 smem_f4[];
  const int h = p.h, w = p.w, hd = p.hd, n = h * w, hw = h + w, hp = (hd + 15) / 16 * 16, nt = hp / 16;
  const int tid = threadIdx.x, group = tid / kGroup, warp = (tid % kGroup) >> 5, lane = tid & 31;
  const int ra = 16 * (warp & 1), half = warp >> 1, cg = lane & 3;  // keys, and half of the columns, of this warp's products
  const int keys[2] = {ra + (lane >> 2), ra + (lane >> 2) + 8};      // this thread's keys
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
  float dk[8][4], dv[8][4];  // columns 8 (half nt + j) ..
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[j][e] = dv[j][e] = 0.f;
  // the bias rows of this thread's keys (past n: any key's, unused)
  const float *rh[2], *rw[2];
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int key = min(k0 + keys[a], n - 1), kh = key / w, kw = key - kh * w;
    rh[a] = p.rel + (bh * hw + kh) * p.np + 16 * half + 2 * cg;
    rw[a] = p.rel + (bh * hw + h + kw) * p.np + 16 * half + 2 * cg;
  }
  const float* ds = p.dsum + bh * p.np + 16 * half + 2 * cg;
  __syncthreads();
  for (int r0 = kQueries * group; r0 < n; r0 += kQueries * G) {
    // (the workspace rows are padded: the vectors stay inside them; what is read past n is not used)
    float2 bias[2][2], dsum[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      dsum[j] = __ldg(reinterpret_cast<const float2*>(ds + r0 + 8 * j));
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const float2 x = __ldg(reinterpret_cast<const float2*>(rh[a] + r0 + 8 * j));
        const float2 y = __ldg(reinterpret_cast<const float2*>(rw[a] + r0 + 8 * j));
        bias[j][a] = make_float2(x.x + y.x, x.y + y.y);
      }
    }
    group_sync(group);
    load_transposed<T, kQueries>(Qs, kS32, qb, r0, n, hd);
    load_transposed<T, kQueries>(Os, kS32, dob, r0, n, hd);
    group_sync(group);
    float s[2][4], dp[2][4];
    dot_tile<2, kS32>(s, Ks, ra, Qs, 16 * half, hp);
    dot_tile<2, kS32>(dp, Vs, ra, Os, 16 * half, hp);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 16 * half + 8 * j + 2 * cg;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const bool ok = k0 + keys[a] < n, in0 = ok && r0 + r < n, in1 = ok && r0 + r + 1 < n;
        const float p0 = in0 ? exp2f(fmaf(s[j][2 * a], c2, bias[j][a].x)) : 0.f;
        const float p1 = in1 ? exp2f(fmaf(s[j][2 * a + 1], c2, bias[j][a].y)) : 0.f;
        *reinterpret_cast<float2*>(&Ps[keys[a] * kS32 + r]) = make_float2(p0, p1);
        *reinterpret_cast<float2*>(&Ds[keys[a] * kS32 + r]) =
            make_float2(in0 ? p0 * (dp[j][2 * a] - dsum[j].x) : 0.f, in1 ? p1 * (dp[j][2 * a + 1] - dsum[j].y) : 0.f);
      }
    }
    group_sync(group);
    FragA f[4];
    load_a<false, kS32>(f, Ps, ra);
    mul_tile<kS32>(dv, f, Os, 8 * half * nt, nt);
    load_a<false, kS32>(f, Ds, ra);
    mul_tile<kS32>(dk, f, Qs, 8 * half * nt, nt);
  }
  group_sync(group);
  join_groups<G>(dv, Qs, own, group, nt);
  join_groups<G>(dk, Qs + 4 * nt * kGroup, own, group, nt);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int key = k0 + keys[e >> 1];
    if (e / (4 / G) == group && key < n) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = 8 * (half * nt + j) + 2 * cg + (e & 1);
        if (j < nt && d < hd) {
          static_cast<T*>(p.dv)[(bh * n + key) * hd + d] = from_f<T>(dv[j][e]);
          static_cast<T*>(p.dkt)[(bh * hd + d) * n + key] = from_f<T>(dk[j][e] * p.scale);
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
