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

constexpr int kThreads = 256;
constexpr int kBK = 64;        // keys per tile
constexpr int kStride = 68;    // floats between the rows of a 64-wide tile: 16-byte reads, 8 rows hit 32 banks
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

// Dynamic shared memory of the two kernels, in floats.
__host__ __device__ inline size_t dq_smem_floats(int bq, int h, int w, int hd) {
  return (size_t)2 * hd * (bq + 4) + (size_t)2 * hd * kStride + (size_t)bq * kStride + (size_t)2 * bq * (h + w) + bq;
}
__host__ __device__ inline size_t dkv_smem_floats(int hd) { return (size_t)4 * hd * kStride + (size_t)2 * kBK * kStride; }

// Rows r0 .. r0 + ROWS - 1 of src [n][hd], transposed into dst[d][r] (row stride `stride`); rows past n are 0. A warp to a
// row, a batch of loads in flight (the stores must not come between them).
template <typename T, int ROWS>
__device__ __forceinline__ void load_transposed(float* dst, int stride, const T* src, int r0, int n, int hd) {
  constexpr int kWarps = kThreads / 32, B = ROWS / kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = lane; d < hd; d += 32) {
    float v[B];
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int r = r0 + warp + kWarps * k;
      v[k] = r < n ? to_f(src[(long)r * hd + d]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < B; ++k) dst[d * stride + warp + kWarps * k] = v[k];
  }
}
// Columns k0 .. k0 + 63 of src [hd][n] into dst[d][k]; columns past n are 0.
template <typename T>
__device__ __forceinline__ void load_columns(float* dst, const T* src, int k0, int n, int hd) {
  const int k = threadIdx.x % kBK;
  constexpr int kStep = kThreads / kBK, B = 8;
  for (int d0 = threadIdx.x / kBK; d0 < hd; d0 += kStep * B) {
    float v[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int d = d0 + kStep * j;
      v[j] = d < hd && k0 + k < n ? to_f(src[(long)d * n + k0 + k]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (d0 + kStep * j < hd) dst[(d0 + kStep * j) * kStride + k] = v[j];
  }
}

// acc[a][b] += sum_d A[d][ra + a] B[d][cb + b]
template <int RA>
__device__ __forceinline__ void dot_tile(float (&acc)[RA][4], const float* A, int sa, int ra, const float* B, int cb, int hd) {
#pragma unroll 4
  for (int d = 0; d < hd; ++d) {
    float av[RA];
#pragma unroll
    for (int a = 0; a < RA; a += 2) {
      const float2 t = *reinterpret_cast<const float2*>(&A[d * sa + ra + a]);
      av[a] = t.x;
      av[a + 1] = t.y;
    }
    const float4 bv = *reinterpret_cast<const float4*>(&B[d * kStride + cb]);
#pragma unroll
    for (int a = 0; a < RA; ++a) {
      acc[a][0] = fmaf(av[a], bv.x, acc[a][0]);
      acc[a][1] = fmaf(av[a], bv.y, acc[a][1]);
      acc[a][2] = fmaf(av[a], bv.z, acc[a][2]);
      acc[a][3] = fmaf(av[a], bv.w, acc[a][3]);
    }
  }
}

// acc[a][c] += sum over the tile's 64 columns x of M[ra + a][x] B[tx + 16c][x]
template <int RA>
__device__ __forceinline__ void mul_tile(float (&acc)[RA][8], const float* M, int ra, const float* B, int tx, int hd) {
#pragma unroll 2
  for (int x = 0; x < kBK; x += 4) {
    float4 m[RA];
#pragma unroll
    for (int a = 0; a < RA; ++a) m[a] = *reinterpret_cast<const float4*>(&M[(ra + a) * kStride + x]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int d = tx + 16 * c;
      if (d < hd) {
        const float4 b = *reinterpret_cast<const float4*>(&B[d * kStride + x]);
#pragma unroll
        for (int a = 0; a < RA; ++a) {
          acc[a][c] = fmaf(m[a].x, b.x, acc[a][c]);
          acc[a][c] = fmaf(m[a].y, b.y, acc[a][c]);
          acc[a][c] = fmaf(m[a].z, b.z, acc[a][c]);
          acc[a][c] = fmaf(m[a].w, b.w, acc[a][c]);
        }
      }
    }
  }
}

// dQ, the bias gradients and what the key walk reads. A CTA takes query tiles blockIdx.x, + gridDim.x, ...
// of 16 RQ rows; thread (ty, tx) owns rows ty RQ .. + RQ - 1 and keys 4 tx .. + 3 of every key tile.
template <typename T, int RQ>
__global__ void __launch_bounds__(kThreads) bwd_dq_simt(Args p) {
  constexpr int BQ = 16 * RQ, QS = BQ + 4;
  extern __shared__ float4 smem_f4[];
  const int h = p.h, w = p.w, hd = p.hd, n = h * w, hw = h + w;
  float* Qs = reinterpret_cast<float*>(smem_f4);  // [hd][QS]
  float* Os = Qs + hd * QS;                       // dO [hd][QS]
  float* Ks = Os + hd * QS;                       // [hd][kStride]
  float* Vs = Ks + hd * kStride;                  // [hd][kStride]
  float* Ds = Vs + hd * kStride;                  // dS [BQ][kStride]
  float* rel = Ds + BQ * kStride;                 // [h + w][BQ]
  float* drel = rel + hw * BQ;                    // [h + w][BQ]: dRh, dRw
  float* dsum = drel + hw * BQ;                   // [BQ]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ty = tid >> 4, tx = tid & 15;
  const int qtiles = (n + BQ - 1) / BQ, tr = table_rows(h, w);
  const T* table = static_cast<const T*>(p.table);
  float* part = p.partial + (long)blockIdx.x * tr * hd;
  const float c2 = p.scale * kLog2e;
  int first = p.first;
  if (first && (long)blockIdx.x >= p.bh * qtiles)
    for (int idx = tid; idx < tr * hd; idx += kThreads) part[idx] = 0.f;

  for (long tile = blockIdx.x; tile < p.bh * qtiles; tile += gridDim.x) {
    const long bh = tile / qtiles;
    const int r0 = (int)(tile - bh * qtiles) * BQ;
    const T* qb = static_cast<const T*>(p.q) + bh * n * hd;
    const T* ob = static_cast<const T*>(p.out) + bh * n * hd;
    const T* dob = static_cast<const T*>(p.dout) + bh * n * hd;
    const T* ktb = static_cast<const T*>(p.kt) + bh * (long)hd * n;
    const T* vb = static_cast<const T*>(p.v) + bh * n * hd;
    __syncthreads();  // the previous tile's shared memory has been read
    load_transposed<T, BQ>(Qs, QS, qb, r0, n, hd);
    load_transposed<T, BQ>(Os, QS, dob, r0, n, hd);
    for (int r = warp; r < BQ; r += kThreads / 32) {
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
    __syncthreads();
    for (int idx = tid; idx < hw * BQ; idx += kThreads) {
      const int r = idx % BQ, c = idx / BQ, row = r0 + r;
      float a = 0.f;
      if (row < n) {
        const int i = row / w, j = row - i * w;
        const T* t = table + (long)(c < h ? i - c + h - 1 : 2 * h - 1 + j - (c - h) + w - 1) * hd;
        for (int d = 0; d < hd; ++d) a = fmaf(Qs[d * QS + r], to_f(t[d]), a);
        a *= kLog2e;
        if (c < h) a -= p.lse[bh * n + row] * kLog2e;
        p.rel[(bh * hw + c) * p.np + row] = a;
      }
      rel[c * BQ + r] = a;
      drel[c * BQ + r] = 0.f;
    }
    float acc[RQ][8];
#pragma unroll
    for (int a = 0; a < RQ; ++a)
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[a][c] = 0.f;

    for (int k0 = 0; k0 < n; k0 += kBK) {
      __syncthreads();  // the previous key tile's Ks and dS have been read
      load_columns<T>(Ks, ktb, k0, n, hd);
      load_transposed<T, kBK>(Vs, kStride, vb, k0, n, hd);
      __syncthreads();
      float s[RQ][4], dp[RQ][4];
#pragma unroll
      for (int a = 0; a < RQ; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) s[a][b] = dp[a][b] = 0.f;
      dot_tile<RQ>(s, Qs, QS, ty * RQ, Ks, tx * 4, hd);
      dot_tile<RQ>(dp, Os, QS, ty * RQ, Vs, tx * 4, hd);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int key = k0 + tx * 4 + b, kh = key / w, kw = key - kh * w;
#pragma unroll
        for (int a = 0; a < RQ; ++a) {
          const int r = ty * RQ + a;
          float ds = 0.f;
          if (key < n && r0 + r < n)
            ds = exp2f(fmaf(s[a][b], c2, rel[kh * BQ + r] + rel[(h + kw) * BQ + r])) * (dp[a][b] - dsum[r]);
          Ds[r * kStride + tx * 4 + b] = ds;
        }
      }
      __syncthreads();
      // the bias gradients: every (row, kh) and (row, kw) adds its keys of this tile
      const int kend = min(k0 + kBK, n), kh0 = k0 / w, kh1 = (kend - 1) / w;
      for (int idx = tid; idx < (kh1 - kh0 + 1 + w) * BQ; idx += kThreads) {
        const int r = idx % BQ, c = idx / BQ;
        float s2 = 0.f;
        if (c <= kh1 - kh0) {
          const int kh = kh0 + c;
          for (int k = max(k0, kh * w); k < min(kend, (kh + 1) * w); ++k) s2 += Ds[r * kStride + k - k0];
          drel[kh * BQ + r] += s2;
        } else {
          const int kw = c - (kh1 - kh0 + 1);
          int k = kh0 * w + kw;
          if (k < k0) k += w;
          for (; k < kend; k += w) s2 += Ds[r * kStride + k - k0];
          drel[(h + kw) * BQ + r] += s2;
        }
      }
      mul_tile<RQ>(acc, Ds, ty * RQ, Ks, tx, hd);
    }
    __syncthreads();
#pragma unroll
    for (int a = 0; a < RQ; ++a) {
      const int r = ty * RQ + a, row = r0 + r;
      if (row < n) {
        const int i = row / w, j = row - i * w;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int d = tx + 16 * c;
          if (d < hd) {
            float g = acc[a][c] * p.scale;
            for (int kh = 0; kh < h; ++kh) g = fmaf(drel[kh * BQ + r], to_f(table[(long)(i - kh + h - 1) * hd + d]), g);
            for (int kw = 0; kw < w; ++kw)
              g = fmaf(drel[(h + kw) * BQ + r], to_f(table[(long)(2 * h - 1 + j - kw + w - 1) * hd + d]), g);
            static_cast<T*>(p.dq)[(bh * n + row) * hd + d] = from_f<T>(g);
          }
        }
      }
    }
    // this CTA's share of dtable
    const int rows = min(BQ, n - r0);
    for (int idx = tid; idx < tr * hd; idx += kThreads) {
      const int t = idx / hd, d = idx - t * hd;
      const bool is_h = t < 2 * h - 1;
      float g = 0.f;
      int i = r0 / w, j = r0 - i * w;
      for (int r = 0; r < rows; ++r) {
        const int c = is_h ? i + h - 1 - t : j + w - 1 - (t - (2 * h - 1));
        if (c >= 0 && c < (is_h ? h : w)) g = fmaf(drel[(is_h ? c : h + c) * BQ + r], Qs[d * QS + r], g);
        if (++j == w) {
          j = 0;
          ++i;
        }
      }
      part[idx] = first ? g : part[idx] + g;
    }
    first = 0;
  }
}

// dK and dV: one CTA per head and 64 keys, walking the query tiles.
template <typename T>
__global__ void __launch_bounds__(kThreads) bwd_dkv_simt(Args p) {
  extern __shared__ float4 smem_f4[];
  const int h = p.h, w = p.w, hd = p.hd, n = h * w, hw = h + w;
  float* Ks = reinterpret_cast<float*>(smem_f4);
  float* Vs = Ks + hd * kStride;
  float* Qs = Vs + hd * kStride;
  float* Os = Qs + hd * kStride;
  float* Ps = Os + hd * kStride;   // P^T [key][query]
  float* Ds = Ps + kBK * kStride;  // dS^T [key][query]
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int ktiles = (n + kBK - 1) / kBK;
  const long bh = blockIdx.x / ktiles;
  const int k0 = (int)(blockIdx.x - bh * ktiles) * kBK;
  const T* qb = static_cast<const T*>(p.q) + bh * n * hd;
  const T* dob = static_cast<const T*>(p.dout) + bh * n * hd;
  const float c2 = p.scale * kLog2e;
  load_columns<T>(Ks, static_cast<const T*>(p.kt) + bh * (long)hd * n, k0, n, hd);
  load_transposed<T, kBK>(Vs, kStride, static_cast<const T*>(p.v) + bh * n * hd, k0, n, hd);
  float dk[4][8], dv[4][8];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < 8; ++c) dk[a][c] = dv[a][c] = 0.f;
  for (int r0 = 0; r0 < n; r0 += kBK) {
    __syncthreads();
    load_transposed<T, kBK>(Qs, kStride, qb, r0, n, hd);
    load_transposed<T, kBK>(Os, kStride, dob, r0, n, hd);
    __syncthreads();
    const float4 d4 = __ldg(reinterpret_cast<const float4*>(p.dsum + bh * p.np + r0) + tx);
    const float dsum[4] = {d4.x, d4.y, d4.z, d4.w};
    float s[4][4], dp[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) s[a][b] = dp[a][b] = 0.f;
    dot_tile<4>(s, Ks, kStride, ty * 4, Qs, tx * 4, hd);
    dot_tile<4>(dp, Vs, kStride, ty * 4, Os, tx * 4, hd);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int key = k0 + ty * 4 + a, kh = key / w, kw = key - kh * w;
      // (the workspace rows are padded: the vectors stay inside them)
      const bool ok = key < n;
      const float4 rh = ok ? __ldg(reinterpret_cast<const float4*>(p.rel + (bh * hw + kh) * p.np + r0) + tx) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 rw = ok ? __ldg(reinterpret_cast<const float4*>(p.rel + (bh * hw + h + kw) * p.np + r0) + tx) : rh;
      const float bias[4] = {rh.x + rw.x, rh.y + rw.y, rh.z + rw.z, rh.w + rw.w};
      float pr[4], g[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const bool in = ok && r0 + tx * 4 + b < n;
        pr[b] = in ? exp2f(fmaf(s[a][b], c2, bias[b])) : 0.f;
        g[b] = in ? pr[b] * (dp[a][b] - dsum[b]) : 0.f;
      }
      *reinterpret_cast<float4*>(&Ps[(ty * 4 + a) * kStride + tx * 4]) = make_float4(pr[0], pr[1], pr[2], pr[3]);
      *reinterpret_cast<float4*>(&Ds[(ty * 4 + a) * kStride + tx * 4]) = make_float4(g[0], g[1], g[2], g[3]);
    }
    __syncthreads();
    mul_tile<4>(dv, Ps, ty * 4, Os, tx, hd);
    mul_tile<4>(dk, Ds, ty * 4, Qs, tx, hd);
  }
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const int key = k0 + ty * 4 + a;
    if (key < n) {
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

// dtable[e] = the CTAs' partial sums added in a fixed order. A block takes 32 elements; its 32 warps share the slots.
template <typename T>
__global__ void __launch_bounds__(1024) bwd_table_reduce(const float* __restrict__ partial, T* __restrict__ dtable,
                                                        int slots, int elems) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  sm100::wait_previous_launch();
  float s = 0.f;
  if (e < elems)
#pragma unroll 8
    for (int k = warp; k < slots; k += 32) s += partial[(long)k * elems + e];
  red[warp][lane] = s;
  __syncthreads();
  s = red[lane][warp];  // warp w adds element w's 32 shares
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int f = blockIdx.x * 32 + warp;
  if (lane == 0 && f < elems) dtable[f] = from_f<T>(s);
}

}  // namespace bwd
}  // namespace samrs
