// relpos_simt.cuh - CUDA-core kernels of the rel-pos attention path.
//
//  * relpos_attn_simt: fused flash-style attention with the decomposed rel-pos bias, any (h, w, hd<=128),
//    any dtype. It is the f32 path (f32 FMA arithmetic, expf) and the path for shapes the tensor-core
//    kernels do not cover. Math: src/kernels.rs:131-225 (cpu::TiledAttention), i.e.
//        x[r,k] = scale * q_r . kt[:,k] + q_r . Th[i-kh+h-1] + q_r . Tw[j-kw+w-1],  out_r = softmax_k(x) . v
//    computed with an online softmax over 64-key tiles, so no score row is ever stored.
//    Bound by the instructions issued: 16 multiplications of a lane for two 16-byte reads of shared memory, two CTAs of 8
//    warps to an SM to hide the loads. The bias takes the table's rows for keys (a dot product per row and grid line, a
//    table row to a lane, took longer than the attention). 30 heads of 7 x 11 x 80, f32: 27 us; 10 heads of
//    45 x 50 x 80: 0.99 ms in f32, 16 TFLOP/s, 1.12 in bf16.
//  * relpos_softmax_rows: the materialising probs-only op (src/kernels.rs:12-43 / 62-105,
//    kernels/sam.cu:44-106): one CTA per score row, two passes over the row (max/sum, then write).
//  * qkv_split: bias add + head split + K transpose (src/kernels.rs:234-263, kernels/sam.cu:108-128).
#pragma once
#include "common.cuh"

namespace samrs {

constexpr int kSimtBQ = 64;   // query rows per CTA
constexpr int kSimtBK = 64;   // keys per tile
constexpr int kSimtThreads = 256;
constexpr int kSimtMaxHd = 128;
constexpr int kSimtStride = 68;  // floats between the rows of a 64-wide tile: 16-byte reads, and 8 rows hit 32 banks

// How relpos_attn_simt lays out and loads its tiles; the results are the same bits.
//   kSimtPlain  P beside K.
//   kSimtShare  P over K, at a barrier more per tile: where only so two CTAs fit an SM. (4000 heads of 14 x 14 x 112, f32:
//               5.5 ms, 7.3 with one CTA; where two fit in any case it is 4 to 19 % slower from 8 x 8 on.)
//   kSimtTiny   P over K, and a head is one tile of few rows: only the rows that exist are loaded, all at once, and the bias
//               is a dot product per grid line (the table's few rows would cost a pass of 64 keys). (4000 heads of
//               1 x 1 x 64, bf16: 121 us against 215, of 5 x 5 x 64: 234 against 276.)
enum SimtForm { kSimtPlain, kSimtShare, kSimtTiny };
constexpr int kSimtTinyLines = 10;                                // h + w of a tiny grid: 25 tokens at most
constexpr size_t kSimtTwoCtas = (228 * 1024 / 2 - 1024) / 4;      // floats of a CTA of which two fit an SM

// Dynamic shared memory (floats) of relpos_attn_simt.
__host__ __device__ inline size_t simt_smem_floats(SimtForm form, int h, int w, int hd) {
  const size_t tile = (size_t)kSimtStride * hd, p = (size_t)kSimtStride * kSimtBQ;
  return 2 * tile + (form == kSimtPlain ? tile + p : tile > p ? tile : p) + (size_t)kSimtBQ * (h + w);
}
inline SimtForm simt_form(int h, int w, int hd) {
  if (h + w <= kSimtTinyLines) return kSimtTiny;
  return simt_smem_floats(kSimtPlain, h, w, hd) > kSimtTwoCtas && simt_smem_floats(kSimtShare, h, w, hd) <= kSimtTwoCtas
             ? kSimtShare
             : kSimtPlain;
}

// Rows r0 .. r0 + 63 of src [n][hd], transposed into dst[d][r]; rows past n are 0. A warp takes 4 rows x 8 columns at a time
// (whole sectors; the stores hit 32 banks), a batch of loads in flight.
template <typename T>
__device__ __forceinline__ void simt_load_rows(float* dst, const T* __restrict__ src, int r0, int n, int hd) {
  const int lane = threadIdx.x & 31, r = 4 * (threadIdx.x >> 5) + (lane >> 3);
  for (int d0 = lane & 7; d0 < hd; d0 += 32) {
    float v[4][2];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = r0 + r + 32 * k, d = d0 + 8 * e;
        v[e][k] = row < n && d < hd ? to_f(src[(long)row * hd + d]) : 0.f;
      }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (d0 + 8 * e < hd) dst[(d0 + 8 * e) * kSimtStride + r + 32 * k] = v[e][k];
  }
}
// s[a][b] = sum_d A[d][ra + a] B[d][cb + b], d ascending
__device__ __forceinline__ void simt_dot(float (&s)[4][4], const float* A, int ra, const float* B, int cb, int hd) {
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) s[a][b] = 0.f;
#pragma unroll 4
  for (int d = 0; d < hd; ++d) {
    const float4 qa = *reinterpret_cast<const float4*>(&A[d * kSimtStride + ra]);
    const float4 kb = *reinterpret_cast<const float4*>(&B[d * kSimtStride + cb]);
    const float qv[4] = {qa.x, qa.y, qa.z, qa.w};
    const float kv[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) s[a][b] = fmaf(qv[a], kv[b], s[a][b]);
  }
}

// grid.x = bh * ceil(n / 64); 256 threads. Thread (ty, tx) = (tid / 16, tid % 16) owns score rows
// ty*4..ty*4+3 x key columns tx*4..tx*4+3 of each tile, and output rows ty*4.. x columns tx + 16c.
template <typename T, SimtForm kForm>
__global__ void __launch_bounds__(kSimtThreads) relpos_attn_simt(const T* __restrict__ q, const T* __restrict__ kt,
                                                                 const T* __restrict__ v,
                                                                 const T* __restrict__ table, T* __restrict__ out,
                                                                 int h, int w, int hd, float scale,
                                                                 float* __restrict__ lse) {
  extern __shared__ float4 smem_f4[];
  float* smem = reinterpret_cast<float*>(smem_f4);
  const int n = h * w;
  const int qtiles = (n + kSimtBQ - 1) / kSimtBQ;
  const long bh = blockIdx.x / qtiles;
  const int r0 = (blockIdx.x % qtiles) * kSimtBQ;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;

  float* Qs = smem;                              // [hd][kSimtStride]
  float* Ks = Qs + kSimtStride * hd;             // K, before the keys the table's rows [hd][kSimtStride]
  float* Vs = Ks + kSimtStride * (kForm == kSimtPlain ? hd : max(hd, kSimtBQ));  // [hd][kSimtStride]
  float* Ps = kForm == kSimtPlain ? Vs + kSimtStride * hd : Ks;                  // [64][kSimtStride]
  float* rh_s = kForm == kSimtPlain ? Ps + kSimtBQ * kSimtStride : Vs + kSimtStride * hd;  // [64][h]
  float* rw_s = rh_s + kSimtBQ * h;                                                        // [64][w]

  const T* qb = q + (bh * n) * hd;
  const T* ktb = kt + bh * (long)hd * n;
  const T* vb = v + (bh * n) * hd;

  if constexpr (kForm == kSimtTiny) {
    for (int idx = tid; idx < n * hd; idx += kSimtThreads) {
      const int r = idx / hd, d = idx - r * hd, kd = idx / n, k = idx - kd * n;
      const float x = to_f(qb[idx]), y = to_f(ktb[idx]), z = to_f(vb[idx]);
      Qs[d * kSimtStride + r] = x;
      Ks[kd * kSimtStride + k] = y;
      Vs[d * kSimtStride + r] = z;
    }
    for (int d = tid; d < hd; d += kSimtThreads)
      for (int k = n; k & 3; ++k) Vs[d * kSimtStride + k] = 0.f;  // (P is zero there)
    __syncthreads();
    for (int idx = tid; idx < n * (h + w); idx += kSimtThreads) {
      const int r = idx % n, c = idx / n, i = r / w, j = r - i * w;
      const bool is_h = c < h;
      const T* line = table + (long)(is_h ? i + h - 1 - c : 2 * h - 1 + j + w - 1 - (c - h)) * hd;
      float u = 0.f;
#pragma unroll 4
      for (int d = 0; d < hd; ++d) u = fmaf(Qs[d * kSimtStride + r], to_f(line[d]), u);
      (is_h ? rh_s + r * h + c : rw_s + r * w + c - h)[0] = u;
    }
  } else {
    simt_load_rows(Qs, qb, r0, n, hd);
    // Rel-pos bias vectors of every row of the tile: rh_s[r][kh] = q_r . Th[i-kh+h-1], rw_s[r][kw] = q_r . Tw[j-kw+w-1]: the
    // table's rows pass like keys, and each product that a row has a key for goes to its place.
    const int tr = 2 * h - 1 + 2 * w - 1;
    int ri[4], rj[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      ri[a] = (r0 + ty * 4 + a) / w;
      rj[a] = (r0 + ty * 4 + a) % w;
    }
    for (int t0 = 0; t0 < tr; t0 += kSimtBK) {
      __syncthreads();
      simt_load_rows(Ks, table, t0, tr, hd);
      __syncthreads();
      float u[4][4];
      simt_dot(u, Qs, ty * 4, Ks, tx * 4, hd);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int t = t0 + tx * 4 + b;
        const bool is_h = t < 2 * h - 1;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int c = is_h ? ri[a] + h - 1 - t : rj[a] + w - 1 - (t - (2 * h - 1));
          if (t < tr && c >= 0 && c < (is_h ? h : w)) (is_h ? rh_s + (ty * 4 + a) * h : rw_s + (ty * 4 + a) * w)[c] = u[a][b];
        }
      }
    }
  }

  const int hdc = (hd + 15) / 16;  // output columns per thread (<= 8)
  float o[4][8];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < 8; ++c) o[a][c] = 0.f;
  float m_run[4], l_run[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    m_run[a] = -INFINITY;
    l_run[a] = 0.f;
  }

  for (int k0 = 0; k0 < n; k0 += kSimtBK) {
    __syncthreads();  // previous tile's Ks/Vs/Ps fully consumed (and rh/rw written on the first pass)
    if constexpr (kForm != kSimtTiny) {
      const int k = tid % kSimtBK;
      for (int d0 = tid / kSimtBK; d0 < hd; d0 += 32) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = d0 + 4 * j < hd && k0 + k < n ? to_f(ktb[(long)(d0 + 4 * j) * n + k0 + k]) : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (d0 + 4 * j < hd) Ks[(d0 + 4 * j) * kSimtStride + k] = x[j];
      }
      simt_load_rows(Vs, vb, k0, n, hd);
      __syncthreads();
    }

    float s[4][4];
    simt_dot(s, Qs, ty * 4, Ks, tx * 4, hd);
    if (kForm != kSimtPlain) __syncthreads();  // K has been read: P may go over it
    // bias + scale, masked keys -> -inf
    int khs[4], kws[4];
    bool valid[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int key = k0 + tx * 4 + b;
      valid[b] = key < n;
      khs[b] = key / w;
      kws[b] = key - khs[b] * w;
    }
    float alpha[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int r = ty * 4 + a;
      float mt = -INFINITY;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float x = -INFINITY;
        if (valid[b]) x = s[a][b] * scale + rh_s[r * h + khs[b]] + rw_s[r * w + kws[b]];
        s[a][b] = x;
        mt = fmaxf(mt, x);
      }
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, off));
      const float m_new = fmaxf(m_run[a], mt);
      alpha[a] = expf(m_run[a] - m_new);  // exp(-inf) = 0 on the first tile
      m_run[a] = m_new;
      float ls = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        s[a][b] = expf(s[a][b] - m_new);
        ls += s[a][b];
      }
      *reinterpret_cast<float4*>(&Ps[r * kSimtStride + tx * 4]) = make_float4(s[a][0], s[a][1], s[a][2], s[a][3]);
      l_run[a] = l_run[a] * alpha[a] + ls;
    }
    __syncthreads();
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 8; ++c) o[a][c] *= alpha[a];
    const int kmax = min(kSimtBK, n - k0);  // (the last step of 4 may run over it: zeros of P and V)
#pragma unroll 2
    for (int k = 0; k < kmax; k += 4) {
      float4 pv[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) pv[a] = *reinterpret_cast<const float4*>(&Ps[(ty * 4 + a) * kSimtStride + k]);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int d = tx + 16 * c;
        if (c < hdc && d < hd) {
          const float4 vv = *reinterpret_cast<const float4*>(&Vs[d * kSimtStride + k]);
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            o[a][c] = fmaf(pv[a].x, vv.x, o[a][c]);
            o[a][c] = fmaf(pv[a].y, vv.y, o[a][c]);
            o[a][c] = fmaf(pv[a].z, vv.z, o[a][c]);
            o[a][c] = fmaf(pv[a].w, vv.w, o[a][c]);
          }
        }
      }
    }
  }
  // Row sums are split over the 16 lanes of a row.
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    float l = l_run[a];
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const float inv = 1.f / l;
    const int row = r0 + ty * 4 + a;
    if (row < n) {
      if (lse && tx == 0) lse[bh * n + row] = m_run[a] + logf(l);  // log of the row's softmax sum
      T* orow = out + (bh * n + row) * hd;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int d = tx + 16 * c;
        if (c < hdc && d < hd) orow[d] = from_f<T>(o[a][c] * inv);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Probs-only rel-pos softmax: one CTA of 256 threads per score row.
// ------------------------------------------------------------------------------------------------
constexpr int kSoftmaxThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kSoftmaxThreads) relpos_softmax_rows(const T* __restrict__ s,
                                                                       const T* __restrict__ q,
                                                                       const T* __restrict__ table,
                                                                       T* __restrict__ out, int h, int w, int hd,
                                                                       float scale) {
  extern __shared__ float4 smem_f4[];
  float* sm = reinterpret_cast<float*>(smem_f4);
  float* qs = sm;        // [hd]
  float* rh = qs + hd;   // [h]
  float* rw = rh + h;    // [w]
  __shared__ float red_m[kSoftmaxThreads / 32], red_l[kSoftmaxThreads / 32];
  const int n = h * w;
  const long row = blockIdx.x;
  const int rem = (int)(row % n), i = rem / w, j = rem % w;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int d = tid; d < hd; d += kSoftmaxThreads) qs[d] = to_f(q[row * hd + d]);
  __syncthreads();
  // one warp per bias dot product
  for (int c = warp; c < h + w; c += kSoftmaxThreads / 32) {
    const bool is_h = c < h;
    const T* tr = is_h ? table + (long)(i - c + h - 1) * hd : table + (long)(2 * h - 1 + j - (c - h) + w - 1) * hd;
    float a = 0.f;
    for (int d = lane; d < hd; d += 32) a = fmaf(qs[d], to_f(tr[d]), a);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
    if (lane == 0) (is_h ? rh[c] : rw[c - h]) = a;
  }
  __syncthreads();
  const T* sr = s + row * n;
  // pass 1: per-thread running (max, sum), then a block merge
  float m = -INFINITY, l = 0.f;
  for (int k = tid; k < n; k += kSoftmaxThreads) {
    const int kh = k / w, kw = k - kh * w;
    const float x = to_f(sr[k]) * scale + rh[kh] + rw[kw];
    if (x > m) {
      l = l * expf(m - x) + 1.f;
      m = x;
    } else {
      l += expf(x - m);
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, off);
    const float l2 = __shfl_xor_sync(0xffffffffu, l, off);
    const float mm = fmaxf(m, m2);
    l = (m == -INFINITY ? 0.f : l * expf(m - mm)) + (m2 == -INFINITY ? 0.f : l2 * expf(m2 - mm));
    m = mm;
  }
  if (lane == 0) {
    red_m[warp] = m;
    red_l[warp] = l;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int wi = 0; wi < kSoftmaxThreads / 32; ++wi) M = fmaxf(M, red_m[wi]);
  float L = 0.f;
#pragma unroll
  for (int wi = 0; wi < kSoftmaxThreads / 32; ++wi)
    if (red_m[wi] != -INFINITY) L += red_l[wi] * expf(red_m[wi] - M);
  const float inv = 1.f / L;
  T* orow = out + row * n;
  for (int k = tid; k < n; k += kSoftmaxThreads) {
    const int kh = k / w, kw = k - kh * w;
    const float x = to_f(sr[k]) * scale + rh[kh] + rw[kw];
    orow[k] = from_f<T>(expf(x - M) * inv);
  }
}

// ------------------------------------------------------------------------------------------------
// qkv split. Each CTA takes one window and one head (blockIdx.x = win * nh + head) and a chunk of
// 32 tokens (blockIdx.y); the K block is transposed through shared memory so that both the reads of
// y and the writes of q, kt and v are coalesced.
// ------------------------------------------------------------------------------------------------
constexpr int kSplitTok = 32;

template <typename T>
__global__ void __launch_bounds__(256) qkv_split_kernel(const T* __restrict__ y, const T* __restrict__ bias,
                                                        T* __restrict__ outp, long tokens, int n, int nh, int hd) {
  extern __shared__ float4 smem_f4[];
  float* kbuf = reinterpret_cast<float*>(smem_f4);  // [kSplitTok][hd + 1]
  const long bhx = blockIdx.x;
  const long win = bhx / nh;
  const int head = (int)(bhx % nh);
  const int tok0 = blockIdx.y * kSplitTok;
  if (tok0 >= n) return;
  const int ntok = min(kSplitTok, n - tok0);
  const long c = (long)nh * hd;
  const long plane = tokens * c;
  T* qo = outp;
  T* ko = outp + plane;
  T* vo = outp + 2 * plane;
  const int tid = threadIdx.x;
  const int hdp = hd + 1;
  for (int idx = tid; idx < ntok * hd; idx += 256) {
    const int t = idx / hd, d = idx % hd;
    const long tokg = win * n + tok0 + t;
    const T* yrow = y + tokg * 3 * c;
    const long cq = (long)head * hd + d;
    qo[(bhx * n + tok0 + t) * hd + d] = from_f<T>(to_f(yrow[cq]) + to_f(bias[cq]));
    vo[(bhx * n + tok0 + t) * hd + d] = from_f<T>(to_f(yrow[2 * c + cq]) + to_f(bias[2 * c + cq]));
    kbuf[t * hdp + d] = to_f(yrow[c + cq]) + to_f(bias[c + cq]);
  }
  __syncthreads();
  for (int idx = tid; idx < ntok * hd; idx += 256) {
    const int d = idx / ntok, t = idx % ntok;
    ko[(bhx * hd + d) * n + tok0 + t] = from_f<T>(kbuf[t * hdp + d]);
  }
}

}  // namespace samrs
