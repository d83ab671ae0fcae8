// layernorm_bwd.cuh - gradients of LayerNorm (layernorm.cuh): y = xh * weight + bias, xh = (x - mean) rstd.
//   g = dy weight,  dx = rstd (g - mean(g) - xh mean(g xh)) (+ dres),  dweight = sum over rows of dy xh,
//   dbias = sum over rows of dy. Statistics are recomputed from x in f32, as the forward pass takes them.
// dres, where given, is the gradient of the residual stream the norm reads from (x + f(norm(x))): adding it here
// saves a pass over dx.
//
// Bound by memory: x, dy (and dres) read once, dx written once. One warp per row, the row's x and dy held in
// registers; each lane owns the same columns of every row it meets, so its share of dweight and dbias stays in
// registers too. The warps of a CTA add their shares in warp order, a second small launch adds the CTAs' in
// CTA order: the result does not depend on scheduling.
#pragma once
#include "common.cuh"

namespace samrs {
namespace lnb {

constexpr int kThreads = 256;
constexpr int kMaxCtas = 592;  // partial sums in the workspace
constexpr int kMaxCols = 2048; // widest row of the register kernel (64 columns per lane)

// V consecutive elements as they sit in memory.
template <typename T, int V>
struct Vec {
  static_assert(V * sizeof(T) == 16 || V == 1, "16-byte vectors or single elements");
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = u; }
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[e]);
    } else {
      T t;
      *reinterpret_cast<uint16_t*>(&t) = (uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu);
      return to_f(t);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(f[i]);
      } else {
        const T lo = from_f<T>(f[2 * i]), hi = from_f<T>(f[2 * i + 1]);
        w[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | ((uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16);
      }
    }
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
struct Vec<T, 1> {
  T t;
  __device__ __forceinline__ void load(const T* p) { t = *p; }
  __device__ __forceinline__ void zero() { t = from_f<T>(0.f); }
  __device__ __forceinline__ void store(T* p) const { *p = t; }
  __device__ __forceinline__ float get(int) const { return to_f(t); }
  __device__ __forceinline__ void set(const float (&f)[1]) { t = from_f<T>(f[0]); }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rows of up to 32 V NCH columns. partial: [gridDim.x][2][c] (dweight, dbias).
template <typename T, int V, int NCH>
__global__ void __launch_bounds__(kThreads) ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                         const T* __restrict__ wt, const T* dres, T* dx,
                                                         float* __restrict__ partial, long rows, int c, float eps) {
  extern __shared__ float sums[];  // [2][c]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long step = (long)gridDim.x * (kThreads / 32);
  float aw[NCH][V], ab[NCH][V];
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) aw[k][e] = ab[k][e] = 0.f;

  const float inv_c = 1.f / c;
  for (long row = blockIdx.x * (long)(kThreads / 32) + warp; row < rows; row += step) {
    const T *xr = x + row * c, *yr = dy + row * c;
    Vec<T, V> vx[NCH], vy[NCH];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int col = V * (lane + 32 * k);
      if (col < c) {
        vx[k].load(xr + col);
        vy[k].load(yr + col);
      } else {
        vx[k].zero();
        vy[k].zero();
      }
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) s += vx[k].get(e);
    const float mean = warp_sum(s) * inv_c;
    float q = 0.f, s1 = 0.f, s2 = 0.f;  // sums of (x - mean)^2, g, g (x - mean)
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int col = V * (lane + 32 * k);
      if (col < c) {
        Vec<T, V> vw;
        vw.load(wt + col);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = vx[k].get(e) - mean, g = vy[k].get(e) * vw.get(e);
          q = fmaf(d, d, q);
          s1 += g;
          s2 = fmaf(g, d, s2);
        }
      }
    }
    q = warp_sum(q);
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    const float rstd = rsqrtf(q * inv_c + eps);
    const float m1 = s1 * inv_c, m2 = s2 * inv_c * rstd;  // mean(g), mean(g xh)
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int col = V * (lane + 32 * k);
      if (col < c) {
        Vec<T, V> vw, vr, vo;
        vw.load(wt + col);
        if (dres) vr.load(dres + row * c + col);
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float y = vy[k].get(e), xh = (vx[k].get(e) - mean) * rstd;
          o[e] = rstd * (y * vw.get(e) - m1 - xh * m2);
          if (dres) o[e] += vr.get(e);
          aw[k][e] = fmaf(y, xh, aw[k][e]);
          ab[k][e] += y;
        }
        vo.set(o);
        vo.store(dx + row * c + col);
      }
    }
  }
  for (int wv = 0; wv < kThreads / 32; ++wv) {
    if (warp == wv) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const int col = V * (lane + 32 * k);
        if (col < c) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sums[col + e] = wv ? sums[col + e] + aw[k][e] : aw[k][e];
            sums[c + col + e] = wv ? sums[c + col + e] + ab[k][e] : ab[k][e];
          }
        }
      }
    }
    __syncthreads();
  }
  for (int idx = threadIdx.x; idx < 2 * c; idx += kThreads) partial[(long)blockIdx.x * 2 * c + idx] = sums[idx];
}

// Rows of any width, one CTA per row: dx, and the row's mean and rstd for ln_bwd_cols.
template <typename T>
__global__ void __launch_bounds__(kThreads) ln_bwd_rows(const T* __restrict__ dy, const T* __restrict__ x,
                                                       const T* __restrict__ wt, const T* dres, T* dx,
                                                       float2* __restrict__ stats, long rows, int c, float eps) {
  __shared__ float red[3][kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto block_sum3 = [&](float& a, float& b, float& d) {
    a = warp_sum(a);
    b = warp_sum(b);
    d = warp_sum(d);
    __syncthreads();
    if (lane == 0) {
      red[0][warp] = a;
      red[1][warp] = b;
      red[2][warp] = d;
    }
    __syncthreads();
    a = b = d = 0.f;
    for (int k = 0; k < kThreads / 32; ++k) {
      a += red[0][k];
      b += red[1][k];
      d += red[2][k];
    }
  };
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * c, *yr = dy + row * c;
    float s = 0.f, z0 = 0.f, z1 = 0.f;
    for (int i = threadIdx.x; i < c; i += kThreads) s += to_f(xr[i]);
    block_sum3(s, z0, z1);
    const float mean = s / c;
    float q = 0.f, s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < c; i += kThreads) {
      const float d = to_f(xr[i]) - mean, g = to_f(yr[i]) * to_f(wt[i]);
      q = fmaf(d, d, q);
      s1 += g;
      s2 = fmaf(g, d, s2);
    }
    block_sum3(q, s1, s2);
    const float rstd = rsqrtf(q / c + eps), m1 = s1 / c, m2 = s2 / c * rstd;
    for (int i = threadIdx.x; i < c; i += kThreads) {
      const float xh = (to_f(xr[i]) - mean) * rstd;
      float o = rstd * (to_f(yr[i]) * to_f(wt[i]) - m1 - xh * m2);
      if (dres) o += to_f(dres[row * c + i]);
      dx[row * c + i] = from_f<T>(o);
    }
    if (threadIdx.x == 0) stats[row] = make_float2(mean, rstd);
  }
}

// dweight and dbias of wide rows: a CTA takes 32 columns (its 8 warps share the rows) and a slice of the rows.
// partial: [gridDim.y][2][c].
template <typename T>
__global__ void __launch_bounds__(kThreads) ln_bwd_cols(const T* __restrict__ dy, const T* __restrict__ x,
                                                       const float2* __restrict__ stats, float* __restrict__ partial,
                                                       long rows, int c) {
  __shared__ float red[2][kThreads / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float a = 0.f, b = 0.f;
  if (col < c)
    for (long row = blockIdx.y * (long)(kThreads / 32) + warp; row < rows; row += (long)gridDim.y * (kThreads / 32)) {
      const float2 st = stats[row];
      const float y = to_f(dy[row * c + col]);
      a = fmaf(y, (to_f(x[row * c + col]) - st.x) * st.y, a);
      b += y;
    }
  red[0][warp][lane] = a;
  red[1][warp][lane] = b;
  __syncthreads();
  if (warp == 0 && col < c) {
    for (int k = 1; k < kThreads / 32; ++k) {
      a += red[0][k][lane];
      b += red[1][k][lane];
    }
    partial[(long)blockIdx.y * 2 * c + col] = a;
    partial[(long)blockIdx.y * 2 * c + c + col] = b;
  }
}

// dweight | dbias = the partial sums in a fixed order: a block takes 32 of the 2c sums, its 8 warps share the slots.
template <typename T>
__global__ void __launch_bounds__(kThreads) ln_bwd_reduce(const float* __restrict__ partial, T* __restrict__ dwt,
                                                         T* __restrict__ dbs, int slots, int c) {
  __shared__ float red[kThreads / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (e < 2 * c)
#pragma unroll 4
    for (int k = warp; k < slots; k += kThreads / 32) s += partial[(long)k * 2 * c + e];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && e < 2 * c) {
    for (int k = 1; k < kThreads / 32; ++k) s += red[k][lane];
    (e < c ? dwt[e] : dbs[e - c]) = from_f<T>(s);
  }
}

}  // namespace lnb
}  // namespace samrs
