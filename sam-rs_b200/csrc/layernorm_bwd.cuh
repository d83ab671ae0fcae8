// layernorm_bwd.cuh - gradients of LayerNorm (layernorm.cuh): y = xh * weight + bias, xh = (x - mean) rstd.
//   g = dy weight,  dx = rstd (g - mean(g) - xh mean(g xh)) (+ dres),  dweight = sum over rows of dy xh,
//   dbias = sum over rows of dy. Statistics are recomputed from x in f32, as the forward pass takes them.
// dres, where given, is the gradient of the residual stream the norm reads from (x + f(norm(x))): adding it here
// saves a pass over dx.
//
// Bound by memory: x, dy (and dres) read once, dx written once. A row belongs to W = ceil(c / 256) warps, 8 columns to a
// lane; a CTA holds as many such groups as 32 warps allow, each walking rows of its own with the next row's loads in
// flight (the lanes' registers are few, so an SM keeps 30 warps of loads going). The warps of a group meet twice per
// row (mean, then the three sums that need it). A lane meets the same columns in every row, so its share of dweight and
// dbias stays in registers; the groups of a CTA add theirs in order, and a second small launch adds the CTAs' in
// order: the result does not depend on scheduling.
#pragma once
#include "common.cuh"

namespace samrs {
namespace lnb {

constexpr int kThreads = 256;   // of the wide-row kernels
constexpr int kMaxCtas = 592;   // partial sums in the workspace
constexpr int kMaxCols = 8192;  // widest row of ln_bwd_kernel (32 warps)
constexpr int kPerLane = 8;     // columns of a lane

__host__ __device__ constexpr int row_warps(int c) { return (c + 32 * kPerLane - 1) / (32 * kPerLane); }
// Groups per CTA: up to 32 warps, and up to the 15 named barriers besides the CTA's own (one-warp groups need none).
__host__ __device__ constexpr int groups(int c) {
  return row_warps(c) == 1 ? 16 : 32 / row_warps(c) < 15 ? 32 / row_warps(c) : 15;
}

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

// partial: [gridDim.x][2][c] (dweight, dbias). Element e of a lane: column V (32 W e / V + lane of the group) + e % V.
template <typename T, int V>
__global__ void __launch_bounds__(1024, 1) ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                        const T* __restrict__ wt, const T* dres, T* dx,
                                                        float* __restrict__ partial, long rows, int c, float eps) {
  constexpr int NV = kPerLane / V;
  extern __shared__ float sums[];  // [groups][2][c]
  __shared__ float red[2][32][4];  // [parity][warp]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int W = row_warps(c), G = blockDim.x / 32 / W;
  const int grp = warp / W, gl = (warp - grp * W) * 32 + lane;  // group, lane of the group
  const long step = (long)gridDim.x * G;
  const float inv_c = 1.f / c;
  int col[NV];
  bool in[NV];
  Vec<T, V> vw[NV];
  float aw[NV][V], ab[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    col[k] = V * (k * 32 * W + gl);
    in[k] = col[k] < c;
    if (in[k])
      vw[k].load(wt + col[k]);
    else
      vw[k].zero();
#pragma unroll
    for (int e = 0; e < V; ++e) aw[k][e] = ab[k][e] = 0.f;
  }
  // the sums of a, b, d over the group's lanes
  auto group_sum = [&](int parity, float& a, float& b, float& d, int count) {
    a = warp_sum(a);
    if (count == 3) {
      b = warp_sum(b);
      d = warp_sum(d);
    }
    if (W == 1) return;
    if (lane == 0) {
      red[parity][warp][0] = a;
      red[parity][warp][1] = b;
      red[parity][warp][2] = d;
    }
    asm volatile("bar.sync %0, %1;" ::"r"(grp + 1), "r"(32 * W) : "memory");
    a = b = d = 0.f;
    for (int k = 0; k < W; ++k) {
      const float4 t = *reinterpret_cast<const float4*>(red[parity][grp * W + k]);
      a += t.x;
      b += t.y;
      d += t.z;
    }
  };
  Vec<T, V> nx[NV], ny[NV], nr[NV];
  auto load_row = [&](long row) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (in[k] && row < rows) {
        nx[k].load(x + row * c + col[k]);
        ny[k].load(dy + row * c + col[k]);
        if (dres) nr[k].load(dres + row * c + col[k]);
      } else {
        nx[k].zero();
        ny[k].zero();
      }
    }
  };
  long row = blockIdx.x * (long)G + grp;
  load_row(row);
  for (; row < rows; row += step) {
    float fx[NV][V], fy[NV][V], fr[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        fx[k][e] = nx[k].get(e);
        fy[k][e] = ny[k].get(e);
        fr[k][e] = dres && in[k] ? nr[k].get(e) : 0.f;
      }
    load_row(row + step);
    float s = 0.f, z0 = 0.f, z1 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) s += fx[k][e];
    group_sum(0, s, z0, z1, 1);
    const float mean = s * inv_c;
    float q = 0.f, s1 = 0.f, s2 = 0.f;  // sums of (x - mean)^2, g, g (x - mean)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = in[k] ? fx[k][e] - mean : 0.f, g = fy[k][e] * vw[k].get(e);
        fx[k][e] = d;
        q = fmaf(d, d, q);
        s1 += g;
        s2 = fmaf(g, d, s2);
      }
    group_sum(1, q, s1, s2, 3);
    const float rstd = rsqrtf(q * inv_c + eps);
    const float m1 = s1 * inv_c, m2 = s2 * inv_c * rstd;  // mean(g), mean(g xh)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = fx[k][e] * rstd;
        o[e] = rstd * (fy[k][e] * vw[k].get(e) - m1 - xh * m2) + fr[k][e];
        aw[k][e] = fmaf(fy[k][e], xh, aw[k][e]);
        ab[k][e] += fy[k][e];
      }
      if (in[k]) {
        Vec<T, V> vo;
        vo.set(o);
        vo.store(dx + row * c + col[k]);
      }
    }
  }
  float* own = sums + (size_t)grp * 2 * c;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (in[k])
#pragma unroll
      for (int e = 0; e < V; ++e) {
        own[col[k] + e] = aw[k][e];
        own[c + col[k] + e] = ab[k][e];
      }
  __syncthreads();
  for (int idx = threadIdx.x; idx < 2 * c; idx += blockDim.x) {
    float t = sums[idx];
    for (int k = 1; k < G; ++k) t += sums[(size_t)k * 2 * c + idx];
    partial[(long)blockIdx.x * 2 * c + idx] = t;
  }
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

// dweight | dbias = the partial sums in a fixed order: a block takes 32 of the 2c sums, its 32 warps share the slots.
template <typename T>
__global__ void __launch_bounds__(1024) ln_bwd_reduce(const float* __restrict__ partial, T* __restrict__ dwt,
                                                     T* __restrict__ dbs, int slots, int c) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (e < 2 * c)
#pragma unroll 8
    for (int k = warp; k < slots; k += 32) s += partial[(long)k * 2 * c + e];
  red[warp][lane] = s;
  __syncthreads();
  s = red[lane][warp];  // warp w adds column w's 32 shares
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int f = blockIdx.x * 32 + warp;
  if (lane == 0 && f < 2 * c) (f < c ? dwt[f] : dbs[f - c]) = from_f<T>(s);
}

}  // namespace lnb
}  // namespace samrs
