// layernorm_bwd.cuh - gradients of LayerNorm (layernorm.cuh): y = xh * weight + bias, xh = (x - mean) rstd.
//   g = dy weight,  dx = rstd (g - mean(g) - xh mean(g xh)) (+ dres),  dweight = sum over rows of dy xh,
//   dbias = sum over rows of dy. Statistics are recomputed from x in f32, as the forward pass takes them.
// dres, where given, is the gradient of the residual stream the norm reads from (x + f(norm(x))): adding it here
// saves a pass over dx.
//
// Bound by memory: x, dy (and dres) read once, dx written once; next by instructions, of which a row split over several
// warps costs three times as many as a row to a warp (reductions, meetings). So a warp takes a whole row, up to 64
// columns to a lane (wider rows are split over W warps, which meet twice per row: mean, then the three sums that need
// it). A block of rows, one per warp, is contiguous in memory and comes by bulk copies into a ring of shared memory,
// 150 to 200 KB in flight per SM, which registers could not hold (rows that do not begin and end on 16 bytes come by
// plain loads). A lane meets the same columns in every row, so its share of dweight and dbias stays in registers; the warps
// of a CTA add theirs in order, and a second small launch adds the CTAs' in order: the result does not depend on
// scheduling.
// 32768 x 768 bf16 with dres: 43 us and 3 for the sums, 4.4 TB/s; 4096 x 1280 bf16: 15 and 3 us, 1.7 TB/s, where filling
// the ring, four rows to a warp and adding the warps' columns follow one another. f32 with dres: 4096 x 768 16 and 3 us,
// 32768 x 768 73 and 3, 5.3 TB/s; 4096 x 1280 32 and 3.
#pragma once
#include "common.cuh"
#include "sm100.cuh"

#include <type_traits>

namespace samrs {
namespace lnb {

constexpr int kThreads = 256;   // of the wide-row kernels
constexpr int kMaxCtas = 592;   // partial sums in the workspace
constexpr int kMaxCols = 7 * 64 * 32;  // widest row of ln_bwd_kernel
constexpr int kMaxStages = 8;

// Columns per lane (8, 16, ... 48, 64) of rows of c columns, the warps of a CTA besides the producer (about 3 registers
// per column and 40 more have to fit; at 40 columns 11 warps of 16-bit rows do, and take 15.2 us for 4096 x 1280 where 9 take
// 17.3, while f32 rows then spill, 22.8 us against 21.6), and the warps of a row. `es`: bytes of an element.
__host__ __device__ constexpr int per_lane(int c) { return c > 1536 ? 64 : c > 256 ? (c + 255) / 256 * 8 : 8; }
__host__ __device__ constexpr int cta_warps(int pl, int es) {
  return pl == 8 ? 23 : pl == 16 ? 19 : pl == 24 ? 15 : pl == 32 ? 11 : pl == 40 ? (es == 2 ? 11 : 9) : 7;
}
__host__ __device__ constexpr int row_warps(int c) { return (c + 32 * per_lane(c) - 1) / (32 * per_lane(c)); }
// Rows in work at a time: as many as registers allow, and with the ring, fewer where two stages of them would not fit
// `room` bytes of shared memory otherwise (f32 rows with dres from 512 columns on).
__host__ __device__ constexpr int groups(int c, int es) { return cta_warps(per_lane(c), es) / row_warps(c); }
__host__ __device__ constexpr int ring_groups(int c, int es, int tensors, int room) {
  int g = groups(c, es);
  while (g > 1 && 2 * g * c * es * tensors > room) --g;
  return g;
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
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return __uint_as_float(e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e >> 1]));
      return e & 1 ? f.y : f.x;
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = __float_as_uint(f[i]);
      else
        w[i] = sm100::pack2(f[2 * i], f[2 * i + 1], std::is_same<T, __nv_bfloat16>::value);
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
  __device__ __forceinline__ void set(const float* f) { t = from_f<T>(f[0]); }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Bars {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t meet[8];  // the warps of a row
  int abort_flag;
};

// partial: [gridDim.x][2][c] (dweight, dbias). Element e of a lane: column V (32 W (e / V) + lane of the row) + e % V.
// V > 1: the last warp is the producer of the ring of `stages` blocks. V = 1: plain loads, no producer.
// kFull: as many rows in work as registers allow, a constant up to 48 columns to a lane (3 % of 4096 x 768 f32).
template <typename T, int V, int PL, bool kFull>
__global__ void __launch_bounds__(32 * (cta_warps(PL, sizeof(T)) + 1), 1)
    ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ wt, const T* dres, T* dx,
                  float* __restrict__ partial, long rows, int c, float eps, int rows_in_work, int stages) {
  using namespace sm100;
  constexpr int NV = PL / V, N2 = PL / 2;
  constexpr bool kRing = V > 1;
  extern __shared__ float4 smem_f4[];  // the ring; at the end [groups][2][c] f32
  uint8_t* ring = reinterpret_cast<uint8_t*>(smem_f4);
  __shared__ float4 red[2][8];  // [parity][warp]
  __shared__ Bars bars;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int W = PL == 64 ? row_warps(c) : 1;
  const int G = PL < 64 && kFull ? cta_warps(PL, sizeof(T)) : rows_in_work;
  const int row_bytes = c * (int)sizeof(T), block_bytes = G * row_bytes;
  const int tensors = dres ? 3 : 2;
  const long blocks = (rows + G - 1) / G;
  if (__syncthreads_or(threadIdx.x == 0 && device_faulted())) return;
  if (threadIdx.x == 0) {
    for (int k = 0; k < stages; ++k) {
      mbar_init(&bars.full[k], 1);
      mbar_init(&bars.empty[k], W * G);
    }
    for (int k = 0; k < 8; ++k) mbar_init(&bars.meet[k], W);
    bars.abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  volatile int* abort_flag = &bars.abort_flag;
  const int grp = warp / W, gl = (warp - grp * W) * 32 + lane;  // row of the block, lane of the row
  float2 aw[N2], ab[N2];
#pragma unroll
  for (int k = 0; k < N2; ++k) aw[k] = ab[k] = make_float2(0.f, 0.f);
  auto col = [&](int k) { return V * (k * 32 * W + gl); };

  if (warp == W * G) {
    if (kRing && lane == 0) {
      Armed copies;
      int st = 0;
      uint32_t ph = 1;
      for (long b = blockIdx.x; b < blocks; b += gridDim.x, ++copies.n) {
        if (copies.n >= stages && !mbar_wait_hot(&bars.empty[st], ph, abort_flag)) break;
        const int n = (int)(rows - b * G < G ? rows - b * G : G) * row_bytes;
        uint8_t* dst = ring + (size_t)st * tensors * block_bytes;
        mbar_arrive_expect_tx(&bars.full[st], tensors * n);
        bulk_load(dst, x + b * G * c, n, &bars.full[st]);
        bulk_load(dst + block_bytes, dy + b * G * c, n, &bars.full[st]);
        if (dres) bulk_load(dst + 2 * block_bytes, dres + b * G * c, n, &bars.full[st]);
        if (++st == stages) st = 0, ph ^= 1;
      }
      copies.pending(stages, [&](int k, uint32_t parity) { mbar_drain(&bars.full[k], parity); });
    }
  } else if (warp < W * G) {
    const float inv_c = 1.f / c;
    uint32_t meets = 0;
    // the sums of a, b, d over the row's lanes (false: a wait has run out somewhere)
    auto row_sum = [&](int parity, float& a, float& b, float& d, bool three) {
      a = warp_sum(a);
      if (three) {
        b = warp_sum(b);
        d = warp_sum(d);
      }
      if (PL < 64 || W == 1) return true;
      if (lane == 0) {
        red[parity][warp] = make_float4(a, b, d, 0.f);
        mbar_arrive(&bars.meet[grp]);
      }
      if (!__all_sync(0xffffffffu, mbar_wait_hot(&bars.meet[grp], meets++ & 1, abort_flag))) return false;
      a = b = d = 0.f;
      for (int k = 0; k < W; ++k) {
        const float4 t = red[parity][grp * W + k];
        a += t.x;
        b += t.y;
        d += t.z;
      }
      return true;
    };
    // this lane's elements 2e, 2e + 1 of its vector k
    auto pair = [](const Vec<T, V>& lo, const Vec<T, V>& hi, int e) { return make_float2(lo.get(2 * e % V), hi.get((2 * e + 1) % V)); };
    int st = 0;
    uint32_t ph = 0;
    for (long row = (long)blockIdx.x * G + grp; row - grp < rows; row += (long)gridDim.x * G) {
      const T *xr = x + row * c, *yr = dy + row * c, *rr = dres + row * c;
      if constexpr (kRing) {
        if (!__all_sync(0xffffffffu, mbar_wait_hot(&bars.full[st], ph, abort_flag))) break;
        xr = reinterpret_cast<const T*>(ring + (size_t)st * tensors * block_bytes) + grp * c;
        yr = xr + G * c;
        rr = yr + G * c;
      }
      bool okk = true;
      if (row < rows) {
        float2 d[N2];
        constexpr int VP = V > 1 ? V / 2 : 1;  // pairs that a step of the loops below covers (V = 1: two vectors, one pair)
        constexpr int KS = V > 1 ? 1 : 2;
        auto load2 = [&](const T* p, int k, Vec<T, V>& lo, Vec<T, V>& hi) {
          lo.zero();
          if (col(k) < c) lo.load(p + col(k));
          if constexpr (V > 1) {
            hi = lo;
          } else {
            hi.zero();
            if (col(k + 1) < c) hi.load(p + col(k + 1));
          }
        };
        float2 t = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < NV; k += KS) {
          Vec<T, V> lo, hi;
          load2(xr, k, lo, hi);
#pragma unroll
          for (int e = 0; e < VP; ++e) {
            d[k * V / 2 + e] = pair(lo, hi, e);
            t = add2(t, d[k * V / 2 + e]);
          }
        }
        float s = t.x + t.y, z0 = 0.f, z1 = 0.f;
        okk = row_sum(0, s, z0, z1, false);
        const float mean = s * inv_c;
        const float2 nm = make_float2(-mean, -mean);
        float2 q = make_float2(0.f, 0.f), g1 = q, g2 = q;  // sums of (x - mean)^2, g, g (x - mean)
#pragma unroll
        for (int k = 0; k < NV; k += KS) {
          Vec<T, V> ylo, yhi, wlo, whi;
          load2(yr, k, ylo, yhi);
          load2(wt, k, wlo, whi);
#pragma unroll
          for (int e = 0; e < VP; ++e) {
            const int f = k * V / 2 + e;
            const float2 y = pair(ylo, yhi, e), w = pair(wlo, whi, e);
            d[f] = add2(d[f], nm);
            if (col(k) >= c) d[f].x = 0.f;  // past the row
            if (col(k + KS - 1) >= c) d[f].y = 0.f;
            const float2 g = mul2(y, w);
            q = fma2(d[f], d[f], q);
            g1 = add2(g1, g);
            g2 = fma2(g, d[f], g2);
          }
        }
        float qs = q.x + q.y, s1 = g1.x + g1.y, s2 = g2.x + g2.y;
        okk = okk && row_sum(1, qs, s1, s2, true);
        const float rstd = rsqrtf(qs * inv_c + eps);
        // dx = rstd (g - mean(g) - xh mean(g xh)), mean(g xh) = rstd s2 / c. (No power of rstd is formed: rows of tiny
        // deviation with eps = 0 have a rstd whose square or cube overflows, and finite gradients.)
        const float c0 = -s1 * inv_c, c1 = -(s2 * inv_c * rstd);
        const float2 c02 = make_float2(c0, c0), c12 = make_float2(c1, c1), r2 = make_float2(rstd, rstd);
#pragma unroll
        for (int k = 0; k < NV; k += KS) {
          Vec<T, V> ylo, yhi, wlo, whi, rlo, rhi;
          load2(yr, k, ylo, yhi);
          load2(wt, k, wlo, whi);
          if (dres) load2(rr, k, rlo, rhi);
          float o[2 * VP];
#pragma unroll
          for (int e = 0; e < VP; ++e) {
            const int f = k * V / 2 + e;
            const float2 y = pair(ylo, yhi, e), w = pair(wlo, whi, e);
            float2 v = mul2(fma2(mul2(d[f], r2), c12, fma2(y, w, c02)), r2);
            if (dres) v = add2(v, pair(rlo, rhi, e));
            o[2 * e] = v.x;
            o[2 * e + 1] = v.y;
            aw[f] = fma2(mul2(y, r2), d[f], aw[f]);
            ab[f] = add2(ab[f], y);
          }
          Vec<T, V> vo;
          if (okk && col(k) < c) {
            vo.set(o);
            vo.store(dx + row * c + col(k));
          }
          if constexpr (V == 1) {
            if (okk && col(k + 1) < c) {
              vo.set(o + 1);
              vo.store(dx + row * c + col(k + 1));
            }
          }
        }
      }
      if constexpr (kRing) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.empty[st]);
        if (++st == stages) st = 0, ph ^= 1;
      }
      if (!okk) break;
    }
  }
  __syncthreads();  // the ring has been read
  float* sums = reinterpret_cast<float*>(smem_f4);
  if (warp < W * G) {
    float* own = sums + (size_t)grp * 2 * c;
#pragma unroll
    for (int f = 0; f < PL; f += V > 1 ? 4 : 1) {
      const int at = col(f / V) + f % V;
      if (at < c) {
        if constexpr (V > 1) {  // (c is a multiple of V, and V of 4)
          *reinterpret_cast<float4*>(own + at) = make_float4(aw[f / 2].x, aw[f / 2].y, aw[f / 2 + 1].x, aw[f / 2 + 1].y);
          *reinterpret_cast<float4*>(own + c + at) = make_float4(ab[f / 2].x, ab[f / 2].y, ab[f / 2 + 1].x, ab[f / 2 + 1].y);
        } else {
          own[at] = f & 1 ? aw[f / 2].y : aw[f / 2].x;
          own[c + at] = f & 1 ? ab[f / 2].y : ab[f / 2].x;
        }
      }
    }
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
  sm100::wait_previous_launch();
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
