// clip_grad.cuh - the global norm of many gradient tensors and their clipping:
//   norm = sqrt(sum over all tensors of g^2),  out = g min(1, max_norm / (norm + 1e-6)).
// Bound by memory: every gradient is read for the norm and once more for the scaling, and written once. Two
// launches for up to kMaxTensors tensors, however many there are: the list of tensors travels in the kernels'
// parameters, and a CTA takes fixed pieces of kPiece elements of whichever tensor they fall in. Squares are
// added in f32 within a thread's part of a piece and in f64 beyond, in an order that does not depend on
// scheduling; every CTA of the second launch adds the first one's sums itself, which costs it less than a
// third launch would. That launch walks the pieces backwards, so that it begins with what the first one left
// in L2, and leaves in-place tensors alone where the factor is 1.
#pragma once
#include "common.cuh"

namespace samrs {
namespace clip {

constexpr int kThreads = 512;
constexpr int kPiece = 16384;  // elements
constexpr int kMaxTensors = 512;
constexpr int kMaxCtas = 592;

struct List {
  const void* src[kMaxTensors];
  void* dst[kMaxTensors];
  int64_t numel[kMaxTensors];
  int first[kMaxTensors];  // the tensor's first piece
  uint8_t src_type[kMaxTensors], dst_type[kMaxTensors];  // SAMRS_F32 / F16 / BF16
  int count, pieces;
};
static_assert(sizeof(List) <= 32000, "kernel parameters");

__device__ __forceinline__ int find(const List& l, int piece) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= piece)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ void unpack(uint4 u, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else {
      T lo, hi;
      *reinterpret_cast<uint16_t*>(&lo) = (uint16_t)(w[i] & 0xFFFFu);
      *reinterpret_cast<uint16_t*>(&hi) = (uint16_t)(w[i] >> 16);
      f[2 * i] = to_f(lo);
      f[2 * i + 1] = to_f(hi);
    }
  }
}

// A piece's 16-byte vectors per thread, all loaded before the first is used.
template <typename T>
__host__ __device__ constexpr int vectors() { return kPiece * (int)sizeof(T) / 16 / kThreads; }

// Sum of squares of n elements, this thread's part of them.
template <typename T>
__device__ __forceinline__ float square_sum(const T* g, int n) {
  constexpr int V = 16 / sizeof(T), NV = vectors<T>();
  float s = 0.f;
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(g) & 15) == 0) {
    const uint4* g4 = reinterpret_cast<const uint4*>(g);
    const int nv = n / V;
    uint4 u[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = threadIdx.x + k * kThreads;
      u[k] = i < nv ? __ldg(g4 + i) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[V];
      unpack<T>(u[k], f);
#pragma unroll
      for (int e = 0; e < V; ++e) s = fmaf(f[e], f[e], s);
    }
    done = nv * V;
  }
  for (int i = done + threadIdx.x; i < n; i += kThreads) {
    const float f = to_f(g[i]);
    s = fmaf(f, f, s);
  }
  return s;
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ List l, double* __restrict__ partial) {
  __shared__ double red[kThreads / 32];
  double s = 0.;
  for (int piece = blockIdx.x; piece < l.pieces; piece += gridDim.x) {
    const int t = find(l, piece);
    const int64_t at = (int64_t)(piece - l.first[t]) * kPiece;
    const int n = (int)(l.numel[t] - at < kPiece ? l.numel[t] - at : kPiece);
    if (l.src_type[t] == 0)
      s += square_sum(static_cast<const float*>(l.src[t]) + at, n);
    else if (l.src_type[t] == 1)
      s += square_sum(static_cast<const __half*>(l.src[t]) + at, n);
    else
      s += square_sum(static_cast<const __nv_bfloat16*>(l.src[t]) + at, n);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kThreads / 32; ++k) s += red[k];
    partial[blockIdx.x] = s;
  }
}

template <typename T, typename O>
__device__ __forceinline__ void scale_piece(const T* g, O* o, int n, float f) {
  constexpr int V = 16 / sizeof(T), NV = vectors<T>();
  int done = 0;
  // 16-byte loads; as many elements leave as one or two 16-byte stores, or one 8-byte store. The stores are marked as
  // not read again soon, so that they leave the gradients that wait for their turn in L2.
  if (((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(o)) & 15) == 0) {
    const uint4* g4 = reinterpret_cast<const uint4*>(g);
    const int nv = n / V;
    uint4 u[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = threadIdx.x + k * kThreads;
      if (i < nv) u[k] = __ldcs(g4 + i);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = threadIdx.x + k * kThreads;
      if (i >= nv) break;
      float x[V];
      unpack<T>(u[k], x);
      if constexpr (sizeof(O) == 4) {
#pragma unroll
        for (int e = 0; e < V; e += 4)
          __stcs(reinterpret_cast<float4*>(o) + i * (V / 4) + e / 4,
                 make_float4(x[e] * f, x[e + 1] * f, x[e + 2] * f, x[e + 3] * f));
      } else {
        uint32_t w[V / 2];
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const O lo = from_f<O>(x[e] * f), hi = from_f<O>(x[e + 1] * f);
          w[e / 2] = (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | ((uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16);
        }
        if constexpr (V == 8)
          __stcs(reinterpret_cast<uint4*>(o) + i, make_uint4(w[0], w[1], w[2], w[3]));
        else
          __stcs(reinterpret_cast<uint2*>(o) + i, make_uint2(w[0], w[1]));
      }
    }
    done = nv * V;
  }
  for (int i = done + threadIdx.x; i < n; i += kThreads) o[i] = from_f<O>(to_f(g[i]) * f);
}

template <typename T>
__device__ __forceinline__ void scale_to(const List& l, int t, int64_t at, int n, float f) {
  const T* g = static_cast<const T*>(l.src[t]) + at;
  if (l.dst_type[t] == 0)
    scale_piece(g, static_cast<float*>(l.dst[t]) + at, n, f);
  else if (l.dst_type[t] == 1)
    scale_piece(g, static_cast<__half*>(l.dst[t]) + at, n, f);
  else
    scale_piece(g, static_cast<__nv_bfloat16*>(l.dst[t]) + at, n, f);
}

__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ List l, const double* __restrict__ partial,
                                                        int slots, float max_norm, float* __restrict__ norm) {
  __shared__ float factor;
  if (threadIdx.x < 32) {
    double s = 0.;
    for (int k = threadIdx.x; k < slots; k += 32) s += partial[k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) {
      const float total = (float)sqrt(s);
      const float c = max_norm / (total + 1e-6f);
      factor = c > 1.f ? 1.f : c;  // a NaN stays one
      if (blockIdx.x == 0) *norm = total;
    }
  }
  __syncthreads();
  const float f = factor;
  for (int piece = l.pieces - 1 - blockIdx.x; piece >= 0; piece -= gridDim.x) {
    const int t = find(l, piece);
    if (f == 1.f && l.src[t] == l.dst[t]) continue;
    const int64_t at = (int64_t)(piece - l.first[t]) * kPiece;
    const int n = (int)(l.numel[t] - at < kPiece ? l.numel[t] - at : kPiece);
    if (l.src_type[t] == 0)
      scale_to<float>(l, t, at, n, f);
    else if (l.src_type[t] == 1)
      scale_to<__half>(l, t, at, n, f);
    else
      scale_to<__nv_bfloat16>(l, t, at, n, f);
  }
}

}  // namespace clip
}  // namespace samrs
