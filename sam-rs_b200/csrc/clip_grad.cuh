// clip_grad.cuh - the global norm of many gradient tensors and their clipping:
//   norm = sqrt(sum over all tensors of g^2),  out = g min(1, max_norm / (norm + 1e-6)).
// Bound by memory: every gradient is read for the norm and once more for the scaling, and written once. Two
// launches for up to kMaxTensors tensors: the list of tensors travels in the kernels' parameters. A CTA per SM takes
// every gridDim-th piece of 16 KB of whichever tensors they fall in; the pieces come by bulk copies into a ring of
// kStages of them (192 KB in flight per SM). Squares are added in f32 within a thread's part of a piece and in f64
// beyond, in an order that does not depend on scheduling; every CTA of the second launch adds the first one's sums
// itself, which costs it less than a third launch would. That launch takes the pieces from the last to the first, so
// that it begins with what the first one left in L2. Where the factor is 1, tensors clipped in place are left alone.
// 52 tensors of 79 million bf16 to f32: 38 + 91 us, 4.9 TB/s of what is moved (the gradients are read twice, L2 holds too
// little of them); 39 small f32 tensors: 4 + 4 us, and about 35 of the host's for the list.
#pragma once
#include "common.cuh"
#include "sm100.cuh"

#include <type_traits>

namespace samrs {
namespace clip {

constexpr int kThreads = 256;  // and a producer warp, which also finds the pieces for the others
constexpr int kPieceBytes = 16384;
constexpr int kStages = 12;
constexpr int kSmemBytes = kStages * kPieceBytes + 128;
constexpr int kMaxTensors = 512;
constexpr int kMaxCtas = 592;

struct List {
  const void* src[kMaxTensors];
  void* dst[kMaxTensors];
  int64_t numel[kMaxTensors];
  int first[kMaxTensors];  // the tensor's first piece
  uint8_t src_type[kMaxTensors], dst_type[kMaxTensors];  // SAMRS_F32 / F16 / BF16
  int count, pieces;
  int in_place;  // every tensor is clipped in place
};
static_assert(sizeof(List) <= 32000, "kernel parameters");

__host__ __device__ constexpr int piece_elems(int type) { return kPieceBytes / (type == 0 ? 4 : 2); }

struct Bars {
  uint64_t full[kStages], empty[kStages], factor;
  int abort_flag;
};

template <typename T>
__device__ __forceinline__ void unpack(uint4 u, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}

// Where a piece begins, how much of it there is, and how much of it comes by the ring (the rest, and all of a piece that
// does not begin on 16 bytes, is read directly). `t` is a tensor at or near the piece's.
struct Piece {
  const uint8_t* src;
  uint8_t* dst;
  int n, ring, src_type, dst_type;  // n, ring: elements
};
__device__ __forceinline__ Piece piece_at(const List& l, int piece, int& t) {
  while (l.first[t] > piece) --t;
  while (t + 1 < l.count && l.first[t + 1] <= piece) ++t;
  Piece p;
  p.src_type = l.src_type[t];
  p.dst_type = l.dst_type[t];
  const int size = p.src_type == 0 ? 4 : 2, each = piece_elems(p.src_type);
  const int64_t at = (int64_t)(piece - l.first[t]) * each;
  p.src = static_cast<const uint8_t*>(l.src[t]) + at * size;
  p.dst = static_cast<uint8_t*>(l.dst[t]) + at * (p.dst_type == 0 ? 4 : 2);
  p.n = (int)(l.numel[t] - at < each ? l.numel[t] - at : each);
  p.ring = (reinterpret_cast<uintptr_t>(p.src) & 15) ? 0 : p.n / (16 / size) * (16 / size);
  return p;
}

template <typename T>
__device__ __forceinline__ float square_sum(const Piece& p, const uint4* u) {
  constexpr int V = 16 / sizeof(T);
  float s = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < p.ring / V; i += kThreads) {
    float f[V];
    unpack<T>(u[i], f);
#pragma unroll
    for (int e = 0; e < V; ++e) s = fmaf(f[e], f[e], s);
  }
  const T* g = reinterpret_cast<const T*>(p.src);
  for (int i = p.ring + threadIdx.x; i < p.n; i += kThreads) {
    const float f = to_f(g[i]);
    s = fmaf(f, f, s);
  }
  return s;
}

// The stores are marked as not read again soon, so that they leave the gradients that wait for their turn in L2.
template <typename T, typename O>
__device__ __forceinline__ void scale_piece(const Piece& p, const uint4* u, float f) {
  constexpr int V = 16 / sizeof(T);
  O* o = reinterpret_cast<O*>(p.dst);
  const bool wide = (reinterpret_cast<uintptr_t>(o) & 15) == 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < p.ring / V; i += kThreads) {
    float x[V];
    unpack<T>(u[i], x);
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] *= f;
    if (!wide) {
#pragma unroll
      for (int e = 0; e < V; ++e) o[i * V + e] = from_f<O>(x[e]);
    } else if constexpr (sizeof(O) == 4) {
#pragma unroll
      for (int e = 0; e < V; e += 4)
        __stcs(reinterpret_cast<float4*>(o) + i * (V / 4) + e / 4, make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]));
    } else {
      uint32_t w[V / 2];
#pragma unroll
      for (int e = 0; e < V; e += 2) w[e / 2] = sm100::pack2(x[e], x[e + 1], std::is_same<O, __nv_bfloat16>::value);
      if constexpr (V == 8)
        __stcs(reinterpret_cast<uint4*>(o) + i, make_uint4(w[0], w[1], w[2], w[3]));
      else
        __stcs(reinterpret_cast<uint2*>(o) + i, make_uint2(w[0], w[1]));
    }
  }
  const T* g = reinterpret_cast<const T*>(p.src);
  for (int i = p.ring + threadIdx.x; i < p.n; i += kThreads) o[i] = from_f<O>(to_f(g[i]) * f);
}

template <typename T>
__device__ __forceinline__ void scale_to(const Piece& p, const uint4* u, float f) {
  if (p.dst_type == 0)
    scale_piece<T, float>(p, u, f);
  else if (p.dst_type == 1)
    scale_piece<T, __half>(p, u, f);
  else
    scale_piece<T, __nv_bfloat16>(p, u, f);
}

// kScale = false: the CTA's sum of squares to partial[blockIdx.x]. kScale = true: the norm from the `slots` partial sums,
// and the scaling.
template <bool kScale>
__global__ void __launch_bounds__(kThreads + 32, 1) clip_kernel(const __grid_constant__ List l, double* __restrict__ partial,
                                                               int slots, float max_norm, float* __restrict__ norm) {
  using namespace sm100;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  __shared__ Bars bars;
  __shared__ double red[kThreads / 32];
  __shared__ float factor;
  __shared__ Piece found[kStages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (__syncthreads_or(threadIdx.x == 0 && device_faulted())) return;
  if (threadIdx.x == 0) {
    for (int k = 0; k < kStages; ++k) {
      mbar_init(&bars.full[k], 1);
      mbar_init(&bars.empty[k], kThreads / 32);
    }
    mbar_init(&bars.factor, 1);
    bars.abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (kScale) wait_previous_launch();
  volatile int* abort_flag = &bars.abort_flag;
  const int mine = l.pieces > (int)blockIdx.x ? (l.pieces - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  auto piece_of = [&](int k) { return blockIdx.x + (kScale ? mine - 1 - k : k) * gridDim.x; };
  double s = 0.;
  float f = 0.f;

  if (warp == kThreads / 32) {
    if (lane == 0) {
      int t = 0;
      Armed copies;
      // tensors clipped in place are not even read where the factor is 1
      const bool go = !kScale || !l.in_place || mbar_wait_hot(&bars.factor, 0, abort_flag);
      if (go && !(kScale && l.in_place && factor == 1.f)) {
        for (; copies.n < mine; ++copies.n) {
          const int st = copies.n % kStages;
          if (copies.n >= kStages && !mbar_wait_hot(&bars.empty[st], ((copies.n / kStages) - 1) & 1, abort_flag)) break;
          const Piece p = piece_at(l, piece_of(copies.n), t);
          const uint32_t bytes = p.ring * (p.src_type == 0 ? 4 : 2);
          found[st] = p;
          if (bytes) {
            mbar_arrive_expect_tx(&bars.full[st], bytes);
            bulk_load(ring + st * kPieceBytes, p.src, bytes, &bars.full[st]);
          } else {
            mbar_arrive(&bars.full[st]);
          }
        }
      }
      copies.pending(kStages, [&](int k, uint32_t parity) { mbar_drain(&bars.full[k], parity); });
    }
  } else {
    bool work = true;
    if constexpr (kScale) {
      for (int k = threadIdx.x; k < slots; k += kThreads) s += partial[k];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) red[warp] = s;
      asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
      if (threadIdx.x == 0) {
        for (int k = 1; k < kThreads / 32; ++k) s += red[k];
        const float total = (float)sqrt(s);
        const float c = max_norm / (total + 1e-6f);
        factor = c > 1.f ? 1.f : c;  // a NaN stays one
        mbar_arrive(&bars.factor);
        if (blockIdx.x == 0) *norm = total;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
      f = factor;
      work = !(l.in_place && f == 1.f);
    }
    int st = 0;
    uint32_t ph = 0;
    for (int it = 0; it < mine && work; ++it) {
      if (!__all_sync(0xffffffffu, mbar_wait_hot(&bars.full[st], ph, abort_flag))) break;
      const Piece p = found[st];
      const uint4* u = reinterpret_cast<const uint4*>(ring + st * kPieceBytes);
      if constexpr (kScale) {
        if (f != 1.f || p.src != p.dst) {
          if (p.src_type == 0)
            scale_to<float>(p, u, f);
          else if (p.src_type == 1)
            scale_to<__half>(p, u, f);
          else
            scale_to<__nv_bfloat16>(p, u, f);
        }
      } else {
        if (p.src_type == 0)
          s += square_sum<float>(p, u);
        else if (p.src_type == 1)
          s += square_sum<__half>(p, u);
        else
          s += square_sum<__nv_bfloat16>(p, u);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.empty[st]);
      if (++st == kStages) st = 0, ph ^= 1;
    }
  }
  if constexpr (!kScale) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0 && warp < kThreads / 32) red[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < kThreads / 32; ++k) s += red[k];
      partial[blockIdx.x] = s;
    }
  }
}

}  // namespace clip
}  // namespace samrs
