// relpos_bwd.cuh - host side of the attention's backward pass: workspace layout, kernel selection, launches.
#pragma once
#include <algorithm>

#include "common.cuh"
#include "relpos_bwd_simt.cuh"
#include "relpos_bwd_tc.cuh"
#include "relpos_tc.cuh"

namespace samrs {
namespace bwd {

// One partial sum of dtable per CTA of a persistent grid; at most two such CTAs share an SM.
constexpr int kMaxSlots = 296;
// Heads are taken in groups whose per-head arrays fit this many bytes: the workspace of a large batch stays
// bounded, and a group is still far more work than its launches cost.
constexpr int64_t kGroupBytes = (int64_t)256 << 20;

struct Plan {
  int64_t group;       // heads per group
  int64_t rel_bytes, dsum_bytes, partial_bytes;
  int64_t e_bytes, kt_bytes, amax_bytes;  // the tensor-core kernels' 0/1 matrix, padded kt, row norms
  int64_t total;
};

inline int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }
inline int round16(int x) { return (x + 15) / 16 * 16; }

// The shapes that the tensor-core kernels are written for (whether one fits shared memory too: dq_layout).
inline bool tc_shape(int h, int w, int hd, int dtype) { return dtype != 0 && hd % 16 == 0 && h <= 64 && w <= 64; }

inline Plan make_plan(int64_t bh, int h, int w, int hd, int dtype) {
  Plan p{};
  const int n = h * w;
  const int64_t np = padded_rows(n);
  const bool tc = tc_shape(h, w, hd, dtype);
  const int64_t rel = (int64_t)(h + w) * np * 4, dsum = np * 4;
  const int64_t kt = tc && n % 8 != 0 ? (int64_t)hd * ((n + 7) / 8 * 8) * 2 : 0;
  p.group = std::max<int64_t>(1, std::min<int64_t>(bh, kGroupBytes / (rel + dsum + kt)));
  p.rel_bytes = round256(p.group * rel);
  p.dsum_bytes = round256(p.group * dsum);
  p.partial_bytes = round256((int64_t)kMaxSlots * table_rows(h, w) * hd * 4);
  if (tc) {
    p.e_bytes = round256((int64_t)round16(h + w) * np * 2);
    p.kt_bytes = round256(p.group * kt);
    p.amax_bytes = round256(p.group * 8);
  }
  p.total = p.rel_bytes + p.dsum_bytes + p.partial_bytes + p.e_bytes + p.kt_bytes + p.amax_bytes;
  return p;
}

// 0, or an error for the caller to word: 1 shared memory, 2 grid.
template <typename T, int RQ>
int launch_dq_simt(const Args& a, int slots, int max_smem, cudaStream_t st) {
  const size_t smem = dq_smem_floats(16 * RQ, a.h, a.w, a.hd) * sizeof(float);
  if ((int)smem > max_smem) return 1;
  auto kern = bwd_dq_simt<T, RQ>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return 1;
  kern<<<slots, kThreads, smem, st>>>(a);
  return 0;
}

template <typename T>
int launch_simt(const Args& a, int slots, int max_smem, cudaStream_t st) {
  const int n = a.h * a.w;
  const int64_t ktiles = (n + kBK - 1) / kBK;
  if (a.bh * ktiles > 0x7fffffffLL) return 2;
  // 64 query rows per CTA where the bias rows of so many fit beside the tiles, else 32
  int rc = launch_dq_simt<T, 4>(a, slots, max_smem, st);
  if (rc == 1) rc = launch_dq_simt<T, 2>(a, slots, max_smem, st);
  if (rc) return rc;
  const size_t smem = dkv_smem_floats(a.hd) * sizeof(float);
  auto kern = bwd_dkv_simt<T>;
  if ((int)smem > max_smem ||
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return 1;
  kern<<<(unsigned)(a.bh * ktiles), kThreads, smem, st>>>(a);
  return 0;
}

// ------------------------------------------------------------------------------------ tensor cores
// 4-D map over a row-major [heads, rows, hd] 16-bit tensor whose box is `box_rows` rows x hd elements, laid out in shared
// memory as hd / 16 chunks of [rows][32 B]: dims (16, rows, hd / 16, heads). Past the tensor: zeros.
inline int make_chunk_map(CUtensorMap* map, bool bf16, const void* base, int hd, uint64_t rows, uint64_t heads, int box_hd,
                          uint32_t box_rows) {
  tcg::EncodeTiledFn fn = tcg::encode_fn();
  if (!fn) return 2;
  cuuint64_t dims[4] = {16, rows, (cuuint64_t)hd / 16, heads};
  cuuint64_t strides[3] = {(cuuint64_t)hd * 2, 32, rows * hd * 2};
  cuuint32_t box[4] = {16, box_rows, (cuuint32_t)box_hd / 16, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims,
            strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : 3;
}

// The same without the heads: dims (16, rows, hd / 16).
inline int make_chunk_map3(CUtensorMap* map, bool bf16, const void* base, int hd, uint64_t rows, int box_hd,
                           uint32_t box_rows) {
  tcg::EncodeTiledFn fn = tcg::encode_fn();
  if (!fn) return 2;
  cuuint64_t dims[3] = {16, rows, (cuuint64_t)hd / 16};
  cuuint64_t strides[2] = {(cuuint64_t)hd * 2, 32};
  cuuint32_t box[3] = {16, box_rows, (cuuint32_t)box_hd / 16};
  cuuint32_t es[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims,
            strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : 3;
}

// 3-D map of `elem` type with dims (d0, d1, d2), the row stride given in bytes, 128-byte swizzle.
inline int make_sw128_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t d0, uint64_t d1, uint64_t d2,
                          uint64_t row_bytes, uint32_t box0, uint32_t box1) {
  tcg::EncodeTiledFn fn = tcg::encode_fn();
  if (!fn) return 2;
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {row_bytes, row_bytes * d1};
  cuuint32_t box[3] = {box0, box1, 1};
  cuuint32_t es[3] = {1, 1, 1};
  return fn(map, type, 3, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : 3;
}

constexpr int kBarBytes = 512, kSlackBytes = 1024;  // barriers; rounding of the shared memory's base
static_assert(sizeof(TcBars) <= kBarBytes, "barrier block");

// Shared memory and TMEM of bwd_dq_tc, false if the shape does not fit; returns the bytes in `smem`.
inline bool dq_layout(TcArgs& t, int HD, int h, int w, bool w64, int max_smem, int* smem) {
  const int E = w64 ? 0 : round16(h + w);
  if (HD + E > 256) return false;
  t.e_rows = E;
  t.halves = table_rows(h, w) > 128 ? 2 : 1;
  const int t_s = 2 * HD + E;
  if (t_s + 128 > 512) return false;
  t.nbuf = t_s + 256 <= 512 ? 2 : 1;
  const int rel = (std::max((h + w) * 512, 2048) + 1023) / 1024 * 1024;
  t.off_tab = rel;
  t.off_q = t.off_tab + t.halves * 256 * HD;
  t.off_stage = t.off_q + 256 * HD;
  t.stage_bytes = (2 * HD + E) * 128;
  const int avail = max_smem - kSlackBytes - kBarBytes - t.off_stage, g = t.halves * 32768;
  t.nstages = std::min(4, avail / t.stage_bytes);
  if (g > avail || t.nstages < 1) return false;
  t.nbuf = std::min(t.nbuf, t.nstages);
  t.off_bar = t.off_stage + std::max(t.nstages * t.stage_bytes, g);
  *smem = t.off_bar + kBarBytes + kSlackBytes;
  return true;
}

// The key block of bwd_dkv_tc: th x tw = 128 with the fewest blocks over the grid, then with the fewest bias rows.
inline void dkv_block(TcArgs& t, int h, int w) {
  int best = 0x7fffffff;
  for (int tw = 1; tw <= 128; tw *= 2) {
    const int th = 128 / tw, nh = (h + th - 1) / th, nw = (w + tw - 1) / tw;
    const int cost = nh * nw * 1024 + th + tw;
    if (cost < best) {
      best = cost;
      t.th = th, t.tw = tw, t.tiles_h = nh, t.tiles_w = nw;
    }
  }
}

template <typename T, int HD>
int launch_tc_hd(TcArgs t, void* e, void* ktp, int slots, int max_smem, cudaStream_t st) {
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr CUtensorMapDataType type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const Args& a = t.a;
  const int h = a.h, w = a.w, n = h * w, hd = a.hd;
  const uint64_t bh = (uint64_t)a.bh;
  const bool w64 = w == 64;
  int smem = 0;
  if (!dq_layout(t, HD, h, w, w64, max_smem, &smem)) return 1;
  const void* kt = a.kt;
  int ktn = n;
  if (n % 8 != 0) {  // the TMA wants rows of a multiple of 16 bytes
    ktn = (n + 7) / 8 * 8;
    const int64_t total = a.bh * hd * (int64_t)ktn;
    bwd_pad_rows<<<(unsigned)std::min<int64_t>((total + 511) / 512, 2368), 512, 0, st>>>(
        static_cast<const uint16_t*>(a.kt), static_cast<uint16_t*>(ktp), a.bh * hd, n, ktn);
    kt = ktp;
  }
  CUtensorMap mk, mv, me, mq, mt, mq64, mo64, mh, mw;
  int rc = make_sw128_map(&mk, type, kt, n, hd, bh, (uint64_t)ktn * 2, 64, HD);
  if (!rc) rc = make_chunk_map(&mv, bf16, a.v, hd, n, bh, HD, kStep);
  if (!rc) rc = make_sw128_map(&me, type, w64 ? kt : e, w64 ? n : a.np, w64 ? hd : t.e_rows, 1, w64 ? (uint64_t)ktn * 2 : a.np * 2,
                               64, w64 ? 16 : t.e_rows);
  if (!rc) rc = make_chunk_map(&mq, bf16, a.q, hd, n, bh, HD, 128);
  if (!rc) rc = make_chunk_map3(&mt, bf16, a.table, hd, table_rows(h, w), HD, 128);
  if (rc) return 10 + rc;
  auto dq = w64 ? bwd_dq_tc<T, HD, true> : bwd_dq_tc<T, HD, false>;
  if (cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return 1;
  dq<<<slots, kTcThreads, smem, st>>>(mk, mv, me, mq, mt, t);

  dkv_block(t, h, w);
  const int64_t grid = a.bh * t.tiles_h * t.tiles_w;
  if (grid > 0x7fffffffLL) return 2;
  t.stage_bytes = dkv_stage_bytes(HD, t.th, t.tw);
  t.nstages = std::min(4, (max_smem - kBarBytes - kSlackBytes) / t.stage_bytes);
  if (t.nstages < 2) return 1;
  t.off_bar = t.nstages * t.stage_bytes;
  const int smem2 = t.off_bar + kBarBytes + kSlackBytes;
  rc = make_chunk_map(&mq64, bf16, a.q, hd, n, bh, HD, kStep);
  if (!rc) rc = make_chunk_map(&mo64, bf16, a.dout, hd, n, bh, HD, kStep);
  if (!rc) rc = make_sw128_map(&mh, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a.rel, a.np, h + w, bh, (uint64_t)a.np * 4, 32, t.th);
  if (!rc) rc = make_sw128_map(&mw, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a.rel, a.np, h + w, bh, (uint64_t)a.np * 4, 32, t.tw);
  if (rc) return 10 + rc;
  auto dkv = bwd_dkv_tc<T, HD>;
  if (cudaFuncSetAttribute(dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, smem2) != cudaSuccess) return 1;
  dkv<<<(unsigned)grid, kTcThreads, smem2, st>>>(mq64, mo64, mh, mw, t);
  return 0;
}

// The narrowest kernel that holds hd columns (further columns are zeros).
template <typename T>
int launch_tc(const TcArgs& t, void* e, void* ktp, int slots, int max_smem, cudaStream_t st) {
  const int hd = t.a.hd;
  if (hd <= 32) return launch_tc_hd<T, 32>(t, e, ktp, slots, max_smem, st);
  if (hd <= 64) return launch_tc_hd<T, 64>(t, e, ktp, slots, max_smem, st);
  if (hd <= 80) return launch_tc_hd<T, 80>(t, e, ktp, slots, max_smem, st);
  if (hd <= 96) return launch_tc_hd<T, 96>(t, e, ktp, slots, max_smem, st);
  return launch_tc_hd<T, 128>(t, e, ktp, slots, max_smem, st);
}

inline int tc_width(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 80 ? 80 : hd <= 96 ? 96 : 128; }

// Whether the tensor-core kernels take this call: shape, 16-byte aligned tensors (TMA and vector accesses), and a scale
// whose inverse is a finite factor of G.
inline bool tc_ok(const Args& a, int dtype, int max_smem) {
  if (!tc_shape(a.h, a.w, a.hd, dtype)) return false;
  const void* ptrs[] = {a.q, a.kt, a.v, a.table, a.out, a.dout, a.dq, a.dkt, a.dv};
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  const float s = a.scale < 0 ? -a.scale : a.scale;
  if (!(s >= 0x1p-20f && s <= 0x1p20f)) return false;
  TcArgs t{};
  int smem = 0;
  return dq_layout(t, tc_width(a.hd), a.h, a.w, a.w == 64, max_smem, &smem);
}

// The whole backward pass of bh >= 1 heads. `a` holds the whole batch's pointers, the workspace is cut here. Returns 0,
// 1 shared memory, 2 grid, 10 + a tensor map error.
template <typename T>
int launch_bwd(Args a, int64_t bh, void* workspace, const Plan& plan, bool tc, int num_sms, int max_smem, cudaStream_t st) {
  const int64_t n = (int64_t)a.h * a.w, per_head = n * a.hd;
  char* ws = static_cast<char*>(workspace);
  auto cut = [&](int64_t bytes) {
    char* at = ws;
    ws += bytes;
    return at;
  };
  a.rel = reinterpret_cast<float*>(cut(plan.rel_bytes));
  a.dsum = reinterpret_cast<float*>(cut(plan.dsum_bytes));
  a.partial = reinterpret_cast<float*>(cut(plan.partial_bytes));
  void* e = cut(plan.e_bytes);
  void* ktp = cut(plan.kt_bytes);
  unsigned int* amax = reinterpret_cast<unsigned int*>(cut(plan.amax_bytes));
  a.np = padded_rows((int)n);
  const Args whole = a;
  const int64_t qtiles = tc ? (n + 127) / 128 : (n + 63) / 64;
  const int slots = (int)std::min<int64_t>(std::min<int64_t>(plan.group, bh) * qtiles, std::min(num_sms, kMaxSlots));
  if (tc && a.w != 64) {
    const int rows = round16(a.h + a.w);
    bwd_indicator<<<std::min((rows * a.np + 255) / 256, 592), 256, 0, st>>>(
        static_cast<uint16_t*>(e), rows, a.np, a.h, a.w, std::is_same<T, __half>::value ? 0x3C00 : 0x3F80);
  }
  for (int64_t b0 = 0; b0 < bh; b0 += plan.group) {
    a.bh = std::min(plan.group, bh - b0);
    a.first = b0 == 0;
    a.q = static_cast<const T*>(whole.q) + b0 * per_head;
    a.kt = static_cast<const T*>(whole.kt) + b0 * per_head;
    a.v = static_cast<const T*>(whole.v) + b0 * per_head;
    a.out = static_cast<const T*>(whole.out) + b0 * per_head;
    a.dout = static_cast<const T*>(whole.dout) + b0 * per_head;
    a.lse = whole.lse + b0 * n;
    a.dq = static_cast<T*>(whole.dq) + b0 * per_head;
    a.dkt = static_cast<T*>(whole.dkt) + b0 * per_head;
    a.dv = static_cast<T*>(whole.dv) + b0 * per_head;
    int rc;
    if constexpr (sizeof(T) == 2) {
      if (tc) {
        TcArgs t{};
        t.a = a;
        if constexpr (std::is_same<T, __half>::value) {
          const float s = a.scale < 0 ? -a.scale : a.scale;
          t.amax = amax;
          t.gain = 8192.f * std::min(1.f, s);  // G holds sums of dS over scale
          if (cudaMemsetAsync(amax, 0, a.bh * 8, st) != cudaSuccess) return 0;  // the caller reads the error
          const dim3 grid((unsigned)a.bh, (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + 31) / 32, 592 / a.bh)));
          bwd_row_norms<<<grid, 256, 0, st>>>(static_cast<const __half*>(a.dout), static_cast<const __half*>(a.v), amax, (int)n,
                                              a.hd);
        }
        rc = launch_tc<T>(t, e, ktp, slots, max_smem, st);
      } else {
        rc = launch_simt<T>(a, slots, max_smem, st);
      }
    } else {
      rc = launch_simt<T>(a, slots, max_smem, st);
    }
    if (rc) return rc;
  }
  const int elems = table_rows(a.h, a.w) * a.hd;
  bwd_table_reduce<T><<<(elems + 31) / 32, 256, 0, st>>>(a.partial, static_cast<T*>(a.dtable), slots, elems);
  return 0;
}

}  // namespace bwd
}  // namespace samrs
