// relpos_bwd.cuh - host side of the attention's backward pass: workspace layout, kernel selection, launches.
#pragma once
#include <algorithm>

#include "common.cuh"
#include "relpos_bwd_simt.cuh"
#include "relpos_bwd_tc.cuh"
#include "relpos_tc.cuh"

namespace samrs {
namespace bwd {

// One partial sum of dtable per CTA of a persistent grid: one CTA per SM at least, more where that stays small.
constexpr int kMinSlots = 148, kMaxSlots = 592;
constexpr int64_t kPartialBytes = (int64_t)32 << 20;
// Heads are taken in groups whose per-head arrays fit this many bytes: the workspace of a large batch stays
// bounded, and a group is still far more work than its launches cost.
constexpr int64_t kGroupBytes = (int64_t)256 << 20;

struct Plan {
  int64_t group;       // heads per group
  int slots;           // partial sums of dtable
  int64_t rel_bytes, dsum_bytes, partial_bytes;
  int64_t rw_bytes, kt_bytes, amax_bytes;  // the tensor-core kernels' rw, padded kt, row norms
  int64_t total;
};

inline int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }

// The shapes that the tensor-core kernels are written for (whether one fits shared memory too: dq_layout).
inline bool tc_shape(int h, int w, int hd, int dtype) { return dtype != 0 && hd % 16 == 0 && h <= 64 && w <= 64; }

// Blocks of a head in bwd_prepare's row norms: 128 rows at least to each.
inline int norm_blocks(int n) { return std::min(16, (n + 127) / 128); }

inline Plan make_plan(int64_t bh, int h, int w, int hd, int dtype) {
  Plan p{};
  const int n = h * w;
  const int64_t np = padded_rows(n);
  const bool tc = tc_shape(h, w, hd, dtype);
  // (the tensor-core kernels keep rw apart, and pad both to 16 rows)
  const int64_t rel = (int64_t)(tc ? round_up(h, 16) : h + w) * np * 4, dsum = np * 4;
  const int64_t rw = tc ? (int64_t)round_up(w, 16) * np * 4 : 0;
  const int64_t kt = tc && w % 8 != 0 ? (int64_t)hd * h * round_up(w, 8) * 2 : 0;
  // the SIMT kernels may run in place of the tensor-core ones (misaligned tensors): room for either
  const int64_t either = std::max(rel + rw, (int64_t)(h + w) * np * 4);
  p.group = std::max<int64_t>(1, std::min<int64_t>(bh, kGroupBytes / (either + dsum + kt)));
  p.rel_bytes = round256(p.group * rel);
  p.rw_bytes = round256(p.group * (either - rel));
  p.dsum_bytes = round256(p.group * dsum);
  const int64_t sum = (int64_t)table_rows(h, w) * hd * 4;
  p.slots = (int)std::max<int64_t>(kMinSlots, std::min<int64_t>(kMaxSlots, kPartialBytes / sum));
  p.partial_bytes = round256(p.slots * sum);
  if (tc) {
    p.kt_bytes = round256(p.group * kt);
    p.amax_bytes = round256(p.group * 8 * norm_blocks(n));
  }
  p.total = p.rel_bytes + p.rw_bytes + p.dsum_bytes + p.partial_bytes + p.kt_bytes + p.amax_bytes;
  return p;
}

// How a CUDA-core kernel runs: groups of warps to a CTA (0: it does not fit), CTAs resident at once.
struct SimtRun {
  int groups, resident;
};
// Groups that share a tile cost memory for their own buffers, and save the tile's; 16 warps are resident in any case where
// that fits (launch bounds). What counts is the steps that one group takes in all rounds of tiles.
template <typename Smem>
SimtRun simt_run(int64_t tiles, int steps, Smem smem_floats, int most, int num_sms, int max_smem) {
  SimtRun best{0, 0};
  int64_t least = 0;
  for (int g = 1; g <= 4; g *= 2) {
    const int64_t smem = smem_floats(g) * 4;
    if (smem > max_smem) break;
    const int per_sm = (int)std::min<int64_t>(4 / g, (max_smem + 1024) / (smem + 1024));  // (1 KB of each CTA is the system's)
    const int resident = std::min(per_sm * num_sms, most);
    const int64_t cost = (tiles + resident - 1) / resident * ((steps + g - 1) / g);
    if (best.groups == 0 || cost < least) best = {g, resident}, least = cost;
  }
  return best;
}
inline SimtRun simt_dq(int64_t bh, int h, int w, int hd, int num_sms, int max_smem) {
  const int n = h * w;
  return simt_run(bh * ((n + kBR - 1) / kBR), (n + kKeys - 1) / kKeys, [=](int g) { return dq_smem_floats(g, h, w, hd); },
                  kMaxSlots, num_sms, max_smem);
}

template <typename Kernel>
bool launch_simt_as(Kernel kern, const Args& a, unsigned grid, int groups, int64_t smem_floats, cudaStream_t st) {
  const int smem = (int)smem_floats * 4;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
  kern<<<grid, kGroup * groups, smem, st>>>(a);
  return true;
}

// 0, or an error for the caller to word: 1 shared memory, 2 grid.
template <typename T>
int launch_simt(const Args& a, int groups, int slots, int num_sms, int max_smem, cudaStream_t st) {
  const int n = a.h * a.w, hd = a.hd;
  const int64_t ktiles = a.bh * ((n + kBR - 1) / kBR);
  if (ktiles > 0x7fffffffLL) return 2;
  const SimtRun kv = simt_run(ktiles, (n + kQueries - 1) / kQueries, [=](int g) { return dkv_smem_floats(g, hd); },
                              0x7fffffff, num_sms, max_smem);
  auto dq = groups == 1 ? bwd_dq_simt<T, 1> : groups == 2 ? bwd_dq_simt<T, 2> : bwd_dq_simt<T, 4>;
  auto dkv = kv.groups == 1 ? bwd_dkv_simt<T, 1> : kv.groups == 2 ? bwd_dkv_simt<T, 2> : bwd_dkv_simt<T, 4>;
  if (kv.groups == 0 || !launch_simt_as(dq, a, slots, groups, dq_smem_floats(groups, a.h, a.w, hd), st) ||
      !launch_simt_as(dkv, a, (unsigned)ktiles, kv.groups, dkv_smem_floats(kv.groups, hd), st))
    return 1;
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

// The general form: `rank` dims, strides in bytes from the second dim on.
inline int make_map_nd(CUtensorMap* map, CUtensorMapDataType type, const void* base, int rank, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle sw) {
  tcg::EncodeTiledFn fn = tcg::encode_fn();
  if (!fn) return 2;
  const cuuint32_t es[5] = {1, 1, 1, 1, 1};
  return fn(map, type, rank, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : 3;
}

constexpr int kBarBytes = 512, kSlackBytes = 1024;  // barriers; rounding of the shared memory's base
static_assert(sizeof(TcBars) <= kBarBytes, "barrier block");

// Shared memory and TMEM of bwd_dq_tc, false if the shape does not fit; returns the bytes in `smem`.
inline bool dq_layout(TcArgs& t, int HD, int h, int w, int max_smem, int* smem) {
  const int hp = blocks_h(h, w) * kBandH, wp = bands(w) * kBandW;
  t.halves = table_rows(h, w) > 128 ? 2 : 1;
  const int t_s = 2 * HD + wp;
  if (t_s + 128 > 512) return false;
  t.nbuf = t_s + 256 <= 512 ? 2 : 1;
  t.stage_bytes = 2 * HD * 128;
  const int rel = (hp + wp) * 512, g = t.halves * 32768, drh = std::max(hp * 512, 2048);
  const int fixed = drh + kEBytes + t.halves * 256 * HD + 256 * HD + kBarBytes + kSlackBytes;
  // G's two terms side by side where that leaves room for three stages
  // (the region holds dO and O before rel and G, and with drh the rows of dtable after them)
  const int least = std::max(std::max(rel, 512 * HD), table_rows(h, w) * (4 * HD + 16) - drh);
  int work = round_up(std::max(least, 2 * g), 1024);
  t.split = max_smem - fixed - work >= 3 * t.stage_bytes;
  if (!t.split) work = round_up(std::max(least, g), 1024);
  t.nstages = std::min(4, (max_smem - fixed - work) / t.stage_bytes);
  if (max_smem < fixed + work || t.nstages < 1) return false;
  t.nbuf = std::min(t.nbuf, t.nstages);
  t.off_drh = work;
  t.off_e = round_up(t.off_drh + drh, 1024);
  t.off_tab = t.off_e + kEBytes;
  t.off_q = t.off_tab + t.halves * 256 * HD;
  t.off_stage = t.off_q + 256 * HD;
  t.off_bar = t.off_stage + t.nstages * t.stage_bytes;
  *smem = t.off_bar + kBarBytes + kSlackBytes;
  return *smem <= max_smem;
}

// The key block of bwd_dkv_tc: 8 x 16 or 16 x 8, whichever takes fewer blocks.
inline void dkv_block(TcArgs& t, int h, int w) {
  const int a = (h + 7) / 8 * ((w + 15) / 16), b = (h + 15) / 16 * ((w + 7) / 8);
  t.th = b < a ? 16 : 8;
  t.tw = 128 / t.th;
  t.tiles_h = (h + t.th - 1) / t.th;
  t.tiles_w = (w + t.tw - 1) / t.tw;
}

template <typename T, int HD>
int launch_tc_hd(TcArgs t, void* ktp, int slots, int ctas, int max_smem, cudaStream_t st) {
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr CUtensorMapDataType type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const Args& a = t.a;
  const int h = a.h, w = a.w, n = h * w, hd = a.hd;
  const uint64_t bh = (uint64_t)a.bh;
  int smem = 0;
  if (!dq_layout(t, HD, h, w, max_smem, &smem)) return 1;
  const void* kt = a.kt;
  int ktw = w;
  if (w % 8 != 0) {  // the TMA wants rows of a multiple of 16 bytes
    ktw = round_up(w, 8);
    kt = ktp;
  }
  PrepArgs prep{a.kt, a.dout, a.v, ktp, const_cast<float*>(t.amax), (unsigned)(a.bh * hd * h), w, ktw, n, hd, 0, t.norm_blocks};
  prep.pad_blocks = ktw == w ? 0 : (int)((a.bh * hd * h * (ktw / 8) + 1023) / 1024);
  const int64_t prep_blocks = prep.pad_blocks + (t.amax ? a.bh * t.norm_blocks : 0);
  CUtensorMap mk, mv, mq, md, mo, mt, mq64, mo64, mh, mw;
  const cuuint64_t kdims[4] = {(cuuint64_t)w, (cuuint64_t)hd, (cuuint64_t)h, bh};
  const cuuint64_t kstr[3] = {(cuuint64_t)h * ktw * 2, (cuuint64_t)ktw * 2, (cuuint64_t)hd * h * ktw * 2};
  const cuuint32_t kbox[4] = {kBandW, HD, kBandH, 1};
  int rc = make_map_nd(&mk, type, kt, 4, kdims, kstr, kbox, CU_TENSOR_MAP_SWIZZLE_32B);
  const cuuint64_t vdims[5] = {16, (cuuint64_t)w, (cuuint64_t)h, (cuuint64_t)hd / 16, bh};
  const cuuint64_t vstr[4] = {(cuuint64_t)hd * 2, (cuuint64_t)w * hd * 2, 32, (cuuint64_t)n * hd * 2};
  const cuuint32_t vbox[5] = {16, kBandW, kBandH, HD / 16, 1};
  if (!rc) rc = make_map_nd(&mv, type, a.v, 5, vdims, vstr, vbox, CU_TENSOR_MAP_SWIZZLE_32B);
  if (!rc) rc = make_chunk_map(&mq, bf16, a.q, hd, n, bh, HD, 128);
  if (!rc) rc = make_chunk_map(&md, bf16, a.dout, hd, n, bh, HD, 128);
  if (!rc) rc = make_chunk_map(&mo, bf16, a.out, hd, n, bh, HD, 128);
  if (!rc) rc = make_chunk_map3(&mt, bf16, a.table, hd, table_rows(h, w), HD, 128);
  if (rc) return 10 + rc;
  auto dq = bwd_dq_tc<T, HD>;
  if (cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return 1;
  if (prep_blocks > 0) {
    bwd_prepare<<<(unsigned)prep_blocks, 256, 0, st>>>(prep);
    launch_dependent(dq, slots, kTcThreads, smem, st, mk, mv, mq, md, mo, mt, t);
  } else {
    dq<<<slots, kTcThreads, smem, st>>>(mk, mv, mq, md, mo, mt, t);
  }

  dkv_block(t, h, w);
  const int64_t grid = a.bh * t.tiles_h * t.tiles_w;
  if (grid > 0x7fffffffLL) return 2;
  constexpr int kStage = dkv_stage_bytes(HD);
  t.nstages = std::min(4, (max_smem - kBarBytes - kSlackBytes) / kStage);
  t.off_bar = t.nstages * kStage;
  const int smem2 = t.off_bar + kBarBytes + kSlackBytes;
  rc = make_chunk_map(&mq64, bf16, a.q, hd, n, bh, HD, kStep);
  if (!rc) rc = make_chunk_map(&mo64, bf16, a.dout, hd, n, bh, HD, kStep);
  const cuuint64_t hdims[2] = {(cuuint64_t)a.np, bh * round_up(h, 16)}, hstr[1] = {(cuuint64_t)a.np * 4};
  const cuuint32_t hbox[2] = {kStep, (cuuint32_t)t.th};
  if (!rc) rc = make_map_nd(&mh, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a.rel, 2, hdims, hstr, hbox, CU_TENSOR_MAP_SWIZZLE_NONE);
  const cuuint64_t wdims[2] = {(cuuint64_t)a.np, bh * round_up(w, 16)};
  const cuuint32_t wbox[2] = {32, (cuuint32_t)t.tw};
  if (!rc) rc = make_map_nd(&mw, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, t.rw, 2, wdims, hstr, wbox, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return 10 + rc;
  auto dkv = bwd_dkv_tc<T, HD>;
  if (cudaFuncSetAttribute(dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, smem2) != cudaSuccess) return 1;
  launch_dependent(dkv, (unsigned)std::min<int64_t>(grid, ctas), kTcThreads, smem2, st, mq64, mo64, mh, mw, t);
  return 0;
}

// The narrowest kernel that holds hd columns (further columns are zeros).
template <typename T>
int launch_tc(const TcArgs& t, void* ktp, int slots, int ctas, int max_smem, cudaStream_t st) {
  const int hd = t.a.hd;
  if (hd <= 32) return launch_tc_hd<T, 32>(t, ktp, slots, ctas, max_smem, st);
  if (hd <= 64) return launch_tc_hd<T, 64>(t, ktp, slots, ctas, max_smem, st);
  if (hd <= 80) return launch_tc_hd<T, 80>(t, ktp, slots, ctas, max_smem, st);
  if (hd <= 96) return launch_tc_hd<T, 96>(t, ktp, slots, ctas, max_smem, st);
  return launch_tc_hd<T, 128>(t, ktp, slots, ctas, max_smem, st);
}

inline int tc_width(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 80 ? 80 : hd <= 96 ? 96 : 128; }

// Whether the tensor-core kernels take this call: shape, 16-byte aligned tensors (TMA and vector accesses), and a scale
// whose inverse is a sane factor of G.
inline bool tc_ok(const Args& a, int dtype, int max_smem) {
  if (!tc_shape(a.h, a.w, a.hd, dtype)) return false;
  const void* ptrs[] = {a.q, a.kt, a.v, a.table, a.out, a.dout, a.dq, a.dkt, a.dv};
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  const float s = a.scale < 0 ? -a.scale : a.scale;
  if (!(s >= 0x1p-12f && s <= 0x1p12f)) return false;
  TcArgs t{};
  int smem = 0;
  return dq_layout(t, tc_width(a.hd), a.h, a.w, max_smem, &smem);
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
  a.rel = reinterpret_cast<float*>(cut(plan.rel_bytes));  // (SIMT: runs on into rw's room)
  float* rw = reinterpret_cast<float*>(cut(plan.rw_bytes));
  a.dsum = reinterpret_cast<float*>(cut(plan.dsum_bytes));
  a.partial = reinterpret_cast<float*>(cut(plan.partial_bytes));
  void* ktp = cut(plan.kt_bytes);
  float* amax = reinterpret_cast<float*>(cut(plan.amax_bytes));
  a.np = padded_rows((int)n);
  const Args whole = a;
  const int64_t rows = tc ? 128 : kBR, qtiles = (n + rows - 1) / rows;
  const SimtRun simt = simt_dq(std::min<int64_t>(plan.group, bh), a.h, a.w, a.hd, num_sms, max_smem);
  if (!tc && simt.groups == 0) return 1;
  const int resident = tc ? std::min(num_sms, kMinSlots) : simt.resident;
  const int slots = (int)std::min<int64_t>(std::min<int64_t>(plan.group, bh) * qtiles, std::min(resident, plan.slots));
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
        t.rw = rw;
        if constexpr (std::is_same<T, __half>::value) {
          const float s = a.scale < 0 ? -a.scale : a.scale;
          t.amax = amax;
          t.norm_blocks = norm_blocks((int)n);
          t.gain = 8192.f * std::min(1.f, s);  // G holds sums of dS over scale
        }
        rc = launch_tc<T>(t, ktp, slots, num_sms, max_smem, st);
      } else {
        rc = launch_simt<T>(a, simt.groups, slots, num_sms, max_smem, st);
      }
    } else {
      rc = launch_simt<T>(a, simt.groups, slots, num_sms, max_smem, st);
    }
    if (rc) return rc;
  }
  const int elems = table_rows(a.h, a.w) * a.hd;
  launch_dependent(bwd_table_reduce<T>, (elems + 31) / 32, 512, 0, st, static_cast<const float*>(a.partial),
                   static_cast<T*>(a.dtable), slots, elems);
  return 0;
}

}  // namespace bwd
}  // namespace samrs
