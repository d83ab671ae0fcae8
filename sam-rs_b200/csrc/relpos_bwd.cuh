// relpos_bwd.cuh - host side of the attention's backward pass: workspace layout, kernel selection, launches.
#pragma once
#include <algorithm>

#include "common.cuh"
#include "relpos_bwd_simt.cuh"

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
  int64_t total;
};

inline int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }

inline Plan make_plan(int64_t bh, int h, int w, int hd) {
  Plan p;
  const int64_t np = padded_rows(h * w);
  const int64_t rel = (int64_t)(h + w) * np * 4, dsum = np * 4;
  p.group = std::max<int64_t>(1, std::min<int64_t>(bh, kGroupBytes / (rel + dsum)));
  p.rel_bytes = round256(p.group * rel);
  p.dsum_bytes = round256(p.group * dsum);
  p.partial_bytes = round256((int64_t)kMaxSlots * table_rows(h, w) * hd * 4);
  p.total = p.rel_bytes + p.dsum_bytes + p.partial_bytes;
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

// The whole backward pass of bh >= 1 heads. `a` holds the whole batch's pointers, the workspace is cut here.
template <typename T>
int launch_bwd(Args a, int64_t bh, void* workspace, const Plan& plan, int num_sms, int max_smem, cudaStream_t st) {
  const int64_t n = (int64_t)a.h * a.w, per_head = n * a.hd;
  char* ws = static_cast<char*>(workspace);
  a.rel = reinterpret_cast<float*>(ws);
  a.dsum = reinterpret_cast<float*>(ws + plan.rel_bytes);
  a.partial = reinterpret_cast<float*>(ws + plan.rel_bytes + plan.dsum_bytes);
  a.np = padded_rows((int)n);
  const Args whole = a;
  const int64_t qtiles = (n + 63) / 64;
  const int slots = (int)std::min<int64_t>(std::min<int64_t>(plan.group, bh) * qtiles, std::min(num_sms, kMaxSlots));
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
    const int rc = launch_simt<T>(a, slots, max_smem, st);
    if (rc) return rc;
  }
  const int elems = table_rows(a.h, a.w) * a.hd;
  bwd_table_reduce<T><<<(elems + 31) / 32, 256, 0, st>>>(a.partial, static_cast<T*>(a.dtable), slots, elems);
  return 0;
}

}  // namespace bwd
}  // namespace samrs
