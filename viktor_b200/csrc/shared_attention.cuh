// Decode attention for rows that share prefixes: row b of group g (group_offsets[g] <= b < group_offsets[g + 1])
// attends the prefix g, stored once, and its own tail, stored in pages.
//
//   out[b, h, :] = sum_j p_j v_j,  p = softmax_j(scale * q[b, h] . k_j),  j in prefix(g) then tail(b),  KV head h / (H / HK)
//
// A row with nothing to attend gives 0 (lse -inf); rows behind the last group are not touched.
#pragma once

#include "vk_common.cuh"

namespace vk {
namespace sattn {

struct Args {
  const void* q;               // [B, H, D], row stride stride_q
  const void* k_prefix;        // [P, S, HK, D], strides stride_kb, stride_ks (elements)
  const void* v_prefix;
  const int32_t* prefix_lens;  // [P]
  const int32_t* offsets;      // [P + 1]
  const void* k_pages;         // [n_pages, page, HK, D], page stride stride_pp (elements)
  const void* v_pages;
  const int32_t* table;        // [B, max_pages], row stride stride_table
  const int32_t* tail_lens;    // [B]
  void* out;                   // [B, H, D]
  float* lse;                  // [B, H] or NULL
  int64_t stride_q, stride_kb, stride_ks, stride_pp, stride_table;
  int B, H, HK, P, S, n_pages, page_shift, max_pages;
  float scale;
};

// Reports group offsets that do not ascend from 0 to at most B.  Spread over the threads of the grid.
VK_DEV void check_offsets(const Args& a) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t g = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; g < a.P; g += step) {
    const int lo = a.offsets[g], hi = a.offsets[g + 1];
    if (lo > hi || hi > a.B || (g == 0 && lo != 0)) raise_error(ERR_BOUNDS);
  }
}

// One warp per (row, query head), one position at a time: the plain restatement of the formula.
template <typename T, int D>
__global__ void __launch_bounds__(128) rows_kernel(Args a) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  check_offsets(a);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (item >= static_cast<int64_t>(a.B) * a.H) return;
  const int b = static_cast<int>(item / a.H), h = static_cast<int>(item % a.H), kvh = h / (a.H / a.HK);
  int g = 0;
  while (g < a.P && a.offsets[g + 1] <= b) ++g;
  if (g == a.P) return;  // behind the last group
  const T* qp = static_cast<const T*>(a.q) + b * a.stride_q + h * D + lane * PER;
  float q[PER], o[PER], m = -INFINITY, l = 0.f;
  for (int i = 0; i < PER; ++i) {
    q[i] = to_f32<T>(qp[i]) * a.scale;
    o[i] = 0.f;
  }
  const int np = checked_len(a.prefix_lens[g], a.S);
  const int nt = checked_len(a.tail_lens[b], a.max_pages << a.page_shift);
  for (int j = 0; j < np + nt; ++j) {
    int64_t off;
    const T *kp, *vp;
    if (j < np) {
      off = g * a.stride_kb + j * a.stride_ks;
      kp = static_cast<const T*>(a.k_prefix);
      vp = static_cast<const T*>(a.v_prefix);
    } else {
      const int t = j - np;
      int page = a.table[b * a.stride_table + (t >> a.page_shift)];
      if (page < 0 || page >= a.n_pages) {
        raise_error(ERR_BOUNDS);
        page = 0;
      }
      off = page * a.stride_pp + static_cast<int64_t>(t & ((1 << a.page_shift) - 1)) * a.HK * D;
      kp = static_cast<const T*>(a.k_pages);
      vp = static_cast<const T*>(a.v_pages);
    }
    off += kvh * D + lane * PER;
    float s = 0.f;
    for (int i = 0; i < PER; ++i) s += q[i] * to_f32<T>(kp[off + i]);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - mu), p = expf(s - mu);
    l = l * f + p;
    for (int i = 0; i < PER; ++i) o[i] = o[i] * f + p * to_f32<T>(vp[off + i]);
    m = mn;
  }
  T* op = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.H + h) * D + lane * PER;
  for (int i = 0; i < PER; ++i) op[i] = from_f32<T>(l > 0.f ? o[i] / l : l);  // l NaN stays NaN, l 0 gives 0
  if (a.lse && lane == 0) a.lse[static_cast<int64_t>(b) * a.H + h] = l > 0.f || l != l ? m + logf(l) : -INFINITY;
}

}  // namespace sattn
}  // namespace vk
