// Penalties for repeated tokens, biases and grammar masks on logits, one pass:
//
//   c = how often v stands in history[b, 0 .. history_lens[b])
//   l = c > 0 ? (logit > 0 ? logit / repetition : logit * repetition) : logit
//   out = allowed ? l - frequency * c - presence * (c > 0) + bias : -inf
//
// Bound by HBM: every logit is read and written once.
#pragma once

#include "vk_common.cuh"

namespace vk {
namespace logit {

constexpr int kSlice = 8192;  // vocabulary entries of a CTA, counted in shared memory
constexpr int kThreads = 256;

struct Args {
  const void* logits;  // [B, V], row stride ld
  void* out;           // [B, V], row stride ld_out
  int64_t ld, ld_out;
  const int64_t* history;  // [B, T], row stride ld_history; ids outside 0..V-1 count for nothing
  const int32_t* history_lens;
  int64_t ld_history;
  const float* repetition;  // [B] each, or NULL
  const float* presence;
  const float* frequency;
  const float* bias;        // row stride ld_bias (0: one for all rows), or NULL
  int64_t ld_bias;
  const uint32_t* mask;     // [masks, ld_mask] words, bit v % 32 of word v / 32, or NULL
  int64_t ld_mask;
  const int32_t* mask_index;  // [B] row of mask, -1: none; NULL: row b (or 0 of a single one)
  int masks;
  int B, V, T;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) penalize_kernel(Args a) {
  __shared__ int counts[kSlice];
  const int slices = (a.V + kSlice - 1) / kSlice;
  const int b = blockIdx.x / slices, v0 = blockIdx.x % slices * kSlice, n = min(kSlice, a.V - v0);
  pdl_wait();
  for (int i = threadIdx.x; i < n; i += kThreads) counts[i] = 0;
  __syncthreads();
  if (a.history) {
    const int len = checked_len(a.history_lens[b], a.T);
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const int64_t t = a.history[b * a.ld_history + i] - v0;
      if (t >= 0 && t < n) atomicAdd(&counts[t], 1);
    }
  }
  __syncthreads();
  const uint32_t* mask = nullptr;
  if (a.mask) {
    int m = a.mask_index ? a.mask_index[b] : a.masks == 1 ? 0 : b;
    if (m < -1 || m >= a.masks) {
      raise_error(ERR_BOUNDS);
      m = -1;
    }
    if (m >= 0) mask = a.mask + m * a.ld_mask;
  }
  const float rep = a.repetition ? a.repetition[b] : 1.f, pres = a.presence ? a.presence[b] : 0.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  const T* in = static_cast<const T*>(a.logits) + b * a.ld;
  T* out = static_cast<T*>(a.out) + b * a.ld_out;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int v = v0 + i, c = counts[i];
    float l = to_f32<T>(in[v]);
    if (c > 0) {
      if (a.repetition) l = l > 0.f ? l / rep : l * rep;
      l = l - freq * c - pres;
    }
    if (a.bias) l += a.bias[b * a.ld_bias + v];
    if (mask && !(mask[v >> 5] >> (v & 31) & 1)) l = -INFINITY;
    out[v] = from_f32<T>(l);
  }
}

}  // namespace logit
}  // namespace vk
