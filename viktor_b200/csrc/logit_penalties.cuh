// Penalties for repeated tokens, biases and grammar masks on logits, one pass:
//
//   c = how often v stands in history[b, 0 .. history_lens[b])
//   l = c > 0 ? (logit > 0 ? logit / repetition : logit * repetition) : logit
//   out = allowed ? l - frequency * c - presence * (c > 0) + bias : -inf
//
// (the quotient as a product with 1 / repetition: half a step of float32 more, and no branches).
// Bound by HBM: every logit is read and written once.  A CTA takes a slice of one row.  It counts the row's tokens that fall
// into the slice in shared memory (whole numbers, so the order of the atomics does not show), in 16 bits while no count
// can pass them: 16384 counters take 32 KB, five CTAs share an SM and hide one another's counting.  The logits stream through
// registers, the next vectors of 16 bytes of every thread under way; vectors without a token of the history skip the penalties.
// 512 x 131072 float32 with 2048 tokens, bias and masks: 105 us, 0.79 of the copy rate (84 us without the history, bias
// and mask; slices of 8192: 109 us; of 32768 in 512 threads at 3 CTAs an SM, with 40 registers each: 121 us).
#pragma once

#include <type_traits>

#include "vk_common.cuh"

namespace vk {
namespace logit {

constexpr int kThreads = 256;
constexpr int kMostSmem = 32768;  // bytes of counters

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
  int slices, slice;  // slice: elements of a CTA, a multiple of kThreads * VEC
  bool wide;          // counters of 32 bits
};

// VEC elements (16 bytes) at a time where the rows of logits and out lie alike relative to 16 bytes, else one.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// Elements e .. e + VEC - 1 of a row; those outside 0..V-1 are left out.
template <typename T, int VEC>
VK_DEV Vec<T, VEC> load_vec(const T* row, int e, int V) {
  Vec<T, VEC> x;
  if (e >= 0 && e + VEC <= V) return *reinterpret_cast<const Vec<T, VEC>*>(row + e);
#pragma unroll
  for (int i = 0; i < VEC; ++i) x.v[i] = e + i >= 0 && e + i < V ? row[e + i] : from_f32<T>(0.f);
  return x;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, 5) penalize_kernel(Args a) {
  constexpr int kStep = kThreads * VEC, kDepth = VEC == 8 ? 1 : 2;  // vectors under way in each thread (48 registers)
  extern __shared__ __align__(16) uint32_t counts[];
  const int b = blockIdx.x / a.slices, s = blockIdx.x % a.slices, tid = threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const T* in = static_cast<const T*>(a.logits) + b * a.ld;
  T* out = static_cast<T*>(a.out) + b * a.ld_out;
  // vectors start at 16-byte boundaries: the row's first one may begin before the row
  const int e0 = s * a.slice - (VEC == 1 ? 0 : static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T)));
  const int e1 = min(e0 + a.slice, a.V);
  if (e0 >= a.V) return;
  int e = e0 + tid * VEC;
  Vec<T, VEC> ahead[kDepth];
#pragma unroll
  for (int i = 0; i < kDepth; ++i) ahead[i] = load_vec<T, VEC>(in, e + i * kStep, e1);
  const uint32_t* mask = nullptr;
  if (a.mask) {
    int m = a.mask_index ? a.mask_index[b] : a.masks == 1 ? 0 : b;
    if (m < -1 || m >= a.masks) {
      raise_error(ERR_BOUNDS);
      m = -1;
    }
    if (m >= 0) mask = a.mask + m * a.ld_mask;
  }
  // the slice's mask bits, bit i % 32 of word i / 32 for element e0 + i
  uint32_t* bits = counts + (a.history ? (a.wide ? a.slice : a.slice / 2) : 0);
  for (int i = tid; i < a.slice / 32; i += kThreads) {
    uint32_t w = 0xffffffffu;
    if (mask) {
      const int at = e0 + i * 32, lo = at >> 5, last = (a.V - 1) >> 5;  // (at >> 5 rounds down: -1 before the row)
      const uint32_t w0 = lo >= 0 && lo <= last ? __ldg(mask + lo) : 0u, w1 = (at & 31) && lo < last ? __ldg(mask + lo + 1) : 0u;
      w = __funnelshift_r(w0, w1, at);
    }
    bits[i] = w;
  }
  const float rep = a.repetition ? a.repetition[b] : 1.f, pres = a.presence ? a.presence[b] : 0.f;
  // the quotient by rep: a product with 1 / (rep 2^k), then with 2^k, k 64 or -64 where the inverse of rep is no normal number, otherwise 0
  const float two_k = fabsf(rep) < 1.17549435e-38f ? 18446744073709551616.f : fabsf(rep) > 8.5e37f ? 5.42101086e-20f : 1.f;
  const float inv = 1.f / (rep * two_k), freq = a.frequency ? a.frequency[b] : 0.f;
  const float* bias = a.bias ? a.bias + b * a.ld_bias : nullptr;
  if (a.history) {
    const int64_t* h = a.history + b * a.ld_history;
    constexpr int kAhead = 4;  // tokens a thread has under way; the first ones do not wait for the length
    int64_t t[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) t[u] = u * kThreads + tid < a.T ? h[u * kThreads + tid] : -1;
    const int len = checked_len(a.history_lens[b], a.T);
    const int words = a.wide ? a.slice : a.slice / 2;
    for (int i = tid * 4; i < words; i += kThreads * 4) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int base = 0; base < len; base += kThreads * kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = base + u * kThreads + tid, next = i + kThreads * kAhead;
        const int64_t at = t[u] - e0;
        if (i < len && t[u] >= 0 && at >= 0 && t[u] < e1) {
          if (a.wide)
            atomicAdd(&counts[at], 1u);
          else
            atomicAdd(&counts[at >> 1], at & 1 ? 65536u : 1u);
        }
        t[u] = next < len ? h[next] : -1;
      }
    }
  }
  __syncthreads();
  const bool bias_whole = bias && VEC > 1 && (reinterpret_cast<uintptr_t>(bias + e0) & 15) == 0;
  // l += bias, for a vector whose elements all lie in the slice (WHOLE) or not
  auto add_bias = [&](int e, float (&l)[VEC], auto is_whole) {
    constexpr bool WHOLE = decltype(is_whole)::value;
#pragma unroll
    for (int i = 0; i < VEC; ++i) l[i] = 0.f;
    if (!bias) return;
    if (WHOLE && bias_whole) {
#pragma unroll
      for (int i = 0; i + 3 < VEC; i += 4) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(bias + e + i));
        l[i] = f.x;
        l[i + 1] = f.y;
        l[i + 2] = f.z;
        l[i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (WHOLE || (e + i >= 0 && e + i < e1)) l[i] = __ldg(bias + e + i);
    }
  };
  // the vector's results from its logits and biases
  auto finish = [&](Vec<T, VEC> x, int e, const float (&add)[VEC], auto is_whole) {
    constexpr bool WHOLE = decltype(is_whole)::value;
    const int at = e - e0;
    float l[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) l[i] = to_f32<T>(x.v[i]);
    if (a.history) {
      constexpr int kWords = VEC == 1 ? 1 : VEC / 2;  // of 16-bit counters
      uint32_t w[kWords], any = 0;
      if (!a.wide) {
        if (VEC == 1) {
          w[0] = counts[at >> 1] >> (at & 1) * 16 & 0xffffu;
        } else {
#pragma unroll
          for (int i = 0; i + 1 < kWords; i += 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(counts + at / 2 + i);
            w[i] = u.x;
            w[i + 1] = u.y;
          }
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) any |= w[i];
      } else {
        any = 1;
      }
      if (any) {  // hardly ever: most vectors hold no token of the history
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const uint32_t c = a.wide ? counts[at + i] : w[i / 2] >> i % 2 * 16 & 0xffffu;
          if (c > 0) l[i] = (l[i] > 0.f ? l[i] * inv * two_k : l[i] * rep) - freq * c - pres;
        }
      }
    }
    const uint32_t allowed = bits[at >> 5] >> (at & 31);  // VEC divides 32: one word
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (bias) l[i] += add[i];
      x.v[i] = from_f32<T>(allowed & 1u << i ? l[i] : -INFINITY);
    }
    if (WHOLE) {
      *reinterpret_cast<Vec<T, VEC>*>(out + e) = x;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (e + i >= 0 && e + i < e1) out[e + i] = x.v[i];
    }
  };
  if (e0 >= 0) {  // steps whose vectors are whole in every thread
    const int whole = (e1 - e0) / kStep;
    for (int k = 0; k + kDepth <= whole; k += kDepth, e += kDepth * kStep) {
      Vec<T, VEC> now[kDepth];
      float add[kDepth][VEC];
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        now[i] = ahead[i];
        add_bias(e + i * kStep, add[i], std::true_type{});
      }
#pragma unroll
      for (int i = 0; i < kDepth; ++i) ahead[i] = load_vec<T, VEC>(in, e + (kDepth + i) * kStep, e1);
#pragma unroll
      for (int i = 0; i < kDepth; ++i) finish(now[i], e + i * kStep, add[i], std::true_type{});
    }
  }
#pragma unroll 1
  for (; e < e1; e += kStep) {
    const Vec<T, VEC> x = ahead[0];
#pragma unroll
    for (int i = 0; i + 1 < kDepth; ++i) ahead[i] = ahead[i + 1];
    ahead[kDepth - 1] = load_vec<T, VEC>(in, e + kDepth * kStep, e1);
    float add[VEC];
    add_bias(e, add, std::false_type{});
    if (e + VEC > 0) finish(x, e, add, std::false_type{});
  }
}

}  // namespace logit
}  // namespace vk
