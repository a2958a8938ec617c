// Decode attention for rows that share prefixes: row b of group g (group_offsets[g] <= b < group_offsets[g + 1])
// attends the prefix g, stored once, and its own tail, stored in pages.
//
//   out[b, h, :] = sum_j p_j v_j,  p = softmax_j(scale * q[b, h] . k_j),  j in prefix(g) then tail(b),  KV head h / (H / HK)
//
// A row with nothing to attend gives 0 (lse -inf); rows behind the last group are not touched.
//
// Prefix and tails are split over CTAs, each with a running maximum and sum (base 2); a last kernel joins the partial results,
// in a fixed order, so equal calls give equal bits and nothing in the workspace outlives a call.
//  * few rows of a group and KV head (up to 32 of D 64, 16 of D 128 on average), and every tail: split_kernel, on the warp tensor
//    cores, bound by HBM.  256 groups of 4 rows, prefixes to 2049, tails to 1100 (451 MB): 77 us, 5.9 TB/s.  4 rows x 16 heads
//    on 131071 positions (537 MB): 91 us, 5.9 TB/s.
//  * more rows: wide_kernel, on the 5th-generation tensor cores, bound by the exponentials and the steps around them.
// The mean is what the host knows.  Whole calls in bf16 on prefixes of 2049, split_kernel / wide_kernel: 256 groups of 4 rows x 8
// heads on 2 of D 64 (16 rows) 77 / 112 us, of 8 rows (32) 85 / 107, of 9 rows (36) 99 / 107, of 16 rows (64) 107 / 120; 128
// groups of 16 rows 69 / 67 us, 32 groups of 32 rows (128) 50 / 44 us; D 128, 256 groups of 4 rows (16) 128 / 159 us.  One group of
// 256 rows among 200 of one: 62 / 83 us.
#pragma once

#include <type_traits>

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
};

constexpr int kThreads = 128;  // 4 warps
constexpr int kStages = 2;     // of each warp's own ring

// Work of one launch: prefix items (tile of rows, KV head, chunk) first, then tail items (row, KV head, tile of heads, chunk).
// Partial results go to slot [split][b * H + h], prefix chunks first.
struct Plan {
  int prefix_tiles;   // at most; group g's tiles begin at floor(offset_g * r / rows) + g
  int prefix_splits, prefix_chunk;
  int tail_tiles;     // tiles of 16 heads of one (row, KV head)
  int tail_splits, tail_chunk;
  int prefix_items, tail_items;
  bool behind_wide;   // launched right behind wide_kernel of the same call
  float scale_log2;
  float* ws_o;        // [prefix_splits + tail_splits][B * H][D]
  float2* ws_ml;      // [prefix_splits + tail_splits][B * H]: reference (below, of scores in base 2) and sum
};

template <typename T>
VK_DEV void mma_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
VK_DEV void mma_16816<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  mma_bf16_16816(d, a, b0, b1);
}
template <>
VK_DEV void mma_16816<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two values rounded to the type.
template <typename T>
VK_DEV uint32_t pack2(float x, float y);
template <>
VK_DEV uint32_t pack2<__nv_bfloat16>(float x, float y) {
  return pack_bf16x2(x, y);
}
template <>
VK_DEV uint32_t pack2<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Probabilities are taken relative to a reference: the largest score so far (base 2) less kDrop, followed only when that is passed by
// more than kLag, so that most tiles need no rescaling.  They lie below 2^(kDrop + kLag) and are rounded to the type for the
// product with V, their sum is not.  bf16 has the exponents of float32: any reference will do.  fp16 is normal down to 2^-14 and
// ends at 2^16: with the reference 11 below the maximum a probability keeps its 11 bits down to 2^-25 of the largest, and is off
// by at most 2^-36 of it below (with the maximum for a reference: 2^-14 and 2^-25, and next to one dominant position with a
// small value the others were lost); a longer lag would take that room away.
template <typename T>
struct Ref {
  static constexpr float kDrop = std::is_same<T, __half>::value ? 11.f : 0.f;
  static constexpr float kLag = std::is_same<T, __half>::value ? 4.f : 8.f;
};

// 16 bytes from global to shared memory; the second form: zeros where !use.
VK_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
VK_DEV void cp_async16(uint32_t dst, const void* src, bool use) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(use ? 16 : 0) : "memory");
}
VK_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
VK_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Positions a warp takes at a time: 4 KB of K and of V.
template <int D>
struct Tile {
  static constexpr int kPos = 2048 / D;              // 32 or 16
  static constexpr int kHalf = kPos * D * 2;         // bytes of K or V
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kWarp = kStages * kStage;
  static constexpr int kSmem = 4 * kWarp;
  // byte offset of 16-byte chunk c of position p; chunks of eight neighbouring positions lie in different banks
  static VK_DEV uint32_t at(int p, int c) { return p * (D * 2) + ((c ^ (p & 7)) << 4); }
};

// Where the keys and values of an item come from.
template <typename T>
struct Source {
  const T* k;
  const T* v;
  int64_t stride;          // of a position, in elements (prefix)
  const int32_t* table;    // page ids (tail)
  int64_t stride_page;
  int page_shift, n_pages;
};

// Loads positions p .. p + kPos - 1 (those at or past end: zeros) into one stage.  page: this lane's page id, that of
// position p + lane.  Where a tile lies in one piece (a prefix, or pages of at least kPos tokens) a lane's addresses are one base
// and constant steps.
template <typename T, int D, bool PAGED>
VK_DEV void load_tile(const Source<T>& s, uint32_t stage, int p, int end, int page) {
  constexpr int kChunks = D / 8, kRows = 32 / kChunks, kPos = Tile<D>::kPos, kLoads = kPos / kRows;
  const int lane = threadIdx.x & 31, c = lane % kChunks, r0 = lane / kChunks, mask = (1 << s.page_shift) - 1;
  if (!PAGED || mask >= kPos - 1) {
    int64_t off = PAGED ? __shfl_sync(0xffffffffu, page, 0) * s.stride_page + static_cast<int64_t>(p & mask) * s.stride : p * s.stride;
    off += r0 * s.stride + c * 8;
    const T *k = s.k + off, *v = s.v + off;
    const int64_t step = kRows * s.stride;
    if (p + kPos <= end) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t to = stage + Tile<D>::at(r0 + i * kRows, c);
        cp_async16(to, k + i * step);
        cp_async16(to + Tile<D>::kHalf, v + i * step);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t to = stage + Tile<D>::at(r0 + i * kRows, c);
        const bool use = p + r0 + i * kRows < end;
        cp_async16(to, use ? k + i * step : s.k, use);
        cp_async16(to + Tile<D>::kHalf, use ? v + i * step : s.v, use);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = r0 + i * kRows, pos = p + r;
      const int pg = __shfl_sync(0xffffffffu, page, r);
      const bool use = pos < end;
      const int64_t off = use ? pg * s.stride_page + static_cast<int64_t>(pos & mask) * s.stride + c * 8 : 0;
      const uint32_t to = stage + Tile<D>::at(r, c);
      cp_async16(to, s.k + off, use);
      cp_async16(to + Tile<D>::kHalf, s.v + off, use);
    }
  }
}

// The page of position pos, 0 (and a report) where the table names none.
template <typename T>
VK_DEV int page_at(const Source<T>& s, int pos, int end) {
  if (pos >= end) return 0;
  const int pg = s.table[pos >> s.page_shift];
  if (pg >= 0 && pg < s.n_pages) return pg;
  raise_error(ERR_BOUNDS);
  return 0;
}

// Online softmax of 16 * MT rows (a row is one query head of one token) over the tiles first, first + step, ... of the
// positions begin .. end - 1; q: the rows' operand fragments.  The warp's ring: kStages stages at `ring`.
//
// Scores, probabilities and the result stay in registers (m16n8k16: the accumulator of the first product is the operand of
// the second); a tile is bound by its 8 KB from HBM, which kStages - 1 tiles of every warp in flight keep coming.
template <typename T, int D, int MT, bool PAGED>
VK_DEV void attend(const Source<T>& s, uint32_t ring, int begin, int end, int first, int step, float scale_log2,
                   const uint32_t (&q)[MT][D / 16][4], float (&o)[MT][D / 8][4], float (&m)[MT][2], float (&l)[MT][2]) {
  constexpr int kPos = Tile<D>::kPos, kN = kPos / 8;
  const int lane = threadIdx.x & 31, t4 = lane & 3, j = lane >> 3, rr = lane & 7;
#pragma unroll
  for (int a = 0; a < MT; ++a) {
    m[a][0] = m[a][1] = -INFINITY;
    l[a][0] = l[a][1] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[a][i][0] = o[a][i][1] = o[a][i][2] = o[a][i][3] = 0.f;
  }
  const int tiles = (end - begin + kPos - 1) / kPos;
  const int own_pos = lane % kPos;  // (16 positions: the upper lanes repeat the lower ones)
  int page = 0, next = first;
  if (PAGED) page = page_at(s, begin + next * kPos + own_pos, end);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (next < tiles) {
      load_tile<T, D, PAGED>(s, ring + i * Tile<D>::kStage, begin + next * kPos, end, page);
      next += step;
      if (PAGED) page = page_at(s, begin + next * kPos + own_pos, end);
    }
    cp_async_commit();
  }
  int stage = 0;
  for (int t = first; t < tiles; t += step) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    {
      const int to = stage == 0 ? kStages - 1 : stage - 1;  // the stage that was read last
      if (next < tiles) {
        load_tile<T, D, PAGED>(s, ring + to * Tile<D>::kStage, begin + next * kPos, end, page);
        next += step;
        if (PAGED) page = page_at(s, begin + next * kPos + own_pos, end);
      }
      cp_async_commit();
    }
    const uint32_t kb = ring + stage * Tile<D>::kStage, vb = kb + Tile<D>::kHalf;
    stage = stage == kStages - 1 ? 0 : stage + 1;
    // ---- S = Q K^T ----
    float sc[MT][kN][4];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
      for (int n = 0; n < kN; ++n) sc[a][n][0] = sc[a][n][1] = sc[a][n][2] = sc[a][n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int n = 0; n < kN; n += 2) {
        uint32_t b[4];
        ldsm_x4(kb + Tile<D>::at(n * 8 + (j >> 1) * 8 + rr, ks * 2 + (j & 1)), b[0], b[1], b[2], b[3]);
#pragma unroll
        for (int a = 0; a < MT; ++a) {
          mma_16816<T>(sc[a][n], q[a][ks], b[0], b[1]);
          mma_16816<T>(sc[a][n + 1], q[a][ks], b[2], b[3]);
        }
      }
    // ---- softmax in base 2 ----
    const int pos0 = begin + t * kPos;
    const bool partial = pos0 + kPos > end;
    uint32_t pr[MT][kN][2];
#pragma unroll
    for (int a = 0; a < MT; ++a) {
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if (partial) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (pos0 + n * 8 + 2 * t4 + (e & 1) >= end) sc[a][n][e] = -INFINITY;
        }
        mx0 = fmaxf(mx0, fmaxf(sc[a][n][0], sc[a][n][1]));
        mx1 = fmaxf(mx1, fmaxf(sc[a][n][2], sc[a][n][3]));
      }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
      }
      mx0 = mx0 * scale_log2 - Ref<T>::kDrop;
      mx1 = mx1 * scale_log2 - Ref<T>::kDrop;
      const float mn0 = mx0 > m[a][0] + Ref<T>::kLag || m[a][0] == -INFINITY ? mx0 : m[a][0];
      const float mn1 = mx1 > m[a][1] + Ref<T>::kLag || m[a][1] == -INFINITY ? mx1 : m[a][1];
      const float mu0 = mn0 == -INFINITY ? 0.f : mn0, mu1 = mn1 == -INFINITY ? 0.f : mn1;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const float p0 = fast_exp2(fmaf(sc[a][n][0], scale_log2, -mu0)), p1 = fast_exp2(fmaf(sc[a][n][1], scale_log2, -mu0));
        const float p2 = fast_exp2(fmaf(sc[a][n][2], scale_log2, -mu1)), p3 = fast_exp2(fmaf(sc[a][n][3], scale_log2, -mu1));
        s0 += p0 + p1;
        s1 += p2 + p3;
        pr[a][n][0] = pack2<T>(p0, p1);
        pr[a][n][1] = pack2<T>(p2, p3);
      }
      if (__any_sync(0xffffffffu, mn0 != m[a][0] || mn1 != m[a][1])) {
        const float f0 = fast_exp2(m[a][0] - mu0), f1 = fast_exp2(m[a][1] - mu1);
        l[a][0] *= f0;
        l[a][1] *= f1;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[a][i][0] *= f0;
          o[a][i][1] *= f0;
          o[a][i][2] *= f1;
          o[a][i][3] *= f1;
        }
        m[a][0] = mn0;
        m[a][1] = mn1;
      }
      l[a][0] += s0;
      l[a][1] += s1;
    }
    // ---- O += P V ----
#pragma unroll
    for (int n = 0; n < kN; n += 2)
#pragma unroll
      for (int i = 0; i < D / 8; i += 2) {
        uint32_t b[4];
        ldsm_x4_t(vb + Tile<D>::at(n * 8 + (j & 1) * 8 + rr, i + (j >> 1)), b[0], b[1], b[2], b[3]);
#pragma unroll
        for (int a = 0; a < MT; ++a) {
          const uint32_t pa[4] = {pr[a][n][0], pr[a][n][1], pr[a][n + 1][0], pr[a][n + 1][1]};
          mma_16816<T>(o[a][i], pa, b[0], b[1]);
          mma_16816<T>(o[a][i + 1], pa, b[2], b[3]);
        }
      }
    __syncwarp();  // the stage may be loaded again
  }
  cp_async_wait<0>();
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) l[a][e] += __shfl_xor_sync(0xffffffffu, l[a][e], x);
}

// Operand fragments of 16 * MT rows: row x is query head kvh * r + x % r of token b0 + x / r, x0 <= x < x1.
template <typename T, int D, int MT>
VK_DEV void load_q(const Args& a, int b0, int kvh, int r, int x0, int x1, uint32_t (&q)[MT][D / 16][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int x = x0 + i * 16 + e * 8 + g;
      const bool use = x < x1;
      const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) +
                                                            (use ? (b0 + x / r) * a.stride_q + (kvh * r + x % r) * D : 0));
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        q[i][ks][e] = use ? p[ks * 8 + t4] : 0u;
        q[i][ks][e + 2] = use ? p[ks * 8 + t4 + 4] : 0u;
      }
    }
}

// Joins the WI warps of an item (through shared memory, which their rings have left) and writes the rows' partial results.
template <int D, int MT, int WI>
VK_DEV void store_partial(const Args& a, const Plan& pl, uint8_t* smem, int split, int b0, int kvh, int r, int x0, int x1,
                          float (&o)[MT][D / 8][4], float (&m)[MT][2], float (&l)[MT][2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int64_t base = static_cast<int64_t>(split) * a.B * a.H;
  if (WI == 1) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int x = x0 + i * 16 + e * 8 + g;
        if (x >= x1) continue;
        const int64_t row = base + static_cast<int64_t>(b0 + x / r) * a.H + kvh * r + x % r;
        if (t4 == 0) pl.ws_ml[row] = make_float2(m[i][e], l[i][e]);
        float* op = pl.ws_o + row * D + 2 * t4;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(op + d * 8) = make_float2(o[i][d][2 * e], o[i][d][2 * e + 1]);
      }
    return;
  }
  constexpr int kRows = 16 * MT;
  float* so = reinterpret_cast<float*>(smem);                      // [4][kRows][D]
  float2* sml = reinterpret_cast<float2*>(so + 4 * kRows * D);     // [4][kRows]
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int x = i * 16 + e * 8 + g;
      if (t4 == 0) sml[warp * kRows + x] = make_float2(m[i][e], l[i][e]);
      float* op = so + (warp * kRows + x) * D + 2 * t4;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(op + d * 8) = make_float2(o[i][d][2 * e], o[i][d][2 * e + 1]);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * (D / 4); i += kThreads) {
    const int x = i / (D / 4), d = i % (D / 4) * 4;
    if (x0 + x >= x1) break;
    float mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, sml[w * kRows + x].x);
    float4 ot = make_float4(0.f, 0.f, 0.f, 0.f);
    const float mu = mt == -INFINITY ? 0.f : mt;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 ml = sml[w * kRows + x];
      const float f = fast_exp2(ml.x - mu);
      const float4 v = *reinterpret_cast<const float4*>(so + (w * kRows + x) * D + d);
      lt += f * ml.y;
      ot.x += f * v.x;
      ot.y += f * v.y;
      ot.z += f * v.z;
      ot.w += f * v.w;
    }
    const int64_t row = base + static_cast<int64_t>(b0 + (x0 + x) / r) * a.H + kvh * r + (x0 + x) % r;
    if (d == 0) pl.ws_ml[row] = make_float2(mt, lt);
    *reinterpret_cast<float4*>(pl.ws_o + row * D + d) = ot;
  }
}

// An item without positions: sums of zero.
VK_DEV void store_nothing(const Args& a, const Plan& pl, int split, int b0, int kvh, int r, int x0, int x1, int thread,
                          int threads) {
  for (int x = x0 + thread; x < x1; x += threads)
    pl.ws_ml[(static_cast<int64_t>(split) * a.B + b0 + x / r) * a.H + kvh * r + x % r] = make_float2(-INFINITY, 0.f);
}

template <typename T, int D, int MT, int WI, bool PAGED>
VK_DEV void run_item(const Args& a, const Plan& pl, uint8_t* smem, const Source<T>& s, int split, int begin, int end, int b0,
                     int kvh, int r, int x0, int x1) {
  const int warp = threadIdx.x >> 5;
  if (begin >= end) {
    if (WI == 1)
      store_nothing(a, pl, split, b0, kvh, r, x0, x1, threadIdx.x & 31, 32);
    else
      store_nothing(a, pl, split, b0, kvh, r, x0, x1, threadIdx.x, kThreads);
    return;
  }
  uint32_t q[MT][D / 16][4];
  load_q<T, D, MT>(a, b0, kvh, r, x0, x1, q);
  float o[MT][D / 8][4], m[MT][2], l[MT][2];
  attend<T, D, MT, PAGED>(s, smem_u32(smem) + warp * Tile<D>::kWarp, begin, end, WI == 1 ? 0 : warp, WI, pl.scale_log2, q, o,
                          m, l);
  store_partial<D, MT, WI>(a, pl, smem, split, b0, kvh, r, x0, x1, o, m, l);
}

// The rows of a prefix item: rows x0 .. x1 - 1 (numbered as in load_q) of the group g, whose prefix has len positions; x0 >= x1:
// none.
struct Rows {
  int g, b0, len, kvh, split, x0, x1;
};
// The item of this CTA of `threads` threads with tiles of kRows rows; found: shared.  Every thread looks at every threads-th
// group (one round of loads for up to `threads` groups); the one whose group's tiles hold this one (group g's begin at
// floor(offset_g * r / kRows) + g) says so.  Offsets that do not ascend can give a tile to several groups: the first thread
// to say so has it, so that the record is always of one group, whose rows lie in 0 .. B - 1.
template <int kRows, int threads>
VK_DEV Rows find_rows(const Args& a, const Plan& pl, Rows* found) {
  constexpr int kNone = 0x7fffffff;
  const int r = a.H / a.HK;
  int item = blockIdx.x;
  const int split = item % pl.prefix_splits;
  item /= pl.prefix_splits;
  const int kvh = item % a.HK, tile = item / a.HK;
  if (threadIdx.x == 0) {
    found->x0 = kNone;
    found->x1 = 0;
  }
  __syncthreads();
  for (int g = threadIdx.x; g < a.P; g += threads) {
    const int lo = a.offsets[g], hi = a.offsets[g + 1], length = a.prefix_lens[g];
    if (lo < 0 || lo > hi || hi > a.B || (g == 0 && lo != 0)) {
      raise_error(ERR_BOUNDS);  // they have to ascend from 0 to at most B
      continue;
    }
    const int first = static_cast<int>(static_cast<int64_t>(lo) * r / kRows) + g;
    const int64_t x0 = static_cast<int64_t>(tile - first) * kRows, all = static_cast<int64_t>(hi - lo) * r;
    if (x0 < 0 || x0 >= all) continue;
    if (atomicCAS(&found->x0, kNone, static_cast<int>(x0)) != kNone) continue;
    found->x1 = static_cast<int>(x0 + kRows < all ? x0 + kRows : all);
    found->g = g;
    found->b0 = lo;
    found->len = checked_len(length, a.S);
    found->kvh = kvh;
    found->split = split;
  }
  __syncthreads();
  return *found;
}

// The tail item of this CTA, or of this warp.
template <typename T, int D, int WT>
VK_DEV void tail_item(const Args& a, const Plan& pl, uint8_t* smem) {
  const int r = a.H / a.HK, per = WT == 1 ? 4 : 1;  // items of a CTA
  int item = (blockIdx.x - pl.prefix_items) * per + (WT == 1 ? threadIdx.x >> 5 : 0);
  if (item >= pl.tail_items) return;
  const int split = item % pl.tail_splits;
  item /= pl.tail_splits;
  const int tile = item % pl.tail_tiles;
  item /= pl.tail_tiles;
  const int kvh = item % a.HK, b = item / a.HK;
  const int rows = a.offsets[a.P], length = a.tail_lens[b];
  if (b >= rows) return;  // behind the last group
  Source<T> s{};
  s.k = static_cast<const T*>(a.k_pages) + kvh * D;
  s.v = static_cast<const T*>(a.v_pages) + kvh * D;
  s.stride = static_cast<int64_t>(a.HK) * D;
  s.table = a.table + b * a.stride_table;
  s.stride_page = a.stride_pp;
  s.page_shift = a.page_shift;
  s.n_pages = a.n_pages;
  const int len = checked_len(length, a.max_pages << a.page_shift), begin = split * pl.tail_chunk;
  run_item<T, D, 1, WT, true>(a, pl, smem, s, pl.prefix_splits + split, begin, min(begin + pl.tail_chunk, len), b, kvh, r,
                              tile * 16, min(tile * 16 + 16, r));
}

// MT: 16-row tiles of a prefix item.  WT: warps of a tail item.
template <typename T, int D, int MT, int WT>
__global__ void __launch_bounds__(kThreads, 3) split_kernel(Args a, Plan pl) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Rows found;
  // Tails do not read what wide_kernel writes, and wide_kernel lets this one start only after its own wait for what came
  // before: so behind it the tails need not wait.  The wait comes last, for the kernel that joins both, and in every CTA: one that is
  // done keeps its place until the prefix is, so that only as many tails run beside it as find a place at first.
  if (!pl.behind_wide) pdl_wait();
  pdl_launch_dependents();
  if (static_cast<int>(blockIdx.x) < pl.prefix_items) {
    const Rows w = find_rows<16 * MT, kThreads>(a, pl, &found);
    if (w.x0 < w.x1) {
      Source<T> s{};
      s.k = static_cast<const T*>(a.k_prefix) + w.g * a.stride_kb + w.kvh * D;
      s.v = static_cast<const T*>(a.v_prefix) + w.g * a.stride_kb + w.kvh * D;
      s.stride = a.stride_ks;
      const int begin = w.split * pl.prefix_chunk;
      run_item<T, D, MT, 4, false>(a, pl, smem, s, w.split, begin, min(begin + pl.prefix_chunk, w.len), w.b0, w.kvh, a.H / a.HK,
                                   w.x0, w.x1);
    }
  } else {
    tail_item<T, D, WT>(a, pl, smem);
  }
  if (pl.behind_wide) pdl_wait();
}

// ---- wide groups -------------------------------------------------------------------------------------------------
// Prefix attention of up to 256 rows of one group and KV head on the 5th-generation tensor cores, one CTA per SM:
//   warp 0      TMA: 64-position tiles of K and V, one after another, into a ring of units
//   warps 1, 10 MMA issue of two streams s = 0, 1, each with 128 x 64 scores, two buffers of probabilities and a 128 x D result in
//               TMEM: S_s = Q K_j^T, then, once the softmax has put P there, O_s += P V_j
//   warps 2-5   softmax of stream 0, one row per thread; warps 6-9 of stream 1
// More than 128 rows: the streams are the two halves of the rows and share every tile.  Otherwise they take the even and the
// odd tiles for the same rows and are joined at the end.
//
// A batch of MMAs takes some 600 cycles more from issue to completion than its work (256 cycles), so nothing a stream's softmax
// waits for may hang on its last result: the scores of tile c + 1 are issued as soon as those of c are in registers, and P
// has a place of its own, twice.  A tile takes some 1700 cycles, the exponentials of both streams (768 of them on their pipe)
// and the steps around them; its MMAs take 1024.  256 rows of 32 heads on 32768 positions, D 128, fp16: 148 to 156 us on several cards, some
// 900 TFLOP/s.
// (P over the scores, in two buffers, which hung on the last result: 5 % more; one buffer of 128 positions and MMAs issued behind a
// branch on the lane: 181 us.)
template <int D>
struct Wide {
  static constexpr int kThreads = 352;
  static constexpr int kRows = 128;                     // of a stream
  static constexpr int kPos = 64;
  static constexpr int kUnit = kPos * D * 2;            // bytes of a K or V tile
  static constexpr int kSub = kPos * 128;               // bytes of 64 of its columns
  static constexpr int kQ = kRows * D * 2;              // bytes of a stream's queries
  // A multiple of four: then a unit of the ring always holds tiles of the same one of two streams that take turns, and the stream
  // sees every phase of its barrier.  (A barrier's parity tells a phase from the next, not from the one after: with ten units a
  // stream saw every other phase, and took a tile whose predecessor was late in coming for its own.)
  static constexpr int kUnits = D == 128 ? 8 : 16;
  static_assert(kUnits % 4 == 0, "tiles of one stream in one unit of the ring");
  static constexpr int kRing = 2 * kQ;                  // behind the queries
  static constexpr int kBars = kRing + kUnits * kUnit;
  static constexpr int kSmem = kBars + 512 + 1024;
  static constexpr uint32_t kColO = 256;                // S_s: 128 s; P_s: 128 s + 64 + 32 (tile & 1); O_s: kColO + D s
  static constexpr uint32_t kCols = 512;
};

// Shared-memory descriptor of a tile with rows of 128 bytes (128-byte swizzle, 8-row atoms 1024 bytes apart); across: bytes to
// the next 64 columns of an MN-major operand.  Adding n to it moves it by 16 n bytes.
VK_DEV uint64_t sdesc_tile(uint32_t saddr, uint32_t across) {
  constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);  // stride, descriptor version, swizzle
  return static_cast<uint64_t>(hi) << 32 | (saddr >> 4) | (across >> 4) << 16;
}

// Largest of three, NaN if one is.
VK_DEV float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of two values, -inf..16, on the FMA pipes, for a part of the probabilities: the SM takes 16 exponentials a cycle but 128 FMAs.
// x is split into a whole number n (by adding 1.5 * 2^23) and f in -0.5..0.5; 2^f by the polynomial of degree 5 with the
// smallest largest relative error on that range (fitted in float64 by reweighted least squares: 2^-23.7; in float32
// arithmetic 2^-22.1); n goes into the exponent bits.  Below -127 the result is 2^-149.  NaN gives some number: the caller
// looks for it in the maximum.
VK_DEV float2 poly_exp2(float2 x) {
  x = make_float2(fmaxf(x.x, -127.f), fmaxf(x.y, -127.f));
  const float2 magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f);
  const float2 t = __fadd2_rn(x, magic), n = __fadd2_rn(t, minus);
  const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
  float2 p = make_float2(0.0013276472454890609f, 0.0013276472454890609f);
  p = __ffma2_rn(p, f, make_float2(0.009675540961325169f, 0.009675540961325169f));
  p = __ffma2_rn(p, f, make_float2(0.05550713092088699f, 0.05550713092088699f));
  p = __ffma2_rn(p, f, make_float2(0.24022120237350464f, 0.24022120237350464f));
  p = __ffma2_rn(p, f, make_float2(0.6931469440460205f, 0.6931469440460205f));
  p = __ffma2_rn(p, f, make_float2(1.0000001192092896f, 1.0000001192092896f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

template <typename T, int D>
__global__ void __launch_bounds__(Wide<D>::kThreads, 1)
    wide_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, Args a, Plan pl) {
  using W = Wide<D>;
  constexpr uint32_t kF16 = sizeof(T) == 2 && std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + W::kBars);
  uint64_t* u_full = q_full + 1;
  uint64_t* u_empty = u_full + W::kUnits;
  uint64_t* s_full = u_empty + W::kUnits;  // [2] scores in TMEM
  uint64_t* s_free = s_full + 2;           // [2] scores read
  uint64_t* p_full = s_free + 2;           // [2][2] stream, tile & 1: probabilities in TMEM, result rescaled
  uint64_t* o_full = p_full + 4;           // [2][2] product done
  uint64_t* tmem_free = o_full + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_free + 1);
  Rows* found = reinterpret_cast<Rows*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int r = a.H / a.HK;

  pdl_wait();
  pdl_launch_dependents();
  const Rows w = find_rows<2 * W::kRows, W::kThreads>(a, pl, found);
  if (w.x0 >= w.x1) return;
  const bool both = w.x1 - w.x0 > W::kRows;  // the streams share the tiles
  const int begin = w.split * pl.prefix_chunk, end = min(begin + pl.prefix_chunk, w.len);
  if (begin >= end) {
    store_nothing(a, pl, w.split, w.b0, w.kvh, r, w.x0, w.x1, threadIdx.x, W::kThreads);
    return;
  }
  const int tiles = (end - begin + W::kPos - 1) / W::kPos;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    for (int i = 0; i < W::kUnits; ++i) {
      mbar_init(&u_full[i], 1);
      mbar_init(&u_empty[i], both ? 2 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(tmem_free, 8);
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, W::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int u = 0;
      for (; u < 2 * tiles; ++u) {
        const int slot = u % W::kUnits;
        if (u >= W::kUnits && !mbar_wait(&u_empty[slot], ((u / W::kUnits) & 1) ^ 1)) {
          raise_error(ERR_WAIT_EMPTY);
          break;
        }
        uint8_t* to = smem + W::kRing + slot * W::kUnit;
        const CUtensorMap* map = u & 1 ? &tmV : &tmK;
        mbar_expect_tx(&u_full[slot], W::kUnit);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(to + c * W::kSub, map, &u_full[slot], c * 64, w.kvh, begin + (u >> 1) * W::kPos, w.g);
      }
      // no load may be under way when the CTA ends, whatever the other warps have given up on
      for (int i = u > W::kUnits ? u - W::kUnits : 0; i < u; ++i)
        if (!mbar_wait(&u_full[i % W::kUnits], (i / W::kUnits) & 1)) raise_error(ERR_WAIT_FULL);
    }
  } else if (warp == 1 || warp == 10) {
    // ---------------- MMA issue of one stream: the whole warp in step, one lane issues ----------------
    const int s = warp == 1 ? 0 : 1;
    constexpr uint32_t kTypes = kF16 ? (1u << 7) | (1u << 10) : 0u;  // fp16 operands: clear the bf16 format bits
    constexpr uint32_t idesc_s = idesc_bf16_f32(W::kRows, W::kPos) & ~kTypes;
    constexpr uint32_t idesc_o = (idesc_bf16_f32(W::kRows, D) & ~kTypes) | (1u << 16);  // V is MN-major
    const uint32_t one = elect_one();
    const int n = __shfl_sync(0xffffffffu, tiles, 0), last = __shfl_sync(0xffffffffu, end - begin, 0) - (n - 1) * W::kPos;
    const bool share = __shfl_sync(0xffffffffu, static_cast<int>(both), 0);
    const uint32_t base = __shfl_sync(0xffffffffu, smem_u32(smem), 0), bars = base + W::kBars;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const auto at = [&](const uint64_t* bar0, int i) {  // shared address of a barrier
      return bars + static_cast<uint32_t>(bar0 - q_full + i) * 8;
    };
    bool late = !mbar_wait(q_full, 0);
    const auto wait = [&](uint64_t* bar, uint32_t parity) { late |= !mbar_wait(bar, parity); };
    // units of K are the even ones, of V the odd ones; kUnits is even
    struct Cursor {
      int slot;
      uint32_t phase;
      VK_DEV void next() {
        slot += 2;
        if (slot >= W::kUnits) {
          slot -= W::kUnits;
          phase ^= 1;
        }
      }
    };
    Cursor k{0, 0}, v{1, 0};
    const int mine = share ? n : (n + 1 - s) / 2, step = share ? 1 : 2;  // tiles of this stream
    if (!share && s == 1) {
      k.next();
      v.next();
    }
    const uint64_t qd = sdesc_tile(base + (share ? s : 0) * W::kQ, 16);
    const auto release = [&](Cursor& u) {
      umma_commit_if(one, at(u_empty, u.slot));
      for (int i = 0; i < step; ++i) u.next();
    };
    const auto scores = [&] {  // of the stream's next tile
      wait(&u_full[k.slot], k.phase);
      tc_fence_after();
      const uint64_t kd = sdesc_tile(base + W::kRing + k.slot * W::kUnit, 16);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
        umma_ss_if(one, tm + s * 128, qd + ks / 4 * (16384 / 16) + 2 * (ks % 4), kd + ks / 4 * (W::kSub / 16) + 2 * (ks % 4),
                   idesc_s, ks != 0);
      umma_commit_if(one, at(s_full, s));
      release(k);
    };
    if (mine > 0) scores();
    for (int c = 0; c < mine; ++c) {
      if (c + 1 < mine) {
        wait(&s_free[s], c & 1);
        scores();
      }
      wait(&u_full[v.slot], v.phase);
      if (last < W::kPos && c * step + (share ? 0 : s) == n - 1) {  // what lies behind the prefix may hold anything, and 0 * NaN is NaN
        for (int i = lane; i < (W::kPos - last) * (D / 8); i += 32) {
          const int pos = last + i / (D / 8), ch = i % (D / 8);
          *reinterpret_cast<uint4*>(smem + W::kRing + v.slot * W::kUnit + ch / 8 * W::kSub + pos * 128 + ch % 8 * 16) =
              make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
      }
      wait(&p_full[2 * s + (c & 1)], (c >> 1) & 1);
      tc_fence_after();
      const uint64_t vd = sdesc_tile(base + W::kRing + v.slot * W::kUnit, W::kSub);
#pragma unroll
      for (int ks = 0; ks < W::kPos / 16; ++ks)
        umma_ts_if(one, tm + W::kColO + s * D, tm + s * 128 + 64 + (c & 1) * 32 + ks * 8, vd + ks * (2048 / 16), idesc_o, (c | ks) != 0);
      umma_commit_if(one, at(o_full, 2 * s + (c & 1)));
      release(v);
      if (__any_sync(0xffffffffu, late)) break;
    }
    if (late) raise_error(ERR_WAIT_FULL);
  } else {
    // ---------------- softmax ----------------
    const int s = (warp - 2) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int x = w.x0 + (both ? s * W::kRows : 0) + row;  // this thread's row of the group
    const bool used = x < w.x1;
    const int token = w.b0 + x / r, h = w.kvh * r + x % r;
    // the stream's queries (of joined streams each loads a half of the rows): a warp takes its rows one after another, so that its
    // lanes read whole rows (a row per thread: 5 us)
    {
      constexpr int kChunks = D / 8, kAt = 32 / kChunks;  // 16-byte chunks of a row, rows at a time
      const int64_t mine = used ? token * a.stride_q + h * D : -1;
      uint4 v[kChunks];
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int64_t off = __shfl_sync(0xffffffffu, mine, i * kAt + lane / kChunks);
        v[i] = make_uint4(0, 0, 0, 0);
        if (off >= 0 && (both || i * 2 / kChunks == s))
          v[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + off) + lane % kChunks);
      }
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int ro = quarter * 32 + i * kAt + lane / kChunks, c = lane % kChunks;
        if (both || i * 2 / kChunks == s)
          *reinterpret_cast<uint4*>(smem + (both ? s : 0) * W::kQ + c / 8 * 16384 + ro * 128 + (((c & 7) ^ (ro & 7)) << 4)) = v[i];
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t to = tmem + W::kColO + s * D + lanes;
    const int mine = both ? tiles : (tiles + 1 - s) / 2;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const uint32_t ts = tmem + s * 128 + lanes;
    // The product of the c-th tile is done.  The scores of tile c are issued behind the product c - 2: when they are there, its
    // buffer of P is free, and of the phases of o_full[c & 1] none but that of tile c - 1 or c can be open.
    auto wait_product = [&](int c) { return __all_sync(0xffffffffu, mbar_wait(&o_full[2 * s + (c & 1)], (c >> 1) & 1)); };
    for (int c = 0; c < mine; ++c) {
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[s], c & 1));
      if (!ok) break;
      tc_fence_after();
      float v[W::kPos];
#pragma unroll
      for (int i = 0; i < W::kPos; i += 16) tmem_ld16(ts + i, v + i);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[s]);
      const int left = end - begin - (both ? c : 2 * c + s) * W::kPos;
      if (left < W::kPos) {
#pragma unroll
        for (int i = 0; i < W::kPos; ++i)
          if (i >= left) v[i] = -INFINITY;
      }
      float mx4[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mx4[k] = max3_nan(v[k], v[k + 4], v[k + 8]);
#pragma unroll
        for (int i = 12; i < W::kPos; i += 8) mx4[k] = i + 4 < W::kPos ? max3_nan(mx4[k], v[i + k], v[i + k + 4]) : max3_nan(mx4[k], v[i + k], v[i + k]);
      }
      const float mx = max3_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * pl.scale_log2 - Ref<T>::kDrop;
      const float m_new = mx > m + Ref<T>::kLag || m == -INFINITY ? fmaxf(m, mx) : m;
      const float mu = m_new == -INFINITY ? 0.f : m_new;
      const float2 sc2 = make_float2(pl.scale_log2, pl.scale_log2), nm2 = make_float2(-mu, -mu);
      float2 rs4[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c0 = 0; c0 < W::kPos; c0 += 32) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float2 t = __ffma2_rn(make_float2(v[c0 + i], v[c0 + i + 1]), sc2, nm2);
          const bool poly = i % 8 == 2;  // every fourth pair (the call above with its tails: none 217 us, every fourth 215, every other one 224)
          const float2 p = poly ? poly_exp2(t) : make_float2(fast_exp2(t.x), fast_exp2(t.y));
          rs4[(i >> 1) & 3] = __fadd2_rn(rs4[(i >> 1) & 3], p);
          pk[i / 2] = pack2<T>(p.x, p.y);
        }
        tmem_st16(ts + 64 + (c & 1) * 32 + c0 / 2, pk);
      }
      const float2 rs2 = __fadd2_rn(__fadd2_rn(rs4[0], rs4[1]), __fadd2_rn(rs4[2], rs4[3]));
      const float alpha = fast_exp2(m - mu);
      if (c > 0 && !__all_sync(0xffffffffu, alpha == 1.f)) {
        ok = wait_product(c - 1);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          float o[32];
          uint32_t ob[32];
          tmem_ld16(to + c0, o);
          tmem_ld16(to + c0 + 16, o + 16);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ob[i] = __float_as_uint(o[i] * alpha);
          tmem_st16(to + c0, ob);
          tmem_st16(to + c0 + 16, ob + 16);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[2 * s + (c & 1)]);
      l = alpha * l + rs2.x + rs2.y;
      if (!(mx < INFINITY)) l = NAN;  // a score that is NaN or inf
      m = m_new;
    }
    if (mine > 0 && ok) ok = wait_product(mine - 1);
    if (!ok && lane == 0) raise_error(ERR_WAIT_ACCUM);
    tc_fence_after();
    // joined streams: stream 1 hands its result over in the queries' place (every product that reads them is done: its own, and
    // those of stream 0 before stream 0 reads)
    float* other = reinterpret_cast<float*>(smem);  // [D][128]
    float2* other_ml = reinterpret_cast<float2*>(smem + W::kRing);  // [128], over the ring's first unit
    if (!both) {
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (s == 1 && mine > 0) {
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          float o[32];
          tmem_ld16(to + c0, o);
          tmem_ld16(to + c0 + 16, o + 16);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) other[(c0 + i) * 128 + row] = o[i];
        }
      }
      if (s == 1) other_ml[row] = make_float2(m, l);
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    if (both || s == 0) {
      float f0 = 1.f, f1 = 0.f;
      if (!both && tiles > 1) {
        const float2 ml = other_ml[row];
        const float mn = fmaxf(m, ml.x), mu = mn == -INFINITY ? 0.f : mn;
        f0 = fast_exp2(m - mu);
        f1 = fast_exp2(ml.x - mu);
        l = l * f0 + ml.y * f1;
        m = mn;
      }
      // the warp's 32 rows, a half of the columns at a time, turned in shared memory so that a row is written in one piece
      // (straight from the threads' rows: 5 us more for every CTA).  Its place: this warp's part of the stream's queries, or of
      // the ring behind other_ml where the queries' place holds the other stream's result.
      float4* turn = reinterpret_cast<float4*>(smem + (both ? s * W::kQ : W::kRing + W::kUnit) + quarter * (W::kQ / 4));
      constexpr int kC = D / 8;  // float4s of half a row
      const int64_t slot = (static_cast<int64_t>(w.split) * a.B + token) * a.H + h;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int c0 = 0; c0 < D / 2; c0 += 32) {
          float o[32];
          tmem_ld16(to + half * (D / 2) + c0, o);
          tmem_ld16(to + half * (D / 2) + c0 + 16, o + 16);
          tmem_wait_ld();
          if (!both && tiles > 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = o[i] * f0 + other[(half * (D / 2) + c0 + i) * 128 + row] * f1;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            turn[lane * kC + (((c0 + i) / 4) ^ (lane & 7))] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
        __syncwarp();
#pragma unroll 4
        for (int i = lane; i < 32 * kC; i += 32) {
          const int ro = i / kC, c = i % kC;
          const int64_t to_slot = __shfl_sync(0xffffffffu, used ? slot : -1, ro);
          if (to_slot >= 0)
            *reinterpret_cast<float4*>(pl.ws_o + to_slot * D + half * (D / 2) + c * 4) = turn[ro * kC + (c ^ (ro & 7))];
        }
        __syncwarp();
      }
      if (used) pl.ws_ml[slot] = make_float2(m, l);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(tmem_free);
  }
  if (warp == 1) {
    if (!mbar_wait(tmem_free, 0) && lane == 0) raise_error(ERR_WAIT_ACCUM);
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, W::kCols);
  }
}

// Joins the partial results of a row and head: W warps each take every W-th run of 32 splits.  A warp's lanes take the weights of
// 32 splits at once; then their values come four loads at a time.
template <typename T, int D, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W) join_kernel(Args a, Plan pl, int splits) {
  constexpr int PER = D / 32;
  using V = typename std::conditional<PER == 2, float2, float4>::type;
  __shared__ V so[W][32];
  __shared__ float2 sml[W];
  const int lane = threadIdx.x & 31, warp = W == 1 ? 0 : threadIdx.x >> 5;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t rows = static_cast<int64_t>(a.B) * a.H;
  const int64_t row = W == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= rows || row / a.H >= a.offsets[a.P]) return;
  float m = -INFINITY, l = 0.f, o[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = 0.f;
  for (int s0 = warp * 32; s0 < splits; s0 += W * 32) {
    const int n = min(32, splits - s0);
    const float2 ml = lane < n ? __ldcg(&pl.ws_ml[(s0 + lane) * rows + row]) : make_float2(-INFINITY, 0.f);
    float mn = ml.x;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
    mn = fmaxf(mn, m);
    const float mu = mn == -INFINITY ? 0.f : mn, f = fast_exp2(m - mu);
    const float weight = ml.y == 0.f ? 0.f : fast_exp2(ml.x - mu);
    l = l * f + ml.y * weight;  // this lane's share
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] *= f;
    m = mn;
    const uint32_t there = __ballot_sync(0xffffffffu, ml.y != 0.f);  // (NaN too) elsewhere no values were written
    const V* at = reinterpret_cast<const V*>(pl.ws_o + (s0 * rows + row) * D) + lane;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float wk = __shfl_sync(0xffffffffu, weight, k);
      if (!(there >> k & 1)) continue;
      const V v = __ldcg(at + k * (rows * 32));
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] += wk * reinterpret_cast<const float*>(&v)[i];
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  if (W > 1) {
#pragma unroll
    for (int i = 0; i < PER; ++i) reinterpret_cast<float*>(&so[warp][lane])[i] = o[i];
    if (lane == 0) sml[warp] = make_float2(m, l);
    __syncthreads();
    if (warp) return;
    for (int w = 1; w < W; ++w) {
      const float2 ml = sml[w];
      if (ml.y == 0.f) continue;
      const float mn = fmaxf(m, ml.x), mu = mn == -INFINITY ? 0.f : mn;
      const float fa = fast_exp2(m - mu), fb = fast_exp2(ml.x - mu);
      l = l * fa + ml.y * fb;
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] = o[i] * fa + reinterpret_cast<const float*>(&so[w][lane])[i] * fb;
      m = mn;
    }
  }
  T* op = static_cast<T*>(a.out) + row * D + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; i += 2) *reinterpret_cast<uint32_t*>(op + i) = l == 0.f ? 0u : pack2<T>(o[i] / l, o[i + 1] / l);
  if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;  // (of one position m + log2 l is exact)
}

}  // namespace sattn
}  // namespace vk
