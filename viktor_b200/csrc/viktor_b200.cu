// C ABI of the viktor_b200 kernels (declared in include/viktor_b200.h).  Single translation unit: the kernel
// headers are included here so that all kernels share one device error word without relocatable device code.
#include <algorithm>
#include <cstring>
#include <type_traits>
#include <utility>

#include "decode_attention.cuh"
#include "elementwise.cuh"
#include "gemm_tc.cuh"
#include "kv_pages.cuh"
#include "logit_penalties.cuh"
#include "prefill_attention.cuh"
#include "shared_attention.cuh"
#include "stitch_host.h"
#include "vk_host.cuh"

namespace vk {

static int g_pdl = 1;

#ifndef VK_ATTN_MAX_CHUNK
#define VK_ATTN_MAX_CHUNK 1024
#endif

// Per-device record of kernels whose dynamic shared-memory limit has been raised.  The first launch of each
// kernel on a device must happen outside stream capture (engines warm up eagerly before capturing).
// most_shared: the SM keeps as much of its memory as shared memory as it can while the kernel runs, so that as many CTAs as its
// 228 KB hold are resident whatever ran before.
template <typename K>
static bool ensure_smem(K kernel, int bytes, bool most_shared = false) {
  struct Entry {
    const void* fn;
    uint64_t mask;
  };
  static Entry table[64];
  static int used = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  const void* fn = reinterpret_cast<const void*>(kernel);
  int i = 0;
  for (; i < used; ++i)
    if (table[i].fn == fn) break;
  if (i < used && (table[i].mask & bit)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (most_shared && cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                          cudaSharedmemCarveoutMaxShared) != cudaSuccess)
    return false;
  if (i == used) {
    if (used == 64) return true;
    table[used++] = Entry{fn, 0};
  }
  table[i].mask |= bit;
  return true;
}

template <typename... KArgs, typename... Args>
static int launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, void* stream, int cluster_x,
                  Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attrs[2];
  int na = 0;
  if (g_pdl) {
    attrs[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  if (cluster_x > 1) {
    attrs[na].id = cudaLaunchAttributeClusterDimension;
    attrs[na].val.clusterDim.x = cluster_x;
    attrs[na].val.clusterDim.y = 1;
    attrs[na].val.clusterDim.z = 1;
    ++na;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = na;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  if (e != cudaSuccess) {
    fprintf(stderr, "viktor_b200: launch failed: %s\n", cudaGetErrorString(e));
    return VK_ERR_CUDA;
  }
  return VK_OK;
}

// SMs of the current device (cached per device); 0 if the runtime cannot tell.
static int device_sm_count() {
  static int sm_count[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!sm_count[dev] && cudaDeviceGetAttribute(&sm_count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sm_count[dev];
}

static inline unsigned blocks_for(int64_t n, int per) { return static_cast<unsigned>((n + per - 1) / per); }

static inline int log2_of(int power) {
  int k = 0;
  while ((1 << k) < power) ++k;
  return k;
}

constexpr int64_t kSmallM = 4096;  // decode-sized GEMMs: narrow tiles + split-K clusters; prefill: wide tiles

// ---- GEMM dispatch ----------------------------------------------------------------------------------------
template <int BN, int EPI, int NK>
static int run_gemm_nk(const void* A, const void* B, int64_t M, int N, int K, const gemm::EpiArgs& ep, int n_tiles,
                       int64_t b_rows, void* stream) {
  using gemm::SmemLayout;
  const int nkb = K / gemm::BK / NK;
  int cap = gemm::max_stages_for(BN);
  if (M <= kSmallM) {
    cap = gemm::kMaxStages;
    while (cap > 2 && SmemLayout(BN, NK, cap, EPI).total > gemm::kSmemBudget) --cap;
  }
  const int stages = nkb < cap ? nkb : cap;
  const SmemLayout L(BN, NK, stages, EPI);
  CUtensorMap ta, tb;
  const uint32_t b_box = EPI == gemm::SWIGLU ? BN / 2 : BN;
  if (!make_map_kmajor(&ta, A, static_cast<uint64_t>(M), K, K, gemm::BM)) return VK_ERR_ARG;
  if (!make_map_kmajor(&tb, B, static_cast<uint64_t>(b_rows), K, K, b_box)) return VK_ERR_ARG;
  auto kern = gemm::gemm_kernel<BN, EPI, NK>;
  if (!ensure_smem(kern, gemm::kSmemBudget)) return VK_ERR_CUDA;
  dim3 grid(NK, n_tiles, static_cast<unsigned>((M + gemm::BM - 1) / gemm::BM));
  return launch(kern, grid, dim3(gemm::kThreads), L.total, stream, NK, ta, tb, static_cast<int>(M), N, K, stages,
                ep);
}

// Split-K factor for small-M GEMMs.  A decode GEMM is bound by latency (load round trips, the epilogue), not
// by throughput, so it is split over K as far as one wave allows: the largest power of two, at most
// VK_MAX_SPLITK (a build-time tuning constant, 8 by default), with tiles x splits CTAs on at most one SM each
// and every split at least two 64-wide K blocks.  (Measured on B200, full decode steps with two row groups in
// one CUDA graph: a second wave costs more than the shorter K loop saves, and one-block splits cost more in
// the reduction than they save in the K loop.)
#ifndef VK_MAX_SPLITK
#define VK_MAX_SPLITK 8
#endif
static int pick_nk(int64_t M, int n_tiles, int K) {
  const int64_t tiles = n_tiles * ((M + gemm::BM - 1) / gemm::BM);
  const int kb = K / gemm::BK;
  const int sms = device_sm_count();
  int nk = 1;
  while (nk < VK_MAX_SPLITK && tiles * nk * 2 <= sms && kb % (nk * 2) == 0 && kb / (nk * 2) >= 2) nk *= 2;
  return nk;
}

template <int BN, int EPI>
static int run_gemm(const void* A, const void* B, int64_t M, int N, int K, const gemm::EpiArgs& ep, int n_tiles,
                    int64_t b_rows, int nk, void* stream) {
  if (M <= 0 || M > (int64_t(1) << 31) - 128) return VK_ERR_ARG;
  if (K <= 0 || K % gemm::BK != 0 || (K / gemm::BK) % nk != 0) return VK_ERR_ARG;
  if (!aligned16(A) || !aligned16(B)) return VK_ERR_ARG;
  switch (nk) {
    case 1: return run_gemm_nk<BN, EPI, 1>(A, B, M, N, K, ep, n_tiles, b_rows, stream);
    case 2: return run_gemm_nk<BN, EPI, 2>(A, B, M, N, K, ep, n_tiles, b_rows, stream);
    case 4: return run_gemm_nk<BN, EPI, 4>(A, B, M, N, K, ep, n_tiles, b_rows, stream);
    case 8: return run_gemm_nk<BN, EPI, 8>(A, B, M, N, K, ep, n_tiles, b_rows, stream);
    default: return VK_ERR_ARG;
  }
}

// Large-M GEMMs (prefill): the persistent BN = 256 kernel when N fits its tiles.
#ifndef VK_PERSISTENT_GEMM
#define VK_PERSISTENT_GEMM 1
#endif
template <int EPI>
static bool persistent_fits(int64_t M, int N) {
  if (!VK_PERSISTENT_GEMM || M <= 0 || M > (int64_t(1) << 31) - 128) return false;
  return EPI == gemm::SWIGLU ? (N / 2) % (gemm::kPBN / 2) == 0 && N % 2 == 0 : N % gemm::kPBN == 0;
}

template <int EPI>
static int run_gemm_persistent(const void* A, const void* B, int64_t M, int N, int K, const gemm::EpiArgs& ep,
                               int64_t b_rows, void* stream) {
  if (K <= 0 || K % gemm::BK != 0) return VK_ERR_ARG;
  if (!aligned16(A) || !aligned16(B)) return VK_ERR_ARG;
  CUtensorMap ta, tb;
  const uint32_t b_box = EPI == gemm::SWIGLU ? gemm::kPBN / 2 : gemm::kPBN;
  if (!make_map_kmajor(&ta, A, static_cast<uint64_t>(M), K, K, gemm::BM)) return VK_ERR_ARG;
  if (!make_map_kmajor(&tb, B, static_cast<uint64_t>(b_rows), K, K, b_box)) return VK_ERR_ARG;
  const int sms = device_sm_count();
  if (sms <= 0) return VK_ERR_CUDA;
  const int64_t n_tiles = (EPI == gemm::SWIGLU ? N / 2 : N) / b_box;
  const int64_t tiles = n_tiles * ((M + gemm::BM - 1) / gemm::BM);
  auto kern = gemm::gemm_persistent_kernel<EPI>;
  if (!ensure_smem(kern, gemm::kPSmemBytes)) return VK_ERR_CUDA;
  return launch(kern, dim3(static_cast<unsigned>(tiles < sms ? tiles : sms)), dim3(gemm::kPThreads),
                gemm::kPSmemBytes, stream, 1, ta, tb, static_cast<int>(M), N, K, ep);
}

static gemm::EpiArgs epi_zero() {
  gemm::EpiArgs e;
  memset(&e, 0, sizeof(e));
  return e;
}

// Failure-path probe: one CTA whose first thread waits on an mbarrier that nothing arrives on (no copy in flight,
// no other thread involved).  The bounded wait gives up after limit_ns, the thread records ERR_WAIT_FULL exactly
// as a pipeline wait that ran out does, writes how long it waited and the kernel returns normally.
__global__ void bounded_wait_probe_kernel(uint64_t limit_ns, unsigned long long* waited_ns) {
  __shared__ __align__(8) uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint64_t t0 = globaltimer();
    const bool done = mbar_wait_for(&bar, 0, limit_ns);
    if (!done) raise_error(ERR_WAIT_FULL);
    if (waited_ns) *waited_ns = globaltimer() - t0;
  }
}


}  // namespace vk

using namespace vk;

extern "C" {

int vk_version(void) { return 100; }

int vk_read_device_errors(uint32_t* bits, int clear) {
  if (!bits) return VK_ERR_ARG;
  if (cudaMemcpyFromSymbol(bits, vk::g_error_word, sizeof(uint32_t)) != cudaSuccess) return VK_ERR_CUDA;
  if (clear) {
    const uint32_t z = 0;
    if (cudaMemcpyToSymbol(vk::g_error_word, &z, sizeof(uint32_t)) != cudaSuccess) return VK_ERR_CUDA;
  }
  return VK_OK;
}

int vk_set_pdl(int enable) {
  vk::g_pdl = enable ? 1 : 0;
  return VK_OK;
}

int vk_test_bounded_wait(uint64_t limit_ns, unsigned long long* waited_ns, void* stream) {
  if (limit_ns == 0 || limit_ns > vk::kWaitLimitNs) return VK_ERR_ARG;
  bounded_wait_probe_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(limit_ns, waited_ns);
  return cudaGetLastError() == cudaSuccess ? VK_OK : VK_ERR_CUDA;
}

int vk_add_rmsnorm(void* x, const void* delta, const void* w, void* h, int64_t n, int d, float eps, void* stream) {
  if (n < 0 || d != 512 || !x || !w || !h) return n == 0 ? VK_OK : VK_ERR_ARG;
  if (n == 0) return VK_OK;
  if (!aligned16(x) || !aligned16(w) || !aligned16(h) || (delta && !aligned16(delta))) return VK_ERR_ARG;
  return launch(ew::rmsnorm_rows_kernel<512>, dim3(blocks_for(n, 8)), dim3(256), 0, stream, 1,
                static_cast<__nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(delta),
                static_cast<const int64_t*>(nullptr), static_cast<const __nv_bfloat16*>(nullptr), int64_t(0),
                static_cast<const __nv_bfloat16*>(w), static_cast<__nv_bfloat16*>(h), n, eps);
}

int vk_embed_rmsnorm(const int64_t* tok, const void* emb, int64_t vocab, const void* w, void* x, void* h, int64_t n,
                     int d, float eps, void* stream) {
  if (n == 0) return VK_OK;
  if (n < 0 || d != 512 || !tok || !emb || !w || !x || !h || vocab <= 0) return VK_ERR_ARG;
  if (!aligned16(emb) || !aligned16(w) || !aligned16(x) || !aligned16(h)) return VK_ERR_ARG;
  return launch(ew::rmsnorm_rows_kernel<512>, dim3(blocks_for(n, 8)), dim3(256), 0, stream, 1,
                static_cast<__nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(nullptr), tok,
                static_cast<const __nv_bfloat16*>(emb), vocab, static_cast<const __nv_bfloat16*>(w),
                static_cast<__nv_bfloat16*>(h), n, eps);
}

int vk_qkv_rope_cache(const void* qkv, const void* q_norm_w, const void* k_norm_w, const float* cos,
                      const float* sin, int rope_len, const int32_t* pos, const int32_t* rope_pos,
                      const int32_t* seq, void* q, void* k_cache, void* v_cache, void* k_out, void* v_out,
                      int64_t n, int64_t stride_cb, int64_t stride_cs, int cache_rows, int cache_len, float eps,
                      int n_heads, int n_kv_heads, int head_dim, void* stream) {
  if (n == 0) return VK_OK;
  if (head_dim != 64 || n_heads <= 0 || n_kv_heads <= 0) return VK_ERR_UNSUPPORTED;
  if (n < 0 || !qkv || !q_norm_w || !k_norm_w || !cos || !sin || !pos || !seq || !q || !k_cache || !v_cache)
    return VK_ERR_ARG;
  if (!aligned16(qkv) || !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || stride_cs % 8 ||
      stride_cb % 8 || (k_out && !aligned16(k_out)) || (v_out && !aligned16(v_out)))
    return VK_ERR_ARG;
  const int64_t threads = n * (n_heads + 2 * n_kv_heads);
  return launch(ew::qkv_rope_cache_kernel, dim3(blocks_for(threads, 128)), dim3(128), 0, stream, 1,
                static_cast<const __nv_bfloat16*>(qkv), static_cast<const __nv_bfloat16*>(q_norm_w),
                static_cast<const __nv_bfloat16*>(k_norm_w), cos, sin, rope_len, pos, rope_pos, seq,
                static_cast<__nv_bfloat16*>(q), static_cast<__nv_bfloat16*>(k_cache),
                static_cast<__nv_bfloat16*>(v_cache), static_cast<__nv_bfloat16*>(k_out),
                static_cast<__nv_bfloat16*>(v_out), n, stride_cb, stride_cs, cache_rows, cache_len, eps, n_heads,
                n_kv_heads);
}

// Shared body of vk_linear / vk_linear_rmsnorm: plain or SwiGLU GEMM, bf16 or f32 out, optional folded norm.
static int linear_impl(const void* x, const float* ssq, float eps, const void* w, void* y, int64_t M, int N, int K,
                       int swiglu, int out_f32, void* stream) {
  if (M == 0) return VK_OK;
  if (!x || !w || !y || N <= 0 || M < 0) return VK_ERR_ARG;
  if (ssq && (K != 512 || !aligned16(ssq))) return VK_ERR_ARG;
  gemm::EpiArgs ep = epi_zero();
  ep.y = y;
  ep.ssq_in = ssq;
  ep.eps = eps;
  if (swiglu) {
    if (out_f32 || N % 2) return VK_ERR_ARG;
    const int F = N / 2;
    ep.ldy = F;
    ep.n_valid = F;
    if (M <= kSmallM) {
      if (F % 64) return VK_ERR_ARG;
      // narrow tiles (32 outputs) while they fit in one wave, for more CTAs in flight; else 64 outputs
      if ((F / 32) * ((M + gemm::BM - 1) / gemm::BM) <= device_sm_count())
        return run_gemm<64, gemm::SWIGLU>(x, w, M, N, K, ep, F / 32, N, pick_nk(M, F / 32, K), stream);
      return run_gemm<128, gemm::SWIGLU>(x, w, M, N, K, ep, F / 64, N, pick_nk(M, F / 64, K), stream);
    }
    if (F % 64) return VK_ERR_ARG;
    if (persistent_fits<gemm::SWIGLU>(M, N)) return run_gemm_persistent<gemm::SWIGLU>(x, w, M, N, K, ep, N, stream);
    return run_gemm<128, gemm::SWIGLU>(x, w, M, N, K, ep, F / 64, N, 1, stream);
  }
  ep.ldy = N;
  ep.n_valid = N;
  if (out_f32) {
    if (N <= 16) return run_gemm<16, gemm::STORE_F32>(x, w, M, N, K, ep, 1, N, pick_nk(M, 1, K), stream);
    const int nt = (N + 127) / 128;
    return run_gemm<128, gemm::STORE_F32>(x, w, M, N, K, ep, nt, N, M <= kSmallM ? pick_nk(M, nt, K) : 1, stream);
  }
  if (N <= 64 || M <= kSmallM) {
    const int nt = (N + 63) / 64;
    return run_gemm<64, gemm::STORE_BF16>(x, w, M, N, K, ep, nt, N, M <= kSmallM ? pick_nk(M, nt, K) : 1, stream);
  }
  if (persistent_fits<gemm::STORE_BF16>(M, N))
    return run_gemm_persistent<gemm::STORE_BF16>(x, w, M, N, K, ep, N, stream);
  return run_gemm<128, gemm::STORE_BF16>(x, w, M, N, K, ep, (N + 127) / 128, N, 1, stream);
}

int vk_linear(const void* x, const void* w, void* y, int64_t M, int N, int K, int swiglu, int out_f32,
              void* stream) {
  return linear_impl(x, nullptr, 0.f, w, y, M, N, K, swiglu, out_f32, stream);
}

int vk_linear_rmsnorm(const void* x, const float* ssq, float eps, const void* w_folded, void* y, int64_t M, int N,
                      int K, int swiglu, int out_f32, void* stream) {
  if (M != 0 && !ssq) return VK_ERR_ARG;
  return linear_impl(x, ssq, eps, w_folded, y, M, N, K, swiglu, out_f32, stream);
}

int vk_swiglu(const void* gu, void* out, int64_t n, int F, void* stream) {
  if (n == 0) return VK_OK;
  if (!gu || !out || n < 0 || F <= 0) return VK_ERR_ARG;
  return launch(ew::swiglu_kernel, dim3(blocks_for(n * F, 256)), dim3(256), 0, stream, 1,
                static_cast<const __nv_bfloat16*>(gu), static_cast<__nv_bfloat16*>(out), n, F);
}

// Fields shared by the selection entry points (viktor/triton_ops.py:172-209, viktor/engine.py:79-89).
static ew::GreedyArgs greedy_args(const float* logits, int64_t ld_logits, const float* bias, const uint8_t* is_tail,
                                  const uint8_t* is_homo, int homo_stop, int64_t* tok, int64_t* run, int64_t* pos,
                                  const int64_t* plen, const int64_t* rope_off, int64_t* out, int64_t out_stride,
                                  int64_t out_cols, int32_t* pos32, int32_t* seqlens, int32_t* rpos32, int B, int V,
                                  int eos, int pad, const void* emb, void* x, float* ssq) {
  ew::GreedyArgs a;
  memset(&a, 0, sizeof(a));
  a.logits = logits;
  a.ld_logits = ld_logits;
  a.bias = bias;
  a.is_tail = is_tail;
  a.is_homo = is_homo;
  a.homo_stop = homo_stop;
  a.tok = tok;
  a.run = run;
  a.pos = pos;
  a.plen = plen;
  a.rope_off = rope_off;
  a.out = out;
  a.out_stride = out_stride;
  a.out_cols = out_cols;
  a.pos32 = pos32;
  a.seqlens = seqlens;
  a.rpos32 = rpos32;
  a.B = B;
  a.V = V;
  a.eos = eos;
  a.pad = pad;
  a.emb = static_cast<const __nv_bfloat16*>(emb);
  a.x = static_cast<__nv_bfloat16*>(emb ? x : nullptr);
  a.ssq = ssq;
  a.temperature = 1.f;
  return a;
}

static bool greedy_state_ok(const float* bias, const uint8_t* is_tail, const uint8_t* is_homo, const int64_t* tok,
                            const int64_t* run, const int64_t* pos, const int64_t* plen, const int64_t* rope_off,
                            const int64_t* out, const int32_t* pos32, const int32_t* seqlens, const int32_t* rpos32,
                            int B, int V, const void* emb, const void* x, const float* ssq) {
  return B > 0 && V > 0 && bias && is_tail && is_homo && tok && run && pos && plen && rope_off && out && pos32 &&
         seqlens && rpos32 && (!emb || (x && ssq));
}

int vk_greedy_update(const float* logits, int64_t ld_logits, const float* bias, const uint8_t* is_tail,
                     const uint8_t* is_homo, int homo_stop, int64_t* tok, int64_t* run, int64_t* pos,
                     const int64_t* plen, const int64_t* rope_off, int64_t* out, int64_t out_stride,
                     int64_t out_cols, int32_t* pos32, int32_t* seqlens, int32_t* rpos32, int B, int V, int eos,
                     int pad, const void* emb, void* x, float* ssq, void* stream) {
  if (B == 0) return VK_OK;
  if (!logits || !greedy_state_ok(bias, is_tail, is_homo, tok, run, pos, plen, rope_off, out, pos32, seqlens, rpos32,
                                  B, V, emb, x, ssq))
    return VK_ERR_ARG;
  const ew::GreedyArgs a = greedy_args(logits, ld_logits, bias, is_tail, is_homo, homo_stop, tok, run, pos, plen,
                                       rope_off, out, out_stride, out_cols, pos32, seqlens, rpos32, B, V, eos, pad,
                                       emb, x, ssq);
  return launch(ew::greedy_kernel<512>, dim3(B), dim3(128), 0, stream, 1, a);
}

int vk_prefill_plan(const int32_t* lens, int n, int row0, int pos_scale, int64_t total, int32_t* cu,
                    int32_t* frame_idx, int64_t* last, int32_t* pos, int32_t* seq, int32_t* rpos, int32_t* lengths,
                    void* stream) {
  if (n <= 0 || n > ew::kPlanMaxSeq || row0 < 0 || pos_scale < 1 || total < n || total > (int64_t(1) << 31) - 1 ||
      !lens || !cu || !last || !pos || !seq || !lengths || (total > n && !frame_idx))
    return VK_ERR_ARG;
  ew::PlanArgs a;
  a.lens = lens;
  a.n = n;
  a.row0 = row0;
  a.pos_scale = pos_scale;
  a.total = total;
  a.cu = cu;
  a.frame_idx = frame_idx;
  a.last = last;
  a.pos = pos;
  a.seq = seq;
  a.rpos = rpos;
  a.lengths = lengths;
  const int sms = device_sm_count();
  if (sms <= 0) return VK_ERR_CUDA;
  const int64_t want = (total + ew::kPlanThreads - 1) / ew::kPlanThreads;
  const unsigned grid = static_cast<unsigned>(want < 2 * sms ? want : 2 * sms);
  return launch(ew::prefill_plan_kernel, dim3(grid), dim3(ew::kPlanThreads), 0, stream, 1, a);
}

int vk_sample_update(const float* logits, int64_t ld_logits, const float* bias, const uint8_t* is_tail,
                     const uint8_t* is_homo, int homo_stop, int64_t* tok, int64_t* run, int64_t* pos,
                     const int64_t* plen, const int64_t* rope_off, int64_t* out, int64_t out_stride,
                     int64_t out_cols, int32_t* pos32, int32_t* seqlens, int32_t* rpos32, int B, int V, int eos,
                     int pad, const void* emb, void* x, float* ssq, const float* noise, int64_t ld_noise,
                     float temperature, void* stream) {
  if (B == 0) return VK_OK;
  if (!logits || !greedy_state_ok(bias, is_tail, is_homo, tok, run, pos, plen, rope_off, out, pos32, seqlens, rpos32,
                                  B, V, emb, x, ssq) ||
      !noise || ld_noise < V || !(temperature > 0.f) || !(temperature < INFINITY))
    return VK_ERR_ARG;
  ew::GreedyArgs a = greedy_args(logits, ld_logits, bias, is_tail, is_homo, homo_stop, tok, run, pos, plen, rope_off,
                                 out, out_stride, out_cols, pos32, seqlens, rpos32, B, V, eos, pad, emb, x, ssq);
  a.noise = noise;
  a.ld_noise = ld_noise;
  a.temperature = temperature;
  return launch(ew::greedy_kernel<512>, dim3(B), dim3(128), 0, stream, 1, a);
}

int vk_head_select(const void* x_final, const float* ssq_final, float eps, const void* head_w, const float* bias,
                   const uint8_t* is_tail, const uint8_t* is_homo, int homo_stop, int64_t* tok, int64_t* run,
                   int64_t* pos, const int64_t* plen, const int64_t* rope_off, int64_t* out, int64_t out_stride,
                   int64_t out_cols, int32_t* pos32, int32_t* seqlens, int32_t* rpos32, int B, int V, int eos, int pad,
                   const void* emb, void* x, float* ssq, const float* noise, int64_t ld_noise, float temperature,
                   const int64_t* limit, int shrink_done, void* stream) {
  if (B == 0) return VK_OK;
  if (!x_final || !ssq_final || !head_w || V > ew::kHeadMaxV || !aligned16(x_final) || !aligned16(ssq_final) ||
      !aligned16(head_w) ||
      !greedy_state_ok(bias, is_tail, is_homo, tok, run, pos, plen, rope_off, out, pos32, seqlens, rpos32, B, V, emb,
                       x, ssq))
    return VK_ERR_ARG;
  if (noise && (ld_noise < V || !(temperature > 0.f) || !(temperature < INFINITY))) return VK_ERR_ARG;
  ew::GreedyArgs a = greedy_args(nullptr, 0, bias, is_tail, is_homo, homo_stop, tok, run, pos, plen, rope_off, out,
                                 out_stride, out_cols, pos32, seqlens, rpos32, B, V, eos, pad, emb, x, ssq);
  a.head_x = static_cast<const __nv_bfloat16*>(x_final);
  a.head_ssq = ssq_final;
  a.head_w = static_cast<const __nv_bfloat16*>(head_w);
  a.head_eps = eps;
  a.limit = limit;
  a.shrink_done = shrink_done ? 1 : 0;
  if (noise) {
    a.noise = noise;
    a.ld_noise = ld_noise;
    a.temperature = temperature;
  }
  return launch(ew::greedy_kernel<512>, dim3(B), dim3(128), 0, stream, 1, a);
}

size_t vk_decode_attention_workspace_bytes(int nq, int S) {
  if (nq <= 0 || S <= 0) return 0;
  const size_t splits = (S + attn::kMinChunk - 1) / attn::kMinChunk;
  const size_t counters = ((size_t)nq * 4 + 255) / 256 * 256;
  const size_t ml = ((size_t)nq * splits * 8 * 2 * 4 + 255) / 256 * 256;
  const size_t o = (size_t)nq * splits * 8 * 64 * 4;
  return counters + ml + o;
}

// TMA maps of one layer of the KV cache, [rows][S][2 heads][64] bf16: boxes of box_pos positions x one head.
static bool make_cache_maps(CUtensorMap* mk, CUtensorMap* mv, const void* k, const void* v, int cache_rows, int S,
                            int64_t stride_kb, int64_t stride_ks, uint32_t box_pos = 64) {
  uint64_t dims[4] = {64, 2, static_cast<uint64_t>(S), static_cast<uint64_t>(cache_rows)};
  uint64_t strides[3] = {128, static_cast<uint64_t>(stride_ks) * 2, static_cast<uint64_t>(stride_kb) * 2};
  uint32_t box[4] = {64, 1, box_pos, 1};
  return make_map_bf16(mk, k, 4, dims, strides, box, true) && make_map_bf16(mv, v, 4, dims, strides, box, true);
}

int vk_decode_attention(const void* q, const void* k_cache, const void* v_cache, const int32_t* lengths, void* out,
                        int nq, int row0, int cache_rows, int S, int64_t stride_kb, int64_t stride_ks,
                        void* workspace, size_t workspace_bytes, void* stream) {
  if (nq == 0) return VK_OK;
  if (nq < 0 || !q || !k_cache || !v_cache || !lengths || !out || !workspace || S <= 0 || row0 < 0 ||
      row0 + nq > cache_rows || stride_ks < 128 || stride_kb < stride_ks * S)
    return VK_ERR_ARG;
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace)) return VK_ERR_ARG;
  if (workspace_bytes < vk_decode_attention_workspace_bytes(nq, S)) return VK_ERR_ARG;
  CUtensorMap mk, mv;
  if (!make_cache_maps(&mk, &mv, k_cache, v_cache, cache_rows, S, stride_kb, stride_ks)) return VK_ERR_ARG;
  const int splits = (S + attn::kMinChunk - 1) / attn::kMinChunk;  // workspace slots per query
  const int sms = device_sm_count();
  if (sms <= 0) return VK_ERR_CUDA;
  // longest split that still fills every SM with its two resident CTAs (judged on the cache length); at most
  // VK_ATTN_MAX_CHUNK positions (a build-time tuning constant)
  int chunk = VK_ATTN_MAX_CHUNK;
  while (chunk > attn::kMinChunk && static_cast<int64_t>(nq) * ((S + chunk - 1) / chunk) < 2 * sms) chunk /= 2;
  attn::DecodeArgs a;
  memset(&a, 0, sizeof(a));
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lengths = lengths;
  a.row0 = row0;
  a.nq = nq;
  a.max_splits = splits;
  a.S = S;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.counters = reinterpret_cast<int*>(ws);
  const size_t counters = ((size_t)nq * 4 + 255) / 256 * 256;
  a.ws_ml = reinterpret_cast<float*>(ws + counters);
  a.ws_o = reinterpret_cast<float*>(ws + counters + ((size_t)nq * splits * 8 * 2 * 4 + 255) / 256 * 256);
  a.scale_log2 = 0.125f * 1.4426950408889634f;
  a.chunk = chunk;
  if (!ensure_smem(attn::decode_attn_kernel, attn::kSmemBytes)) return VK_ERR_CUDA;
  return launch(attn::decode_attn_kernel, dim3((S + chunk - 1) / chunk, nq), dim3(attn::kThreads), attn::kSmemBytes,
                stream, 1, mk, mv, a);
}

// ---- int8 prefix KV ------------------------------------------------------------------------------------------
// Split plan of decode_attn_i8_kernel: bf16 splits of `chunk` positions and at most n8max int8 splits of about
// 2 x chunk positions (the same bytes per CTA), the longest chunk that still fills every SM twice.
struct I8Plan {
  int chunk, n8max, n16max;
};
static I8Plan i8_plan(int nq, int S8, int max_tail, int sms) {
  I8Plan p{};
  for (int c = 1024;; c /= 2) {
    p.chunk = c;
    p.n8max = (S8 + 2 * c - 1) / (2 * c);
    p.n16max = (max_tail + c - 1) / c;
    if (c == 128 || static_cast<int64_t>(nq) * (p.n8max + p.n16max) >= 2 * sms) break;
  }
  return p;
}
static size_t i8_slots_bound(int S8, int max_tail) { return (S8 + 255) / 256 + (max_tail + 127) / 128; }

size_t vk_decode_attention_i8_workspace_bytes(int nq, int S8, int max_tail) {
  if (nq <= 0 || S8 <= 0 || max_tail <= 0) return 0;
  const size_t splits = i8_slots_bound(S8, max_tail);
  const size_t counters = ((size_t)nq * 4 + 255) / 256 * 256;
  const size_t ml = ((size_t)nq * splits * 8 * 2 * 4 + 255) / 256 * 256;
  return counters + ml + (size_t)nq * splits * 8 * 64 * 4;
}

int vk_kv_quantize(const void* k_cache, const void* v_cache, int cache_rows, int S, int64_t stride_kb,
                   int64_t stride_ks, const int32_t* starts, int row0, int n, void* k8, void* v8t, float* sk,
                   float* sv, int S8, void* stream) {
  if (n == 0) return VK_OK;
  if (n < 0 || !k_cache || !v_cache || !starts || !k8 || !v8t || !sk || !sv || S <= 0 || row0 < 0 ||
      row0 + n > cache_rows || S8 <= 0 || S8 % 128 != 0 || stride_ks < 128 || stride_ks % 8 != 0 ||
      stride_kb < stride_ks * S || stride_kb % 8 != 0)
    return VK_ERR_ARG;
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k8) || !aligned16(v8t) || !aligned16(sk) ||
      !aligned16(sv))
    return VK_ERR_ARG;
  attn::QuantArgs a;
  a.k = static_cast<const __nv_bfloat16*>(k_cache);
  a.v = static_cast<const __nv_bfloat16*>(v_cache);
  a.stride_kb = stride_kb;
  a.stride_ks = stride_ks;
  a.starts = starts;
  a.row0 = row0;
  a.n = n;
  a.S = S;
  a.S8 = S8;
  a.k8 = static_cast<uint8_t*>(k8);
  a.v8t = static_cast<uint8_t*>(v8t);
  a.sk = sk;
  a.sv = sv;
  return launch(attn::kv_quantize_kernel, dim3(n, 2), dim3(attn::kQuantThreads), 0, stream, 1, a);
}

int vk_decode_attention_i8(const void* q, const void* k_cache, const void* v_cache, const void* k8,
                           const void* v8t, const float* sk, const float* sv, const int32_t* starts,
                           const int32_t* lengths, void* out, int nq, int row0, int cache_rows, int S,
                           int64_t stride_kb, int64_t stride_ks, int S8, int max_tail, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (nq == 0) return VK_OK;
  if (nq < 0 || !q || !k_cache || !v_cache || !k8 || !v8t || !sk || !sv || !starts || !lengths || !out ||
      !workspace || S <= 0 || row0 < 0 || row0 + nq > cache_rows || stride_ks < 128 || stride_kb < stride_ks * S ||
      S8 <= 0 || S8 % 128 != 0 || max_tail <= 0 || max_tail > S)
    return VK_ERR_ARG;
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || !aligned16(sk) || !aligned16(sv))
    return VK_ERR_ARG;
  if (workspace_bytes < vk_decode_attention_i8_workspace_bytes(nq, S8, max_tail)) return VK_ERR_ARG;
  CUtensorMap mk, mv, mk8, mv8;
  if (!make_cache_maps(&mk, &mv, k_cache, v_cache, cache_rows, S, stride_kb, stride_ks)) return VK_ERR_ARG;
  {
    uint64_t dims[3] = {128, static_cast<uint64_t>(S8), static_cast<uint64_t>(cache_rows)};
    uint64_t strides[2] = {128, static_cast<uint64_t>(S8) * 128};
    uint32_t box[3] = {128, attn::kTile8, 1};
    if (!make_map_u8(&mk8, k8, 3, dims, strides, box, true)) return VK_ERR_ARG;
  }
  {
    uint64_t dims[4] = {attn::kTile8, 128, static_cast<uint64_t>(S8 / attn::kTile8), static_cast<uint64_t>(cache_rows)};
    uint64_t strides[3] = {attn::kTile8, attn::kTile8 * 128, static_cast<uint64_t>(S8) * 128};
    uint32_t box[4] = {attn::kTile8, 128, 1, 1};
    if (!make_map_u8(&mv8, v8t, 4, dims, strides, box, true)) return VK_ERR_ARG;
  }
  const int sms = device_sm_count();
  if (sms <= 0) return VK_ERR_CUDA;
  const I8Plan plan = i8_plan(nq, S8, max_tail, sms);
  attn::DecodeArgs a;
  memset(&a, 0, sizeof(a));
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lengths = lengths;
  a.row0 = row0;
  a.nq = nq;
  a.max_splits = plan.n8max + plan.n16max;
  a.S = S;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.counters = reinterpret_cast<int*>(ws);
  const size_t counters = ((size_t)nq * 4 + 255) / 256 * 256;
  a.ws_ml = reinterpret_cast<float*>(ws + counters);
  a.ws_o = reinterpret_cast<float*>(ws + counters + ((size_t)nq * a.max_splits * 8 * 2 * 4 + 255) / 256 * 256);
  a.scale_log2 = 0.125f * 1.4426950408889634f;
  a.chunk = plan.chunk;
  a.starts = starts;
  a.n8max = plan.n8max;
  a.max_tail = max_tail;
  a.sk = sk;
  a.sv = sv;
  a.S8 = S8;
  if (!ensure_smem(attn::decode_attn_i8_kernel, attn::kSmemBytes8)) return VK_ERR_CUDA;
  return launch(attn::decode_attn_i8_kernel, dim3(nq, plan.n8max + plan.n16max), dim3(attn::kThreads),
                attn::kSmemBytes8, stream, 1, mk, mv, mk8, mv8, a);
}

}  // extern "C"

// ---- allocation-free decode attention -----------------------------------------------------------------------
// The split-K workspace of vk_decode_attention_noalloc: sized for 256 queries over 4096 cache positions (16
// splits of 256).  Zero at module load; each call clears the tickets it uses before the kernel runs.
namespace vk {
constexpr int kNoAllocMaxQ = 256;
constexpr int kNoAllocMaxS = 4096;
constexpr size_t kNoAllocSplits = (kNoAllocMaxS + attn::kMinChunk - 1) / attn::kMinChunk;
constexpr size_t kNoAllocBytes = 1024 + 256 * kNoAllocSplits * 8 * 2 * 4 + 256 * kNoAllocSplits * 8 * 64 * 4;
static __device__ __align__(256) uint8_t g_noalloc_attn_scratch[kNoAllocBytes];
}  // namespace vk

extern "C" {

int vk_decode_attention_noalloc(const void* q, const void* k_cache, const void* v_cache, const int32_t* lengths,
                                void* out, int nq, int row0, int cache_rows, int S, int64_t stride_kb,
                                int64_t stride_ks, void* stream) {
  if (nq == 0) return VK_OK;
  if (nq < 0 || nq > vk::kNoAllocMaxQ || S <= 0 || S > vk::kNoAllocMaxS) {
    fprintf(stderr,
            "viktor_b200: vk_decode_attention_noalloc supports at most %d queries and %d cache positions "
            "(got %d queries, %d positions); use vk_decode_attention with a caller-provided workspace\n",
            vk::kNoAllocMaxQ, vk::kNoAllocMaxS, nq, S);
    return VK_ERR_ARG;
  }
  const size_t need = vk_decode_attention_workspace_bytes(nq, S);
  if (need > vk::kNoAllocBytes) return VK_ERR_ARG;
  // Device address of the array, looked up once per device with that device current (host code cannot use the
  // symbol itself as a device pointer).
  static void* scratch[64] = {nullptr};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return VK_ERR_CUDA;
  // the array used is the current device's: a stream of another device would run against memory it cannot see
  int stream_dev = dev;
  if (cudaStreamGetDevice(static_cast<cudaStream_t>(stream), &stream_dev) != cudaSuccess) return VK_ERR_CUDA;
  if (stream_dev != dev) {
    fprintf(stderr, "viktor_b200: vk_decode_attention_noalloc: the stream belongs to device %d, the current device "
                    "is %d\n", stream_dev, dev);
    return VK_ERR_ARG;
  }
  if (!scratch[dev]) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, vk::g_noalloc_attn_scratch) != cudaSuccess || !p) {
      fprintf(stderr, "viktor_b200: cannot resolve the decode-attention scratch array on device %d\n", dev);
      return VK_ERR_CUDA;
    }
    scratch[dev] = p;
  }
  // the per-query tickets must start at zero (an earlier aborted call could have left them set)
  const size_t tickets = ((size_t)nq * 4 + 255) / 256 * 256;
  if (cudaMemsetAsync(scratch[dev], 0, tickets, static_cast<cudaStream_t>(stream)) != cudaSuccess)
    return VK_ERR_CUDA;
  return vk_decode_attention(q, k_cache, v_cache, lengths, out, nq, row0, cache_rows, S, stride_kb, stride_ks,
                             scratch[dev], vk::kNoAllocBytes, stream);
}

int vk_test_noalloc_poison(void* stream) {
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, vk::g_noalloc_attn_scratch) != cudaSuccess || !p) return VK_ERR_CUDA;
  const size_t tickets = static_cast<size_t>(vk::kNoAllocMaxQ) * 4;
  if (cudaMemsetAsync(p, 0x5A, tickets, static_cast<cudaStream_t>(stream)) != cudaSuccess) return VK_ERR_CUDA;
  return VK_OK;
}

int vk_prefill_attention(const void* q, const void* k_cache, const void* v_cache, const int32_t* cu_seqlens,
                         int nseq, int max_seqlen, int64_t n_tok, int row0, int cache_rows, int S,
                         int64_t stride_kb, int64_t stride_ks, void* out, void* stream) {
  if (nseq == 0 || n_tok == 0) return VK_OK;
  if (nseq < 0 || !q || !k_cache || !v_cache || !cu_seqlens || !out || max_seqlen <= 0 || max_seqlen > S ||
      row0 < 0 || row0 + nseq > cache_rows || stride_ks < 128 || stride_kb < stride_ks * S)
    return VK_ERR_ARG;
  if (!aligned16(q) || !aligned16(out)) return VK_ERR_ARG;
  CUtensorMap mq, mk, mv;
  {
    uint64_t dims[3] = {64, 8, static_cast<uint64_t>(n_tok)};
    uint64_t strides[2] = {128, 1024};
    uint32_t box[3] = {64, 1, pattn::kBQ};
    if (!make_map_bf16(&mq, q, 3, dims, strides, box, true)) return VK_ERR_ARG;
  }
  if (!make_cache_maps(&mk, &mv, k_cache, v_cache, cache_rows, S, stride_kb, stride_ks, pattn::kBK))
    return VK_ERR_ARG;
  pattn::PrefillArgs a;
  a.cu_seqlens = cu_seqlens;
  a.nseq = nseq;
  a.row0 = row0;
  a.n_qtiles = (max_seqlen + pattn::kBQ - 1) / pattn::kBQ;
  a.S = S;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.scale_log2 = 0.125f * 1.4426950408889634f;
  if (!ensure_smem(pattn::prefill_attn_kernel, pattn::kSmemBytes)) return VK_ERR_CUDA;
  return launch(pattn::prefill_attn_kernel, dim3(a.n_qtiles, 8, nseq), dim3(pattn::kThreads), pattn::kSmemBytes,
                stream, 1, mq, mk, mv, a);
}

int vk_linear_qkv_rope_cache(const void* x, const float* ssq, float norm_eps, const void* w_qkv,
                             const void* q_norm_w, const void* k_norm_w, const float* cos, const float* sin,
                             int rope_len, const int32_t* pos, const int32_t* rope_pos, const int32_t* seq, void* q,
                             void* k_cache, void* v_cache, void* k_out, void* v_out, int64_t M, int64_t stride_cb,
                             int64_t stride_cs, int cache_rows, int cache_len, float eps, int n_heads,
                             int n_kv_heads, void* stream) {
  if (M == 0) return VK_OK;
  if (n_heads != 8 || n_kv_heads != 2) return VK_ERR_UNSUPPORTED;
  if (M < 0 || !x || !w_qkv || !q_norm_w || !k_norm_w || !cos || !sin || !pos || !seq || !q || !k_cache ||
      !v_cache)
    return VK_ERR_ARG;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || stride_cs % 8 || stride_cb % 8 ||
      !aligned16(cos) || !aligned16(sin) || (k_out && !aligned16(k_out)) || (v_out && !aligned16(v_out)) ||
      (ssq && !aligned16(ssq)) || !aligned16(q_norm_w) || !aligned16(k_norm_w))
    return VK_ERR_ARG;
  gemm::EpiArgs ep = epi_zero();
  ep.ssq_in = ssq;
  ep.eps = norm_eps;
  ep.q_out = static_cast<__nv_bfloat16*>(q);
  ep.k_cache = static_cast<__nv_bfloat16*>(k_cache);
  ep.v_cache = static_cast<__nv_bfloat16*>(v_cache);
  ep.k_out = static_cast<__nv_bfloat16*>(k_out);
  ep.v_out = static_cast<__nv_bfloat16*>(v_out);
  ep.pos = pos;
  ep.rope_pos = rope_pos;
  ep.seq = seq;
  ep.q_norm_w = static_cast<const __nv_bfloat16*>(q_norm_w);
  ep.k_norm_w = static_cast<const __nv_bfloat16*>(k_norm_w);
  ep.cos = cos;
  ep.sin = sin;
  ep.rope_len = rope_len;
  ep.cache_rows = cache_rows;
  ep.cache_len = cache_len;
  ep.stride_cb = stride_cb;
  ep.stride_cs = stride_cs;
  ep.n_heads = n_heads;
  ep.n_kv_heads = n_kv_heads;
  ep.qk_eps = eps;
  const int N = (n_heads + 2 * n_kv_heads) * 64;
  if (M <= kSmallM)
    return run_gemm<64, gemm::QKV_ROPE>(x, w_qkv, M, N, 512, ep, N / 64, N, pick_nk(M, N / 64, 512), stream);
  if (persistent_fits<gemm::QKV_ROPE>(M, N))
    return run_gemm_persistent<gemm::QKV_ROPE>(x, w_qkv, M, N, 512, ep, N, stream);
  return run_gemm<128, gemm::QKV_ROPE>(x, w_qkv, M, N, 512, ep, N / 128, N, 1, stream);
}

int vk_linear_residual(const void* a, const void* w, void* x, float* ssq_out, int64_t M, int K, void* stream) {
  if (M == 0) return VK_OK;
  if (M < 0 || !a || !w || !x || !ssq_out) return VK_ERR_ARG;
  if (!aligned16(x) || !aligned16(ssq_out)) return VK_ERR_ARG;
  gemm::EpiArgs ep = epi_zero();
  ep.x = static_cast<__nv_bfloat16*>(x);
  ep.ssq_out = ssq_out;
  if (M <= kSmallM) return run_gemm<64, gemm::ADD_RESID>(a, w, M, 512, K, ep, 8, 512, pick_nk(M, 8, K), stream);
  if (persistent_fits<gemm::ADD_RESID>(M, 512))
    return run_gemm_persistent<gemm::ADD_RESID>(a, w, M, 512, K, ep, 512, stream);
  return run_gemm<128, gemm::ADD_RESID>(a, w, M, 512, K, ep, 4, 512, 1, stream);
}

int vk_row_ssq(const void* x, float* ssq, int64_t n, int d, void* stream) {
  if (n == 0) return VK_OK;
  if (!x || !ssq || n < 0 || d != 512 || !aligned16(x)) return VK_ERR_ARG;
  return launch(ew::row_ssq_kernel, dim3(blocks_for(n, 8)), dim3(256), 0, stream, 1,
                static_cast<const __nv_bfloat16*>(x), ssq, n);
}

int vk_ssq_rmsnorm(const void* x, const float* ssq, const void* w, void* h, int64_t n, int d, float eps,
                   void* stream) {
  if (n == 0) return VK_OK;
  if (!x || !ssq || !w || !h || n < 0 || d != 512 || !aligned16(x) || !aligned16(h)) return VK_ERR_ARG;
  return launch(ew::ssq_rmsnorm_kernel, dim3(blocks_for(n * 64, 256)), dim3(256), 0, stream, 1,
                static_cast<const __nv_bfloat16*>(x), ssq, static_cast<const __nv_bfloat16*>(w),
                static_cast<__nv_bfloat16*>(h), n, eps);
}

int vk_linear_add_rmsnorm(const void* a, const void* w, void* x, const void* norm_w, void* h, float* ssq_scratch,
                          int64_t M, int K, float eps, void* stream) {
  int rc = vk_linear_residual(a, w, x, ssq_scratch, M, K, stream);
  if (rc != VK_OK) return rc;
  return vk_ssq_rmsnorm(x, ssq_scratch, norm_w, h, M, 512, eps, stream);
}

int vk_fold_norm_weight(const void* w, const void* norm_w, void* out, int64_t N, int K, void* stream) {
  if (N == 0) return VK_OK;
  if (!w || !norm_w || !out || N < 0 || K <= 0) return VK_ERR_ARG;
  return launch(ew::fold_norm_kernel, dim3(blocks_for(N * K, 256)), dim3(256), 0, stream, 1,
                static_cast<const __nv_bfloat16*>(w), static_cast<const __nv_bfloat16*>(norm_w),
                static_cast<__nv_bfloat16*>(out), N, K);
}

int vk_linear_bias_act(const void* x, const void* w, const void* bias, void* y, int64_t ldy, const int32_t* row_map,
                       int64_t M, int N, int K, int act, void* stream) {
  if (M == 0) return VK_OK;
  if (M < 0 || !x || !w || !bias || !y || N <= 0 || N % 64 || ldy < N || (act != 0 && act != 1)) return VK_ERR_ARG;
  gemm::EpiArgs ep = epi_zero();
  ep.y = y;
  ep.ldy = ldy;
  ep.n_valid = N;
  ep.row_map = row_map;
  ep.bias = static_cast<const __nv_bfloat16*>(bias);
  ep.act = act;
  if (M <= kSmallM) return run_gemm<64, gemm::BIAS_ACT>(x, w, M, N, K, ep, N / 64, N, 1, stream);
  if (persistent_fits<gemm::BIAS_ACT>(M, N))
    return run_gemm_persistent<gemm::BIAS_ACT>(x, w, M, N, K, ep, N, stream);
  return run_gemm<128, gemm::BIAS_ACT>(x, w, M, N, K, ep, (N + 127) / 128, N, 1, stream);
}

int vk_cast_f32_bf16(const float* src, void* dst, int64_t n, void* stream) {
  if (n == 0) return VK_OK;
  if (!src || !dst || n < 0 || !aligned16(src) || (reinterpret_cast<uintptr_t>(dst) & 7)) return VK_ERR_ARG;
  return launch(ew::cast_f32_bf16_kernel, dim3(blocks_for((n + 3) / 4, 256)), dim3(256), 0, stream, 1, src,
                static_cast<__nv_bfloat16*>(dst), n);
}

int vk_gather_rows(const void* src, const int64_t* idx, void* dst, int64_t n, int row_bytes, int64_t src_rows,
                   void* stream) {
  if (n == 0) return VK_OK;
  if (!src || !idx || !dst || n < 0 || row_bytes <= 0 || row_bytes % 16 || !aligned16(src) || !aligned16(dst))
    return VK_ERR_ARG;
  return launch(ew::gather_rows_kernel, dim3(static_cast<unsigned>(n)), dim3(128), 0, stream, 1,
                static_cast<const uint8_t*>(src), idx, static_cast<uint8_t*>(dst), n, row_bytes, src_rows);
}

int vk_copy_rows(const void* src, const int64_t* src_idx, int64_t src_rows, void* dst, const int64_t* dst_idx,
                 int64_t dst_rows, int64_t n, int row_bytes, void* stream) {
  if (n == 0) return VK_OK;
  if (!src || !dst || n < 0 || row_bytes <= 0 || row_bytes % 16 || !aligned16(src) || !aligned16(dst))
    return VK_ERR_ARG;
  return launch(ew::copy_rows_kernel, dim3(static_cast<unsigned>(n)), dim3(128), 0, stream, 1,
                static_cast<const uint8_t*>(src), src_idx, src_rows, static_cast<uint8_t*>(dst), dst_idx, dst_rows, n,
                row_bytes);
}

int vk_scatter_embed(void* x, const int64_t* rows, int64_t n, int64_t x_rows, const void* emb, int64_t token, int d,
                     void* stream) {
  if (n == 0) return VK_OK;
  if (!x || !rows || !emb || n < 0 || d <= 0 || d % 8 || !aligned16(x) || !aligned16(emb) || token < 0)
    return VK_ERR_ARG;
  return launch(ew::scatter_embed_kernel, dim3(static_cast<unsigned>(n)), dim3(64), 0, stream, 1,
                static_cast<__nv_bfloat16*>(x), rows, n, x_rows, static_cast<const __nv_bfloat16*>(emb), token, d);
}

// ---- several candidates of a chunk ------------------------------------------------------------------------------
}  // extern "C"

namespace vk {
// Splits of an axis of `most` positions among `items` independent pieces of work: at least `ctas` pieces, chunks of `shortest` to
// 4096 positions.  ctas is four per SM, of which three are resident (64 KB of shared memory each): the fourth evens out lengths and
// ends, more of them cost more partial results.  Whole calls of 256 groups x 4 rows (prefixes to 2049, tails to 1100) / of 4 rows x
// 16 heads on 131071 positions / of 37 uneven groups: two or three per SM 88 to 89 / 107 / 33.5 us, four 83 / 103 / 33.4 us, eight
// 85 / 104 / 37 us.  (148: the SMs of a B200; the workspace has one size with and without a device.)
static int splits_of(int most, int64_t items, int shortest, int64_t ctas) {
  if (most <= 0) return 0;
  const int64_t want = (ctas + items - 1) / items, top = (most + shortest - 1) / shortest, low = (most + 4095) / 4096;
  return static_cast<int>(std::max(low, std::min(want, top)));
}
static int chunk_of(int most, int splits) { return splits ? ((most + splits - 1) / splits + 31) / 32 * 32 : 32; }

// Splits of wide_kernel's prefixes: the number that finishes first on `sms` CTAs at a time, counted in tiles of 128 positions;
// an item costs six more than its tiles (pipeline fill, partial results: some 12 us).
static int wide_splits(int64_t items, int S, int sms) {
  const int64_t tiles = (S + 127) / 128;
  int64_t best = 0;
  int at = 1;
  for (int64_t s = 1; s <= std::min<int64_t>(tiles, 64); ++s) {
    const int64_t cost = (items * s + sms - 1) / sms * ((tiles + s - 1) / s + 6);
    if (s == 1 || cost < best) {
      best = cost;
      at = static_cast<int>(s);
    }
  }
  return at;
}

// Positions of a prefix and a tail together.  Chunks end less than 2^15 behind them (64 splits of wide_kernel are rounded up to 128
// positions, some 600 of split_kernel to 32, or chunks have 4096) and loads look a few tiles further: all below 2^31.
constexpr int64_t kMostPositions = (int64_t(1) << 31) - (1 << 16);

struct SharedPlan {
  bool wide;
  int mt, wt;
  sattn::Plan p;
  int64_t prefix_items, tail_items;
};
static SharedPlan shared_plan(int B, int H, int HK, int D, int P, int S, int max_tail) {
  SharedPlan r;
  memset(&r, 0, sizeof(r));
  const int64_t ratio = H / HK, rows = B * ratio, ctas = 4 * 148;
  r.wide = rows > (D == 64 ? 32 : 16) * static_cast<int64_t>(P);
  if (r.wide) {
    r.p.prefix_tiles = static_cast<int>(P + rows / 256);
    r.p.prefix_splits = wide_splits(std::max<int64_t>(P, (rows + 255) / 256) * HK, S, 148);
    r.p.prefix_chunk = ((S + r.p.prefix_splits - 1) / r.p.prefix_splits + 127) / 128 * 128;
  } else {
    r.mt = rows > 16 * static_cast<int64_t>(P) ? 2 : 1;
    r.p.prefix_tiles = static_cast<int>(P + rows / (16 * r.mt));
    r.p.prefix_splits = splits_of(S, static_cast<int64_t>(r.p.prefix_tiles) * HK, 128, ctas);
    r.p.prefix_chunk = chunk_of(S, r.p.prefix_splits);
  }
  r.p.tail_tiles = static_cast<int>((ratio + 15) / 16);
  const int64_t pieces = static_cast<int64_t>(B) * HK * r.p.tail_tiles;
  r.wt = pieces >= 4 * ctas ? 1 : 4;
  r.p.tail_splits = splits_of(max_tail, r.wt == 1 ? pieces / 4 : pieces, 128, ctas);
  r.p.tail_chunk = chunk_of(max_tail, r.p.tail_splits);
  r.prefix_items = static_cast<int64_t>(r.p.prefix_tiles) * HK * r.p.prefix_splits;
  r.tail_items = pieces * r.p.tail_splits;
  return r;
}

template <typename T, int D, int MT, int WT>
static int shared_split(const sattn::Args& a, const sattn::Plan& p, unsigned grid, void* stream) {
  auto kern = sattn::split_kernel<T, D, MT, WT>;
  const int smem = std::max(sattn::Tile<D>::kSmem, 4 * 16 * MT * (D + 2) * 4);
  if (!ensure_smem(kern, smem, true)) return VK_ERR_CUDA;
  return launch(kern, dim3(grid), dim3(sattn::kThreads), smem, stream, 1, a, p);
}

template <typename T, int D>
static int shared_run(const sattn::Args& a, SharedPlan r, void* stream) {
  const int64_t tails = r.wt == 1 ? (r.tail_items + 3) / 4 : r.tail_items;
  if (r.prefix_items + tails >= (int64_t(1) << 31) || r.tail_items >= (int64_t(1) << 31)) return VK_ERR_ARG;
  int rc = VK_OK;
  if (r.wide) {
    CUtensorMap mk, mv;
    const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const uint64_t dims[4] = {D, static_cast<uint64_t>(a.HK), static_cast<uint64_t>(a.S), static_cast<uint64_t>(a.P)};
    const uint64_t strides[3] = {D * 2, static_cast<uint64_t>(a.stride_ks) * 2, static_cast<uint64_t>(a.stride_kb) * 2};
    const uint32_t box[4] = {64, 1, sattn::Wide<D>::kPos, 1};
    if (!make_map(&mk, type, a.k_prefix, 4, dims, strides, box, true) || !make_map(&mv, type, a.v_prefix, 4, dims, strides, box, true))
      return VK_ERR_ARG;
    auto kern = sattn::wide_kernel<T, D>;
    if (!ensure_smem(kern, sattn::Wide<D>::kSmem)) return VK_ERR_CUDA;
    rc = launch(kern, dim3(static_cast<unsigned>(r.prefix_items)), dim3(sattn::Wide<D>::kThreads), sattn::Wide<D>::kSmem, stream, 1,
                mk, mv, a, r.p);
    r.prefix_items = 0;
    r.p.behind_wide = true;
  }
  r.p.prefix_items = static_cast<int>(r.prefix_items);
  const unsigned n = static_cast<unsigned>(r.prefix_items + tails);
  constexpr int MT2 = D == 64 ? 2 : 1;  // (two 16-row tiles of 128 columns do not fit the registers)
  if (rc == VK_OK && n)
    rc = r.mt == 2 ? (r.wt == 1 ? shared_split<T, D, MT2, 1>(a, r.p, n, stream) : shared_split<T, D, MT2, 4>(a, r.p, n, stream))
                   : (r.wt == 1 ? shared_split<T, D, 1, 1>(a, r.p, n, stream) : shared_split<T, D, 1, 4>(a, r.p, n, stream));
  if (rc != VK_OK) return rc;
  const int splits = r.p.prefix_splits + r.p.tail_splits;
  const unsigned rows = static_cast<unsigned>(static_cast<int64_t>(a.B) * a.H);
  // one warp per row and head, or eight where there are many splits and rows alone do not fill the SMs
  return splits > 32 ? launch(sattn::join_kernel<T, D, 8>, dim3(rows), dim3(256), 0, stream, 1, a, r.p, splits)
                     : launch(sattn::join_kernel<T, D, 1>, dim3(blocks_for(rows, 4)), dim3(128), 0, stream, 1, a, r.p, splits);
}

template <typename T, int VEC>
static int penalize_launch(logit::Args a, void* stream) {
  constexpr int kStep = logit::kThreads * VEC;
  // the longest slice whose counters fit, or shorter ones where those would leave SMs idle (three CTAs each)
  a.wide = a.T > 65535;
  int64_t slice = logit::kMostSmem / (a.wide ? 4 : 2);
  while (slice > kStep && static_cast<int64_t>(a.B) * ((a.V + slice - 1) / slice) < 3 * 148) slice = std::max<int64_t>(slice / 2, kStep);
  const int64_t need = static_cast<int64_t>(a.V) + VEC - 1;
  slice = std::min<int64_t>(slice, (need + kStep - 1) / kStep * kStep);
  a.slice = static_cast<int>(slice);
  a.slices = static_cast<int>((need + slice - 1) / slice);
  const int64_t ctas = static_cast<int64_t>(a.slices) * a.B;
  if (ctas >= (int64_t(1) << 31)) return VK_ERR_ARG;
  auto kern = logit::penalize_kernel<T, VEC>;
  const int64_t smem = (a.history ? slice * (a.wide ? 4 : 2) : 0) + slice / 8;
  if (!ensure_smem(kern, logit::kMostSmem + logit::kMostSmem / 16)) return VK_ERR_CUDA;
  return launch(kern, dim3(static_cast<unsigned>(ctas)), dim3(logit::kThreads), smem, stream, 1, a);
}

template <typename T>
static int penalize_run(const logit::Args& a, void* stream) {
  const uintptr_t off = reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.out);
  if (off % 16 || (a.B > 1 && (a.ld - a.ld_out) * static_cast<int64_t>(sizeof(T)) % 16)) return penalize_launch<T, 1>(a, stream);
  return penalize_launch<T, 16 / sizeof(T)>(a, stream);
}

}  // namespace vk

extern "C" {

size_t vk_shared_attention_workspace_bytes(int B, int H, int HK, int D, int P, int S, int max_tail) {
  if (B <= 0 || H <= 0 || HK <= 0 || H % HK || D <= 0 || P <= 0 || S <= 0 || max_tail < 0 ||
      static_cast<int64_t>(S) + max_tail > kMostPositions)
    return 0;
  const SharedPlan r = shared_plan(B, H, HK, D, P, S, max_tail);
  return static_cast<size_t>(r.p.prefix_splits + r.p.tail_splits) * B * H * (D + 2) * 4;
}

int vk_shared_attention(const void* q, int64_t stride_q, int dtype, const void* k_prefix, const void* v_prefix,
                        const int32_t* prefix_lens, const int32_t* group_offsets, int P, int S, int64_t stride_kb,
                        int64_t stride_ks, const void* k_pages, const void* v_pages, int n_pages, int page,
                        int64_t stride_pp, const int32_t* page_table, int max_pages, int64_t stride_table,
                        const int32_t* tail_lens, void* out, float* lse, int B, int H, int HK, int D, float scale,
                        void* workspace, size_t workspace_bytes, void* stream) {
  if (B == 0) return VK_OK;
  if (B < 0 || P <= 0 || S <= 0 || H <= 0 || HK <= 0 || H % HK || n_pages <= 0 || max_pages < 0 || page < 8 ||
      page > 256 || (page & (page - 1)) || !(scale > 0.f) || !(scale < INFINITY))
    return VK_ERR_ARG;
  if ((D != 64 && D != 128) || (dtype != VK_BF16 && dtype != VK_F16)) return VK_ERR_UNSUPPORTED;
  if (!q || !k_prefix || !v_prefix || !prefix_lens || !group_offsets || !k_pages || !v_pages || !tail_lens || !out ||
      !workspace || (max_pages && !page_table))
    return VK_ERR_ARG;
  const int64_t token = static_cast<int64_t>(HK) * D, cap = int64_t(1) << 31;
  if (static_cast<int64_t>(B) * H >= cap || static_cast<int64_t>(max_pages) * page + S > kMostPositions ||
      stride_q < static_cast<int64_t>(H) * D || stride_q % 8 || stride_ks < token || stride_ks % 8 ||
      stride_kb < stride_ks * S || stride_kb % 8 || stride_pp < token * page || stride_pp % 8 ||
      stride_table < max_pages)
    return VK_ERR_ARG;
  if (!aligned16(q) || !aligned16(k_prefix) || !aligned16(v_prefix) || !aligned16(k_pages) || !aligned16(v_pages) ||
      !aligned16(out) || !aligned16(workspace) ||
      workspace_bytes < vk_shared_attention_workspace_bytes(B, H, HK, D, P, S, max_pages * page))
    return VK_ERR_ARG;
  sattn::Args a;
  memset(&a, 0, sizeof(a));
  a.q = q;
  a.k_prefix = k_prefix;
  a.v_prefix = v_prefix;
  a.prefix_lens = prefix_lens;
  a.offsets = group_offsets;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.table = page_table;
  a.tail_lens = tail_lens;
  a.out = out;
  a.lse = lse;
  a.stride_q = stride_q;
  a.stride_kb = stride_kb;
  a.stride_ks = stride_ks;
  a.stride_pp = stride_pp;
  a.stride_table = stride_table;
  a.B = B;
  a.H = H;
  a.HK = HK;
  a.P = P;
  a.S = S;
  a.n_pages = n_pages;
  a.page_shift = log2_of(page);
  a.max_pages = max_pages;
  SharedPlan r = shared_plan(B, H, HK, D, P, S, max_pages * page);
  r.p.tail_items = static_cast<int>(r.tail_items);
  r.p.scale_log2 = scale * 1.4426950408889634f;
  r.p.ws_o = static_cast<float*>(workspace);
  r.p.ws_ml = reinterpret_cast<float2*>(r.p.ws_o + static_cast<size_t>(r.p.prefix_splits + r.p.tail_splits) * B * H * D);
  if (dtype == VK_BF16)
    return D == 64 ? shared_run<__nv_bfloat16, 64>(a, r, stream) : shared_run<__nv_bfloat16, 128>(a, r, stream);
  return D == 64 ? shared_run<__half, 64>(a, r, stream) : shared_run<__half, 128>(a, r, stream);
}

// Scratch of the page calls, one region after another: ints, then the moves.
static size_t pages_ints(int rows, int max_pages, int n_pages, int n) {
  return static_cast<size_t>(rows) + 2 * static_cast<size_t>(n_pages) + 3 * static_cast<size_t>(n) +
         static_cast<size_t>(n) * max_pages + 4;
}
size_t vk_pages_workspace_bytes(int rows, int max_pages, int n_pages, int n) {
  if (rows <= 0 || max_pages <= 0 || n_pages <= 0 || n < 0) return 0;
  return 4 * pages_ints(rows, max_pages, n_pages, n) + sizeof(pages::Move) * (static_cast<size_t>(n) + n_pages / 2 + 1);
}

static bool pool_ok(const int32_t* table, const int32_t* refs, int rows, int max_pages, int n_pages, int page) {
  return table && refs && rows > 0 && max_pages > 0 && n_pages > 0 && page >= 8 && page <= 256 && !(page & (page - 1)) &&
         static_cast<int64_t>(rows) * max_pages < (int64_t(1) << 31) &&
         static_cast<int64_t>(max_pages) * page < (int64_t(1) << 31);
}
// Grid of 256-thread CTAs over `cells`, one cell per thread while that fills the SMs less than eight times over.
static unsigned cells_grid(int64_t cells) { return static_cast<unsigned>(std::min<int64_t>((cells + 255) / 256, 8 * 148)); }
static pages::Pool pool_of(int32_t* table, int32_t* lens, int32_t* refs, int rows, int max_pages, int n_pages, int page) {
  return pages::Pool{table, lens, refs, rows, max_pages, n_pages, log2_of(page)};
}

int vk_pages_extend(int32_t* table, int32_t* lens, int32_t* refs, int rows, int max_pages, int n_pages, int page,
                    const int32_t* list, int n, int count, int32_t* page_out, int32_t* slot_out, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (n == 0) return VK_OK;
  if (!pool_ok(table, refs, rows, max_pages, n_pages, page) || !lens || n < 0 || (!list && n != rows) || count <= 0 ||
      count > max_pages * page || static_cast<int64_t>(n) * count >= (int64_t(1) << 31) || !page_out || !slot_out || !workspace || !aligned16(workspace) ||
      workspace_bytes < vk_pages_workspace_bytes(rows, max_pages, n_pages, n))
    return VK_ERR_ARG;
  pages::ExtendArgs a;
  a.p = pool_of(table, lens, refs, rows, max_pages, n_pages, page);
  a.list = list;
  a.n = n;
  a.count = count;
  a.page = page_out;
  a.slot = slot_out;
  a.claim = static_cast<int32_t*>(workspace);
  a.first = a.claim + rows;
  a.len = a.first + n;
  a.free_list = a.len + n;
  const int64_t cells = static_cast<int64_t>(n) * count;
  const bool few = cells <= pages::kFewCells;
  const int rc = launch(pages::extend_kernel, dim3(1), dim3(pages::kPlanThreads), 0, stream, 1, a, few);
  if (rc != VK_OK || few) return rc;
  return launch(pages::extend_cells_kernel, dim3(cells_grid(cells)), dim3(256), 0, stream, 1, a);
}

}  // extern "C"

namespace vk {
template <typename Also>
static int copy_pages(const pages::CopyArgs& c, int64_t most, const Also& also, void* stream) {
  const int sms = device_sm_count();
  if (sms <= 0) return VK_ERR_CUDA;
  const int64_t units = most * c.layers * 2;
  return launch(pages::copy_kernel<Also>, dim3(static_cast<unsigned>(units < 8 * sms ? units : 8 * sms)),
                dim3(pages::kCopyThreads), 0, stream, 1, c, also);
}
}  // namespace vk

extern "C" {

int vk_pages_fork(int32_t* table, int32_t* lens, int32_t* refs, int rows, int max_pages, int n_pages, int page,
                  const int32_t* src, const int32_t* dst, int n, void* k, void* v, int layers, int token_bytes,
                  void* workspace, size_t workspace_bytes, void* stream) {
  if (n == 0) return VK_OK;
  if (!pool_ok(table, refs, rows, max_pages, n_pages, page) || !lens || n < 0 || !src || !dst || !k || !v ||
      layers <= 0 || token_bytes <= 0 || token_bytes % 16 || !aligned16(k) || !aligned16(v) || !workspace ||
      !aligned16(workspace) || workspace_bytes < vk_pages_workspace_bytes(rows, max_pages, n_pages, n) ||
      static_cast<int64_t>(n) * max_pages >= (int64_t(1) << 31))
    return VK_ERR_ARG;
  pages::ForkArgs a;
  a.p = pool_of(table, lens, refs, rows, max_pages, n_pages, page);
  a.src = src;
  a.dst = dst;
  a.n = n;
  a.claim = static_cast<int32_t*>(workspace);
  a.state = a.claim + rows;
  a.len = a.state + n;
  a.free_list = a.len + n;
  a.stage = a.free_list + n;
  a.moves = reinterpret_cast<pages::Move*>(static_cast<int32_t*>(workspace) + pages_ints(rows, max_pages, n_pages, n));
  const int64_t cells = static_cast<int64_t>(n) * max_pages;
  const bool few = cells <= pages::kFewCells;
  int rc = launch(pages::fork_kernel, dim3(1), dim3(pages::kPlanThreads), 0, stream, 1, a, few);
  if (rc == VK_OK && !few) rc = launch(pages::fork_stage_kernel, dim3(cells_grid(cells)), dim3(256), 0, stream, 1, a);
  if (rc != VK_OK) return rc;
  pages::CopyArgs c;
  c.k = static_cast<uint8_t*>(k);
  c.v = static_cast<uint8_t*>(v);
  c.moves = a.moves;
  c.count = nullptr;
  c.n = n;
  c.layers = layers;
  c.token_bytes = token_bytes;
  c.page_bytes = static_cast<int64_t>(token_bytes) * page;
  c.layer_bytes = c.page_bytes * n_pages;
  return few ? copy_pages(c, n, pages::JustCopy{}, stream) : copy_pages(c, n, pages::ForkWrite{a}, stream);
}

int vk_pages_free(int32_t* table, int32_t* lens, int32_t* refs, int rows, int max_pages, int n_pages,
                  const int32_t* list, int n, void* stream) {
  if (n == 0) return VK_OK;
  if (!pool_ok(table, refs, rows, max_pages, n_pages, 8) || !lens || n < 0 || (!list && n != rows)) return VK_ERR_ARG;
  return launch(pages::free_kernel, dim3(blocks_for(n, 8)), dim3(256), 0, stream, 1,
                pool_of(table, lens, refs, rows, max_pages, n_pages, 8), list, n);
}

int vk_pages_compact(int32_t* table, int32_t* refs, int rows, int max_pages, int n_pages, int page, void* k, void* v,
                     int layers, int token_bytes, int32_t* live, void* workspace, size_t workspace_bytes, void* stream) {
  if (!pool_ok(table, refs, rows, max_pages, n_pages, page) || !k || !v || layers <= 0 || token_bytes <= 0 ||
      token_bytes % 16 || !aligned16(k) || !aligned16(v) || !live || !workspace || !aligned16(workspace) ||
      workspace_bytes < vk_pages_workspace_bytes(rows, max_pages, n_pages, 0))
    return VK_ERR_ARG;
  pages::CompactArgs a;
  a.p = pool_of(table, nullptr, refs, rows, max_pages, n_pages, page);
  a.counts = static_cast<int32_t*>(workspace);
  a.holes = a.counts + 4;
  a.goes = a.holes + n_pages;
  a.moves = reinterpret_cast<pages::Move*>(static_cast<int32_t*>(workspace) + pages_ints(rows, max_pages, n_pages, 0));
  a.live = live;
  const int rc = launch(pages::compact_kernel, dim3(1), dim3(pages::kPlanThreads), 0, stream, 1, a);
  if (rc != VK_OK) return rc;
  pages::CopyArgs c;
  c.k = static_cast<uint8_t*>(k);
  c.v = static_cast<uint8_t*>(v);
  c.moves = a.moves;
  c.count = a.counts;
  c.n = 0;
  c.layers = layers;
  c.token_bytes = token_bytes;
  c.page_bytes = static_cast<int64_t>(token_bytes) * page;
  c.layer_bytes = c.page_bytes * n_pages;
  return copy_pages(c, n_pages / 2 + 1, pages::Renumber{a.p, a.goes, a.counts + 1}, stream);
}

int vk_penalize_logits(const void* logits, void* out, int dtype, int64_t ld, int64_t ld_out, int B, int V,
                       const int64_t* history, const int32_t* history_lens, int T, int64_t ld_history,
                       const float* repetition, const float* presence, const float* frequency, const float* bias,
                       int64_t ld_bias, const uint32_t* mask, int64_t ld_mask, int masks, const int32_t* mask_index,
                       void* stream) {
  if (B == 0) return VK_OK;
  if (dtype < VK_BF16 || dtype > VK_F32) return VK_ERR_UNSUPPORTED;
  if (B < 0 || V <= 0 || V > 1 << 30 || !logits || !out || ld < V || ld_out < V || (history && (!history_lens || T < 0 || ld_history < T)) ||
      (bias && ld_bias != 0 && ld_bias < V))
    return VK_ERR_ARG;
  if (mask && (masks <= 0 || ld_mask < (V + 31) / 32 || (!mask_index && masks != 1 && masks != B))) return VK_ERR_ARG;
  logit::Args a;
  a.logits = logits;
  a.out = out;
  a.ld = ld;
  a.ld_out = ld_out;
  a.history = T > 0 ? history : nullptr;
  a.history_lens = history_lens;
  a.ld_history = ld_history;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.bias = bias;
  a.ld_bias = ld_bias;
  a.mask = mask;
  a.ld_mask = ld_mask;
  a.mask_index = mask_index;
  a.masks = masks;
  a.B = B;
  a.V = V;
  a.T = T;
  return dtype == VK_F32    ? penalize_run<float>(a, stream)
         : dtype == VK_BF16 ? penalize_run<__nv_bfloat16>(a, stream)
                            : penalize_run<__half>(a, stream);
}

// ---- host-side stitching (no device work) ------------------------------------------------------------------
int vk_align(const char* query, int qlen, const char* target, int tlen, int mode, int k, int* out, char* cigar,
             int cigar_cap) {
  if (qlen < 0 || tlen < 0 || (qlen && !query) || (tlen && !target) || !out || mode < 0 || mode > 2)
    return VK_ERR_ARG;
  if (cigar && cigar_cap < qlen + tlen + 1) return VK_ERR_ARG;
  const vk::stitch::Alignment r = vk::stitch::align(query, qlen, target, tlen, mode, k, cigar != nullptr);
  out[0] = r.dist;
  out[1] = r.start;
  out[2] = r.end;
  if (cigar) {
    const size_t n = r.dist < 0 ? 0 : r.ops.size();
    memcpy(cigar, r.ops.data(), n);
    cigar[n] = 0;
  }
  return VK_OK;
}

int vk_overlap_cut(const char* a, int la, const char* b, int lb, int ov_frames, double rate, int* cut) {
  if (la < 0 || lb < 0 || (la && !a) || (lb && !b) || !cut) return VK_ERR_ARG;
  const vk::stitch::Cut c = vk::stitch::overlap_cut(std::string(a, a + la), std::string(b, b + lb), ov_frames, rate);
  cut[0] = c.a;
  cut[1] = c.b;
  return VK_OK;
}

int vk_stitch(const char* calls, const int64_t* offsets, const int64_t* spans, int n, int stride, char* out,
              int64_t cap, int64_t* out_len) {
  if (n < 0 || stride <= 0 || !out_len || (n && (!calls || !offsets || !spans))) return VK_ERR_ARG;
  std::vector<std::string> cs(n);
  for (int i = 0; i < n; ++i) {
    if (offsets[i + 1] < offsets[i]) return VK_ERR_ARG;
    cs[i].assign(calls + offsets[i], calls + offsets[i + 1]);
  }
  std::string res;
  int64_t cut_prev = 0;
  for (int i = 0; i < n; ++i) {
    const std::string& s = cs[i];
    if (i + 1 < n) {
      const int64_t ov = vk::stitch::floor_div(spans[2 * i + 1] - spans[2 * (i + 1)], stride);
      const int64_t frames = std::max<int64_t>(vk::stitch::floor_div(spans[2 * i + 1] - spans[2 * i], stride), 1);
      const double rate = static_cast<double>(s.size()) / static_cast<double>(frames);
      const vk::stitch::Cut c = vk::stitch::overlap_cut(s, cs[i + 1], static_cast<int>(ov), rate);
      res += vk::stitch::py_slice(s, cut_prev, c.a);
      cut_prev = c.b;
    } else {
      res += vk::stitch::py_slice(s, cut_prev, static_cast<int64_t>(s.size()));
    }
  }
  *out_len = static_cast<int64_t>(res.size());
  if (!out || cap < static_cast<int64_t>(res.size())) return out ? VK_ERR_ARG : VK_OK;
  memcpy(out, res.data(), res.size());
  return VK_OK;
}

}  // extern "C"
