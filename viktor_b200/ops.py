"""PyTorch-facing wrappers of the C ABI, one per op.

The first group keeps the names, arguments and return values of the reference's Triton ops
(viktor/triton_ops.py) and of viktor/decode_attention.py, so code written against those modules ports by
changing the import.  The second group exposes the fused tensor-core forms this package runs on the hot path.
Every wrapper launches on the current CUDA stream of the tensors' device and raises on failure; nothing falls
back to PyTorch.
"""

from __future__ import annotations

import functools

import torch

from ._lib import call, load

_BF16 = torch.bfloat16


def _p(t):
    return None if t is None else t.data_ptr()


def _stream(t: torch.Tensor):
    return torch.cuda.current_stream(t.device).cuda_stream


def _check_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("viktor_b200 ops need CUDA tensors (there is no CPU path)")


# ---------------------------------------------------------------- mirrors of viktor/triton_ops.py
def add_rmsnorm(x, w, eps, delta=None):
    """x [n, d] (updated in place by += delta); returns RMSNorm(x) * w.  (viktor/triton_ops.py:34-40)"""
    _check_cuda(x, w, delta)
    n, d = x.shape
    assert x.dtype == _BF16 and x.is_contiguous() and (delta is None or delta.is_contiguous())
    h = torch.empty_like(x)
    call("vk_add_rmsnorm", _p(x), _p(delta), _p(w), _p(h), n, d, eps, _stream(x))
    return h


def embed_rmsnorm(tok, emb, w, eps):
    """tok [n] token ids -> (x = emb[tok] [n, d], RMSNorm(x) * w).  (viktor/triton_ops.py:163-169)"""
    _check_cuda(tok, emb, w)
    n, d = tok.shape[0], emb.shape[1]
    tok = tok.to(torch.int64).contiguous()
    x = torch.empty(n, d, dtype=emb.dtype, device=emb.device)
    h = torch.empty_like(x)
    call("vk_embed_rmsnorm", _p(tok), _p(emb), emb.shape[0], _p(w), _p(x), _p(h), n, d, eps, _stream(emb))
    return x, h


def qkv_rope_cache(qkv, q_norm_w, k_norm_w, cos, sin, pos, seq, k_cache, v_cache, eps, n_heads, n_kv_heads,
                   head_dim, return_kv=False, rope_pos=None):
    """qkv [n, (H + 2 Hkv) * D]; pos/seq [n] int32; k_cache/v_cache [B, S, Hkv, D] (one layer).
    Returns q [n, H, D] (and packed k, v [n, Hkv, D]).  (viktor/triton_ops.py:94-108)"""
    _check_cuda(qkv, k_cache, v_cache, pos, seq)
    n = qkv.shape[0]
    assert k_cache.stride() == v_cache.stride() and k_cache.stride(-1) == 1 and k_cache.stride(-2) == head_dim
    q = torch.empty(n, n_heads, head_dim, dtype=qkv.dtype, device=qkv.device)
    k = v = None
    if return_kv:
        k = torch.empty(n, n_kv_heads, head_dim, dtype=qkv.dtype, device=qkv.device)
        v = torch.empty_like(k)
    call("vk_qkv_rope_cache", _p(qkv.contiguous()), _p(q_norm_w), _p(k_norm_w), _p(cos), _p(sin), cos.shape[0],
         _p(pos), _p(rope_pos), _p(seq), _p(q), _p(k_cache), _p(v_cache), _p(k), _p(v), n, k_cache.stride(0),
         k_cache.stride(1), k_cache.shape[0], k_cache.shape[1], eps, n_heads, n_kv_heads, head_dim, _stream(qkv))
    return (q, k, v) if return_kv else q


def linear(x, w, swiglu=False, out_dtype=None):
    """x @ w^T on tcgen05 tensor cores.  swiglu: w is gate_up [2F, K] and the result silu(gate) * up [M, F].
    out_dtype: torch.float32 for unrounded logits.  (viktor/triton_ops.py:138-146)"""
    _check_cuda(x, w)
    M, K = x.shape
    N = w.shape[0]
    out_f32 = out_dtype == torch.float32
    y = torch.empty(M, N // 2 if swiglu else N, dtype=torch.float32 if out_f32 else x.dtype, device=x.device)
    call("vk_linear", _p(x.contiguous()), _p(w.contiguous()), _p(y), M, N, K, int(bool(swiglu)), int(out_f32),
         _stream(x))
    return y


def swiglu(gu):
    """gu [n, 2F] (gate | up) -> silu(gate) * up [n, F].  (viktor/triton_ops.py:223-229)"""
    _check_cuda(gu)
    n, f2 = gu.shape
    out = torch.empty(n, f2 // 2, dtype=gu.dtype, device=gu.device)
    call("vk_swiglu", _p(gu.contiguous()), _p(out), n, f2 // 2, _stream(gu))
    return out


def greedy_update(logits, bias, is_tail, is_homo, homo_stop, tok, run, pos, plen, rope_off, out, pos32, seqlens,
                  rpos32, eos, pad, emb=None, x=None, ssq=None):
    """Greedy step bookkeeping in one kernel (viktor/triton_ops.py:200-209).  is_tail / is_homo: bool or uint8
    [V].  With emb/x/ssq also writes the next step's embedding x [B, 512] and its block sums of squares ssq [B, 8]."""
    _check_cuda(logits, tok, out)
    B, V = logits.shape
    it = is_tail.to(torch.uint8) if is_tail.dtype != torch.uint8 else is_tail
    ih = is_homo.to(torch.uint8) if is_homo.dtype != torch.uint8 else is_homo
    call("vk_greedy_update", _p(logits), logits.stride(0), _p(bias), _p(it), _p(ih), int(homo_stop), _p(tok),
         _p(run), _p(pos), _p(plen), _p(rope_off), _p(out), out.stride(0), out.shape[1], _p(pos32), _p(seqlens),
         _p(rpos32), B, V, eos, pad, _p(emb), _p(x), _p(ssq), _stream(logits))


# ---------------------------------------------------------------- mirror of viktor/decode_attention.py
_WS = {}


def decode_attention_workspace(nq: int, S: int, device) -> torch.Tensor:
    """A zero-filled workspace for decode_attention (per-query tickets return to zero after every call)."""
    nbytes = load().vk_decode_attention_workspace_bytes(nq, S)
    return torch.zeros(nbytes, dtype=torch.uint8, device=device)


def decode_attention(q, k, v, lengths, block=64, workspace=None, row0=0):
    """q [B, H, D]; k/v [B', S, Hkv, D] (one layer of the cache, B' >= row0 + B); lengths [B] int32 including
    the current token, 1 <= lengths <= S.  Query b attends cache row row0 + b.  (viktor/decode_attention.py:41-53)"""
    B, H, D = q.shape
    HK = k.shape[2]
    assert q.is_contiguous() and H % HK == 0 and H // HK <= 16 and D == 64
    assert q.dtype == k.dtype == v.dtype == torch.bfloat16
    assert k.stride() == v.stride() and k.stride(-1) == 1 and k.stride(-2) == D
    assert lengths.shape == (B,) and lengths.dtype == torch.int32 and lengths.is_contiguous()
    if (H, HK) != (8, 2):
        raise NotImplementedError("decode attention kernels are built for 8 query / 2 KV heads")
    S = k.shape[1]
    if workspace is None:
        # one implicit workspace per (device, shape, stream): calls on the same stream run one after another;
        # calls on different streams get different workspaces, so they never share split-K tickets or partials
        key = (q.device, B, S, _stream(q))
        workspace = _WS.get(key)
        if workspace is None:
            workspace = _WS[key] = decode_attention_workspace(B, S, q.device)
    out = torch.empty_like(q)
    call("vk_decode_attention", _p(q), _p(k), _p(v), _p(lengths), _p(out), B, row0, k.shape[0], S, k.stride(0),
         k.stride(1), _p(workspace), workspace.numel(), _stream(q))
    return out


# ---------------------------------------------------------------- opt-in INT8 prefix KV (analysis.md:95)
class PrefixKV8:
    """Int8 copy of the prefix of one layer's cache rows: k8 [rows, S8, 128] / v8t [rows, S8 / 128, 128, 128]
    uint8 (excess-128 bytes; v8t channel-major within each tile of 128 positions), sk / sv [rows, 128] float32
    per-channel scales.  S8 is rounded up to a multiple of 128."""

    def __init__(self, rows: int, S8: int, device):
        self.S8 = -(-S8 // 128) * 128
        self.k8 = torch.zeros(rows, self.S8, 128, dtype=torch.uint8, device=device)
        self.v8t = torch.zeros(rows, self.S8 // 128, 128, 128, dtype=torch.uint8, device=device)
        self.sk = torch.zeros(rows, 128, dtype=torch.float32, device=device)
        self.sv = torch.zeros(rows, 128, dtype=torch.float32, device=device)


def kv_quantize(k, v, starts, prefix: PrefixKV8, row0=0):
    """Quantizes positions [0, starts[i]) of cache rows row0 + i of one layer (k/v [B', S, 2, 64] bf16) into
    prefix: per channel s = max|x| / 127, byte = clamp(rint(x / s), -127, 127) + 128."""
    assert k.dtype == v.dtype == torch.bfloat16 and k.stride() == v.stride() and k.stride(-1) == 1
    assert k.shape[2:] == (2, 64) and k.stride(-2) == 64
    assert starts.dtype == torch.int32 and starts.is_contiguous()
    call("vk_kv_quantize", _p(k), _p(v), k.shape[0], k.shape[1], k.stride(0), k.stride(1), _p(starts), row0,
         starts.shape[0], _p(prefix.k8), _p(prefix.v8t), _p(prefix.sk), _p(prefix.sv), prefix.S8, _stream(k))


def decode_attention_i8(q, k, v, prefix: PrefixKV8, starts, lengths, max_tail, workspace=None, row0=0):
    """decode_attention with positions [0, starts[b]) read from the int8 prefix and [starts[b], lengths[b]) from
    the bf16 cache (0 <= starts < lengths, lengths - starts <= max_tail)."""
    B, H, D = q.shape
    assert (H, D) == (8, 64) and q.is_contiguous() and q.dtype == k.dtype == v.dtype == torch.bfloat16
    assert k.stride() == v.stride() and k.stride(-1) == 1 and k.shape[2:] == (2, 64) and k.stride(-2) == 64
    assert starts.dtype == lengths.dtype == torch.int32 and starts.shape == lengths.shape == (B,)
    S = k.shape[1]
    if workspace is None:
        key = ("i8", q.device, B, prefix.S8, max_tail)
        workspace = _WS.get(key)
        if workspace is None:
            nbytes = load().vk_decode_attention_i8_workspace_bytes(B, prefix.S8, max_tail)
            workspace = _WS[key] = torch.zeros(nbytes, dtype=torch.uint8, device=q.device)
    out = torch.empty_like(q)
    call("vk_decode_attention_i8", _p(q), _p(k), _p(v), _p(prefix.k8), _p(prefix.v8t), _p(prefix.sk),
         _p(prefix.sv), _p(starts), _p(lengths), _p(out), B, row0, k.shape[0], S, k.stride(0), k.stride(1),
         prefix.S8, max_tail, _p(workspace), workspace.numel(), _stream(q))
    return out


def prefill_attention(q, k_cache, v_cache, cu_seqlens, max_seqlen, row0=0, out=None):
    """Varlen causal attention (flash_attn_varlen_func(..., causal=True), viktor/fast_decoder.py:73) over K/V
    already in the cache.  q [n_tok, 8, 64] packed by cu_seqlens [nseq + 1] int32; k_cache/v_cache one layer
    [B', S, 2, 64]; sequence b reads cache row row0 + b."""
    n_tok = q.shape[0]
    nseq = cu_seqlens.shape[0] - 1
    if out is None:
        out = torch.empty_like(q)
    call("vk_prefill_attention", _p(q), _p(k_cache), _p(v_cache), _p(cu_seqlens), nseq, int(max_seqlen), n_tok,
         row0, k_cache.shape[0], k_cache.shape[1], k_cache.stride(0), k_cache.stride(1), _p(out), _stream(q))
    return out


# ---------------------------------------------------------------- fused tensor-core forms (hot path)
def fold_norm_weight(w, norm_w):
    """W' = bf16(W * norm_w[None, :]): an RMSNorm weight folded into the GEMM that consumes the norm."""
    out = torch.empty_like(w)
    call("vk_fold_norm_weight", _p(w.contiguous()), _p(norm_w.contiguous()), _p(out), w.shape[0], w.shape[1],
         _stream(w))
    return out


def row_ssq(x, out=None):
    """[n, 8] fp32 sums of squares of the eight 64-column blocks of each row of x [n, 512]."""
    out = out if out is not None else torch.empty(x.shape[0], 8, dtype=torch.float32, device=x.device)
    call("vk_row_ssq", _p(x), _p(out), x.shape[0], x.shape[1], _stream(x))
    return out


def linear_rmsnorm(x, ssq, eps, w_folded, swiglu=False, out_dtype=None):
    """(RMSNorm(x) * w) . W^T given W' = W diag(w) and the row sums of squares of x."""
    M, K = x.shape
    N = w_folded.shape[0]
    out_f32 = out_dtype == torch.float32
    y = torch.empty(M, N // 2 if swiglu else N, dtype=torch.float32 if out_f32 else x.dtype, device=x.device)
    call("vk_linear_rmsnorm", _p(x), _p(ssq), eps, _p(w_folded), _p(y), M, N, K, int(bool(swiglu)), int(out_f32),
         _stream(x))
    return y


def linear_qkv_rope_cache(x, w_qkv, q_norm_w, k_norm_w, cos, sin, pos, seq, k_cache, v_cache, eps, rope_pos=None,
                          q_out=None, return_kv=False, ssq=None, norm_eps=1e-6, n_heads=8, n_kv_heads=2):
    """x [M, 512] . w_qkv^T with the qkv_rope_cache epilogue: returns q [M, H, 64] (and packed k, v).  With ssq,
    x is the residual and w_qkv carries the folded attention-norm weight."""
    M = x.shape[0]
    q = q_out if q_out is not None else torch.empty(M, n_heads, 64, dtype=x.dtype, device=x.device)
    k = v = None
    if return_kv:
        k = torch.empty(M, n_kv_heads, 64, dtype=x.dtype, device=x.device)
        v = torch.empty_like(k)
    call("vk_linear_qkv_rope_cache", _p(x), _p(ssq), norm_eps, _p(w_qkv), _p(q_norm_w), _p(k_norm_w), _p(cos),
         _p(sin), cos.shape[0], _p(pos), _p(rope_pos), _p(seq), _p(q), _p(k_cache), _p(v_cache), _p(k), _p(v), M,
         k_cache.stride(0), k_cache.stride(1), k_cache.shape[0], k_cache.shape[1], eps, n_heads, n_kv_heads,
         _stream(x))
    return (q, k, v) if return_kv else q


def linear_residual(a, w, x, ssq_out=None):
    """x += a . w^T (bf16, in place); returns the new rows' block sums of squares [M, 8]."""
    M, K = a.shape
    ssq = ssq_out if ssq_out is not None else torch.empty(M, 8, dtype=torch.float32, device=a.device)
    call("vk_linear_residual", _p(a), _p(w), _p(x), _p(ssq), M, K, _stream(a))
    return ssq


def linear_add_rmsnorm(a, w, x, norm_w, eps, h_out=None):
    """x += a . w^T (bf16, in place); returns h = RMSNorm(x) * norm_w.  x, h [M, 512]."""
    M, K = a.shape
    h = h_out if h_out is not None else torch.empty_like(x)
    ssq = torch.empty(M, 8, dtype=torch.float32, device=a.device)
    call("vk_linear_add_rmsnorm", _p(a), _p(w), _p(x), _p(norm_w), _p(h), _p(ssq), M, K, eps, _stream(a))
    return h


def linear_bias_act(x, w, bias, act=0, out=None, row_map=None):
    """act(x . w^T + bias) in bf16 (act 0 identity, 1 GELU-erf); row i of the result lands in out[row_map[i]]."""
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    call("vk_linear_bias_act", _p(x), _p(w), _p(bias), _p(out), out.stride(0), _p(row_map), M, N, K, act,
         _stream(x))
    return out


def cast_bf16(src, out=None):
    out = out if out is not None else torch.empty(src.shape, dtype=torch.bfloat16, device=src.device)
    call("vk_cast_f32_bf16", _p(src.contiguous()), _p(out), src.numel(), _stream(src))
    return out


def gather_rows(src, idx, out=None):
    n = idx.shape[0]
    row_bytes = src[0].numel() * src.element_size()
    out = out if out is not None else torch.empty((n,) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device)
    call("vk_gather_rows", _p(src), _p(idx), _p(out), n, row_bytes, src.shape[0], _stream(src))
    return out


def scatter_embed(x, rows, emb, token):
    call("vk_scatter_embed", _p(x), _p(rows), rows.shape[0], x.shape[0], _p(emb), int(token), x.shape[1],
         _stream(x))


# ---------------------------------------------------------------- several candidates of a chunk (no reference counterpart)
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_I32 = torch.int32
_PAGES = (8, 16, 32, 64, 128, 256)
_MOST_POSITIONS = (1 << 31) - (1 << 16)


def _launch(name, device, *args):
    """call() on the current stream of `device`, which need not be the current device."""
    if device.type != "cuda":
        raise ValueError("viktor_b200 ops need CUDA tensors (there is no CPU path)")
    if device.index == torch.cuda.current_device():
        call(name, *args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            call(name, *args, torch.cuda.current_stream(device).cuda_stream)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _same_device(device, *ts):
    for t in ts:
        if t is not None and t.device != device:
            raise ValueError("all tensors must be on one device")


def _ints(name, t, *shape):
    if t.dtype != _I32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 {list(shape)}")


def _cache_strides(shape, stride):
    """(row stride, position stride) in elements of [P, S, HK, D] whose positions are laid out as [HK, D]."""
    P, S, HK, D = shape
    sb, ss, sh, sd = stride
    _need(sd == 1 and (HK == 1 or sh == D), "the last two dimensions of a cache must be contiguous")
    if S == 1:
        ss = HK * D
    if P == 1:
        sb = ss * S
    _need(ss >= HK * D and sb >= ss * S and ss % 8 == 0 and sb % 8 == 0, "positions of a cache that overlap or are not 16-byte "
          "aligned")
    return sb, ss


@functools.lru_cache(maxsize=256)
def _shared_workspace(*sizes):
    return load().vk_shared_attention_workspace_bytes(*sizes)


def shared_prefix_attention(q, k_prefix, v_prefix, prefix_lens, group_offsets, k_pages, v_pages, page_table, tail_lens,
                            scale=None, out=None, return_lse=False, workspace=None):
    """Attention of one query token per row over a prefix that a group of rows shares and the row's own tail.

    q [B, H, D] bf16 or fp16 (D 64 or 128); k_prefix / v_prefix [P, S, HK, D]: one layer of a static cache, one row per
    group; prefix_lens [P] int32; group_offsets [P + 1] int32: rows group_offsets[g] .. group_offsets[g + 1] - 1 belong
    to group g.  k_pages / v_pages [n_pages, page, HK, D]: one layer of a KVPages; page_table [B, max_pages] int32;
    tail_lens [B] int32; S + max_pages * page at most 2^31 - 2^16.  Query head h reads KV head h // (H // HK).  scale: 1 / sqrt(D) by default.

    Returns out [B, H, D], with return_lse also the log of the sum of exponentials [B, H] (float32).  A row with nothing
    to attend gets 0 and -inf; rows behind the last group are not written.  What a cache holds behind a length is not
    used.  No gradients.  workspace: uint8, vk_shared_attention_workspace_bytes; calls that may run at the same time need one each (by
    default every call allocates its own)."""
    q_shape, prefix_shape, pages_shape, table_shape = q.shape, k_prefix.shape, k_pages.shape, page_table.shape
    _need(len(q_shape) == 3 and len(prefix_shape) == len(pages_shape) == 4 and len(table_shape) == 2,
          "q [B, H, D], caches of four dimensions, page_table [B, max_pages]")
    B, H, D = q_shape
    P, S, HK, _ = prefix_shape
    n_pages, page, _, _ = pages_shape
    max_pages = table_shape[1]
    device, dtype = q.device, q.dtype
    _same_device(device, k_prefix, v_prefix, prefix_lens, group_offsets, k_pages, v_pages, page_table, tail_lens, out, workspace)
    _need((dtype is torch.bfloat16 or dtype is torch.float16) and k_prefix.dtype is dtype and v_prefix.dtype is dtype
          and k_pages.dtype is dtype and v_pages.dtype is dtype, "q and the caches must all be bfloat16 or all float16")
    _need(D == 64 or D == 128, "head_dim must be 64 or 128")
    _need(P > 0 and S > 0 and HK > 0 and n_pages > 0 and H > 0 and H % HK == 0, "empty cache, or heads that do not divide")
    _need(page in _PAGES, "pages hold a power of two from 8 to 256 tokens")
    _need(S + max_pages * page <= _MOST_POSITIONS, "S + max_pages * page must be at most 2^31 - 2^16")
    _need(v_prefix.shape == prefix_shape and prefix_shape[3] == D, "k_prefix and v_prefix: [P, S, HK, D]")
    _need(v_pages.shape == pages_shape and pages_shape[2] == HK and pages_shape[3] == D, "k_pages and v_pages: [n_pages, page, "
          "HK, D]")
    _need(page_table.dtype is _I32 and table_shape[0] == B, "page_table: int32 [B, max_pages]")
    _ints("prefix_lens", prefix_lens, P)
    _ints("group_offsets", group_offsets, P + 1)
    _ints("tail_lens", tail_lens, B)
    stride_table, one = page_table.stride()
    if B <= 1:
        stride_table = max_pages
    _need((max_pages < 2 or one == 1) and stride_table >= max_pages, "the rows of page_table must be contiguous and must not "
          "overlap")
    stride_q, sh, one = q.stride()
    if B <= 1:
        stride_q = H * D
    _need(one == 1 and (H == 1 or sh == D), "the heads of a row of q must be contiguous")
    _need(stride_q >= H * D and stride_q % 8 == 0, "the rows of q must be 16-byte aligned and must not overlap")
    kb, ks = _cache_strides(prefix_shape, k_prefix.stride())
    pp, ps = _cache_strides(pages_shape, k_pages.stride())
    _need(v_prefix.stride() == k_prefix.stride() or (kb, ks) == _cache_strides(prefix_shape, v_prefix.stride()),
          "k_prefix and v_prefix must have the same strides")
    _need(ps == HK * D and (v_pages.stride() == k_pages.stride() or (pp, ps) == _cache_strides(pages_shape, v_pages.stride())),
          "pages must be contiguous, with the same strides in k and v")
    scale = D ** -0.5 if scale is None else float(scale)
    _need(0.0 < scale < float("inf"), "scale must be positive and finite")
    q_at = q.data_ptr()
    if out is None:
        out = torch.empty(q_shape, dtype=dtype, device=device)
        out_at = out.data_ptr()
    else:
        out_at = out.data_ptr()
        _need(out.dtype is dtype and out.shape == q_shape and out.is_contiguous(), "out: contiguous, as q")
        _need(B == 0 or out_at + 2 * B * H * D <= q_at or out_at >= q_at + 2 * ((B - 1) * stride_q + H * D), "out must not overlap q")
    lse = torch.empty(B, H, dtype=torch.float32, device=device) if return_lse else None
    if B:
        nbytes = _shared_workspace(B, H, HK, D, P, S, max_pages * page)
        if workspace is None:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        elif not workspace.is_contiguous() or workspace.nbytes < nbytes:
            raise ValueError(f"workspace: {nbytes} contiguous bytes")
        _launch("vk_shared_attention", device, q_at, stride_q, 0 if dtype is torch.bfloat16 else 1, k_prefix.data_ptr(),
                v_prefix.data_ptr(), prefix_lens.data_ptr(), group_offsets.data_ptr(), P, S, kb, ks, k_pages.data_ptr(),
                v_pages.data_ptr(), n_pages, page, pp, page_table.data_ptr(), max_pages, stride_table, tail_lens.data_ptr(), out_at,
                _p(lse), B, H, HK, D, scale, workspace.data_ptr(), workspace.nbytes)
    return (out, lse) if return_lse else out


class KVPages:
    """Tails of the rows of a decode batch in pages: k / v [layers, n_pages, page, HK, D], table [rows, max_pages] int32 (the
    pages of each row, -1 behind its last), lens [rows] int32 (tokens of each row), refs [n_pages] int32 (rows that
    name a page; 0: free).  All but a row's last page are full, and only full pages are shared.  The operations below
    run on the device without a host wait (they may be captured) and follow one another on one stream."""

    def __init__(self, k, v, table, lens, refs):
        _need(k.dim() == 5 and k.shape == v.shape and k.dtype == v.dtype and k.is_contiguous() and v.is_contiguous(),
              "k and v: contiguous [layers, n_pages, page, HK, D] of one type")
        self.layers, self.n_pages, self.page, hk, d = k.shape
        self.token_bytes = hk * d * k.element_size()
        _need(k.numel() > 0 and self.token_bytes % 16 == 0, "a token's K must be a multiple of 16 bytes")
        _need(self.page in _PAGES, "pages hold a power of two from 8 to 256 tokens")
        _need(table.dim() == 2 and table.numel() > 0, "table: int32 [rows, max_pages]")
        self.rows, self.max_pages = table.shape
        _ints("table", table, self.rows, self.max_pages)
        _ints("lens", lens, self.rows)
        _ints("refs", refs, self.n_pages)
        self.device = k.device
        _same_device(k.device, v, table, lens, refs)
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs

    @classmethod
    def empty(cls, layers, n_pages, page, rows, max_pages, n_kv_heads=2, head_dim=64, dtype=_BF16, device="cuda"):
        """A pool whose pages are all free."""
        shape = (layers, n_pages, page, n_kv_heads, head_dim)
        i32 = dict(dtype=_I32, device=device)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   torch.full((rows, max_pages), -1, **i32), torch.zeros(rows, **i32), torch.zeros(n_pages, **i32))

    def _books(self):
        return self.table.data_ptr(), self.lens.data_ptr(), self.refs.data_ptr(), self.rows, self.max_pages, self.n_pages

    def _data(self):
        return self.k.data_ptr(), self.v.data_ptr(), self.layers, self.token_bytes

    def _workspace(self, n):
        nbytes = load().vk_pages_workspace_bytes(self.rows, self.max_pages, self.n_pages, n)
        return torch.empty(nbytes, dtype=torch.uint8, device=self.device)

    def _rows(self, name, rows):
        """(pointer, count) of a list of rows; None stands for all of them."""
        if rows is None:
            return None, self.rows
        n = rows.numel()
        _ints(name, rows, n)
        if rows.device != self.device:
            raise ValueError(f"{name}: on another device than the pages")
        return rows.data_ptr(), n


def pages_extend(pages: KVPages, count=1, rows=None):
    """Makes room for `count` more tokens in each of `rows` (int32 [n]; None: all): lens grows, and the tokens' places come
    back as (page, slot), int32 [n, count] each, to be used as the cache row and position of qkv_rope_cache.  Free pages
    are taken the lowest first, in the order of the rows.  A row that is out of range, named before, full, whose length or
    last page is out of range, or that needs more pages than the rows before it have left is not changed (place -1) and reported by check_device_errors(); in the last
    case later rows that need a page are not served either, even if fewer would have done (rows that need none are)."""
    ptr, n = pages._rows("rows", rows)
    _need(0 < count <= pages.max_pages * pages.page, "count must be 1 to the tokens of a row")
    page, slot = torch.empty(2, n, count, dtype=_I32, device=pages.device).unbind(0)
    if n:
        ws = pages._workspace(n)
        _launch("vk_pages_extend", pages.device, *pages._books(), pages.page, ptr, n, count, page.data_ptr(), slot.data_ptr(),
                ws.data_ptr(), ws.nbytes)
    return page, slot


def pages_fork(pages: KVPages, src, dst):
    """Rows dst[i] (int32 [n]) become copies of rows src[i] as they were before the call.  Full pages are shared; a partly
    filled last page is copied in every layer.  What the dst rows held is released, and given out again from the next
    call on.  src[i] == dst[i] leaves the row as it is.  A row that is out of range, a dst named before, or a src whose length or
    page to be copied is out of range or for which no page is left changes nothing and is reported by check_device_errors()."""
    src_ptr, n = pages._rows("src", src)
    dst_ptr, m = pages._rows("dst", dst)
    _need(src is not None and dst is not None and n == m, "src and dst must have one length")
    if n:
        ws = pages._workspace(n)
        _launch("vk_pages_fork", pages.device, *pages._books(), pages.page, src_ptr, dst_ptr, n, *pages._data(), ws.data_ptr(),
                ws.nbytes)


def pages_free(pages: KVPages, rows=None):
    """`rows` (int32 [n]; None: all) give their pages up and are empty."""
    ptr, n = pages._rows("rows", rows)
    if n:
        _launch("vk_pages_free", pages.device, *pages._books(), ptr, n)


def pages_compact(pages: KVPages):
    """Moves the pages in use to the lowest numbers: those at or above their count go into the free ones below it, both in
    ascending order; table and refs follow.  (A page that only refs names, not the table, is moved as well.)  Returns the
    count, int32 [1] on the device."""
    live = torch.empty(1, dtype=_I32, device=pages.device)
    ws = pages._workspace(0)
    table, _, refs, rows, max_pages, n_pages = pages._books()
    _launch("vk_pages_compact", pages.device, table, refs, rows, max_pages, n_pages, pages.page, *pages._data(), live.data_ptr(),
            ws.data_ptr(), ws.nbytes)
    return live


def penalize_logits(logits, history=None, history_lens=None, repetition=None, presence=None, frequency=None, bias=None,
                    mask=None, mask_index=None, out=None):
    """Penalties for the tokens of each row's history, a bias and a grammar mask, in one pass over the logits [B, V] (float32,
    bfloat16 or float16; computed in float32, rounded once).

    history [B, T] int64 with history_lens [B] int32: with c = how often v is among the row's first history_lens[b]
    tokens (ids outside 0..V-1 count for nothing), l = logit / repetition[b] (logit * repetition[b] where it is not
    positive) if c, then l - frequency[b] * c - presence[b] * (c > 0) + bias ([V] or [B, V]); repetition, presence, frequency
    and bias float32.  mask [M, ceil(V / 32)] int32: bit v % 32 of word v // 32 is 0 where v is forbidden, which gives -inf
    whatever the logit holds; mask_index [B] int32 names each row's mask (-1: none), without it M is B or 1.
    out: as logits (may be logits); returned."""
    shape, dtype, device = logits.shape, logits.dtype, logits.device
    _need(len(shape) == 2 and dtype in _DTYPES, "logits: float32, bfloat16 or float16 [B, V]")
    B, V = shape
    _same_device(device, history, history_lens, repetition, presence, frequency, bias, mask, mask_index, out)
    ld, one = logits.stride()
    if B <= 1:
        ld = V
    _need(0 < V <= 1 << 30 and (V == 1 or one == 1) and ld >= V, "the rows of logits must be contiguous and must not overlap")
    at = logits.data_ptr()
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
        ld_out, out_at = V, out.data_ptr()
    else:
        ld_out, one = out.stride()
        if B <= 1:
            ld_out = V
        out_at, size = out.data_ptr(), out.element_size()
        _need(out.shape == shape and out.dtype is dtype and (V == 1 or one == 1) and ld_out >= V, "out: as logits")
        if out_at != at or ld != ld_out:
            # rows may lie side by side in one buffer, but not over one another
            side = ld == ld_out and V * size <= (out_at - at) % (ld * size) <= (ld - V) * size
            _need(side or out_at + ((B - 1) * ld_out + V) * size <= at or at + ((B - 1) * ld + V) * size <= out_at,
                  "out must be logits or must not overlap it")
    T = ld_history = masks = ld_mask = ld_bias = 0
    if history is not None:
        _need(history.dim() == 2 and history.shape[0] == B and history.dtype is torch.int64 and history_lens is not None,
              "history: int64 [B, T], with history_lens")
        T = history.shape[1]
        ld_history, one = history.stride()
        if B <= 1:
            ld_history = T
        _need((T < 2 or one == 1) and ld_history >= T, "the rows of history must be contiguous and must not overlap")
        _ints("history_lens", history_lens, B)
    else:
        _need(repetition is None and presence is None and frequency is None, "penalties need a history")
    for t in (repetition, presence, frequency):
        if t is not None and (t.dtype is not torch.float32 or t.shape != (B,) or not t.is_contiguous()):
            raise ValueError("repetition, presence and frequency: contiguous float32 [B]")
    if bias is not None:
        _need(bias.dtype is torch.float32 and (bias.shape == (V,) or bias.shape == shape) and (V == 1 or bias.stride(-1) == 1),
              "bias: float32 [V] or [B, V]")
        ld_bias = bias.stride(0) if bias.dim() == 2 and B > 1 else 0
        _need(ld_bias == 0 or ld_bias >= V, "rows of bias that overlap")
    if mask is not None:
        words = -(-V // 32)
        _need(mask.dim() == 2 and mask.dtype is _I32 and mask.shape[0] > 0 and mask.shape[1] == words, "mask: int32 [M, ceil(V / 32)]")
        masks = mask.shape[0]
        ld_mask, one = mask.stride()
        if masks == 1:
            ld_mask = words
        _need((words == 1 or one == 1) and ld_mask >= words, "the rows of mask must be contiguous and must not overlap")
        _need(mask_index is not None or masks in (1, B), "mask: one row, or B, or a mask_index")
    if mask_index is not None:
        _need(mask is not None, "mask_index without a mask")
        _ints("mask_index", mask_index, B)
    if B:
        _launch("vk_penalize_logits", device, at, out_at, _DTYPES[dtype], ld, ld_out, B, V, _p(history) if T else None,
                _p(history_lens), T, ld_history, _p(repetition), _p(presence), _p(frequency), _p(bias), ld_bias, _p(mask), ld_mask, masks,
                _p(mask_index))
    return out
