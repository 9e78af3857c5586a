"""The paged K/V cache of `fa2.kernel.attention_kvcache` in 8 bits (an extension: the reference has no
cache): half the bytes of a 16-bit one, quantised as it is written.

    cache = alloc_kvcache_fp8(num_pages, page_size, heads_kv, head_dim, device)
    kvcache_append_fp8(k, v, cache, block_table, cache_seqlens, cu_seqlens=None)
    out = attention_kvcache_fp8(q, cache, block_table, cache_seqlens, ...)
    k, v = kvcache_read_fp8(cache, block_table, cu_seqlens, total, dtype=torch.bfloat16)

One step of a serving loop: raise cache_seqlens by the new tokens of each sequence, append their K/V,
attend. The three take the same block_table and cache_seqlens. Codes are float8_e4m3fn with one fp32
scale for each row of head_dim values: x is stored as e4m3(x / scale), scale = max|row| / 448, and
stands for code * scale. A row that holds a NaN or an infinity reads back as NaN.

Reports of the kernels (a length longer than the table, a table entry outside the cache, ...) are
raised by fa2.kernel.check_device_errors(), as for attention_kvcache.
"""

import math
from typing import NamedTuple

import torch

from . import _kvlib, _lib
from .kernel import CAUSAL_ALIGNS, LOG2E, _err_word, _sync_check_enabled, check_device_errors


class KVCacheFP8(NamedTuple):
    """k, v: float8_e4m3fn [num_pages, page_size, H_kv, D]; k_scale, v_scale: float32
    [num_pages, page_size, H_kv]. Any strides with adjacent D values on 16-byte boundaries; any
    sequence of four such tensors is taken in its place."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def alloc_kvcache_fp8(num_pages, page_size, heads_kv, head_dim, device=None):
    """An empty cache. Within a page the rows of one head are adjacent in memory (the layout that the
    attention kernels read in whole lines); the tensors are views of shape [pages, row, head, ...]."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    made = [torch.zeros(num_pages, heads_kv, page_size, head_dim, dtype=torch.uint8, device=device)
            .view(torch.float8_e4m3fn).transpose(1, 2) for _ in range(2)]
    made += [torch.zeros(num_pages, heads_kv, page_size, device=device).transpose(1, 2) for _ in range(2)]
    return KVCacheFP8(*made)


def _check_cache(cache):
    assert len(cache) == 4, "cache must be (k, v, k_scale, v_scale)"
    k, v, ks, vs = cache
    assert k.dim() == 4 and v.shape == k.shape, "cache k and v must be [num_pages, page_size, H_kv, D]"
    assert k.dtype == v.dtype == torch.float8_e4m3fn, "cache codes must be float8_e4m3fn"
    assert ks.shape == vs.shape == k.shape[:3], "cache scales must be [num_pages, page_size, H_kv]"
    assert ks.dtype == vs.dtype == torch.float32, "cache scales must be float32"
    assert k.shape[3] in (16, 32, 64, 128), "head_dim must be a power of two in [16, 128]"
    page_size = k.shape[1]
    assert page_size in (16, 32, 64) or (page_size >= 128 and page_size % 128 == 0), "page_size"
    assert k.shape[0] > 0 and k.shape[2] > 0, "the cache has no pages or no heads"
    return k, v, ks, vs


def _fill_cache(c, cache):
    k, v, ks, vs = cache
    c.k, c.v, c.k_scale, c.v_scale = k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()
    if k.stride(3) != 1 or v.stride(3) != 1:
        raise _lib.Fa2Error(_lib.FA2_ERR_LAYOUT, "the D values of a cache row must be adjacent")
    c.k_stride[:], c.v_stride[:] = k.stride()[:3], v.stride()[:3]
    c.ks_stride[:], c.vs_stride[:] = ks.stride(), vs.stride()
    c.num_pages, c.page_size, c.heads_kv, c.head_dim = k.shape


def _check_table(name, block_table, B, *lengths):
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B, \
        "block_table must be int32 [B, pages_per_seq]"
    for t, n in lengths:
        assert t.dtype == torch.int32 and t.shape == (n,), "sequence lengths and their sums must be int32"


def _check_devices(name, *tensors):
    if not all(t.is_cuda for t in tensors):
        raise RuntimeError(f"fa2.kvcache.{name} runs only on an sm_100 CUDA device (no CPU path)")
    if not all(t.device == tensors[0].device for t in tensors):
        raise RuntimeError(f"fa2.kvcache.{name}: all tensors must be on the same CUDA device")


def _no_grad(name, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"fa2.kvcache.{name} is forward only: use it under torch.no_grad()")


def _rows(t):
    """(b, h, n, d) strides of [B, H, N, D] or of packed [total, H, D]."""
    if t.dim() == 4:
        return tuple(int(s) for s in t.stride())
    return (0, int(t.stride(1)), int(t.stride(0)), int(t.stride(2)))


def _table(block_table):
    return block_table if block_table.stride(1) == 1 or block_table.shape[1] <= 1 else block_table.contiguous()


def _dtype(t):
    return _lib.FA2_DTYPE_BF16 if t == torch.bfloat16 else _lib.FA2_DTYPE_FP16


def _run(name, p, device):
    with torch.cuda.device(device):
        _kvlib.launch(name, p, torch.cuda.current_stream(device).cuda_stream)
        if _sync_check_enabled():
            check_device_errors(device)


def kvcache_append_fp8(k, v, cache, block_table, cache_seqlens, cu_seqlens=None):
    """Quantises new K/V rows into their pages. Each sequence's new tokens are its last positions:
    cache_seqlens (int32 [B]) counts them already.

    k, v: [B, H_kv, N, D], N new tokens for every sequence (one with cache_seqlens 0 is skipped: an
    empty slot of a padded batch); or packed [total, H_kv, D] with cu_seqlens (int32 [B + 1] prefix
    sums of the new tokens; rows past its end are ignored). fp16/bf16, any strides. block_table: int32
    [B, pages_per_seq]. Two sequences that share a page may both read it, but the rows that one call
    writes must be distinct. Returns the cache; asynchronous on torch's current stream.
    """
    ck, cv, cks, cvs = _check_cache(cache)
    assert k.dim() == (4 if cu_seqlens is None else 3) and v.shape == k.shape, \
        "k and v must be [B, H_kv, N, D], or [total, H_kv, D] with cu_seqlens"
    assert k.dtype == v.dtype and k.dtype in (torch.float16, torch.bfloat16)
    assert tuple(k.shape[-1:]) == tuple(ck.shape[3:]) and k.shape[1] == ck.shape[2], "k must have the cache's heads and D"
    B = block_table.shape[0] if block_table.dim() else 0
    assert B > 0, "block_table must be int32 [B, pages_per_seq]"
    _check_table("kvcache_append_fp8", block_table, B, (cache_seqlens, B),
                 *([(cu_seqlens, B + 1)] if cu_seqlens is not None else []))
    assert cu_seqlens is not None or k.shape[0] == B, "k's batch must be block_table's"
    _check_devices("kvcache_append_fp8", k, v, ck, cv, cks, cvs, block_table, cache_seqlens,
                   *([cu_seqlens] if cu_seqlens is not None else []))
    _no_grad("kvcache_append_fp8", k, v)
    if k.numel() == 0:
        return cache
    bt, sl = _table(block_table), cache_seqlens.contiguous()
    cu = cu_seqlens.contiguous() if cu_seqlens is not None else None
    p = _kvlib.AppendParams()
    _fill_cache(p.cache, (ck, cv, cks, cvs))
    p.k, p.v = k.data_ptr(), v.data_ptr()
    p.k_in_stride[:], p.v_in_stride[:] = _rows(k), _rows(v)
    p.block_table, p.cache_seqlens, p.err_flag = bt.data_ptr(), sl.data_ptr(), _err_word(k.device).data_ptr()
    p.cu_seqlens = cu.data_ptr() if cu is not None else None
    p.block_table_stride, p.pages_per_seq = bt.stride(0), bt.shape[1]
    p.batch, p.seqlen, p.dtype = B, k.shape[2] if cu is None else k.shape[0], _dtype(k.dtype)
    _run("fa2_kv8_append_sm100", p, k.device)
    return cache


def kvcache_read_fp8(cache, block_table, cu_seqlens, total, dtype=torch.bfloat16):
    """The first n_b keys and values of every sequence, n_b = cu_seqlens[b + 1] - cu_seqlens[b], back in
    16 bits and packed as attention_varlen takes them: (k, v), each [total, H_kv, D]. Rows past
    cu_seqlens[B] are not written; rows of a refused page are zeros. Asynchronous.
    """
    ck, cv, cks, cvs = _check_cache(cache)
    assert dtype in (torch.float16, torch.bfloat16)
    assert block_table.dim() == 2 and block_table.shape[0] > 0, "block_table must be int32 [B, pages_per_seq]"
    B = block_table.shape[0]
    _check_table("kvcache_read_fp8", block_table, B, (cu_seqlens, B + 1))
    assert total >= 0, "total must not be negative"
    _check_devices("kvcache_read_fp8", ck, cv, cks, cvs, block_table, cu_seqlens)
    shape = (int(total), ck.shape[2], ck.shape[3])
    k, v = (torch.empty(shape, dtype=dtype, device=ck.device) for _ in range(2))
    if total == 0:
        return k, v
    bt, cu = _table(block_table), cu_seqlens.contiguous()
    p = _kvlib.ReadParams()
    _fill_cache(p.cache, (ck, cv, cks, cvs))
    p.k_out, p.v_out = k.data_ptr(), v.data_ptr()
    p.block_table, p.cu_seqlens, p.err_flag = bt.data_ptr(), cu.data_ptr(), _err_word(ck.device).data_ptr()
    p.block_table_stride, p.pages_per_seq = bt.stride(0), bt.shape[1]
    p.batch, p.total, p.dtype = B, int(total), _dtype(dtype)
    _run("fa2_kv8_read_sm100", p, ck.device)
    return k, v


def attention_kvcache_fp8(q, cache, block_table, cache_seqlens, max_seqlen_k=None, causal=True, sm_scale=None,
                          causal_align="bottom_right", num_splits=None, cu_seqlens_q=None, max_seqlen_q=None):
    """Attention of new queries over the 8-bit paged cache: attention_kvcache for a KVCacheFP8.

    q: [B, H_q, N_q, D]; or packed [total_q, H_q, D] with cu_seqlens_q (int32 [B + 1]) and max_seqlen_q,
    a bound of the sequences' new tokens, so that prompt chunks and single tokens share a call.
    block_table: int32 [B, pages_per_seq]; cache_seqlens: int32 [B] keys per sequence, bounded by
    max_seqlen_k (default: pages_per_seq * page_size; a longer one is reported as a device error and
    attends to nothing). The causal mask is per sequence, bottom-right by default (the queries are the
    last positions). A query that sees no key gets zeros. num_splits: key ranges that run beside one
    another (None: chosen from the sizes). A query that sees a key of a refused page gets NaN. Returns
    a tensor like q (rows past cu_seqlens_q[B] are not written), asynchronously.
    """
    ck, cv, cks, cvs = _check_cache(cache)
    packed = cu_seqlens_q is not None
    assert q.dim() == (3 if packed else 4), "q must be [B, H_q, N_q, D], or [total_q, H_q, D] with cu_seqlens_q"
    assert q.dtype in (torch.float16, torch.bfloat16)
    H_q, D = q.shape[1], q.shape[-1]
    H_kv = ck.shape[2]
    assert D == ck.shape[3], "q must have the cache's head_dim"
    assert H_q % H_kv == 0, "GQA needs H_q divisible by H_kv"
    assert causal_align in CAUSAL_ALIGNS, f"causal_align must be one of {sorted(CAUSAL_ALIGNS)}"
    assert block_table.dim() == 2 and block_table.shape[0] > 0, "block_table must be int32 [B, pages_per_seq]"
    B = block_table.shape[0]
    _check_table("attention_kvcache_fp8", block_table, B, (cache_seqlens, B),
                 *([(cu_seqlens_q, B + 1)] if packed else []))
    if packed:
        assert max_seqlen_q is not None and max_seqlen_q >= 0, "packed queries need max_seqlen_q"
        n_q = int(max_seqlen_q)
    else:
        assert q.shape[0] == B, "q's batch must be block_table's"
        n_q = q.shape[2]
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    if not sm_scale > 0:
        raise ValueError(f"sm_scale must be positive (the row max is scaled after it is taken), got {sm_scale}")
    _check_devices("attention_kvcache_fp8", q, ck, cv, cks, cvs, block_table, cache_seqlens,
                   *([cu_seqlens_q] if packed else []))
    _no_grad("attention_kvcache_fp8", q)
    if max_seqlen_k is None:
        max_seqlen_k = block_table.shape[1] * ck.shape[1]
    out = torch.empty_like(q)
    if out.numel() == 0 or n_q == 0:
        return out
    if max_seqlen_k == 0 or block_table.shape[1] == 0:
        return out.zero_()
    bt, sl = _table(block_table), cache_seqlens.contiguous()
    cu = cu_seqlens_q.contiguous() if packed else None
    p = _kvlib.AttnParams()
    _fill_cache(p.cache, (ck, cv, cks, cvs))
    p.block_table, p.cache_seqlens, p.err_flag = bt.data_ptr(), sl.data_ptr(), _err_word(q.device).data_ptr()
    p.cu_seqlens_q = cu.data_ptr() if packed else None
    p.block_table_stride, p.pages_per_seq = bt.stride(0), bt.shape[1]
    p.batch, p.heads_q, p.seqlen_q, p.total_q = B, H_q, n_q, q.shape[0] if packed else 0
    p.max_seqlen_k, p.dtype = int(max_seqlen_k), _dtype(q.dtype)
    p.causal, p.causal_align = int(bool(causal)), CAUSAL_ALIGNS[causal_align]
    p.num_splits = 0 if num_splits is None else max(1, int(num_splits))
    p.qk_scale = sm_scale * LOG2E
    qq, oo = q, out
    if not _aligned(q) or not _aligned(out):  # layout copy: rows are moved 16 bytes at a time
        qq = q.clone(memory_format=torch.contiguous_format)
        oo = torch.empty_like(qq)
    p.q, p.o = qq.data_ptr(), oo.data_ptr()
    p.q_stride[:], p.o_stride[:] = _rows(qq), _rows(oo)
    with torch.cuda.device(q.device):
        nbytes = _kvlib.lib().fa2_kv8_attn_sm100_workspace_bytes(p)
        ws = torch.empty(max(0, nbytes), dtype=torch.uint8, device=q.device)  # caching allocator, this stream's
        p.workspace, p.workspace_bytes = ws.data_ptr() if nbytes > 0 else None, max(0, nbytes)
        _kvlib.launch("fa2_kv8_attn_sm100", p, torch.cuda.current_stream(q.device).cuda_stream)
        if oo is not out:
            out.copy_(oo)
        if _sync_check_enabled():
            check_device_errors(q.device)
    return out


def _aligned(t):
    return t.data_ptr() % 16 == 0 and t.stride(-1) == 1 and all(
        n <= 1 or s % 8 == 0 for n, s in zip(t.shape[:-1], t.stride()[:-1]))
