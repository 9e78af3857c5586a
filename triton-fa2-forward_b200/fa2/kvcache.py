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


_DTYPES = (torch.float16, torch.bfloat16)
_workspace_bytes = {}  # of attention_kvcache_fp8, by the sizes that it follows from


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


def _cache_fields(cache):
    """The cache's part of a parameter struct, its [H_kv, D], and its tensors; checked."""
    assert len(cache) == 4, "cache must be (k, v, k_scale, v_scale)"
    k, v, ks, vs = cache
    shape = k.shape
    assert len(shape) == 4 and v.shape == shape, "cache k and v must be [num_pages, page_size, H_kv, D]"
    assert k.dtype == v.dtype == torch.float8_e4m3fn, "cache codes must be float8_e4m3fn"
    pages, page_size, H_kv, D = shape
    assert ks.shape == vs.shape == (pages, page_size, H_kv), "cache scales must be [num_pages, page_size, H_kv]"
    assert ks.dtype == vs.dtype == torch.float32, "cache scales must be float32"
    assert D in (16, 32, 64, 128), "head_dim must be a power of two in [16, 128]"
    assert page_size in (16, 32, 64) or (page_size >= 128 and page_size % 128 == 0), "page_size"
    assert pages > 0 and H_kv > 0, "the cache has no pages or no heads"
    k_st, v_st = k.stride(), v.stride()
    if k_st[3] != 1 or v_st[3] != 1:
        raise _lib.Fa2Error(_lib.FA2_ERR_LAYOUT, "the D values of a cache row must be adjacent")
    fields = (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *k_st[:3], *v_st[:3], *ks.stride(), *vs.stride(),
              pages, page_size, H_kv, D)
    return fields, shape, cache


def _check_table(block_table, *lengths):
    """B of a block table [B, pages_per_seq]; `lengths`: (tensor, entries more than B)."""
    shape = block_table.shape
    assert block_table.dtype == torch.int32 and len(shape) == 2 and shape[0] > 0, \
        "block_table must be int32 [B, pages_per_seq]"
    for t, more in lengths:
        assert t.dtype == torch.int32 and t.shape == (shape[0] + more,), \
            "cache_seqlens must be int32 [B], cu_seqlens int32 [B + 1], B as in block_table"
    return shape[0]


def _check_device(name, *tensors):
    """The index of the one CUDA device that holds the tensors."""
    index = tensors[0].get_device()
    for t in tensors:
        at = t.get_device()
        if at < 0 or index < 0:
            raise RuntimeError(f"fa2.kvcache.{name} runs only on an sm_100 CUDA device (no CPU path)")
        if at != index:
            raise RuntimeError(f"fa2.kvcache.{name}: all tensors must be on the same CUDA device")
    return index


def _no_grad(name, *tensors):
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"fa2.kvcache.{name} is forward only: use it under torch.no_grad()")


def _rows(t):
    """(b, h, n, d) strides of [B, H, N, D] or of packed [total, H, D]."""
    st = t.stride()
    return st if len(st) == 4 else (0, st[1], st[0], st[2])


def _table(block_table):
    return block_table if block_table.stride(1) == 1 or block_table.shape[1] <= 1 else block_table.contiguous()


def _report_word(device):
    """Address of the device's error word of these kernels: not the one of fa2.kernel's, which stop for
    any report in theirs."""
    return _err_word(device).data_ptr() + 4


def _launch(entry, packed, index):
    _kvlib.launch(entry, packed, index)
    if _sync_check_enabled():
        check_device_errors(torch.device("cuda", index))


def kvcache_append_fp8(k, v, cache, block_table, cache_seqlens, cu_seqlens=None):
    """Quantises new K/V rows into their pages. Each sequence's new tokens are its last positions:
    cache_seqlens (int32 [B]) counts them already.

    k, v: [B, H_kv, N, D], N new tokens for every sequence (one with cache_seqlens 0 is skipped: an
    empty slot of a padded batch); or packed [total, H_kv, D] with cu_seqlens (int32 [B + 1] prefix
    sums of the new tokens; rows past its end are ignored). fp16/bf16, any strides. block_table: int32
    [B, pages_per_seq]. Two sequences that share a page may both read it, but the rows that one call
    writes must be distinct. Returns the cache; asynchronous on torch's current stream.
    """
    fields, shape, tensors = _cache_fields(cache)
    k_shape, dtype = k.shape, k.dtype
    assert len(k_shape) == (4 if cu_seqlens is None else 3) and v.shape == k_shape, \
        "k and v must be [B, H_kv, N, D], or [total, H_kv, D] with cu_seqlens"
    assert dtype in _DTYPES and v.dtype == dtype, "k and v must be fp16 or bf16"
    assert k_shape[-1] == shape[3] and k_shape[1] == shape[2], "k and v must have the cache's H_kv and D"
    if cu_seqlens is None:
        B = _check_table(block_table, (cache_seqlens, 0))
        assert k_shape[0] == B, "k and v must have block_table's batch"
        index = _check_device("kvcache_append_fp8", k, v, *tensors, block_table, cache_seqlens)
        cu, n = 0, k_shape[2]
    else:
        B = _check_table(block_table, (cache_seqlens, 0), (cu_seqlens, 1))
        index = _check_device("kvcache_append_fp8", k, v, *tensors, block_table, cache_seqlens, cu_seqlens)
        cu_seqlens = cu_seqlens.contiguous()
        cu, n = cu_seqlens.data_ptr(), k_shape[0]
    _no_grad("kvcache_append_fp8", k, v)
    if n == 0:
        return cache
    bt, sl = _table(block_table), cache_seqlens.contiguous()
    packed = _kvlib.APPEND.pack(
        *fields, k.data_ptr(), v.data_ptr(), *_rows(k), *_rows(v), bt.data_ptr(), sl.data_ptr(), cu,
        _report_word(k.device), bt.stride(0), bt.shape[1], B, n, dtype == torch.bfloat16)
    _launch(_kvlib.lib().fa2_kv8_append_sm100, packed, index)
    return cache


def kvcache_read_fp8(cache, block_table, cu_seqlens, total, dtype=torch.bfloat16):
    """The first n_b keys and values of every sequence, n_b = cu_seqlens[b + 1] - cu_seqlens[b], back in
    16 bits and packed as attention_varlen takes them: (k, v), each [total, H_kv, D]. Rows past
    cu_seqlens[B] are not written; rows of a refused page, or of a sequence that goes past total, are zeros.
    Asynchronous.
    """
    fields, shape, tensors = _cache_fields(cache)
    assert dtype in _DTYPES, "dtype must be fp16 or bf16"
    B = _check_table(block_table, (cu_seqlens, 1))
    total = int(total)
    assert total >= 0, "total must not be negative"
    index = _check_device("kvcache_read_fp8", *tensors, block_table, cu_seqlens)
    device = tensors[0].device
    k = torch.empty((total, shape[2], shape[3]), dtype=dtype, device=device)
    v = torch.empty_like(k)
    if total == 0:
        return k, v
    bt, cu = _table(block_table), cu_seqlens.contiguous()
    packed = _kvlib.READ.pack(
        *fields, k.data_ptr(), v.data_ptr(), bt.data_ptr(), cu.data_ptr(), _report_word(device),
        bt.stride(0), bt.shape[1], B, total, dtype == torch.bfloat16)
    _launch(_kvlib.lib().fa2_kv8_read_sm100, packed, index)
    return k, v


def attention_kvcache_fp8(q, cache, block_table, cache_seqlens, max_seqlen_k=None, causal=True, sm_scale=None,
                          causal_align="bottom_right", num_splits=None, cu_seqlens_q=None, max_seqlen_q=None):
    """Attention of new queries over the 8-bit paged cache: attention_kvcache for a KVCacheFP8.

    q: [B, H_q, N_q, D]; or packed [total_q, H_q, D] with cu_seqlens_q (int32 [B + 1]) and max_seqlen_q,
    a bound of the sequences' new tokens, so that prompt chunks and single tokens share a call.
    block_table: int32 [B, pages_per_seq]; cache_seqlens: int32 [B] keys per sequence, bounded by
    max_seqlen_k (default: pages_per_seq * page_size; a longer one is reported as a device error and
    attends to nothing). The causal mask is per sequence, bottom-right by default (the queries are the
    last positions). A query that sees no key gets zeros, one that sees a key of a refused page NaN.
    With more than 16 rows (queries x heads of a group) a query's values are exact within 2^13 of the
    largest of its row; smaller ones are off by at most 2^-21 (bf16) or 2^-24 (fp16) of that one.
    num_splits: CTAs that share the work for each (sequence, kv head, block of rows); None: chosen from
    the sizes. The same call gives the same bits; another batch around a sequence may cut its keys
    elsewhere and change its last bits. Returns a tensor like q, asynchronously. Not written are rows past
    cu_seqlens_q[B] and, beside a device error, those of a sequence whose sums fall, leave q or give more
    than max_seqlen_q queries (all rows, where sums go back and forth thousands of times).
    """
    fields, shape, tensors = _cache_fields(cache)
    q_shape, dtype = q.shape, q.dtype
    packed = cu_seqlens_q is not None
    assert len(q_shape) == (3 if packed else 4), "q must be [B, H_q, N_q, D], or [total_q, H_q, D] with cu_seqlens_q"
    assert dtype in _DTYPES, "q must be fp16 or bf16"
    _, page_size, H_kv, D = shape
    H_q = q_shape[1]
    assert q_shape[-1] == D, "q must have the cache's head_dim"
    assert H_q % H_kv == 0, "GQA needs H_q divisible by H_kv"
    assert causal_align in CAUSAL_ALIGNS, f"causal_align must be one of {sorted(CAUSAL_ALIGNS)}"
    if packed:
        B = _check_table(block_table, (cache_seqlens, 0), (cu_seqlens_q, 1))
        assert max_seqlen_q is not None and max_seqlen_q >= 0, "packed queries need max_seqlen_q"
        n_q = int(max_seqlen_q)
        index = _check_device("attention_kvcache_fp8", q, *tensors, block_table, cache_seqlens, cu_seqlens_q)
        cu_seqlens_q = cu_seqlens_q.contiguous()
    else:
        B = _check_table(block_table, (cache_seqlens, 0))
        assert q_shape[0] == B, "q must have block_table's batch"
        n_q = q_shape[2]
        index = _check_device("attention_kvcache_fp8", q, *tensors, block_table, cache_seqlens)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    if not sm_scale > 0:
        raise ValueError(f"sm_scale must be positive (the row max is scaled after it is taken), got {sm_scale}")
    _no_grad("attention_kvcache_fp8", q)
    pages_per_seq = block_table.shape[1]
    if max_seqlen_k is None:
        max_seqlen_k = min(pages_per_seq * page_size, 2 ** 31 - 1)
    out = torch.empty_like(q)
    if out.numel() == 0 or n_q == 0:
        return out
    if max_seqlen_k == 0 or pages_per_seq == 0:
        return out.zero_()
    bt, sl = _table(block_table), cache_seqlens.contiguous()
    qq, oo = q, out
    if not _aligned(q) or (out.stride() != q.stride() and not _aligned(out)):  # layout copy: rows are moved 16 bytes at a time
        qq = q.clone(memory_format=torch.contiguous_format)
        oo = torch.empty_like(qq)
    L = _kvlib.lib()
    head = (*fields, qq.data_ptr(), oo.data_ptr(), *_rows(qq), *_rows(oo), bt.data_ptr(), sl.data_ptr(),
            cu_seqlens_q.data_ptr() if packed else 0, _report_word(q.device))
    tail = (bt.stride(0), 0, pages_per_seq, B, H_q, n_q, q_shape[0] if packed else 0, int(max_seqlen_k),
            dtype == torch.bfloat16, bool(causal), CAUSAL_ALIGNS[causal_align],
            0 if num_splits is None else max(1, int(num_splits)), sm_scale * LOG2E, 0)
    sizes = (B, H_q, H_kv, D, n_q, tail[7], tail[11])
    nbytes = _workspace_bytes.get(sizes)
    if nbytes is None:
        nbytes = max(0, L.fa2_kv8_attn_sm100_workspace_bytes(_kvlib.ATTN.pack(*head, 0, 0, *tail)))  # (-1: refused below)
        if nbytes:
            if len(_workspace_bytes) >= 4096:
                _workspace_bytes.clear()
            _workspace_bytes[sizes] = nbytes
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)  # caching allocator, this stream's
    _launch(L.fa2_kv8_attn_sm100, _kvlib.ATTN.pack(*head, ws.data_ptr(), nbytes, *tail), index)
    if oo is not out:
        out.copy_(oo)
    return out


def _aligned(t):
    *st, inner = t.stride()
    if t.data_ptr() % 16 or inner != 1:
        return False
    for n, s in zip(t.shape, st):
        if s % 8 and n > 1:
            return False
    return True
