"""GPU tests of the 8-bit paged K/V cache (fa2.kvcache) against 64-bit forms (oracle.serving).

Tolerances, fixed before the first run.
 * append: the scale and the codes are defined in 32-bit arithmetic with correctly rounded division, so
   they are compared for equality, and against the 64-bit value: a code is off by half an e4m3 step,
   2^-4 of the value or 2^-10 of the scale where it is subnormal, plus 2^-21 for the two divisions.
 * read: code * scale rounds to 32 bits (2^-24) and then to 16 bits (eps / 2), half a subnormal step
   at the bottom of fp16.
 * attention: see `tolerance`.
"""

import math

import pytest
import torch

from fa2 import _lib
from fa2.kernel import attention_varlen, check_device_errors
from fa2.kvcache import KVCacheFP8, alloc_kvcache_fp8, attention_kvcache_fp8, kvcache_append_fp8, kvcache_read_fp8
from fa2.rotary import rotary, rotary_inv_freq
from oracle import serving

pytestmark = pytest.mark.gpu

SUBNORMAL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    check_device_errors()


def randn(*shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def table_for(lens, page_size, seed=0, spare=3):
    """A shuffled block table; entries past a sequence's last page are out of range on purpose."""
    g = torch.Generator().manual_seed(seed)
    per = max(1, max(-(-n // page_size) for n in lens))
    need = [-(-n // page_size) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    bt = torch.full((len(lens), per), 1 << 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[at:at + n]
        at += n
    return bt.cuda(), pages


def poison(cache):
    """NaN codes and NaN scales everywhere: what no sequence wrote must not show."""
    for t in cache[:2]:
        t.view(torch.uint8).fill_(0x7f)
    for t in cache[2:]:
        t.fill_(math.nan)
    return cache


def filled(lens, page_size, H_kv, D, dtype=torch.bfloat16, seed=0, k_size=1.0, v_size=1.0, plain_layout=False):
    """A cache whose sequences hold random rows, through the append operator; NaN everywhere else."""
    bt, pages = table_for(lens, page_size, seed)
    if plain_layout:  # the 16-bit cache's memory order: page, row, head
        made = [torch.zeros(pages, page_size, H_kv, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
        cache = KVCacheFP8(*made, *[torch.zeros(pages, page_size, H_kv, device="cuda") for _ in range(2)])
    else:
        cache = alloc_kvcache_fp8(pages, page_size, H_kv, D)
    poison(cache)
    total = sum(lens)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32).cuda()
    k = (randn(max(1, total), H_kv, D, dtype=torch.float32, seed=seed + 1) * k_size).to(dtype)
    v = (randn(max(1, total), H_kv, D, dtype=torch.float32, seed=seed + 2) * v_size).to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    kvcache_append_fp8(k[:total], v[:total], cache, bt, lens_t, cu_seqlens=cu)
    return cache, bt, lens_t, cu, k, v


# ------------------------------------------------------------------------------------ append
def check_rows(cache, bt, b, first, x_k, x_v):
    """Sequence b's rows from position `first` on hold x_k, x_v [n, H, D]."""
    n, ps = x_k.shape[0], cache[0].shape[1]
    at = torch.arange(first, first + n)
    page, row = bt[b].cpu()[at // ps].long().cuda(), (at % ps).cuda()
    for x, codes, scales in ((x_k, cache[0], cache[2]), (x_v, cache[1], cache[3])):
        want_codes, want_scales = serving.quantise(x)
        got = codes.view(torch.uint8)[page, row].view(torch.float8_e4m3fn).float()
        got_s = scales[page, row]
        assert torch.equal(torch.isnan(got_s), torch.isnan(want_scales))
        fine = ~torch.isnan(want_scales)
        assert torch.equal(got_s[fine], want_scales[fine])
        assert torch.equal(got, want_codes)
        value = got.double() * got_s.double()[..., None]
        err = (value - x.double()).abs()[fine]
        tol = x.double().abs() * (2.0 ** -4 + 2.0 ** -21) + got_s.double()[..., None] * 2.0 ** -10 * (1 + 2.0 ** -21)
        assert (err <= tol[fine]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H_kv", [(128, 8), (64, 3), (32, 1), (16, 5)])
@pytest.mark.parametrize("page_size", [16, 128, 384])
def test_append_packed(dtype, D, H_kv, page_size):
    new, after = [1, 40, 0, 131, 7], [1, 900, 55, 131, 300]
    bt, pages = table_for(after, page_size)
    cache = poison(alloc_kvcache_fp8(pages, page_size, H_kv, D))
    before = [t.view(torch.uint8).clone() if t.dtype == torch.float8_e4m3fn else t.clone() for t in cache]
    cu = torch.tensor([0, 1, 41, 41, 172, 179], dtype=torch.int32).cuda()
    k = randn(190, H_kv, D, dtype=dtype, seed=1)  # eleven rows behind the last sequence
    v = randn(190, H_kv, D, dtype=dtype, seed=2) * 30
    kvcache_append_fp8(k, v, cache, bt, torch.tensor(after, dtype=torch.int32).cuda(), cu_seqlens=cu)
    touched = torch.zeros(pages, page_size, dtype=torch.bool)
    for b, (n, m) in enumerate(zip(new, after)):
        check_rows(cache, bt, b, m - n, k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]])
        for j in range(m - n, m):
            touched[int(bt[b, j // page_size]), j % page_size] = True
    for t, was in zip(cache, before):  # nothing else is written
        now = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
        same = (now == was) | (now != now)
        rest = ~touched.cuda()
        assert same[rest].all()


@pytest.mark.parametrize("N", [1, 3, 130])
def test_append_fixed_length_with_empty_slots(N):
    """[B, H, N, D] views of [B, N, H, D] storage; a sequence of length 0 is an empty slot."""
    B, H_kv, D, ps = 5, 2, 64, 32
    lens = [N + 100, 0, N, N + 31, N + 1]
    bt, pages = table_for(lens, ps)
    cache = poison(alloc_kvcache_fp8(pages, ps, H_kv, D))
    k = randn(B, N, H_kv, D, dtype=torch.bfloat16, seed=1).transpose(1, 2)
    v = randn(B, N, H_kv, D, dtype=torch.bfloat16, seed=2).transpose(1, 2)
    kvcache_append_fp8(k, v, cache, bt, torch.tensor(lens, dtype=torch.int32).cuda())
    for b in (0, 2, 3, 4):
        check_rows(cache, bt, b, lens[b] - N, k[b].transpose(0, 1), v[b].transpose(0, 1))


def test_append_extreme_rows():
    """Zero rows, the largest and smallest values of the type, NaN and infinity, negative maxima."""
    D = 128
    x = randn(16, 1, D, dtype=torch.bfloat16)
    x[0] = 0
    x[1] = 0
    x[1, 0, 3] = 9.2e-41  # the smallest bf16 subnormal
    x[2] = torch.finfo(torch.bfloat16).max
    x[3, 0, 5] = math.nan
    x[4, 0, 6] = math.inf
    x[5, 0, 7] = -math.inf
    x[6, 0, 8] = -1000.0
    x[7] *= 1e-38
    x[8] *= 1e30
    x[9] = -0.0
    bt, pages = table_for([16], 16)
    cache = poison(alloc_kvcache_fp8(pages, 16, 1, D))
    kvcache_append_fp8(x, -x, cache, bt, torch.tensor([16], dtype=torch.int32).cuda(),
                       cu_seqlens=torch.tensor([0, 16], dtype=torch.int32).cuda())
    got_s = cache.k_scale[bt[0, 0].long(), :, 0]
    assert torch.isnan(got_s[3:6]).all() and torch.isfinite(got_s[:3]).all()
    keep = [i for i in range(16) if i != 1]  # a scale of a few subnormal steps: only its codes' bound below
    want_codes, want_s = serving.quantise(x)
    got = cache.k.view(torch.uint8)[bt[0, 0].long()].view(torch.float8_e4m3fn).float()
    assert torch.equal(torch.nan_to_num(got_s[keep]), torch.nan_to_num(want_s[keep, 0]))
    assert torch.equal(got[keep], want_codes[keep])
    # Row 1: a scale of 146 subnormal steps is off by half of one, so its value by 1 / 292.
    assert abs(got[1, 0, 3].double() * got_s[1].double() - x[1, 0, 3].double()) <= x[1, 0, 3].double() * (2.0 ** -4 + 1 / 292)
    back, _ = kvcache_read_fp8(cache, bt, torch.tensor([0, 16], dtype=torch.int32).cuda(), 16)
    assert torch.isnan(back[3:6]).all() and torch.isfinite(back[6:]).all() and (back[0] == 0).all()


def test_append_unaligned_input():
    D, H_kv = 32, 2
    store = randn(20, H_kv, D + 1, dtype=torch.float16)
    k, v = store[..., 1:], store[..., :-1]
    bt, pages = table_for([20], 16)
    cache = alloc_kvcache_fp8(pages, 16, H_kv, D)
    kvcache_append_fp8(k, v, cache, bt, torch.tensor([20], dtype=torch.int32).cuda(),
                       cu_seqlens=torch.tensor([0, 20], dtype=torch.int32).cuda())
    check_rows(cache, bt, 0, 0, k, v)


# ------------------------------------------------------------------------------------ read
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page_size", [(128, 256), (64, 16), (32, 64), (16, 128)])
def test_read_back(dtype, D, page_size):
    lens = [700, 1, 0, 257, 16]
    cache, bt, _, _, _, _ = filled(lens, page_size, 3, D, dtype, seed=3, plain_layout=page_size == 64)
    part = [500, 1, 0, 257, 3]  # prefixes of them
    cu = torch.tensor([0] + list(torch.tensor(part).cumsum(0)), dtype=torch.int32).cuda()
    k, v = kvcache_read_fp8(cache, bt, cu, sum(part) + 9, dtype=dtype)
    for b, n in enumerate(part):
        for got, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
            ref = serving.rows_of(codes, scales, bt, b, n)
            tol = ref.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -23) + SUBNORMAL[dtype]
            assert ((got[cu[b]:cu[b + 1]].double() - ref).abs() <= tol).all()


# ------------------------------------------------------------------------------------ attention
def tolerance(q, weight, spread, small, out, n, v_top):
    """How far the kernel's output may be from the 64-bit one, element by element.

    A score x = sm_scale log2(e) sum q k is a fp32 sum of D exact products and two more roundings,
    subtracted from the maximum: off by at most (D + 8) 2^-23 spread log2(e) (2^-23: a tensor sum may
    truncate), so p is off by ln(2) times that, and 2^-22 for exp2; numerator and denominator both
    have it. P' = p sv 2^k is rounded to fp16: 2^-11, or 2^-31 of the largest |v| for a subnormal
    one, n of them at most. The fp32 sums over n keys: n / 8 * 2^-23 each. The output is rounded
    once: eps / 2, half a subnormal step at the bottom of fp16. What an element is off by is relative
    to weight = sum p |v| / sum p.

    Many rows: a query's values more than 2^10 below its row's largest are off by at most 2^-17 of
    that one (e4m3 terms), which moves a score by 2^-17 small. Their bf16 queries also run on v * 2^k
    rounded to fp16 (half a step: 2^-11 of the value)."""
    D = q.shape[-1]
    folded = 2.0 ** -11 if q.dtype == torch.bfloat16 else 0.0
    dx = (D + 8) * 2.0 ** -23 * spread[..., None] + 2.0 ** -17 * small[..., None] + 2.0 ** -22
    rel = 2.0 ** -11 + folded + 2 * dx + 2 * n / 8 * 2.0 ** -23
    eps = torch.finfo(q.dtype).eps / 2
    return weight * rel * (1 + eps) + eps * out.abs() + n * 2.0 ** -31 * v_top + SUBNORMAL[q.dtype]


def check_attention(q, cache, bt, lens, **kw):
    got = attention_kvcache_fp8(q, cache, bt, lens, **kw)
    plain_kw = {k: kw[k] for k in ("causal", "sm_scale", "causal_align", "cu_seqlens_q") if k in kw}
    out, weight, spread, small = serving.attention(q, cache, bt, lens, **plain_kw)
    n = int(lens.max())
    v_top = max([serving.rows_of(cache[1], cache[3], bt, b, m).abs().max().item() for b, m in enumerate(lens.tolist()) if m] + [0.0])
    assert got.shape == q.shape and got.dtype == q.dtype
    end = q.shape[0] if q.dim() == 4 else int(kw["cu_seqlens_q"][-1])
    err, tol = (got.double() - out).abs()[:end], tolerance(q, weight, spread, small, out, n, v_top)[:end]
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3f} of the tolerance, err {err.max().item():.3e}"
    return got


@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256, 384])
@pytest.mark.parametrize("N_q", [1, 5, 70])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_pages_and_lengths(page_size, N_q, causal):
    lens = [max(n, N_q) for n in (1, 15, 16, 17, 129, 700, 1025)]
    cache, bt, sl, _, _, _ = filled(lens, page_size, 2, 128, seed=page_size)
    check_attention(randn(len(lens), 8, N_q, 128, dtype=torch.bfloat16, seed=9), cache, bt, sl, causal=causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("group", [1, 3, 4, 16, 20])
def test_attention_heads_and_types(dtype, D, group):
    lens = [333, 64, 2049]
    cache, bt, sl, _, _, _ = filled(lens, 64, 2, D, dtype, seed=D + group, plain_layout=group == 3)
    for n in (1, 9):
        check_attention(randn(3, 2 * group, n, D, dtype=dtype, seed=4), cache, bt, sl)


@pytest.mark.parametrize("num_splits", [1, 2, 7, 100])
@pytest.mark.parametrize("N_q", [1, 33])
def test_attention_splits(num_splits, N_q):
    lens = [4000, 33, 1111, 4096]
    cache, bt, sl, _, _, _ = filled(lens, 128, 2, 64, torch.float16, seed=5)
    check_attention(randn(4, 8, N_q, 64, dtype=torch.float16, seed=6), cache, bt, sl, num_splits=num_splits)


@pytest.mark.parametrize("align", ["bottom_right", "top_left"])
@pytest.mark.parametrize("N_q", [40, 300])
def test_attention_masks_that_leave_rows_empty(align, N_q):
    """Sequences with no key, fewer keys than queries, and as many: rows that see nothing are zeros."""
    lens = [0, 1, 17, N_q, N_q + 200]
    cache, bt, sl, _, _, _ = filled(lens, 16, 2, 64, seed=7)
    q = randn(5, 6, N_q, 64, dtype=torch.bfloat16, seed=8)
    for splits in (1, 3):
        out = check_attention(q, cache, bt, sl, causal_align=align, num_splits=splits)
        assert (out[0] == 0).all()
        if align == "bottom_right":
            assert (out[2, :, :N_q - 17] == 0).all()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 16)])
@pytest.mark.parametrize("num_splits", [None, 1, 4])
def test_attention_packed_queries(dtype, D, num_splits):
    """Prompt chunks and single tokens in one call, a sequence without queries, one without keys,
    and rows behind the last sequence."""
    new, lens = [1, 64, 0, 300, 1, 2, 9], [513, 64, 90, 2000, 1, 0, 700]
    cache, bt, sl, _, _, _ = filled(lens, 32, 2, D, dtype, seed=11)
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32).cuda()
    q = randn(sum(new) + 5, 6, D, dtype=dtype, seed=12)
    out = check_attention(q, cache, bt, sl, cu_seqlens_q=cu, max_seqlen_q=300, max_seqlen_k=2000, num_splits=num_splits)
    assert (out[cu[5]:cu[6]] == 0).all()
    check_attention(q, cache, bt, sl, cu_seqlens_q=cu, max_seqlen_q=301, causal=False, num_splits=num_splits)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128)])
def test_attention_long_shares_of_a_ragged_batch(dtype, D):
    """Shares of many tiles and several blocks, so that a block's own cost counts in the line; new tokens
    from none to 300, heads in groups of three, so blocks of 256, of 129 to 255 and of fewer rows."""
    new = [(37 * b * b + 11 * b) % 301 for b in range(40)]
    lens = [max(n, (97 * b * b + 501) % 2300) if b % 9 else n for b, n in enumerate(new)]
    cache, bt, sl, _, _, _ = filled(lens, 64, 2, D, dtype, seed=31)
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32).cuda()
    q = randn(sum(new), 6, D, dtype=dtype, seed=32)
    first = check_attention(q, cache, bt, sl, cu_seqlens_q=cu, max_seqlen_q=300)
    check_attention(q, cache, bt, sl, cu_seqlens_q=cu, max_seqlen_q=300, causal=False)
    assert torch.equal(attention_kvcache_fp8(q, cache, bt, sl, cu_seqlens_q=cu, max_seqlen_q=300), first)


@pytest.mark.parametrize("N_q", [1, 4, 90])
def test_attention_many_sequences(N_q):
    """More sequences than a warp's lanes or the GPU's SMs, every third without a key."""
    lens = [0 if b % 3 == 2 else 1 + (b * 53) % 400 for b in range(330)]
    cache, bt, sl, _, _, _ = filled(lens, 16, 1, 32, seed=33)
    out = check_attention(randn(330, 4, N_q, 32, dtype=torch.bfloat16, seed=34), cache, bt, sl)
    assert (out[2::3] == 0).all()


@pytest.mark.parametrize("N_q", [1, 200])
def test_attention_sizes_of_values(N_q):
    """Values whose scales span 2^40 from row to row, large and tiny scores, zero rows."""
    lens = [900, 350]
    cache, bt, sl, cu, k, v = filled(lens, 64, 2, 128, seed=13)
    g = torch.Generator().manual_seed(1)
    size = 2.0 ** torch.randint(-30, 11, (sum(lens), 1, 1), generator=g).float().cuda()
    v2 = (v[:sum(lens)].float() * size).to(v.dtype)
    v2[::7] = 0
    k2 = k[:sum(lens)].clone()
    k2[::5] = 0
    kvcache_append_fp8(k2, v2, cache, bt, sl, cu_seqlens=cu)
    for s in (1e-3, 1.0, 1e4):
        q = (randn(2, 4, N_q, 128, dtype=torch.float32, seed=14) * s).to(torch.bfloat16)
        q[:, 1] = 0
        check_attention(q, cache, bt, sl)
    check_attention((randn(2, 4, N_q, 128, dtype=torch.float32, seed=15) * 1e-38).to(torch.bfloat16), cache, bt, sl)
    check_attention(randn(2, 4, N_q, 128, dtype=torch.bfloat16, seed=15), cache, bt, sl, sm_scale=0.5)


@pytest.mark.parametrize("N_q", [6, 150])
def test_attention_nonfinite_rows_reach_only_who_sees_them(N_q):
    lens = [400]
    cache, bt, sl, cu, k, v = filled(lens, 32, 1, 128, seed=16)
    k[400 - 2, 0, 3] = math.nan       # the key of the last query but one
    v[400 - 4, 0, 9] = math.inf
    kvcache_append_fp8(k[:400], v[:400], cache, bt, sl, cu_seqlens=cu)
    q = randn(1, 4, N_q, 128, dtype=torch.bfloat16, seed=17)
    out = attention_kvcache_fp8(q, cache, bt, sl)
    assert torch.isnan(out[:, :, N_q - 4:]).all()
    assert torch.isfinite(out[:, :, :N_q - 4]).all()
    clean, *_ = serving.attention(q[:, :, :N_q - 4], cache, bt, sl - 4)
    assert (out[:, :, :N_q - 4].double() - clean).abs().max() < 0.02  # (bounded tightly by the tests above)
    q[0, 2, 1, 5] = math.nan
    out = attention_kvcache_fp8(q, cache, bt, sl)
    assert torch.isnan(out[0, 2, 1]).all() and torch.isfinite(out[0, 1, :N_q - 4]).all()


def test_attention_long_cache():
    """65,536 keys, and offsets past 2^31 bytes from the cache's start."""
    pages, ps, H, D = 9000, 256, 8, 128  # 2.4e9 bytes a tensor
    cache = alloc_kvcache_fp8(pages, ps, H, D)
    lens = [65536, 4097]
    g = torch.Generator().manual_seed(3)
    bt = (pages - 1 - torch.randperm(600, generator=g)[:2 * 256]).view(2, 256).to(torch.int32).cuda()  # the last pages
    k, v = randn(sum(lens), H, D, dtype=torch.bfloat16, seed=1), randn(sum(lens), H, D, dtype=torch.bfloat16, seed=2)
    sl = torch.tensor(lens, dtype=torch.int32).cuda()
    cu = torch.tensor([0, 65536, 65536 + 4097], dtype=torch.int32).cuda()
    kvcache_append_fp8(k, v, cache, bt, sl, cu_seqlens=cu)
    check_rows(cache, bt, 1, 0, k[65536:], v[65536:])
    check_attention(randn(2, 32, 1, D, dtype=torch.bfloat16, seed=4), cache, bt, sl)
    check_attention(randn(2, 32, 40, D, dtype=torch.bfloat16, seed=5), cache, bt, sl)


@pytest.mark.parametrize("N_q", [1, 160])
def test_attention_same_bits_every_time_and_on_strided_queries(N_q):
    lens = [3000, 70]
    cache, bt, sl, _, _, _ = filled([max(n, N_q) for n in lens], 64, 4, 128, seed=18)
    q = randn(2, N_q, 8, 128, dtype=torch.bfloat16, seed=19).transpose(1, 2)
    first = attention_kvcache_fp8(q, cache, bt, sl)
    assert first.stride() == q.stride()
    for _ in range(3):
        assert torch.equal(attention_kvcache_fp8(q, cache, bt, sl), first)
    assert torch.equal(attention_kvcache_fp8(q.contiguous(), cache, bt, sl), first)
    odd = torch.zeros(2, 8, N_q, 131, dtype=torch.bfloat16, device="cuda")[..., 3:]
    odd.copy_(q)
    assert torch.equal(attention_kvcache_fp8(odd, cache, bt, sl), first)
    wide = torch.zeros(2, 2 * bt.shape[1], dtype=torch.int32, device="cuda")
    wide[:, ::2] = bt
    assert torch.equal(attention_kvcache_fp8(q, cache, wide[:, ::2], sl), first)


# ------------------------------------------------------------------------------------ reports
def test_reports_of_lengths_and_pages():
    cache, bt, sl, _, k, v = filled([300, 200], 64, 2, 64, seed=20)
    q = randn(2, 4, 1, 64, dtype=torch.bfloat16, seed=21)
    good = attention_kvcache_fp8(q, cache, bt, sl)

    def reported(status):
        with pytest.raises(RuntimeError, match=f"status {status}:"):
            check_device_errors()

    out = attention_kvcache_fp8(q, cache, bt, sl, max_seqlen_k=256)
    reported(_lib.FA2_ERR_SHAPE)
    assert (out[0] == 0).all()
    for bad in (-1, 6 * 64, 1 << 30):
        out = attention_kvcache_fp8(q, cache, bt, torch.tensor([bad, 200], dtype=torch.int32).cuda(), max_seqlen_k=320)
        reported(_lib.FA2_ERR_SHAPE)
        # As if it had no keys. The other sequence's keys may be cut elsewhere than beside a good one (the
        # sequences share the work as one line), so its sum differs in rounding: both results are
        # within `tolerance` of the same value, none is promised to have the other's bits.
        ref, weight, spread, small = serving.attention(q, cache, bt, torch.tensor([0, 200], dtype=torch.int32).cuda())
        assert (out[0] == 0).all() and (ref[0] == 0).all()
        assert ((out.double() - ref).abs() <= tolerance(q, weight, spread, small, ref, 200, 8.0)).all()
    for page in (-1, cache.k.shape[0], 1 << 30):
        wrong = bt.clone()
        wrong[1, 1] = page
        out = attention_kvcache_fp8(q, cache, wrong, sl)
        reported(_lib.FA2_ERR_PAGE)
        assert torch.equal(out[0], good[0]) and torch.isnan(out[1]).all()
        cu = torch.tensor([0, 300, 500], dtype=torch.int32).cuda()
        kr, _ = kvcache_read_fp8(cache, wrong, cu, 500)
        reported(_lib.FA2_ERR_PAGE)
        assert (kr[364:428] == 0).all() and torch.isfinite(kr).all()
        was = cache.k.view(torch.uint8).clone()
        kvcache_append_fp8(k[:500], v[:500], cache, wrong, sl, cu_seqlens=cu)
        reported(_lib.FA2_ERR_PAGE)
        assert torch.equal(cache.k.view(torch.uint8), was)  # the same rows as before, none elsewhere
    # More new tokens than the length that counts them; a length past the table.
    kvcache_append_fp8(k[:500], v[:500], cache, bt, torch.tensor([299, 200], dtype=torch.int32).cuda(),
                       cu_seqlens=torch.tensor([0, 300, 500], dtype=torch.int32).cuda())
    reported(_lib.FA2_ERR_SHAPE)
    kvcache_append_fp8(k[:2].view(2, 2, 1, 64), v[:2].view(2, 2, 1, 64), cache, bt, torch.tensor([321, 200], dtype=torch.int32).cuda())
    reported(_lib.FA2_ERR_SHAPE)
    # Sums of the query lengths that leave their tensor, fall, or exceed the declared maximum.
    qp = randn(10, 4, 64, dtype=torch.bfloat16, seed=22)
    for cu in ([0, 4, 11], [0, 5, 3], [-1, 4, 10], [0, 9, 10]):
        attention_kvcache_fp8(qp, cache, bt, sl, cu_seqlens_q=torch.tensor(cu, dtype=torch.int32).cuda(), max_seqlen_q=6)
        reported(_lib.FA2_ERR_SHAPE)


# ------------------------------------------------------------------------------------ together
def test_step_of_a_serving_loop():
    """Rotary, append, attention as a decode loop runs them, three steps after a packed prompt; the
    prompt's attention by attention_varlen over the rows read back. Checked step by step in 64 bits."""
    B, H_q, H_kv, D, ps = 3, 8, 2, 64, 16
    prompts = [37, 5, 130]
    bt, pages = table_for([n + 4 for n in prompts], ps)
    cache = poison(alloc_kvcache_fp8(pages, ps, H_kv, D))
    freq, mag = rotary_inv_freq(D, scaling="yarn", factor=4.0, device="cuda")
    cu = torch.tensor([0, 37, 42, 172], dtype=torch.int32).cuda()
    pos = torch.cat([torch.arange(n) for n in prompts]).cuda()
    q, k, v = (randn(172, h, D, dtype=torch.bfloat16, seed=s) for h, s in ((H_q, 1), (H_kv, 2), (H_kv, 3)))
    q, k = rotary(q, k, pos, freq, magnitude=mag)
    lens = torch.tensor(prompts, dtype=torch.int32).cuda()
    kvcache_append_fp8(k, v, cache, bt, lens, cu_seqlens=cu)
    out = check_attention(q, cache, bt, lens, cu_seqlens_q=cu, max_seqlen_q=130)
    kb, vb = kvcache_read_fp8(cache, bt, cu, 172)
    same = attention_varlen(q, kb, vb, cu, cu, 130, 130, causal=True)
    # kb and vb are the cache's values rounded to bf16 (2^-8 or less): scores move by 2^-8 of their size
    # (below 8 here), the values by 2^-8; both outputs round once more.
    assert (out.double() - same.double()).abs().max() <= (2 * 8 * 2.0 ** -8 + 3 * 2.0 ** -8) * vb.double().abs().max()
    for step in range(3):
        lens += 1
        q, k, v = (randn(B, h, 1, D, dtype=torch.bfloat16, seed=10 * step + s) for h, s in ((H_q, 4), (H_kv, 5), (H_kv, 6)))
        q, k = rotary(q, k, (lens - 1)[:, None], freq, magnitude=mag)
        kvcache_append_fp8(k, v, cache, bt, lens)
        check_attention(q, cache, bt, lens)


@pytest.mark.parametrize("N_q", [1, 150])
def test_two_graphs_and_a_side_stream(N_q):
    """Two captured graphs and eager calls with workspaces of their own, replayed in turn and beside
    one another; lengths change between replays."""
    lens = [2000, 600]
    cache, bt, sl, _, _, _ = filled(lens, 64, 2, 128, seed=23)
    qs = [randn(2, 8, N_q, 128, dtype=torch.bfloat16, seed=24 + i) for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for q in qs:
            attention_kvcache_fp8(q, cache, bt, sl, num_splits=5)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(attention_kvcache_fp8(q, cache, bt, sl, num_splits=5))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for change in (0, -37, -400):
        sl.copy_(torch.tensor([2000 + change, 600 + change], dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        eager = attention_kvcache_fp8(qs[0], cache, bt, sl, num_splits=5)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager)
        assert torch.equal(outs[1], attention_kvcache_fp8(qs[1], cache, bt, sl, num_splits=5))
        ref, weight, spread, small = serving.attention(qs[1], cache, bt, sl)
        assert ((outs[1].double() - ref).abs() <= tolerance(qs[1], weight, spread, small, ref, 2000, 8.0)).all()
