"""GPU tests of what the 8-bit cache's attention does beside a report (a refused page, length or sum of
lengths) and when a wait runs out, in the kernel for many rows a kv head as in the one for few."""

import struct

import pytest
import torch

from fa2 import _kvlib, _lib, kvcache
from fa2.kernel import attention, check_device_errors
from fa2.kvcache import attention_kvcache_fp8
from oracle import serving
from test_kvcache_gpu import _no_device_errors, filled, randn, tolerance  # noqa: F401

pytestmark = pytest.mark.gpu

LENS = [1300, 200, 700, 64, 2049]


def reported(status):
    with pytest.raises(RuntimeError, match=f"status {status}:"):
        check_device_errors()


def held(out, q, cache, bt, lens, keep):
    """Sequences `keep` of `out` are within `tolerance` of the 64-bit form; lens: what they may see."""
    ref, weight, spread, small = serving.attention(q, cache, bt, lens)
    ok = (out.double() - ref).abs() <= tolerance(q, weight, spread, small, ref, int(lens.max()), 8.0)
    assert ok[keep].all()


@pytest.mark.parametrize("N_q", [1, 40, 200])  # 2, 80 and 400 rows a kv head
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_refused_page_or_length_leaves_the_others_alone(N_q, dtype):
    cache, bt, sl, _, _, _ = filled(LENS, 64, 2, 64, dtype, seed=20)
    q = randn(len(LENS), 4, N_q, 64, dtype=dtype, seed=21)
    others = [0, 2, 3, 4]
    wrong = bt.clone()
    wrong[1, 0] = cache.k.shape[0]  # every key's way starts there
    out = attention_kvcache_fp8(q, cache, wrong, sl)
    held(out, q, cache, bt, sl, others)
    sees = (torch.arange(N_q) + 200 - N_q >= 0).cuda()
    assert torch.isnan(out[1][:, sees]).all() and (out[1][:, ~sees] == 0).all()
    reported(_lib.FA2_ERR_PAGE)
    for bad in (-1, 64 * bt.shape[1] + 1):
        lens = torch.tensor([LENS[0], bad, *LENS[2:]], dtype=torch.int32).cuda()
        out = attention_kvcache_fp8(q, cache, bt, lens)
        held(out, q, cache, bt, torch.tensor([LENS[0], 0, *LENS[2:]], dtype=torch.int32).cuda(), others)
        assert (out[1] == 0).all()
        reported(_lib.FA2_ERR_SHAPE)


@pytest.mark.parametrize("N_q", [1, 40, 200])
def test_calls_beside_an_uncleared_report(N_q):
    """A report stays until it is asked for; until then later calls give what they give without it, the
    16-bit attention's as well."""
    cache, bt, sl, _, _, _ = filled(LENS, 64, 2, 64, seed=22)
    q = randn(len(LENS), 4, N_q, 64, dtype=torch.bfloat16, seed=23)
    x = [randn(2, 8, 1500, 64, dtype=torch.bfloat16, seed=24 + i) for i in range(3)]
    good, good16 = attention_kvcache_fp8(q, cache, bt, sl), attention(*x)
    wrong = bt.clone()
    wrong[1, 1] = -1
    attention_kvcache_fp8(q, cache, wrong, sl)
    for _ in range(3):
        assert torch.equal(attention_kvcache_fp8(q, cache, bt, sl), good)
        assert torch.equal(attention(*x), good16)
    reported(_lib.FA2_ERR_PAGE)


@pytest.mark.parametrize("dtype,N_q", [(torch.bfloat16, 200), (torch.bfloat16, 40), (torch.float16, 200)])
def test_a_limit_of_one_clock_ends_the_call(dtype, N_q, monkeypatch):
    """Waits that may run out at their first look at the clock: the call ends, with what it had to say or
    with FA2_ERR_TIMEOUT, and the next one is right."""
    cache, bt, sl, _, _, _ = filled(LENS, 64, 2, 128, dtype, seed=25)
    q = randn(len(LENS), 4, N_q, 128, dtype=dtype, seed=26)
    good = attention_kvcache_fp8(q, cache, bt, sl)
    names = [name for name, _ in _kvlib.ATTN.fields]
    before = _kvlib.ATTN.fields[:names.index("timeout_cycles")]
    at = struct.calcsize("@" + "".join(code for _, code in before) + "0q")
    launch = kvcache._launch

    def impatient(entry, packed, index):
        launch(entry, packed[:at] + struct.pack("q", 1) + packed[at + 8:], index)

    monkeypatch.setattr(kvcache, "_launch", impatient)
    for _ in range(5):
        out = attention_kvcache_fp8(q, cache, bt, sl)
        try:
            check_device_errors()
            assert torch.equal(out, good)
        except RuntimeError as e:
            assert f"status {_lib.FA2_ERR_TIMEOUT}:" in str(e)
    monkeypatch.undo()
    assert torch.equal(attention_kvcache_fp8(q, cache, bt, sl), good)


@pytest.mark.parametrize("group,N_q", [(2, 6), (8, 40)])
def test_a_refused_number_of_queries_leaves_the_others_alone(group, N_q):
    """Sums that fall, leave q or exceed the declared maximum."""
    cache, bt, sl, _, _, _ = filled([300, 200, 150], 64, 2, 64, seed=27)
    q = randn(3 * N_q + 3, 2 * group, 64, dtype=torch.bfloat16, seed=28)
    total = q.shape[0]
    for cu, good in (([0, N_q, 2 * N_q + 1, 3 * N_q], [0, 2]), ([0, N_q, N_q - 3, N_q - 3], [0]),
                     ([0, N_q, 2 * N_q, total + 1], [0, 1])):
        cu_t = torch.tensor(cu, dtype=torch.int32).cuda()
        out = attention_kvcache_fp8(q, cache, bt, sl, cu_seqlens_q=cu_t, max_seqlen_q=N_q)
        reported(_lib.FA2_ERR_SHAPE)
        for b in good:
            alone = torch.tensor([0, cu[b + 1] - cu[b]], dtype=torch.int32).cuda()
            ref, weight, spread, small = serving.attention(q[cu[b]:cu[b + 1]], cache, bt[b:b + 1], sl[b:b + 1], cu_seqlens_q=alone)
            got, qs = out[cu[b]:cu[b + 1]], q[cu[b]:cu[b + 1]]
            assert ((got.double() - ref).abs() <= tolerance(qs, weight, spread, small, ref, 300, 8.0)).all()


def test_append_and_read_report_sums_that_fall_or_leave_their_tensor():
    """A sequence that goes past the tensor is left out (read: zeros where its rows are), the others are right;
    sums that fall are reported. 200 sequences: more than a block's threads."""
    lens = [3 + b % 5 for b in range(200)]
    cache, bt, sl, cu, k, v = filled(lens, 16, 2, 64, seed=29)
    total = int(cu[-1])
    held = [t.view(torch.uint8).clone() if t.dtype == torch.float8_e4m3fn else t.clone() for t in cache]

    def unchanged():
        return all(torch.equal(torch.nan_to_num(t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t), torch.nan_to_num(h))
                   for t, h in zip(cache, held))

    kr, vr = kvcache.kvcache_read_fp8(cache, bt, cu, total)
    check_device_errors()
    short = total - 2  # the last sequence has three rows or more
    kvcache.kvcache_append_fp8(k[:short] * 1.0, v[:short] * 1.0, cache, bt, sl, cu_seqlens=cu)
    reported(_lib.FA2_ERR_SHAPE)
    assert unchanged()  # the same rows again, and none of the last sequence's
    changed = k.clone()
    changed[int(cu[-2]):] += 1
    kvcache.kvcache_append_fp8(changed[:short], v[:short], cache, bt, sl, cu_seqlens=cu)
    reported(_lib.FA2_ERR_SHAPE)
    assert unchanged()
    ks, vs = kvcache.kvcache_read_fp8(cache, bt, cu, short)
    reported(_lib.FA2_ERR_SHAPE)
    at = int(cu[-2])
    assert torch.equal(ks[:at], kr[:at]) and torch.equal(vs[:at], vr[:at])
    assert (ks[at:] == 0).all() and (vs[at:] == 0).all()
    for i in (1, 150, 199):
        fallen = cu.clone()
        fallen[i] = fallen[i + 1] + 1
        kvcache.kvcache_read_fp8(cache, bt, fallen, total)
        reported(_lib.FA2_ERR_SHAPE)
        kvcache.kvcache_append_fp8(k[:total], v[:total], cache, bt, sl, cu_seqlens=fallen)
        reported(_lib.FA2_ERR_SHAPE)
    negative = cu.clone()
    negative[0] = -1
    kvcache.kvcache_read_fp8(cache, bt, negative, total)
    reported(_lib.FA2_ERR_SHAPE)
