"""GPU tests of how many bits of the queries the 8-bit cache's attention uses: query rows with one channel far
above the others, for few rows a kv head and for many.

Tolerance: `tolerance` of the other tests, whose term for a query's small values (`small`: the row's
largest value times sum |k|) is replaced by the operator's own bound. Values within 2^13 of their row's largest
are exact (8-bit terms; for up to 16 rows fp16 holds them exactly as well): 0. Below that they are off by at most
2^-21 (bf16) or 2^-24 (fp16) of the largest, of which `tolerance` gets 2^-17 times the given size."""

import pytest
import torch

from fa2.kvcache import attention_kvcache_fp8, kvcache_append_fp8
from oracle import serving
from test_kvcache_gpu import SUBNORMAL, _no_device_errors, filled, randn, tolerance  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N_q", [1, 40, 200])  # 4, 160 and 800 rows a kv head
@pytest.mark.parametrize("D", [128, 64, 16])
@pytest.mark.parametrize("size", [300, 2000, 40000])
def test_queries_with_one_large_channel(dtype, N_q, D, size):
    """The large channel's key is small and nearly the same everywhere, so the scores' differences come from the
    other channels, which must keep their bits beside it."""
    lens = [max(N_q, n) for n in (3, 41, 700)]
    cache, bt, sl, cu, k, v = filled(lens, 64, 2, D, dtype, seed=D)
    k = k[:sum(lens)].clone()
    k[..., 5] = 0.03
    kvcache_append_fp8(k, v[:sum(lens)], cache, bt, sl, cu_seqlens=cu)
    x = randn(len(lens), 8, N_q, D, dtype=torch.float32, seed=40)
    q = (x.sign() * x.abs().clamp(0.25, 4.0)).to(dtype)  # within 2^13 of 2000: 0.25 * 8192 = 2048
    q[..., 5] = size
    scale = 4.0 / D ** 0.5
    got = attention_kvcache_fp8(q, cache, bt, sl, sm_scale=scale)
    out, weight, spread, small = serving.attention(q, cache, bt, sl, sm_scale=scale)
    part = 0.0 if size <= 2000 else 2.0 ** -4 if dtype == torch.bfloat16 else 2.0 ** -7
    err, tol = (got.double() - out).abs(), tolerance(q, weight, spread, small * part, out, max(lens), 8.0)
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3f} of the tolerance, err {err.max().item():.3e}"


def bound(q, rows, weight, spread, small, out, n, v_top):
    """`tolerance` with what the kernel that these rows take has, and no more. Both: scores as fp32 sums of exact
    products ((D + 8) 2^-23 of their size), 2^-22 for exp2, P' in fp16 (2^-11, or 2^-31 of the largest |v| for a
    subnormal one), fp32 sums over the keys, one rounding of the output. More than 16 rows: bf16 queries run on
    v * 2^k in fp16 (2^-11 once more), and the queries' values more than 2^13 below their row's largest are off by
    2^-21 or 2^-24 of it."""
    bf16, D = q.dtype == torch.bfloat16, q.shape[-1]
    dx = (D + 8) * 2.0 ** -23 * spread[..., None] + 2.0 ** -22
    rel = 2.0 ** -11
    if rows > 16:
        dx = dx + (2.0 ** -21 if bf16 else 2.0 ** -24) * small[..., None]
        rel += 2.0 ** -11 if bf16 else 0.0
    rel = rel + 2 * dx + 2 * n / 8 * 2.0 ** -23
    eps = torch.finfo(q.dtype).eps / 2
    return weight * rel * (1 + eps) + eps * out.abs() + n * 2.0 ** -31 * v_top + SUBNORMAL[q.dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("group,N_q", [(1, 1), (4, 1), (8, 1), (3, 4), (16, 1), (5, 5), (4, 40), (3, 100)])
def test_each_kernel_within_its_own_bound(dtype, D, group, N_q):
    """1 to 300 rows a kv head: the kernel for up to 16 is held to what it rounds itself."""
    lens = [max(N_q, n) for n in (1, 5, 300, 2500)]
    cache, bt, sl, _, _, _ = filled(lens, 32, 2, D, dtype, seed=D + group)
    q = randn(len(lens), 2 * group, N_q, D, dtype=dtype, seed=41)
    for kw in (dict(), dict(causal=False, num_splits=3)):
        got = attention_kvcache_fp8(q, cache, bt, sl, **kw)
        out, weight, spread, small = serving.attention(q, cache, bt, sl, causal=kw.get("causal", True))
        err, tol = (got.double() - out).abs(), bound(q, group * N_q, weight, spread, small, out, max(lens), 8.0)
        assert (err <= tol).all(), f"worst {(err / tol).max().item():.3f} of the tolerance, err {err.max().item():.3e}"
