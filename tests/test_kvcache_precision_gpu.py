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
from test_kvcache_gpu import _no_device_errors, filled, randn, tolerance  # noqa: F401

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
