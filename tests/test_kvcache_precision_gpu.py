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


def plain(q, cache, bt, n, sm_scale):
    """One sequence's causal attention in 64 bits: (out, weight, spread, small, top), the first four as
    oracle.serving.attention gives them but over the keys that have any weight (2^-100 of the row's sum), top the
    largest p_ij max|v_j| / sum_j p_ij of a row: what a rounding of a product P V is relative to."""
    k, v = (serving.rows_of(cache[i], cache[i + 2], bt, 0, n) for i in (0, 1))
    H, N_q, D = q.shape[1:]
    group = H // k.shape[1]
    out, weight = torch.zeros(2, *q.shape, dtype=torch.float64, device="cuda")
    spread, small, top = torch.zeros(3, *q.shape[:3], dtype=torch.float64, device="cuda")
    sees = torch.ones(N_q, n, dtype=torch.bool, device="cuda").tril(n - N_q)
    for h in range(H):
        x, key, val = q[0, h].double(), k[:, h // group], v[:, h // group]
        p = torch.softmax((x @ key.T * sm_scale).masked_fill(~sees, -torch.inf), -1)
        p = torch.where(p < 2.0 ** -100, torch.zeros_like(p), p)
        out[0, h], weight[0, h] = p @ val, p @ val.abs()
        spread[0, h] = torch.where(p > 0, x.abs() @ key.abs().T * sm_scale, torch.zeros_like(p)).amax(-1)
        small[0, h] = x.abs().amax(-1) * torch.where(p > 0, key.abs().sum(-1), torch.zeros_like(p)).amax(-1) * sm_scale
        top[0, h] = (p * val.abs().amax(-1)).amax(-1)
    return out, weight, spread, small, top


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N_q", [1, 6, 40, 200])  # 2, 12, 80 and 400 rows a kv head
@pytest.mark.parametrize("D", [128, 64, 16])
@pytest.mark.parametrize("where", ["last", "unheeded", "first", "everywhere", "spread"])
def test_values_far_above_the_others(dtype, N_q, D, where):
    """Value rows up to the type's largest, which some queries do not see or give no weight: they leave those
    queries' outputs as they are. A row of P' is rounded relative to its own largest product: 2^-31 of it and 2^-19
    where the values' scales lie within 2^12 of one another (a common exponent); n keys."""
    n = 900
    cache, bt, sl, cu, k, v = filled([n], 32, 1, D, dtype, seed=50)
    k, v = k[:n].clone(), v[:n].float()
    most = 3e38 if dtype == torch.bfloat16 else 6e4
    v *= 1e-3
    q = randn(1, 2, N_q, D, dtype=dtype, seed=51)
    q[..., 0] = 8
    k[..., 0] = 0.1
    if where == "last":  # seen by the last query alone
        v[n - 1:] = v[n - 1:].sign() * most
    elif where == "unheeded":  # scores far below the others'
        v[[3, 500, 899]] *= most * 1e3 / 8
        k[[3, 500, 899], :, 0] = -40 * D ** 0.5
    elif where == "first":  # a tile of them, soon outweighed
        v[:128] *= most * 1e3 / 8
        k[:128, :, 0] = -40 * D ** 0.5
    elif where == "everywhere":
        v = v.sign() * most
    else:  # sizes over the type's whole range
        g = torch.Generator().manual_seed(52)
        size = torch.rand(n, 1, 1, generator=g).cuda() * 2 - 1
        v *= 1e3 * (2.0 ** (110 * size) if dtype == torch.bfloat16 else 2.0 ** (10 * size))
    kvcache_append_fp8(k, v.clamp(-most, most).to(dtype), cache, bt, sl, cu_seqlens=cu)
    scale = D ** -0.5
    out, weight, spread, small, top = plain(q, cache, bt, n, scale)
    for splits in (None, 1, 3):
        got = attention_kvcache_fp8(q, cache, bt, sl, sm_scale=scale, num_splits=splits)
        tol = bound(q, 2 * N_q, weight, spread, small, out, n, 0.0) + n * 2.0 ** -19 * top[..., None]
        err = (got.double() - out).abs()
        assert (err <= tol).all(), f"worst {(err / tol).nan_to_num(1e9).max().item():.3f} of the tolerance"
