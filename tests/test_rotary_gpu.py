"""GPU tests of fa2.rotary.rotary against its 64-bit definition (oracle.serving.rotary).

Tolerance, fixed before the first run. y = a cos t - c sin t in 32 bits from exact 16-bit a, c: the
reduced angle is rounded once (2^-24 of at most pi radians), sincospi is off by a few units of
2^-24, the magnitude, the products and the sum round four more times; all in all less than
2^-20 * magnitude * (|a| + |c|). Then one rounding to 16 bits: half a step, eps / 2 * |y|, or half
the smallest subnormal step for a tiny fp16 result. The angle itself is formed in 64 bits on both sides
(position * inv_freq to 2^-53 of its size: 1e-7 radians at 10^9 radians, within the 2^-20 for every
position used here).
"""

import pytest
import torch

from fa2.kernel import check_device_errors
from fa2.rotary import rotary, rotary_inv_freq
from oracle.serving import rotary as plain

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def pair_size(x, rd, interleaved, magnitude):
    """|a| + |c| of each rotated value's pair, 0 for the copied ones."""
    s = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    y = x.double().abs()
    if interleaved:
        t = y[..., 0:rd:2] + y[..., 1:rd:2]
        s[..., 0:rd:2], s[..., 1:rd:2] = t, t
    else:
        t = y[..., :rd // 2] + y[..., rd // 2:rd]
        s[..., :rd // 2], s[..., rd // 2:rd] = t, t
    return s * magnitude


def check(y, x, pos, freq, interleaved, inverse, magnitude):
    ref = plain(x, pos, freq, interleaved, inverse, magnitude)
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + TINY[x.dtype]
    tol += pair_size(x, 2 * freq.numel(), interleaved, magnitude) * 2.0 ** -20
    err = (y.double() - ref).abs()
    assert y.dtype == x.dtype and y.shape == x.shape
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3f} of the tolerance"
    return y


def randn(*shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rd", [(128, 128), (64, 32), (32, 32), (16, 16), (128, 96), (64, 6), (80, 80), (6, 4), (7, 2)])
def test_rotary_matches_definition(dtype, interleaved, D, rd):
    B, N, H_q, H_kv = 2, 37, 6, 2
    q, k = randn(B, H_q, N, D, dtype=dtype), randn(B, H_kv, N, D, dtype=dtype, seed=1)
    freq, mag = rotary_inv_freq(rd, device="cuda")
    pos = torch.randint(0, 5000, (B, N), generator=torch.Generator().manual_seed(2)).cuda()
    for inverse in (False, True):
        a, b = rotary(q, k, pos, freq, interleaved=interleaved, inverse=inverse, magnitude=mag)
        check(a, q, pos, freq, interleaved, inverse, mag)
        check(b, k, pos, freq, interleaved, inverse, mag)


@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("far", [0, 131072, 10_000_000])
def test_rotary_packed_far_and_negative_positions(pos_dtype, far):
    total, D = 301, 128
    q, k = randn(total, 4, D, dtype=torch.bfloat16), randn(total, 2, D, dtype=torch.bfloat16, seed=1)
    freq, mag = rotary_inv_freq(D, scaling="yarn", factor=16.0, device="cuda")
    pos = (torch.arange(total) * 7 + far - 3).to(pos_dtype).cuda()
    a, b = rotary(q, k, pos, freq, magnitude=mag)
    check(a, q, pos, freq, False, False, mag)
    check(b, k, pos, freq, False, False, mag)


def test_rotary_strided_in_place_and_shared_positions():
    """[B, N, 3, H, D] storage as a projection leaves it, rotated in place: q and k change, v (the
    bytes between) does not."""
    B, N, H, D = 2, 50, 4, 64
    qkv = randn(B, N, 3, H, D, dtype=torch.float16)
    was = qkv.clone()
    q, k = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
    freq, mag = rotary_inv_freq(32, scaling="linear", factor=4.0, device="cuda")
    pos = torch.arange(100, 100 + N, dtype=torch.int32).cuda()
    a, b = rotary(q, k, pos, freq, magnitude=mag, inplace=True)
    assert a.data_ptr() == q.data_ptr() and b.data_ptr() == k.data_ptr()
    check(q, was[:, :, 0].transpose(1, 2), pos, freq, False, False, mag)
    check(k, was[:, :, 1].transpose(1, 2), pos, freq, False, False, mag)
    assert torch.equal(qkv[:, :, 2], was[:, :, 2])


@pytest.mark.parametrize("shift", [1, 4])
def test_rotary_unaligned_and_inner_strides(shift):
    """Bases and strides that 16-byte loads cannot take, and a d stride of 2."""
    B, N, H, D = 2, 9, 3, 32
    store = randn(B, H, N, D + shift + 3, dtype=torch.bfloat16)
    q = store[..., shift:shift + D]
    freq, mag = rotary_inv_freq(D, device="cuda")
    pos = torch.arange(N).cuda()
    check(rotary(q, None, pos, freq)[0], q, pos, freq, False, False, mag)
    wide = randn(B, H, N, 2 * D, dtype=torch.bfloat16)[..., ::2]
    check(rotary(wide, wide[:, :1], pos, freq, interleaved=True)[1], wide[:, :1], pos, freq, True, False, mag)


def test_rotary_expanded_input_many_tokens():
    """A broadcast key (stride 0) and enough tokens for several heads a thread."""
    N, D = 6000, 128
    q = randn(1, 8, N, D, dtype=torch.bfloat16)
    k = randn(1, 1, N, D, dtype=torch.bfloat16, seed=3).expand(1, 5, N, D)
    freq, mag = rotary_inv_freq(D, scaling="ntk", factor=8.0, device="cuda")
    pos = torch.arange(N).cuda()
    a, b = rotary(q, k, pos, freq, magnitude=mag)
    check(a, q, pos, freq, False, False, mag)
    check(b, k, pos, freq, False, False, mag)


def test_rotary_inverse_is_the_gradient():
    """<g, R x> = <R^T g, x>: inverse=True is the transposed map. Each value is off by half a bf16 step
    of itself (2^-8) and by 2^-20 of its pair, so each side of the identity is off by at most
    (2^-8 + 2^-18) * sum |g| |R x| (or |R^T g| |x|)."""
    q, g = randn(1, 3, 40, 64, dtype=torch.bfloat16), randn(1, 3, 40, 64, dtype=torch.bfloat16, seed=5)
    freq, mag = rotary_inv_freq(48, scaling="yarn", factor=4.0, device="cuda")
    pos = torch.arange(40).cuda() * 31
    y = rotary(q, None, pos, freq, magnitude=mag)[0].double()
    x = rotary(g, None, pos, freq, magnitude=mag, inverse=True)[0].double()
    left, right = (g.double() * y).sum(), (x * q.double()).sum()
    size = (g.double() * y).abs().sum() + (x * q.double()).abs().sum()
    assert abs(left - right) <= (2.0 ** -8 + 2.0 ** -18) * size


def test_rotary_gradient_against_differences():
    """The map is linear, so its directional difference is exact: R (x + h e) - R x = h R e. In fp16
    with x + h e and x exact, both rotations round once (2^-11 of the values, below 4 here); the
    difference over h is off from <column of R> by 2 * 4 * 2^-11 / h."""
    D, h = 16, 2.0
    freq, mag = rotary_inv_freq(D, device="cuda")
    x = (torch.arange(D, dtype=torch.float32) / 16).half().cuda().view(1, 1, 1, D)
    pos = torch.tensor([3]).cuda()
    columns = []
    for d in range(D):
        e = torch.zeros_like(x)
        e[..., d] = h
        columns.append((rotary(x + e, None, pos, freq)[0].double() - rotary(x, None, pos, freq)[0].double()).view(-1) / h)
    jac = torch.stack(columns, 1)  # d y / d x
    for d in range(D):
        g = torch.zeros_like(x)
        g[..., d] = 1
        grad = rotary(g, None, pos, freq, inverse=True)[0].double().view(-1)
        assert (grad - jac[d]).abs().max() <= 2 * 4 * 2.0 ** -11 / h + 2.0 ** -11


def test_rotary_nonfinite_stays_in_its_pair():
    x = randn(1, 2, 8, 32, dtype=torch.bfloat16)
    x[0, 0, 3, 5], x[0, 1, 2, 30] = float("nan"), float("inf")
    freq, mag = rotary_inv_freq(32, device="cuda")
    pos = torch.arange(8).cuda()
    y = rotary(x, None, pos, freq)[0]
    hit = torch.zeros(x.shape, dtype=torch.bool)
    for h, n, d in ((0, 3, 5), (1, 2, 30)):
        hit[0, h, n, d % 16] = hit[0, h, n, d % 16 + 16] = True
    assert (~torch.isfinite(y.cpu()) == hit).all()


def test_rotary_on_a_side_stream_and_in_a_graph():
    q, k = randn(4, 8, 1, 128, dtype=torch.bfloat16), randn(4, 2, 1, 128, dtype=torch.bfloat16, seed=1)
    freq, mag = rotary_inv_freq(128, device="cuda")
    pos = torch.tensor([[3], [900], [17], [0]]).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rotary(q, k, pos, freq)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            a, b = rotary(q, k, pos, freq)
    torch.cuda.current_stream().wait_stream(s)
    pos += 5  # the graph reads its tensors again at every replay
    graph.replay()
    torch.cuda.synchronize()
    check(a, q, pos, freq, False, False, mag)
    check(b, k, pos, freq, False, False, mag)
    check_device_errors()
