"""Rotary positions for the queries and keys of `fa2.kernel` (an extension: the reference has none).

    rotary_inv_freq(rotary_dim, base=10000.0, scaling=None, ...) -> (inv_freq, magnitude)
    rotary(q, k, positions, inv_freq, interleaved=False, inverse=False, magnitude=1.0, inplace=False)

Forward only, like attention(): `inverse=True` applies the transposed map, which is the gradient of
the forward one.
"""

import functools
import math

import torch

from . import _kvlib

SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_inv_freq(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_max_position=4096,
                    beta_fast=32.0, beta_slow=1.0, device=None):
    """Radians a position for each of the rotary_dim / 2 pairs (float64), and the factor on the
    rotated values.

    f_i = base^(-2 i / rotary_dim). Scalings for contexts `factor` times longer than
    original_max_position: "linear" f_i / factor; "ntk" base * factor^(rd / (rd - 2)), which leaves the
    fastest pair and divides the slowest by factor; "yarn" f_i where a pair turns more than beta_fast times
    within original_max_position, f_i / factor where it turns less than beta_slow times, between them a
    linear ramp over the pair's index (from the pair at or before the one, to the pair at or behind the other,
    within [0, rotary_dim - 1] as published), and the magnitude 0.1 ln(factor) + 1.
    """
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not base > 1 or not factor >= 1:
        raise ValueError(f"base must be above 1 and factor at least 1, got {base} and {factor}")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    magnitude = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-2 * i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn" and factor > 1:
        def pair_of(turns):  # the (fractional) pair that turns so often within the original context
            return rotary_dim * math.log(original_max_position / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(0, math.floor(pair_of(beta_fast)))
        # (The end may lie behind the last pair, which then still turns more than beta_slow times.)
        high = min(rotary_dim - 1, math.ceil(pair_of(beta_slow)))
        stretched = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f * (1 - stretched) + f / factor * stretched
        magnitude = 0.1 * math.log(factor) + 1.0
    return f.to(device), magnitude


_DTYPES = (torch.float16, torch.bfloat16)  # the index is the C ABI's Fa2DType
_NONE = (0, 0, 0, 0)


def _strides4(t):
    st = t.stride()
    return st if len(st) == 4 else (0, st[1], st[0], st[2])  # [total, H, D]


def _reaches(terms, target, left):
    """Whether whole numbers lo <= x <= hi exist for the terms (stride, lo, hi) with sum stride * x = target.
    Largest strides first: as long as a stride is longer than what the smaller ones span, at most two x
    each are in question. left: [steps], after which the answer is True."""
    if not terms:
        return target == 0
    left[0] -= 1
    if left[0] < 0:
        return True
    (stride, lo, hi), rest = terms[0], terms[1:]
    least, most = sum(s * a for s, a, _ in rest), sum(s * b for s, _, b in rest)
    first, last = max(lo, -((most - target) // stride)), min(hi, (target - least) // stride)
    return any(_reaches(rest, target - stride * x, left) for x in range(first, last + 1))


@functools.lru_cache(maxsize=4096)
def _share_memory(dims, other=None, distance=0):
    """Whether two values of a tensor of dims ((size, stride), ...) share an address; with the dims of
    another tensor that starts `distance` elements behind it: a value of each. (Layouts that are too tangled to
    tell count as sharing.)"""
    left = [10000]
    if other is None:
        dims = sorted(((s, n) for n, s in dims if n > 1), reverse=True)
        if any(s == 0 for s, _ in dims):
            return True
        # The first index that differs is larger in one of the two values by 1 or more.
        return any(_reaches([(s, 1, n - 1)] + [(t, 1 - m, m - 1) for t, m in dims[i + 1:]], 0, left) for i, (s, n) in enumerate(dims))
    spans = {}
    for n, s in dims:
        if n > 1 and s:
            lo, hi = spans.get(s, (0, 0))
            spans[s] = lo, hi + n - 1
    for n, s in other:
        if n > 1 and s:
            lo, hi = spans.get(s, (0, 0))
            spans[s] = lo - (n - 1), hi
    return _reaches(sorted(((s, lo, hi) for s, (lo, hi) in spans.items()), reverse=True), distance, left)


def _refuse_shared(q, k):
    """Rotation in place: every value of q and k has memory of its own."""
    tensors = [t for t in (q, k) if t is not None and t.numel() > 0]
    dims = [tuple(zip(t.shape, t.stride())) for t in tensors]
    shared = any(_share_memory(d) for d in dims)
    if not shared and len(tensors) == 2:
        shared = _share_memory(dims[0], dims[1], (tensors[1].data_ptr() - tensors[0].data_ptr()) // 2)
    if shared:
        raise ValueError("inplace needs tensors whose values do not share memory (no expanded dimensions or overlapping "
                         "views, no value in both q and k)")


def rotary(q, k, positions, inv_freq, interleaved=False, inverse=False, magnitude=1.0, inplace=False):
    """Turns the pairs of q's and k's heads by position * inv_freq, both in one launch.

    q: [B, H_q, N, D], k: [B, H_kv, N, D] (or None) with positions [B, N] or [N]; or packed along one
    token axis, q [total, H_q, D], k [total, H_kv, D] with positions [total]. fp16/bf16, any strides;
    positions int32 or int64. inv_freq: float64 [rotary_dim / 2] on the same device, rotary_dim <= D;
    values from rotary_dim on pass unchanged. Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) with
    interleaved=True. The angle is formed in 64 bits, so far positions lose nothing.

    inverse=True turns by the negative angle: with the same magnitude, the gradient of the forward
    map. inplace=True writes into q and k themselves, which may be views of one buffer but have no value
    in common. Returns (q', k'); k' is None where k is.
    Asynchronous on torch's current stream.
    """
    dims, dtype = q.dim(), q.dtype
    assert dims in (3, 4), "q must be [B, H, N, D] or [total, H, D]"
    assert dtype in _DTYPES, "q must be fp16 or bf16"
    q_shape, pos_shape = q.shape, positions.shape
    pos_st = positions.stride()
    if dims == 4:
        B, H_q, N, D = q_shape
        assert pos_shape == (B, N) or pos_shape == (N,), "positions must be [B, N] or [N]"
        if len(pos_st) == 1:
            pos_st = (0, *pos_st)
    else:
        B, (N, H_q, D) = 1, q_shape
        assert pos_shape == (N,), "positions must be [total]"
        pos_st = (0, *pos_st)
    H_kv = 0
    if k is not None:
        k_shape = k.shape
        H_kv = k_shape[1] if len(k_shape) > 1 else 0
        assert k.dtype == dtype and k_shape == ((B, H_kv, N, D) if dims == 4 else (N, H_kv, D)), "k must match q"
    pos_dtype = positions.dtype
    assert pos_dtype == torch.int64 or pos_dtype == torch.int32, "positions must be int32 or int64"
    assert inv_freq.dtype == torch.float64 and inv_freq.dim() == 1, "inv_freq must be float64 [rotary_dim / 2]"
    rd = 2 * inv_freq.numel()
    assert 2 <= rd <= D, "inv_freq must have between 1 and D / 2 entries"
    if not 0 < magnitude < 3e38:
        raise ValueError(f"magnitude must be positive and finite, got {magnitude}")
    if inplace:
        _refuse_shared(q, k)
    index = q.get_device()  # -1: not on CUDA
    if index < 0 or positions.get_device() < 0 or inv_freq.get_device() < 0 or (k is not None and k.get_device() < 0):
        raise RuntimeError("fa2.rotary.rotary runs only on an sm_100 CUDA device (no CPU path)")
    if positions.get_device() != index or inv_freq.get_device() != index or (k is not None and k.get_device() != index):
        raise RuntimeError("q, k, positions and inv_freq must be on the same CUDA device")
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
        raise RuntimeError("fa2.rotary.rotary is forward only: use it under torch.no_grad(); "
                           "inverse=True gives the gradient")
    if k is not None and H_kv == 0:
        raise ValueError("k has no heads: pass None")
    if inplace:
        q_out, k_out = q, k
    else:
        q_out, k_out = torch.empty_like(q), None if k is None else torch.empty_like(k)
    if B == 0 or N == 0:
        return q_out, k_out
    if H_q == 0:
        raise ValueError("q has no heads")
    if inv_freq.stride(0) != 1:
        inv_freq = inv_freq.contiguous()
    packed = _kvlib.ROTARY.pack(
        q.data_ptr(), 0 if k is None else k.data_ptr(), q_out.data_ptr(), 0 if k is None else k_out.data_ptr(),
        *_strides4(q), *(_NONE if k is None else _strides4(k)),
        *_strides4(q_out), *(_NONE if k is None else _strides4(k_out)),
        positions.data_ptr(), *pos_st, inv_freq.data_ptr(),
        pos_dtype == torch.int64, B, N, H_q, H_kv, D, rd, dtype == torch.bfloat16,
        bool(interleaved), bool(inverse), magnitude, 0)
    _kvlib.launch(_kvlib.lib().fa2_rotary_sm100, packed, index)
    return q_out, k_out
