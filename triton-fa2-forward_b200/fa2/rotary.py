"""Rotary positions for the queries and keys of `fa2.kernel` (an extension: the reference has none).

    rotary_inv_freq(rotary_dim, base=10000.0, scaling=None, ...) -> (inv_freq, magnitude)
    rotary(q, k, positions, inv_freq, interleaved=False, inverse=False, magnitude=1.0, inplace=False)

Forward only, like attention(): `inverse=True` applies the transposed map, which is the gradient of
the forward one.
"""

import math

import torch

from . import _kvlib, _lib

SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_inv_freq(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_max_position=4096,
                    beta_fast=32.0, beta_slow=1.0, device=None):
    """Radians a position for each of the rotary_dim / 2 pairs (float64), and the factor on the
    rotated values.

    f_i = base^(-2 i / rotary_dim). Scalings for contexts `factor` times longer than
    original_max_position: "linear" f_i / factor; "ntk" base * factor^(rd / (rd - 2)), which leaves the
    fastest pair and divides the slowest by factor; "yarn" f_i where a pair turns more than beta_fast times
    within original_max_position, f_i / factor where it turns less than beta_slow times, a linear
    ramp over the pair's index between, and the magnitude 0.1 ln(factor) + 1.
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
        high = min(rotary_dim // 2 - 1, math.ceil(pair_of(beta_slow)))
        stretched = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f * (1 - stretched) + f / factor * stretched
        magnitude = 0.1 * math.log(factor) + 1.0
    return f.to(device), magnitude


def _strides4(t):
    if t.dim() == 4:
        return tuple(int(s) for s in t.stride())
    return (0, int(t.stride(1)), int(t.stride(0)), int(t.stride(2)))  # [total, H, D]


def _overlaps(t):
    return any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride()))


def rotary(q, k, positions, inv_freq, interleaved=False, inverse=False, magnitude=1.0, inplace=False):
    """Turns the pairs of q's and k's heads by position * inv_freq, both in one launch.

    q: [B, H_q, N, D], k: [B, H_kv, N, D] (or None) with positions [B, N] or [N]; or packed along one
    token axis, q [total, H_q, D], k [total, H_kv, D] with positions [total]. fp16/bf16, any strides;
    positions int32 or int64. inv_freq: float64 [rotary_dim / 2] on the same device, rotary_dim <= D;
    values from rotary_dim on pass unchanged. Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) with
    interleaved=True. The angle is formed in 64 bits, so far positions lose nothing.

    inverse=True turns by the negative angle: with the same magnitude, the gradient of the forward
    map. inplace=True writes into q and k themselves. Returns (q', k'); k' is None where k is.
    Asynchronous on torch's current stream.
    """
    assert q.dim() in (3, 4), "q must be [B, H, N, D] or [total, H, D]"
    assert q.dtype in (torch.float16, torch.bfloat16)
    if q.dim() == 4:
        B, H_q, N, D = q.shape
        assert positions.shape in ((B, N), (N,)), "positions must be [B, N] or [N]"
        pos_stride = (int(positions.stride(0)) if positions.dim() == 2 else 0, int(positions.stride(-1)))
    else:
        B, (N, H_q, D) = 1, q.shape
        assert positions.shape == (N,), "positions must be [total]"
        pos_stride = (0, int(positions.stride(0)))
    if k is not None:
        want = (B, k.shape[1], N, D) if q.dim() == 4 else (N, k.shape[1], D)
        assert k.dim() == q.dim() and tuple(k.shape) == want and k.dtype == q.dtype, "k must match q"
    assert positions.dtype in (torch.int32, torch.int64)
    assert inv_freq.dtype == torch.float64 and inv_freq.dim() == 1
    rd = 2 * inv_freq.numel()
    assert 2 <= rd <= D, "inv_freq must have between 1 and D / 2 entries"
    if not 0 < magnitude < 3e38:
        raise ValueError(f"magnitude must be positive and finite, got {magnitude}")
    tensors = [t for t in (q, k, positions, inv_freq) if t is not None]
    if not all(t.is_cuda for t in tensors):
        raise RuntimeError("fa2.rotary.rotary runs only on an sm_100 CUDA device (no CPU path)")
    if not all(t.device == q.device for t in tensors):
        raise RuntimeError("q, k, positions and inv_freq must be on the same CUDA device")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        raise RuntimeError("fa2.rotary.rotary is forward only: use it under torch.no_grad(); "
                           "inverse=True gives the gradient")
    if inplace:
        if _overlaps(q) or (k is not None and _overlaps(k)):
            raise ValueError("inplace needs tensors whose values do not share memory (no expanded dimensions)")
        q_out, k_out = q, k
    else:
        q_out, k_out = torch.empty_like(q), None if k is None else torch.empty_like(k)
    if q.numel() == 0:
        if k is not None and k.numel() and not inplace:
            raise ValueError("q has no values but k does")
        return q_out, k_out
    if k is not None and k.numel() == 0:
        raise ValueError("k has no heads: pass None")
    freq = inv_freq.contiguous()
    p = _kvlib.RotaryParams()
    p.q, p.q_out = q.data_ptr(), q_out.data_ptr()
    p.q_stride[:], p.q_out_stride[:] = _strides4(q), _strides4(q_out)
    if k is not None:
        p.k, p.k_out = k.data_ptr(), k_out.data_ptr()
        p.k_stride[:], p.k_out_stride[:] = _strides4(k), _strides4(k_out)
    p.positions, p.inv_freq = positions.data_ptr(), freq.data_ptr()
    p.pos_stride[:] = pos_stride
    p.pos_is_64 = int(positions.dtype == torch.int64)
    p.batch, p.seqlen, p.heads_q, p.heads_kv = B, N, H_q, 0 if k is None else k.shape[1]
    p.head_dim, p.rotary_dim = D, rd
    p.dtype = _lib.FA2_DTYPE_BF16 if q.dtype == torch.bfloat16 else _lib.FA2_DTYPE_FP16
    p.interleaved, p.inverse, p.magnitude = int(bool(interleaved)), int(bool(inverse)), float(magnitude)
    with torch.cuda.device(q.device):
        _kvlib.launch("fa2_rotary_sm100", p, torch.cuda.current_stream(q.device).cuda_stream)
    return q_out, k_out
