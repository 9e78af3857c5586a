"""Plain 64-bit forms of the serving operators (rotary positions, the 8-bit paged K/V cache and its
attention), written from their definitions for the tests. Loops over sequences and heads on purpose.
"""

import math

import torch

E4M3_MAX = 448.0


def rotary(x, positions, inv_freq, interleaved=False, inverse=False, magnitude=1.0):
    """x [B, H, N, D] with positions [B, N] or [N], or [total, H, D] with [total]; returns float64."""
    rd = 2 * inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()  # [..., N, rd / 2]
    if inverse:
        angle = -angle
    cos, sin = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    if x.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    elif cos.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    y = x.double().clone()
    first = torch.arange(rd // 2, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else rd // 2)
    a, c = x.double()[..., first], x.double()[..., second]
    y[..., first] = a * cos - c * sin
    y[..., second] = a * sin + c * cos
    return y


def quantise(x):
    """Rows [..., D] -> (code values as float32, scales float32), in the 32-bit arithmetic of the
    definition: scale = max|x| / 448, code = e4m3(x / scale)."""
    x = x.float()
    top = x.abs().amax(-1)
    # A tensor divisor: division by a number is a product with its rounded reciprocal on a GPU.
    scale = torch.where(torch.isfinite(top), top / torch.full_like(top, E4M3_MAX), torch.full_like(top, math.nan))
    some = scale > 0
    q = torch.where(some[..., None], x / scale[..., None], torch.zeros_like(x)).clamp(-E4M3_MAX, E4M3_MAX)
    return q.to(torch.float8_e4m3fn).float(), scale


def rows_of(codes, scales, block_table, b, n):
    """The first n rows of sequence b as float64 [n, H, D]."""
    ps = codes.shape[1]
    pages = block_table[b, : -(-n // ps)].long()
    c = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
    x = c * scales[pages].double()[..., None]
    return x.reshape(-1, *codes.shape[2:])[:n]


def attention(q, cache, block_table, cache_seqlens, causal=True, sm_scale=None, causal_align="bottom_right",
              cu_seqlens_q=None):
    """Returns (out, weight, spread, small): out as the operator defines it, weight = sum_j p_ij |v_j| /
    sum_j p_ij (the same average of the magnitudes, for error bounds), spread [.., H] the largest sum_d
    |q_d k_d| * sm_scale of a row and small [.., H] the largest max_d |q_d| * sum_d |k_d| * sm_scale, all
    float64."""
    k, v, ks, vs = cache
    D = q.shape[-1]
    sm_scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    group = q.shape[1] // k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    spread, small = (torch.zeros(q.shape[:-1], dtype=torch.float64, device=q.device) for _ in range(2))
    lens = [int(n) for n in cache_seqlens.tolist()]
    cu = [int(n) for n in cu_seqlens_q.tolist()] if cu_seqlens_q is not None else None
    for b, n in enumerate(lens):
        rows = slice(cu[b], cu[b + 1]) if cu is not None else None
        qs = q[rows].transpose(0, 1).double() if cu is not None else q[b].double()  # [H_q, n_q, D]
        n_q = qs.shape[1]
        if n == 0 or n_q == 0:
            continue
        keys, vals = rows_of(k, ks, block_table, b, n), rows_of(v, vs, block_table, b, n)
        sees = torch.ones(n_q, n, dtype=torch.bool, device=q.device)
        if causal:
            sees = sees.tril(n - n_q if causal_align == "bottom_right" else 0)
        for h in range(q.shape[1]):
            s = qs[h] @ keys[:, h // group].T * sm_scale
            s = s.masked_fill(~sees, -math.inf)
            p = torch.softmax(s, -1)
            p = torch.where(sees, p, torch.zeros_like(p))  # a row that sees nothing: zeros, not NaN
            val = vals[:, h // group]
            # A key that a row does not see has no part in it, whatever it holds.
            o = torch.stack([p[i, sees[i]] @ val[sees[i]] for i in range(n_q)]) if not torch.isfinite(val).all() else p @ val
            w = p @ val.abs()
            a = (qs[h].abs() @ keys[:, h // group].abs().T * sm_scale).masked_fill(~sees, 0).amax(-1)
            e = qs[h].abs().amax(-1) * keys[:, h // group].abs().sum(-1).amax() * sm_scale
            at = (rows, h) if cu is not None else (b, h)
            out[at], weight[at], spread[at], small[at] = o, w, a, e
    return out, weight, spread, small
