"""Paged attention with a sliding window and sinks in 64 bits, row by row from
the definition: key t is visible to the row at position p iff t <= p and
(t > p - window or t < sinks).  No counterpart in the reference."""
from __future__ import annotations

import torch


def visible(p: int, window: int | None, sinks: int) -> torch.Tensor:
    """Keys that the row at position p sees, in order."""
    if window is None:
        return torch.arange(p + 1)
    first = max(0, p + 1 - window)
    return torch.cat([torch.arange(min(sinks, first)), torch.arange(first, p + 1)])


def attention(q, k, v, ctx: int, window: int | None, sinks: int, scale: float):
    """One sequence: q [rows, Hq, D], k / v [keys, Hkv, D] (any dtype, exact
    values), rows at positions ctx, ctx + 1, ...  Returns the output and, for
    error bounds, sum_t p_t |v_t - o| and the largest sum |q k| scale of a row,
    all float64 [rows, Hq, D] (the last [rows, Hq, 1])."""
    rows, Hq, D = q.shape
    Hkv = k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out, spread, mag = torch.empty(rows, Hq, D).double(), torch.empty(rows, Hq, D).double(), torch.empty(rows, Hq, 1).double()
    for r in range(rows):
        t = visible(ctx + r, window, sinks)
        kt = k[t].repeat_interleave(Hq // Hkv, 1).transpose(0, 1)      # [Hq, n, D]
        vt = v[t].repeat_interleave(Hq // Hkv, 1).transpose(0, 1)
        s = (kt * q[r][:, None]).sum(-1) * scale
        p = torch.softmax(s, -1)[..., None]
        out[r] = (p * vt).sum(1)
        spread[r] = (p * (vt - out[r][:, None]).abs()).sum(1)
        mag[r] = (kt * q[r][:, None]).abs().sum(-1).amax(-1, keepdim=True) * scale
    return out, spread, mag


def bound(out, spread, mag, D: int, keys: int, dtype: torch.dtype, p_bits: float = 0.0):
    """How far the kernels' result may be from the 64-bit one.  A relative
    error e of every weight moves the output by at most e / (1 - e) spread
    (numerator and denominator share the weights).  e: the scores' fp32 sums
    (D + 2 roundings of sum |q k| scale), exp2 and its argument (4 ulp of a score
    in log2 units), the weights' own rounding `p_bits`; then the fp32 sums over
    the keys (weights are positive, so keys * 2^-24 of sum p |v| <= spread + |o|)
    and the output's rounding."""
    u = 2.0 ** -24
    e = (D + 2) * u * mag + 6 * u * (1 + mag) + p_bits
    return e / (1 - e).clamp_min(0.1) * spread + (keys + 8) * u * (spread + out.abs()) + torch.finfo(dtype).eps / 2 * out.abs() \
        + torch.finfo(dtype).smallest_normal
