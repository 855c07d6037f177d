"""Rotary positions in 64 bits from the definition, pair by pair.  The
frequency schedules restate what model configurations mean by ``rope_scaling``;
no counterpart in the reference, which ignores it."""
from __future__ import annotations

import math

import torch


def frequencies(R: int, theta: float, scaling: dict | None):
    """(radians per position of each pair, factor of cos and sin)."""
    out, m = [], 1.0
    kind = scaling["rope_type"] if scaling else None
    if kind == "yarn":
        m = scaling.get("attention_factor") or 0.1 * math.log(scaling["factor"]) + 1
    for i in range(R // 2):
        f = 1.0 / theta ** (2 * i / R)
        if kind == "linear":
            f /= scaling["factor"]
        elif kind == "llama3":
            wave, orig = 2 * math.pi / f, scaling["original_max_position_embeddings"]
            lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
            if wave > orig / lo:
                f /= scaling["factor"]
            elif wave >= orig / hi:
                t = (orig / wave - lo) / (hi - lo)
                f = (1 - t) * f / scaling["factor"] + t * f
        elif kind == "yarn":
            orig = scaling["original_max_position_embeddings"]
            first, last = (R * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(theta))
                           for n in (scaling.get("beta_fast", 32), scaling.get("beta_slow", 1)))
            first, last = max(math.floor(first), 0), min(math.ceil(last), R - 1)
            ramp = min(max((i - first) / max(last - first, 0.001), 0.0), 1.0)
            f = f / scaling["factor"] * ramp + f * (1 - ramp)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64), m


def rotate(x: torch.Tensor, pos: torch.Tensor, freq: torch.Tensor, m: float, R: int, interleaved: bool) -> torch.Tensor:
    """x [n, H, D] at positions [n] -> float64."""
    y = x.double().clone()
    a = pos.double()[:, None] * freq
    c, s = torch.cos(a) * m, torch.sin(a) * m
    for i in range(R // 2):
        d1, d2 = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        x1, x2 = x[..., d1].double(), x[..., d2].double()
        y[..., d1] = x1 * c[:, i, None] - x2 * s[:, i, None]
        y[..., d2] = x1 * s[:, i, None] + x2 * c[:, i, None]
    return y
