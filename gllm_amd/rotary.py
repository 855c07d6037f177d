"""Rotary positions of a model: which dims of a head turn, how they pair up and
by how much per position, scaled for long contexts.

The reference turns half pairs over the whole head at one theta
(``gllm/model/layers/attention.py:76-119``, ``gllm/model/model.py:117-128``) and
ignores a configuration's ``rope_scaling``; this is for models that it does not
cover.  ``paged.rotary_kv_write`` and ``paged.rotary_rotate`` take it.
"""
from __future__ import annotations

import math

import torch


def _need(scaling: dict, key: str) -> float:
    try:
        x = float(scaling[key])
    except (KeyError, TypeError, ValueError):
        raise ValueError(f"rope scaling {scaling!r} needs a number {key!r}") from None
    if not math.isfinite(x) or x <= 0:
        raise ValueError(f"rope scaling {scaling!r}: {key} must be positive")
    return x


class Rotary:
    """``theta``: the base of the frequencies theta^(-2i / rotary_dim).
    ``rotary_dim``: the first dims of the head that turn (None: all of them).
    ``interleaved``: pairs (2i, 2i + 1) instead of (i, i + rotary_dim / 2).
    ``scaling``: None or a model configuration's ``rope_scaling`` (a ``rope_theta``
    or ``partial_rotary_factor`` in it has to agree with the arguments):

    - ``default``: unscaled;
    - ``linear``: positions divided by ``factor``;
    - ``llama3``: pairs that make fewer than ``low_freq_factor`` turns over
      ``original_max_position_embeddings`` positions are divided by ``factor``,
      those that make more than ``high_freq_factor`` are kept, in between both
      are blended;
    - ``yarn``: the same by pair index between ``beta_slow`` (1) and ``beta_fast``
      (32) turns, and cos and sin times ``attention_factor`` (0.1 ln factor + 1);
      ``mscale``, ``mscale_all_dim`` and ``truncate=False`` are refused.

    ``freq``: radians per position of each pair, float64 on ``device``;
    ``factor``: of cos and sin.
    """

    def __init__(self, head_dim: int, *, theta: float = 10000.0, rotary_dim: int | None = None,
                 interleaved: bool = False, scaling: dict | None = None, device="cuda"):
        R = head_dim if rotary_dim is None else rotary_dim
        if head_dim <= 0 or not 0 < R <= head_dim or R % 2:
            raise ValueError(f"rotary_dim {R} must be even, positive and at most head_dim {head_dim}")
        if not (math.isfinite(theta) and theta > 0):
            raise ValueError(f"theta {theta} must be positive")
        self.head_dim, self.rotary_dim, self.interleaved, self.factor = head_dim, R, bool(interleaved), 1.0
        self.freq = self._scaled(theta ** (-2 * torch.arange(R // 2, dtype=torch.float64) / R), theta, scaling).to(device)

    def _scaled(self, base: torch.Tensor, theta: float, scaling: dict | None) -> torch.Tensor:
        if scaling is None:
            return base
        kind = scaling.get("rope_type", scaling.get("type"))
        if kind is None:
            raise ValueError(f"rope scaling {scaling!r} names no rope_type")
        if kind not in ("default", "linear", "llama3", "yarn"):
            raise NotImplementedError(f"rope scaling {kind!r} (default, linear, llama3, yarn)")
        part = scaling.get("partial_rotary_factor")
        if scaling.get("rope_theta", theta) != theta or part is not None and int(self.head_dim * part) != self.rotary_dim:
            raise ValueError(f"rope scaling {scaling!r}: not the theta {theta}, rotary_dim {self.rotary_dim} given")
        if kind == "default":
            return base
        f = _need(scaling, "factor")
        if kind == "linear":
            return base / f
        orig = _need(scaling, "original_max_position_embeddings")
        if kind == "llama3":
            lo, hi = _need(scaling, "low_freq_factor"), _need(scaling, "high_freq_factor")
            if hi <= lo:
                raise ValueError(f"rope scaling {scaling!r}: high_freq_factor must exceed low_freq_factor")
            keep = ((orig * base / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
        else:
            R = self.rotary_dim
            if scaling.get("mscale") or scaling.get("mscale_all_dim") or scaling.get("truncate") is False:
                raise NotImplementedError(f"rope scaling {scaling!r}: mscale, mscale_all_dim and truncate=False")
            def index(turns: float) -> float:          # the pair that makes so many turns
                return R * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
            if theta <= 1:
                raise ValueError(f"yarn needs a theta above 1, got {theta}")
            fast, slow = (_need(scaling, k) if scaling.get(k) is not None else d
                          for k, d in (("beta_fast", 32.0), ("beta_slow", 1.0)))
            lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), R - 1)
            keep = 1 - ((torch.arange(R // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
            self.factor = _need(scaling, "attention_factor") if scaling.get("attention_factor") is not None \
                else 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
        return base * (keep + (1 - keep) / f)

    def tables(self, positions: int, dtype: torch.dtype):
        """cos and sin rows ``[positions, rotary_dim / 2]`` in ``dtype`` for the
        entry points that take tables (``rope_kv_write``, ``paged_attention``'s
        ``rope``, ``Attention.forward``), which turn half pairs of whole heads."""
        if self.interleaved or self.rotary_dim != self.head_dim:
            raise ValueError("tables serve half pairs over the whole head; use paged.rotary_kv_write")
        a = torch.arange(positions, dtype=torch.float64, device=self.freq.device)[:, None] * self.freq
        return (torch.cos(a) * self.factor).to(dtype), (torch.sin(a) * self.factor).to(dtype)
