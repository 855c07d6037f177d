"""The 4-bit KV cache's format in plain torch: each block of 32 dims as fp4 e2m1
codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit) times 2^e, e the least integer
with amax < 7 * 2^e (between -126 and 127); a block with an infinity or NaN has
the scale byte 255 and stands for NaN.  Finite values of an fp16 model stop at
6 * 2^13: the next larger value that a block can stand for, 4 * 2^14, is past
fp16's largest.  No counterpart in the reference."""
from __future__ import annotations

import torch

CODES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                     dtype=torch.float64)


def record_bytes(bs: int, D: int) -> int:
    return -(-bs * (D // 2 + D // 32) // 16) * 16


def quantize(x: torch.Tensor, model: torch.dtype | None = None):
    """x [..., D] of a model of dtype `model` -> (codes uint8 [..., D], scale bytes
    uint8 [..., D / 32])."""
    b = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(b).all(-1)
    if model == torch.float16:
        b = b.clamp(-6.0 * 2 ** 13, 6.0 * 2 ** 13)
    b = torch.where(bad[..., None], torch.zeros_like(b), b)
    amax = b.abs().amax(-1)
    e = torch.full(amax.shape, -126, dtype=torch.int64)
    for i in range(-126, 128):                 # the least e that holds the block
        e = torch.where(amax >= 7 * 2.0 ** (i - 1), torch.maximum(e, torch.tensor(i)), e)
    y = b / torch.exp2(e.double())[..., None]
    # nearest code; between two codes the even one
    d = (y.abs()[..., None] - CODES[:8]).abs()
    best = d.amin(-1, keepdim=True)
    even = (d == best) & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.double().argmax(-1), (d == best).double().argmax(-1))
    code = (code + 8 * torch.signbit(y)).to(torch.uint8)
    byte = torch.where(bad, 255, e + 127).to(torch.uint8)
    return code.flatten(-2), byte


def values(code: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """The float64 values that codes [..., D] and scale bytes [..., D / 32] stand for."""
    s = torch.where(byte == 255, float("nan"), torch.exp2(byte.double() - 127))
    return (CODES[code.long()].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def views(cache: torch.Tensor, bs: int, D: int):
    """Code bytes [NB, Hkv, bs, D / 2] and scale bytes [NB, Hkv, bs, D / 32] of a cache."""
    n = bs * D // 2
    return cache[..., :n].unflatten(-1, (bs, D // 2)), cache[..., n:n + bs * D // 32].unflatten(-1, (bs, D // 32))


def write(cache: torch.Tensor, slots: torch.Tensor, x: torch.Tensor, bs: int, model: torch.dtype | None = None) -> None:
    """Rows x [n, Hkv, D] into their slots of a CPU cache."""
    code, byte = quantize(x, model)
    c, s = views(cache, bs, x.shape[-1])
    c[slots // bs, :, slots % bs] = code[..., 0::2] + 16 * code[..., 1::2]
    s[slots // bs, :, slots % bs] = byte


def read(cache: torch.Tensor, slots: torch.Tensor, bs: int, D: int) -> torch.Tensor:
    """float64 rows [n, Hkv, D] of a CPU cache."""
    c, s = views(cache, bs, D)
    b = c[slots // bs, :, slots % bs]
    return values(torch.stack([b % 16, b // 16], -1).flatten(-2), s[slots // bs, :, slots % bs])
