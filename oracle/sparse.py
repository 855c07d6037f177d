"""Key bounds, block scores, the selection and the attention over selected
blocks in plain torch and 64 bits, from their definitions.  No counterpart in
the reference.

Bounds of a block and KV head: codes floor(least / 2^e), ceil(largest / 2^e) of
every dim, e the least integer from -100 on with the largest magnitude at most
127 * 2^e; past 127 * 2^100, or with an infinity or NaN, the block is open (byte
255, codes 0) and the bounds are infinities.
"""
from __future__ import annotations

import math

import torch


def record_bytes(Hkv: int, D: int) -> int:
    return -(-Hkv * (2 * D + 1) // 16) * 16


def exponent(top: float) -> int | None:
    """None: open."""
    if not math.isfinite(top):
        return None
    for e in range(-100, 101):
        if top <= 127 * 2.0 ** e:
            return e
    return None


def key_bounds(k: torch.Tensor):
    """k [keys, Hkv, D] -> (codes int64 [Hkv, 2, D], bytes int64 [Hkv])."""
    k = k.double()
    n, Hkv, D = k.shape
    codes, byte = torch.zeros(Hkv, 2, D, dtype=torch.int64), torch.full((Hkv,), 255)
    for h in range(Hkv):
        e = exponent(float(k[:, h].abs().max()))       # a NaN's maximum is NaN
        if e is None:
            continue
        codes[h, 0] = torch.floor(k[:, h].amin(0) / 2.0 ** e).long()
        codes[h, 1] = torch.ceil(k[:, h].amax(0) / 2.0 ** e).long()
        byte[h] = e + 128
    return codes, byte


def record(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """The bytes of a record, without its padding."""
    return torch.cat([codes.reshape(-1).to(torch.int8).view(torch.uint8), byte.to(torch.uint8)])


def values(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """float64 bounds of codes [..., 2, D] and bytes [...]."""
    x = codes.double() * torch.exp2(byte.double() - 128)[..., None, None]
    open_ = torch.tensor([-math.inf, math.inf]).double()[:, None]
    return torch.where((byte == 255)[..., None, None], open_, x)


def query_codes(q: torch.Tensor) -> torch.Tensor:
    """Codes (float64) of one KV head's query heads [G, D]: ties to the even one."""
    q = q.double()
    e = exponent(float(q.abs().max()))
    return torch.zeros_like(q) if e is None else torch.round(q / 2.0 ** e)


def scores(q: torch.Tensor, codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """Scores [Hkv, blocks] of one row q [Hq, D] against bounds [blocks, Hkv, 2, D] / [blocks, Hkv]."""
    nb, Hkv = byte.shape
    out = torch.empty(Hkv, nb, dtype=torch.float64)
    for h in range(Hkv):
        c = query_codes(q.reshape(Hkv, -1, q.shape[-1])[h])
        lo, hi = codes[:, h, 0].double(), codes[:, h, 1].double()
        dot = torch.stack([torch.maximum(x * lo, x * hi).sum(-1) for x in c]).amax(0)
        out[h] = torch.where(byte[:, h] == 255, math.inf, dot * torch.exp2(byte[:, h].double() - 128))
    return out


def select(score: torch.Tensor, blocks: int, first: int, recent: int) -> list[int]:
    """The selected of len(score) visible blocks, in order."""
    nb = len(score)
    if nb <= blocks:
        return list(range(nb))
    always = [b for b in range(nb) if b < first or b >= nb - recent]
    rest = sorted((b for b in range(nb) if b not in set(always)), key=lambda b: (-float(score[b]), b))
    return sorted(always + rest[:blocks - len(always)])


def listed(selected, own: int) -> list[int]:
    """The entries of a selection that count: up to the first that is negative,
    not above the one before it, or behind the row's own block."""
    out = []
    for s in selected:
        if s < 0 or s > own or (out and s <= out[-1]):
            break
        out.append(int(s))
    return out


def keys_of(blocks: list[int], pos: int, bs: int) -> torch.Tensor:
    """The keys that a row at position pos sees of its blocks."""
    t = torch.tensor(blocks, dtype=torch.int64)[:, None] * bs + torch.arange(bs)
    t = t.reshape(-1)
    return t[t <= pos]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float):
    """Query heads q [G, D] over keys k / v [keys, D] of their KV head: the output and,
    for error bounds, sum_t p_t |v_t - o| and the largest sum |q k| scale (float64)."""
    q, k, v = q.double(), k.double(), v.double()
    if not len(k):
        z = torch.zeros_like(q)
        return z, z, torch.zeros(len(q), 1).double()
    s = (q[:, None] * k[None]).sum(-1) * scale
    p = torch.softmax(s, -1)[..., None]
    out = (p * v).sum(1)
    return out, (p * (v - out[:, None]).abs()).sum(1), (q[:, None] * k[None]).abs().sum(-1).amax(-1, keepdim=True) * scale
