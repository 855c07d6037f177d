"""Batches of the windowed and 4-bit attention tests: inputs on the CPU, the
oracle's outputs and error bounds for every real row."""
from __future__ import annotations

import math

import torch

from oracle import kv4
from oracle import metadata as om
from oracle import window as ow

BF, F16, F32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


class Batch:
    """ctx / ql: lengths; kv: the cache's dtype, "4" for a 4-bit one.  Packed
    rows, or padded to `stride` rows a sequence."""

    def __init__(self, ctx, ql, Hq=8, Hkv=2, D=64, dtype=BF, kv=None, bs=16, stride=0, seed=0, scale_q=1.0):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.ql, self.L = list(ctx), list(ql), [c + q for c, q in zip(ctx, ql)]
        self.Hq, self.Hkv, self.D, self.dtype, self.bs, self.stride = Hq, Hkv, D, dtype, bs, stride
        self.kv = dtype if kv is None else kv
        nb = sum(-(-x // bs) for x in self.L) + 5
        self.nb = nb
        self.bt = torch.from_numpy(om.random_block_tables(self.L, bs, nb, g))
        self.start = [i * stride for i in range(len(ql))] if stride else [sum(ql[:i]) for i in range(len(ql))]
        rows = len(ql) * stride if stride else sum(ql)
        self.q = (torch.randn(rows, Hq, D, generator=g) * scale_q).to(dtype)
        k, v = torch.randn(nb * bs, Hkv, D, generator=g), torch.randn(nb * bs, Hkv, D, generator=g)
        if self.kv == "4":
            self.kc, self.vc = (torch.randint(0, 256, (nb, Hkv, kv4.record_bytes(bs, D)), generator=g, dtype=torch.uint8)
                                for _ in range(2))
            slots = torch.arange(nb * bs)
            for c, x in ((self.kc, k), (self.vc, v)):
                kv4.write(c, slots, x, bs)
        else:
            self.kc, self.vc = k.to(self.kv), v.to(self.kv)

    def rows(self, cache, i):
        """Sequence i's cached rows, as the model dtype reads them."""
        t = torch.arange(self.L[i])
        slots = self.bt[i, t // self.bs].long() * self.bs + t % self.bs
        x = kv4.read(cache, slots, self.bs, self.D) if self.kv == "4" else cache[slots].double()
        return x.to(self.dtype)

    def check(self, out, window, sinks, what=""):
        out = out.cpu()
        p_bits = 2.0 ** -24 if self.dtype == F32 else 0.0
        mfma = self.dtype != F32 and self.D in (64, 128) and self.kv in (self.dtype, F8, "4")
        if mfma:                               # the weights enter P V in the model dtype
            p_bits = torch.finfo(self.dtype).eps / 2
        for i, (c, n) in enumerate(zip(self.ctx, self.ql)):
            rows = slice(self.start[i], self.start[i] + n)
            scale = 1 / math.sqrt(self.D)
            ref, spread, mag = ow.attention(self.q[rows], self.rows(self.kc, i), self.rows(self.vc, i), c, window, sinks, scale)
            tol = ow.bound(ref, spread, mag, self.D, min(self.L[i], (window or self.L[i]) + sinks), self.dtype, p_bits)
            if mfma and self.dtype == F16:     # weights below 2^-14 of the largest are fp16 subnormals, 2^-25 off each
                tol = tol + self.L[i] * 2.0 ** -25 * 2 * self.rows(self.vc, i).double().abs().max()
            d = (out[rows].double() - ref).abs()
            assert torch.isfinite(out[rows]).all(), f"{what}: sequence {i} not finite"
            worst = (d / tol).max().item()
            assert worst <= 1, f"{what}: sequence {i} (ctx {c}, rows {n}): {worst:.2f} of the bound, |d| {d.max():.3e}"

    def evict(self, window, sinks):
        """Gives the blocks without a visible key to poison: their table entries
        point to a block of NaN, or outside the pool."""
        bt = self.bt.clone()
        seen = [{int(t) // self.bs for r in range(n) for t in ow.visible(c + r, window, sinks)}
                for c, n in zip(self.ctx, self.ql)]
        used = {int(bt[i, b]) for i, s in enumerate(seen) for b in s}
        spare = next(b for b in range(1, self.nb) if b not in used)
        for i, s in enumerate(seen):
            for b in range(-(-self.L[i] // self.bs)):
                if b not in s:
                    bt[i, b] = (-1, spare, 1 << 30)[b % 3]
        kc, vc = self.kc.clone(), self.vc.clone()
        for b in set(range(self.nb)) - used:   # block 0 among them, which stands in for ids outside the pool
            for c in (kc, vc):
                if self.kv == "4":
                    c[b] = 255
                else:
                    c[b * self.bs:(b + 1) * self.bs] = float("nan")
        return bt, kc, vc
