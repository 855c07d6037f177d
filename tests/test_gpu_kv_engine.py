"""The later operators together, as an engine uses them: rotary positions into
a 4-bit cache that windowed attention reads, over many steps with blocks given
back, and the Attention layer with a window and a 4-bit pool."""
import math

import pytest
import torch
import torch.nn.functional as F

import gllm_amd
from gllm_amd import paged
from oracle import kv4
from oracle import rope as orope
from oracle import rotary as orot
from oracle import window as ow

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.mark.parametrize("D,window,sinks", [(64, 40, 3), (128, 33, 0), (128, None, 0)])
def test_prompt_then_decode(D, window, sinks):
    """Three sequences: a prompt chunk each, then decode steps; blocks that the
    window has left go back to the pool and are written by another sequence."""
    Hq, Hkv, bs, steps, B = 8, 2, 8, 24, 3
    g = torch.Generator().manual_seed(D)
    rot = gllm_amd.Rotary(D, theta=500000.0, rotary_dim=D // 2, interleaved=True, device=DEV,
                          scaling={"rope_type": "linear", "factor": 2.0})
    lens = [70, 5, 33]
    nb = 40
    cache = gllm_amd.PagedKVCache(1, Hkv, D, bs, 1, nb * bs, paged.KV4, DEV)
    assert cache.num_blocks == nb
    kc, vc = cache.get_layer_kv_cache(0)
    free, bt = list(range(nb - 1, 0, -1)), torch.zeros(B, 16, dtype=torch.int32)
    ks, vs = [torch.zeros(0, Hkv, D, dtype=torch.float64) for _ in range(B)], [torch.zeros(0, Hkv, D, dtype=torch.float64) for _ in range(B)]
    held, reused = [{} for _ in range(B)], 0
    given = set()
    ctx = [0] * B
    for step in range(steps):
        ql = lens if step == 0 else [1, 3, 1]
        rows = sum(ql)
        q, k, v = (torch.randn(rows, h, D, generator=g).to(BF) for h in (Hq, Hkv, Hkv))
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, ql)])
        slots = []
        for i, (c, n) in enumerate(zip(ctx, ql)):
            for b in range(-(-(c + n) // bs)):
                if b not in held[i] and b * bs + bs > c:
                    held[i][b] = free.pop()
                    reused += held[i][b] in given
                    bt[i, b] = held[i][b]
            slots += [held[i][p // bs] * bs + p % bs for p in range(c, c + n)]
        qr = torch.empty(rows, Hq, D, dtype=BF, device=DEV)
        paged.rotary_kv_write(k.to(DEV), v.to(DEV), pos.to(DEV), rot, kc, vc, torch.tensor(slots, device=DEV), q=q.to(DEV), q_out=qr)
        plan = paged.AttentionPlan(ql, [c + n for c, n in zip(ctx, ql)], num_q_heads=Hq, num_kv_heads=Hkv, head_dim=D,
                                   block_size=bs, dtype=BF, device=DEV, window=window, sinks=sinks)
        out = paged.paged_attention(plan, qr, kc, vc, bt.to(DEV)).cpu()
        kr = kv4.values(*kv4.quantize(orot.rotate(k, pos, rot.freq.cpu(), rot.factor, rot.rotary_dim, True)))
        vr = kv4.values(*kv4.quantize(v))
        at = 0
        for i, (c, n) in enumerate(zip(ctx, ql)):
            ks[i], vs[i] = torch.cat([ks[i], kr[at:at + n]]), torch.cat([vs[i], vr[at:at + n]])
            ref, spread, mag = ow.attention(qr[at:at + n].cpu(), ks[i], vs[i], c, window, sinks, 1 / math.sqrt(D))
            tol = ow.bound(ref, spread, mag, D, c + n, BF, torch.finfo(BF).eps / 2)
            assert ((out[at:at + n].double() - ref).abs() <= tol).all(), f"step {step}, sequence {i}"
            at += n
            ctx[i] = c + n
            if window is not None:              # the next row sees from ctx + 1 - window on
                for b in [b for b in held[i] if (b + 1) * bs <= ctx[i] + 1 - window and b * bs >= sinks]:
                    free.insert(0, held[i][b])
                    free.append(free.pop(0))    # the next block to be taken
                    given.add(held[i].pop(b))
    assert (reused > 0) == (window is not None)


def _layer(window, sinks, kv, Hq=8, Hkv=2, D=64, B=5, Tq=1, bs=16):
    g = torch.Generator().manual_seed(7)
    hid = Hq * D
    L = [Tq, 30 + Tq, 100, 257, 64]
    need = [-(-x // bs) for x in L]
    nb = sum(need) + 1
    perm = torch.randperm(nb - 1, generator=g).int() + 1
    bt, o = torch.zeros(B, max(need), dtype=torch.int32), 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[o:o + n]
        o += n
    pos = torch.tensor([[x - Tq + r for r in range(Tq)] for x in L])
    slots = torch.gather(bt.long(), 1, pos // bs) * bs + pos % bs

    class Cfg:
        num_attn_heads, num_kv_heads, head_dim, hidden_size, dtype = Hq, Hkv, D, hid, BF
    w = {f"model.layers.0.self_attn.{n}_proj.weight": (torch.randn(r, hid, generator=g) / hid ** 0.5).to(BF).to(DEV)
         for n, r in (("q", hid), ("k", Hkv * D), ("v", Hkv * D), ("o", hid))}
    meta = gllm_amd.AttentionMetadata(torch.full((B,), Tq, dtype=torch.int32, device=DEV),
                                      torch.tensor(L, dtype=torch.int32, device=DEV), max(L), bt.to(DEV), None,
                                      slots.to(DEV), None, bs)
    rows = torch.randn(2, nb * bs, Hkv, D, generator=g).to(BF)
    if kv == paged.KV4:
        pool = torch.zeros(2, nb, Hkv, kv4.record_bytes(bs, D), dtype=torch.uint8)
        for i in range(2):
            kv4.write(pool[i], torch.arange(nb * bs), rows[i], bs)
            rows[i] = kv4.read(pool[i], torch.arange(nb * bs), bs, D).to(BF)
    else:
        pool = rows.clone()
    cos, sin = orope.rope_cache(512, D, 500000.0, BF)
    x = torch.randn(B, Tq, hid, generator=g).to(BF).to(DEV)
    att = gllm_amd.Attention(0, Cfg, w, window=window, sinks=sinks)
    return att, x, cos[pos], sin[pos], pool.to(DEV), meta, rows, L, bt, slots


@pytest.mark.parametrize("Tq", [1, 20])
@pytest.mark.parametrize("kv,window,sinks", [(paged.KV4, None, 0), (paged.KV4, 50, 2), (BF, 50, 2)])
def test_attention_layer(Tq, kv, window, sinks):
    att, x, cos, sin, pool, meta, rows, L, bt, slots = _layer(window, sinks, kv, Tq=Tq)
    Hq, Hkv, D, bs = 8, 2, 64, 16
    q, k, v = (F.linear(x, w).view(5, Tq, h, D).cpu() for w, h in ((att.W_q, Hq), (att.W_k, Hkv), (att.W_v, Hkv)))
    got = att.attention(q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), pool, meta).cpu()
    q, k = orope.apply_rope(q, cos, sin), orope.apply_rope(k, cos, sin)
    if kv == paged.KV4:
        k, v = (kv4.values(*kv4.quantize(t)).to(BF) for t in (k, v))
    rows[0][slots.flatten()], rows[1][slots.flatten()] = k.flatten(0, 1), v.flatten(0, 1)
    for i in range(5):
        t = torch.arange(L[i])
        s = bt[i, t // bs].long() * bs + t % bs
        ref, spread, mag = ow.attention(q[i], rows[0][s], rows[1][s], L[i] - Tq, window, sinks, 1 / math.sqrt(D))
        tol = ow.bound(ref, spread, mag, D, L[i], BF, torch.finfo(BF).eps / 2)
        assert ((got[i].double() - ref).abs() <= tol).all(), f"sequence {i}"
    # forward: the same layer with its projections (for bf16 caches possibly fused)
    out = att.forward(x, cos.to(DEV), sin.to(DEV), pool, meta)
    want = F.linear(got.to(DEV).view(5, Tq, -1), att.W_o)
    assert (out.float() - want.float()).abs().max() <= 0.05


def test_layers_with_and_without_a_window_share_a_step():
    """Each window has its own plan on the step's metadata."""
    a, x, cos, sin, pool, meta, *_ = _layer(50, 2, BF)
    b = _layer(None, 0, BF)[0]
    c = _layer(50, 0, BF)[0]
    cs = (cos.to(DEV), sin.to(DEV))
    first = [t.forward(x, *cs, pool, meta) for t in (a, b, c)]
    again = [t.forward(x, *cs, pool, meta) for t in (a, b, c)]
    fresh = [t.forward(x, *cs, pool, _layer(None, 0, BF)[5]) for t in (a, b, c)]
    for f, g, h in zip(first, again, fresh):
        assert torch.equal(f, g) and torch.equal(f, h)
    assert not torch.equal(first[0], first[1]) and not torch.equal(first[0], first[2])
