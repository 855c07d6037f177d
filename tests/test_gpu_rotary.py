"""Rotary positions with the KV write, and the rows of the 4-bit cache, against
the 64-bit oracle."""
import math

import pytest
import torch

import gllm_amd
from gllm_amd import paged
from oracle import kv4
from oracle import rope as orope
from oracle import rotary as orot
from tests.test_rotary_host import LLAMA3, SCALINGS, YARN

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _exact(x, pos, rot):
    return orot.rotate(x, pos, rot.freq.cpu(), rot.factor, rot.rotary_dim, rot.interleaved)


def _size(x, rot):
    """|x1| + |x2| of each element's pair, for the error bounds."""
    R, i = rot.rotary_dim, torch.arange(x.shape[-1])
    partner = torch.where(i >= R, i, i ^ 1 if rot.interleaved else torch.where(i < R // 2, i + R // 2, i - R // 2))
    return (x.double().abs() + x.double()[..., partner].abs()) * rot.factor


def _close(got, want, size, dtype, steps):
    """One rounding to dtype, after arithmetic off by `steps` 2^-24 of `size`."""
    info = torch.finfo(dtype)
    tol = info.eps / 2 * want.abs() * (1 + 2.0 ** -10) + steps * 2.0 ** -24 * size + info.smallest_normal * info.eps / 2
    d = (got.cpu().double() - want).abs()
    assert (d <= tol).all(), f"{(d / tol).max():.2f} of the bound"


def _inputs(n, Hq, Hkv, D, dtype, seed, pmax=100000, amp=3.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = ((torch.randn(n, h, D, generator=g) * amp).to(dtype) for h in (Hq, Hkv, Hkv))
    return q, k, v, torch.randint(0, pmax, (n,), generator=g), g


def _pool(nslots, Hkv, D, kv, bs, g):
    if kv == "4":
        return torch.randint(0, 256, (nslots // bs, Hkv, kv4.record_bytes(bs, D)), generator=g, dtype=torch.uint8)
    return torch.randn(nslots, Hkv, D, generator=g).to(kv)


def _bytes(t):
    return t.cpu().contiguous().view(torch.uint8)


SHAPES = [(128, 128, False), (128, 64, True), (64, 64, True), (64, 16, False), (256, 256, False), (96, 24, False),
          (80, 20, True), (8, 2, False), (40, 40, False)]


@pytest.mark.parametrize("D,R,inter", SHAPES)
@pytest.mark.parametrize("dtype,kv", [(BF, BF), (F16, F16), (F32, F32), (BF, F8), (F32, BF), (F16, F32)])
def test_rotary_kv_write(D, R, inter, dtype, kv):
    for n, scaling in ((1, None), (37, LLAMA3), (70, YARN)):
        print(f"rotary D={D} R={R} inter={inter} {dtype}->{kv} n={n}", flush=True)
        q, k, v, pos, g = _inputs(n, 6, 3, D, dtype, D + R + n)
        rot = gllm_amd.Rotary(D, theta=500000.0, rotary_dim=R, interleaved=inter, scaling=scaling, device=DEV)
        slots = torch.randperm(96, generator=g)[:n]
        kc, vc = _pool(96, 3, D, kv, 16, g), _pool(96, 3, D, kv, 16, g)
        dk, dv, out = kc.to(DEV), vc.to(DEV), torch.empty_like(q).to(DEV)
        paged.rotary_kv_write(k.to(DEV), v.to(DEV), pos.to(DEV), rot, dk, dv, slots.to(DEV), q=q.to(DEV), q_out=out)
        torch.cuda.synchronize()
        _close(out, _exact(q, pos, rot), _size(q, rot), dtype, 3)
        _close(dk[slots.to(DEV)].float(), _exact(k, pos, rot), _size(k, rot), kv, 2.0 ** -20)
        assert torch.equal(_bytes(dv)[slots], _bytes(v.to(kv)))
        rest = torch.ones(96, dtype=torch.bool)
        rest[slots] = False
        assert torch.equal(_bytes(dk)[rest], _bytes(kc)[rest]) and torch.equal(_bytes(dv)[rest], _bytes(vc)[rest])
        same = paged.rotary_rotate(q.to(DEV), pos.to(DEV), rot)
        assert torch.equal(_bytes(same), _bytes(out))


@pytest.mark.parametrize("scaling", SCALINGS)
def test_far_positions(scaling):
    """Angles of 10^9 radians, and positions below zero."""
    q, k, v, pos, g = _inputs(64, 2, 1, 64, F32, 3)
    pos[:20] = torch.randint(0, 2 ** 31 - 1, (20,), generator=g)
    pos[20], pos[21], pos[22], pos[23] = 2 ** 31 - 1, -1, -(2 ** 20), 0
    rot = gllm_amd.Rotary(64, theta=10000.0, scaling=scaling, device=DEV)
    out = paged.rotary_rotate(q.to(DEV), pos.to(DEV), rot)
    torch.cuda.synchronize()
    _close(out, _exact(q, pos, rot), _size(q, rot), F32, 3)
    assert torch.equal(out[23].cpu(), q[23]) or rot.factor != 1.0


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("D,R,inter,bs", [(128, 128, False, 16), (64, 32, True, 16), (256, 64, False, 3), (96, 96, True, 24),
                                          (32, 16, False, 1)])
def test_rotary_write_into_4_bits(dtype, D, R, inter, bs):
    """Codes and scales equal the oracle's from the 64-bit rotation, and the
    rest of the pool stays as it was."""
    for n in (1, 90):
        print(f"rotary 4-bit {dtype} D={D} R={R} bs={bs} n={n}", flush=True)
        q, k, v, pos, g = _inputs(n, 4, 2, D, dtype, D + n)
        k *= torch.exp2(torch.randint(-12, 12, (n, 2, 1), generator=g)).to(dtype)
        rot = gllm_amd.Rotary(D, theta=500000.0, rotary_dim=R, interleaved=inter, device=DEV)
        nslots = 10 * 24 // bs * bs
        slots = torch.randperm(nslots, generator=g)[:n]
        kc, vc = _pool(nslots, 2, D, "4", bs, g), _pool(nslots, 2, D, "4", bs, g)
        dk, dv, out = kc.to(DEV), vc.to(DEV), torch.empty_like(q).to(DEV)
        paged.rotary_kv_write(k.to(DEV), v.to(DEV), pos.to(DEV), rot, dk, dv, slots.to(DEV), q=q.to(DEV), q_out=out)
        torch.cuda.synchronize()
        kv4.write(kc, slots, _exact(k, pos, rot), bs)
        kv4.write(vc, slots, v, bs)
        assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
        _close(out, _exact(q, pos, rot), _size(q, rot), dtype, 3)
        for t in (F32, BF, F16):
            got = paged.kv4_values(dk, slots.to(DEV), D, t)
            assert torch.equal(got.cpu(), kv4.read(kc, slots, bs, D).to(t))


def test_every_bf16_value_in_4_bits():
    """All finite bf16 values in V, 32 of one magnitude range a block, and the
    blocks with an infinity or NaN."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    v = bits.view(BF).view(-1, 1, 64)                 # neighbours share a block
    g = torch.Generator().manual_seed(1)
    mixed = bits.view(BF)[torch.randperm(1 << 16, generator=g)].view(-1, 1, 64)
    v = torch.cat([v, mixed])
    n = v.shape[0]
    rot = gllm_amd.Rotary(64, device=DEV)
    dk, dv = (torch.zeros(n // 16, 1, kv4.record_bytes(16, 64), dtype=torch.uint8, device=DEV) for _ in range(2))
    slots = torch.arange(n)
    paged.rotary_kv_write(torch.zeros_like(v).to(DEV), v.to(DEV), slots.to(DEV), rot, dk, dv, slots.to(DEV))
    torch.cuda.synchronize()
    want = kv4.values(*kv4.quantize(v))
    got = kv4.read(dv.cpu(), slots, 16, 64)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(kv4.views(dv.cpu(), 16, 64)[1].flatten(), kv4.quantize(v)[1].reshape(n // 16, 1, 16, 2).flatten())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 24)])
def test_rope_kv_write_into_4_bits(dtype, D, bs):
    """Table rows: each op rounded to the model dtype, as into any other cache."""
    n = 50
    q, k, v, _, g = _inputs(n, 4, 2, D, dtype, D)
    cos_t, sin_t = orope.rope_cache(256, D, 500000.0, dtype)
    pos = torch.randint(0, 256, (n,), generator=g)
    slots = torch.randperm(240, generator=g)[:n]
    kc, vc = _pool(240, 2, D, "4", bs, g), _pool(240, 2, D, "4", bs, g)
    dk, dv, out = kc.to(DEV), vc.to(DEV), torch.empty_like(q).to(DEV)
    paged.rope_kv_write(k.to(DEV), v.to(DEV), cos_t.to(DEV), sin_t.to(DEV), dk, dv, slots.to(DEV), q=q.to(DEV), q_out=out,
                        rope_rows=pos.to(DEV))
    torch.cuda.synchronize()
    cos, sin = cos_t[pos][None], sin_t[pos][None]
    kv4.write(kc, slots, orope.apply_rope(k[None], cos, sin)[0], bs)
    kv4.write(vc, slots, v, bs)
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
    assert torch.equal(_bytes(out), _bytes(orope.apply_rope(q[None], cos, sin)[0]))


@pytest.mark.parametrize("kv", [BF, "4"])
def test_padded_rows_and_slots_outside(kv):
    """Rows past a sequence's length and slots outside the cache write nothing."""
    B, T, D = 3, 5, 64
    q, k, v, pos, g = _inputs(B * T, 4, 2, D, BF, 7)
    ql = torch.tensor([5, 0, 2], dtype=torch.int32)
    slots = torch.arange(B * T) + 3
    slots[1], slots[2] = -1, 48
    kc, vc = _pool(48, 2, D, kv, 16, g), _pool(48, 2, D, kv, 16, g)
    dk, dv = kc.to(DEV), vc.to(DEV)
    out = torch.full((B, T, 4, D), 7.0, dtype=BF, device=DEV)
    rot = gllm_amd.Rotary(D, device=DEV)
    paged.rotary_kv_write(k.view(B, T, 2, D).to(DEV), v.view(B, T, 2, D).to(DEV), pos.view(B, T).to(DEV), rot, dk, dv,
                          slots.view(B, T).to(DEV), query_lens=ql.to(DEV), q=q.view(B, T, 4, D).to(DEV), q_out=out)
    torch.cuda.synchronize()
    real = torch.tensor([r < ql[b] for b in range(B) for r in range(T)])
    wrote = real & (slots >= 0) & (slots < 48)
    if kv == "4":
        kv4.write(kc, slots[wrote], _exact(k, pos, rot)[wrote], 16)
        kv4.write(vc, slots[wrote], v[wrote], 16)
        assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
        vals = paged.kv4_values(dv, torch.tensor([-1, 48, 3]).to(DEV), D, F32).cpu()
        assert (vals[:2] == 0).all() and torch.equal(vals[2], kv4.read(vc, torch.tensor([3]), 16, D)[0].float())
    else:
        vc[slots[wrote]] = v[wrote]
        assert torch.equal(_bytes(dv), _bytes(vc))
        rest = torch.ones(48, dtype=torch.bool)
        rest[slots[wrote]] = False
        assert torch.equal(_bytes(dk)[rest], _bytes(kc)[rest])
    out = out.view(B * T, 4, D).cpu()
    assert (out[~real] == 7.0).all()
    _close(out[real], _exact(q, pos, rot)[real], _size(q, rot)[real], BF, 3)


def test_strided_rows_in_place_and_many_tokens():
    """q, k and v as slices of one projection, q rotated in place, more tokens
    than one pass of the grid's small form takes."""
    n, D = 3000, 128
    g = torch.Generator().manual_seed(9)
    x = torch.randn(n, 8, D, generator=g).to(BF).to(DEV)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    x0 = x.cpu().clone()
    rot = gllm_amd.Rotary(D, scaling=LLAMA3, device=DEV)
    pos = torch.arange(n)
    kc, vc = torch.zeros(n, 2, D, dtype=BF, device=DEV), torch.zeros(n, 2, D, dtype=BF, device=DEV)
    paged.rotary_kv_write(k, v, pos.to(DEV), rot, kc, vc, pos.to(DEV), q=q, q_out=q)
    torch.cuda.synchronize()
    _close(q, _exact(x0[:, :4], pos, rot), _size(x0[:, :4], rot), BF, 3)
    _close(kc, _exact(x0[:, 4:6], pos, rot), _size(x0[:, 4:6], rot), BF, 2.0 ** -20)
    assert torch.equal(vc.cpu(), x0[:, 6:]) and torch.equal(x[:, 4:].cpu(), x0[:, 4:])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kv", ["same", "4"])
def test_rows_at_odd_places(dtype, kv):
    """Rows that start one element off any vector's alignment, at odd strides."""
    n, D = 9, 64
    g = torch.Generator().manual_seed(4)
    flat = torch.randn(n * (6 * D + 5) + 1, generator=g).to(dtype)
    def rows(t, first, heads):
        return t.as_strided((n, heads, D), (6 * D + 5, D, 1), 1 + first * D)
    q, k, v = (rows(flat, *x) for x in ((0, 2), (2, 2), (4, 2)))
    rot = gllm_amd.Rotary(D, rotary_dim=32, device=DEV)
    pos, slots = torch.arange(n) * 31, torch.arange(n) + 7
    kc, vc = _pool(32, 2, D, dtype if kv == "same" else kv, 16, g), _pool(32, 2, D, dtype if kv == "same" else kv, 16, g)
    dflat, dk, dv = flat.to(DEV), kc.to(DEV), vc.to(DEV)
    dq, dkk, dvv = (rows(dflat, *x) for x in ((0, 2), (2, 2), (4, 2)))
    out_flat = torch.zeros_like(dflat)
    out = rows(out_flat, 0, 2)
    paged.rotary_kv_write(dkk, dvv, pos.to(DEV), rot, dk, dv, slots.to(DEV), q=dq, q_out=out)
    torch.cuda.synchronize()
    _close(out, _exact(q, pos, rot), _size(q, rot), dtype, 3)
    keep = torch.ones_like(flat, dtype=torch.bool)
    rows(keep, 0, 2)[:] = False
    assert (out_flat.cpu()[keep] == 0).all()
    if kv == "4":
        kv4.write(kc, slots, _exact(k, pos, rot), 16)
        kv4.write(vc, slots, v, 16)
        assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
    else:
        _close(dk[slots.to(DEV)], _exact(k, pos, rot), _size(k, rot), dtype, 2.0 ** -20)
        assert torch.equal(dv.cpu()[slots], v)


def test_two_streams():
    """Calls on streams of their own do not meet."""
    parts = []
    for seed in (1, 2):
        q, k, v, pos, g = _inputs(500, 4, 2, 128, BF, seed)
        parts.append((q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV)))
    rot = gllm_amd.Rotary(128, device=DEV)
    slots = torch.arange(500, device=DEV)

    def pools():
        return [torch.zeros(32, 2, kv4.record_bytes(16, 128), dtype=torch.uint8, device=DEV) for _ in range(4)]
    want, got = pools(), pools()
    for i, (q, k, v, pos) in enumerate(parts):
        paged.rotary_kv_write(k, v, pos, rot, want[2 * i], want[2 * i + 1], slots)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in parts]
    for _ in range(5):
        for i, ((q, k, v, pos), st) in enumerate(zip(parts, streams)):
            with torch.cuda.stream(st):
                paged.rotary_kv_write(k, v, pos, rot, got[2 * i], got[2 * i + 1], slots)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_infinities_stay_in_their_block():
    q, k, v, pos, g = _inputs(4, 2, 2, 128, BF, 5)
    k[0, 1, 3], v[1, 0, 40], v[2, 1, 100] = math.inf, math.nan, -math.inf
    rot = gllm_amd.Rotary(128, rotary_dim=64, device=DEV)
    dk, dv = (torch.zeros(1, 2, kv4.record_bytes(16, 128), dtype=torch.uint8, device=DEV) for _ in range(2))
    slots = torch.arange(4).to(DEV)
    paged.rotary_kv_write(k.to(DEV), v.to(DEV), pos.to(DEV), rot, dk, dv, slots)
    kk, vv = (paged.kv4_values(c, slots, 128, F32).cpu() for c in (dk, dv))
    nan = torch.zeros(4, 2, 128, dtype=torch.bool)
    nan[0, 1, :64] = True                     # dims 3 and 35 turn together: both their blocks
    assert torch.equal(kk.isnan(), nan)
    nan[:] = False
    nan[1, 0, 32:64] = nan[2, 1, 96:] = True
    assert torch.equal(vv.isnan(), nan)


@pytest.mark.parametrize("kv", [BF, "4"])
def test_graph_replays(kv):
    q, k, v, pos, g = (x.to(DEV) if torch.is_tensor(x) else x for x in _inputs(20, 4, 2, 64, BF, 6))
    rot = gllm_amd.Rotary(64, device=DEV)
    slots = torch.arange(20, device=DEV) + 5
    kc, vc = _pool(48, 2, 64, kv, 16, g).to(DEV), _pool(48, 2, 64, kv, 16, g).to(DEV)
    out = torch.empty_like(q)
    args = (k, v, pos, rot, kc, vc, slots)
    paged.rotary_kv_write(*args, q=q, q_out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.rotary_kv_write(*args, q=q, q_out=out)
    for i in range(3):
        pos.add_(17)
        k.mul_(-1.5)
        want, k2, v2 = torch.empty_like(q), kc.clone(), vc.clone()
        paged.rotary_kv_write(k, v, pos, rot, k2, v2, slots, q=q, q_out=want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(_bytes(kc), _bytes(k2)) and torch.equal(_bytes(vc), _bytes(v2))


@pytest.mark.parametrize("table", [False, True])
def test_every_fp16_value_in_4_bits(table):
    """All finite fp16 values, neighbours and mixed: rows read in fp16 are finite,
    blocks with an infinity or NaN stay NaN."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    x = bits.view(F16).view(-1, 1, 64)
    g = torch.Generator().manual_seed(1)
    x = torch.cat([x, bits.view(F16)[torch.randperm(1 << 16, generator=g)].view(-1, 1, 64),
                   bits.view(F16).nan_to_num(1.0, 2.0, 3.0)[torch.randperm(1 << 16, generator=g)].view(-1, 1, 64)])
    n = x.shape[0]
    rot = gllm_amd.Rotary(64, device=DEV)
    kc, vc = (torch.zeros(n // 16, 1, kv4.record_bytes(16, 64), dtype=torch.uint8) for _ in range(2))
    dk, dv, slots = kc.to(DEV), vc.to(DEV), torch.arange(n)
    k = x.nan_to_num(1.0, 2.0, 3.0)              # position 0 keeps finite values; NaN would reach its partner
    if table:
        cos, sin = torch.ones(n, 32, dtype=F16, device=DEV), torch.zeros(n, 32, dtype=F16, device=DEV)
        paged.rope_kv_write(k.to(DEV), x.to(DEV), cos, sin, dk, dv, slots.to(DEV))
    else:
        paged.rotary_kv_write(k.to(DEV), x.to(DEV), torch.zeros_like(slots).to(DEV), rot, dk, dv, slots.to(DEV))
    torch.cuda.synchronize()
    for dev, host, rows in ((dk, kc, k), (dv, vc, x)):
        kv4.write(host, slots, rows, 16, F16)
        want = kv4.read(host, slots, 16, 64)
        assert torch.equal(kv4.views(dev.cpu(), 16, 64)[1], kv4.views(host, 16, 64)[1])
        got = kv4.read(dev.cpu(), slots, 16, 64)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
        half = paged.kv4_values(dev, slots.to(DEV), 64, F16).cpu()
        assert torch.equal(half.isnan(), want.isnan()) and torch.equal(half.nan_to_num(7.0), want.to(F16).nan_to_num(7.0))
        assert not half.isinf().any()
    assert not kv4.read(dk.cpu(), slots, 16, 64).isnan().any()


def test_turned_fp16_rows_past_the_largest_value():
    """k rows that the rotation takes past 65,504 are limited, not infinite."""
    g = torch.Generator().manual_seed(3)
    k = ((torch.rand(64, 2, 128, generator=g) - 0.5) * 2 * 65504).to(F16)
    rot = gllm_amd.Rotary(128, scaling=YARN, device=DEV)
    pos = torch.randint(0, 100000, (64,), generator=g)
    kc, vc = (torch.zeros(4, 2, kv4.record_bytes(16, 128), dtype=torch.uint8) for _ in range(2))
    dk, dv, slots = kc.to(DEV), vc.to(DEV), torch.randperm(64, generator=g)
    paged.rotary_kv_write(k.to(DEV), k.to(DEV), pos.to(DEV), rot, dk, dv, slots.to(DEV))
    torch.cuda.synchronize()
    want = _exact(k, pos, rot)
    assert want.abs().max() > 65536
    kv4.write(kc, slots, want, 16, F16)
    kv4.write(vc, slots, k, 16, F16)
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
    assert paged.kv4_values(dk, slots.to(DEV), 128, F16).isfinite().all()
