"""Paged attention over a 4-bit KV cache against the 64-bit oracle on the values
that the cache stands for."""
import pytest
import torch

import gllm_amd
from gllm_amd import paged
from oracle import kv4
from oracle import rope as orope
from oracle import window as ow
from tests.window_helpers import BF, F8, F16, F32, Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DECODE = dict(ctx=[0, 3, 15, 16, 40, 299, 1000, 2500], ql=[1] * 8)


def _plan(b, window=None, sinks=0, **kw):
    return paged.AttentionPlan(b.ql, b.L, num_q_heads=b.Hq, num_kv_heads=b.Hkv, head_dim=b.D, block_size=b.bs,
                               dtype=b.dtype, device=DEV, q_seq_stride=b.stride, window=window, sinks=sinks, **kw)


def _run(b, window=None, sinks=0, bt=None, kc=None, vc=None, rope=None, **kw):
    bt, kc, vc = (x.to(DEV) for x in (b.bt if bt is None else bt, b.kc if kc is None else kc, b.vc if vc is None else vc))
    out = paged.paged_attention(_plan(b, window, sinks, **kw), b.q.to(DEV), kc, vc, bt, rope=rope)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("split", [0, 64, paged.BALANCED])
def test_decode(dtype, D, split):
    for bs in (16, 1, 24, 7):
        print(f"kv4 decode {dtype} D={D} split={split} bs={bs}", flush=True)
        b = Batch(**DECODE, D=D, dtype=dtype, kv="4", bs=bs, seed=D + bs)
        b.check(_run(b, split_tokens=split), None, 0, "kv4 decode")


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 1), (6, 3), (32, 8)])
def test_rows_and_heads(Hq, Hkv):
    n = min(4, 16 // (Hq // Hkv))
    for D in (64, 128):
        b = Batch([0, 14, 130, 777, 1500], [1, n, 1, n, n], Hq=Hq, Hkv=Hkv, D=D, kv="4", stride=5, seed=Hq)
        b.check(_run(b), None, 0, "kv4 rows")


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (128, 24), (64, 5)])
def test_prefill_and_mixed(dtype, D, bs):
    for ctx, ql in (([0, 0, 37, 1000], [33, 200, 77, 130]), ([300, 0, 57, 1000, 5, 2500], [1, 120, 64, 1, 1, 1])):
        print(f"kv4 prefill / mixed {dtype} D={D} bs={bs}", flush=True)
        b = Batch(ctx, ql, D=D, dtype=dtype, kv="4", bs=bs, seed=D + bs)
        b.check(_run(b), None, 0, "kv4 prefill")
        if dtype == BF:
            b.check(_run(b, split_tokens=paged.BALANCED), None, 0, "kv4 mixed, balanced")


@pytest.mark.parametrize("window,sinks", [(1, 0), (17, 4), (129, 20), (600, 64)])
@pytest.mark.parametrize("D", [64, 128])
def test_windows(D, window, sinks):
    for ctx, ql in ((DECODE["ctx"], DECODE["ql"]), ([0, 37, 1000, 700], [150, 77, 64, 1])):
        print(f"kv4 window={window} sinks={sinks} D={D}", flush=True)
        b = Batch(ctx, ql, D=D, kv="4", seed=window + D)
        want = _run(b, window, sinks)
        b.check(want, window, sinks, "kv4 window")
        assert torch.equal(_run(b, window, sinks, *b.evict(window, sinks)), want)


@pytest.mark.parametrize("D", [64, 128])
def test_rope_on_load(D):
    b = Batch([0, 300, 20], [1, 1, 50], D=D, kv="4", seed=D)
    cos, sin = orope.rope_cache(512, D, 500000.0, BF)
    pos = torch.cat([torch.arange(c, c + n) for c, n in zip(b.ctx, b.ql)])
    out = _run(b, rope=(cos.to(DEV), sin.to(DEV), "position"))
    b.q = orope.apply_rope(b.q[None], cos[pos][None], sin[pos][None])[0]
    b.check(out, None, 0, "kv4 rope")


def test_scales_from_end_to_end():
    """Scale bytes across their range of finite scores; a NaN block reaches its
    own head's rows only."""
    b = Batch([100, 40], [1, 1], D=128, kv="4", seed=4)
    codes, scales = kv4.views(b.vc, b.bs, 128)
    g = torch.Generator().manual_seed(1)
    scales[:] = torch.randint(1, 230, scales.shape, generator=g, dtype=torch.uint8)
    b.check(_run(b), None, 0, "kv4 scales")
    slot = int(b.bt[0, 2])
    scales[slot, 1, 5, 2] = 255                       # dims 64..95 of key 37, KV head 1
    out = _run(b).float().cpu()
    nan = torch.zeros(2, 8, 128, dtype=torch.bool)
    nan[0, 4:, 64:96] = True
    assert torch.equal(out.isnan(), nan)


def test_strided_blocks_and_view():
    """K and V as the halves of one pool, as an engine keeps them."""
    b = Batch(**DECODE, D=64, kv="4", seed=6)
    pool = torch.stack([b.kc, b.vc], 1).to(DEV)       # [NB, 2, Hkv, record]
    plan = _plan(b)
    out = paged.paged_attention(plan, b.q.to(DEV), pool[:, 0], pool[:, 1], b.bt.to(DEV))
    torch.cuda.synchronize()
    b.check(out, None, 0, "strided")


@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 128), (BF, 32), (F32, 96), (F16, 160), (BF, 256)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3), (300, 0)])
def test_generic(dtype, D, window, sinks):
    """Model dtypes and head dims of the generic kernel; enough rows for its
    tiled form in the last batch, which a 4-bit cache does not take."""
    for ctx, ql, bs in (([0, 20, 500, 0, 130], [1, 3, 1, 60, 40], 16), ([5, 1000], [1, 1], 7)):
        print(f"kv4 generic {dtype} D={D} window={window} bs={bs}", flush=True)
        b = Batch(ctx, ql, D=D, dtype=dtype, kv="4", bs=bs, seed=D)
        out = _run(b, window, sinks)
        b.check(out, window, sinks, "kv4 generic")
        if window is not None:
            assert torch.equal(_run(b, window, sinks, *b.evict(window, sinks)), out)


def test_generic_many_rows():
    b = Batch([0, 64] * 8, [70, 90] * 8, Hq=32, Hkv=8, D=64, dtype=F32, kv="4", seed=1)
    b.check(_run(b), None, 0, "kv4 generic, many rows")


@pytest.mark.parametrize("kv,D,dtype", [("4", 64, BF), ("4", 128, F16), ("4", 96, F32), (BF, 64, BF), (F8, 128, BF), (F32, 64, F32)])
@pytest.mark.parametrize("bs", [16, 7])
def test_nan_in_slots_that_no_row_sees(kv, D, dtype, bs):
    """Slots behind a sequence's end and beside its window, in blocks that
    hold visible keys too, may hold anything."""
    for ctx, ql in (([0, 3, 40, 299, 1000], [1] * 5), ([0, 37, 500, 5], [150, 77, 40, 1]), ([700, 0], [70, 5])):
        for window, sinks in ((1, 0), (21, 3), (130, 40)) + (((None, 0),) if kv == "4" else ()):
            print(f"unseen NaN {kv} D={D} bs={bs} window={window} {ctx}", flush=True)
            b = Batch(ctx, ql, D=D, dtype=dtype, kv=kv, bs=bs, seed=D + bs)
            want = _run(b, window, sinks)
            b.check(want, window, sinks, "seen")
            bad = torch.ones(b.nb * bs, dtype=torch.bool)
            for i, (c, n) in enumerate(zip(ctx, ql)):
                t = torch.cat([ow.visible(c + r, window, sinks) for r in range(n)])
                bad[b.bt[i, t // bs].long() * bs + t % bs] = False
            bad = bad.nonzero()[:, 0]
            for c in (b.kc, b.vc):
                if kv == "4":
                    kv4.views(c, bs, D)[1][bad // bs, :, bad % bs] = 255
                else:
                    c[bad] = float("nan")
            assert torch.equal(_run(b, window, sinks), want)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, F16), (128, F32)])
def test_blocks_past_4_gib(D, dtype):
    """A pool of more than 4 GiB a tensor: blocks at byte 2^31 and behind 2^32,
    written, read back and attended to."""
    b = Batch([0, 60, 200], [40, 1, 1], Hq=8, Hkv=8, D=D, dtype=dtype, kv="4", seed=D)
    rec = kv4.record_bytes(16, D)
    nb = (1 << 32) // (8 * rec) + b.nb + 7
    far = torch.tensor([nb - 1 - i if i % 3 else (1 << 31) // (8 * rec) + i for i in range(b.nb)])
    print(f"far blocks D={D} {dtype}: {nb} blocks", flush=True)
    kc, vc = (torch.empty(nb, 8, rec, dtype=torch.uint8, device=DEV) for _ in range(2))
    kc[far.to(DEV)], vc[far.to(DEV)] = b.kc.to(DEV), b.vc.to(DEV)
    bt = far[b.bt.long().clamp(0, b.nb - 1)].int()
    for window, sinks in ((None, 0), (50, 2)):
        b.check(_run(b, window, sinks, bt, kc, vc), window, sinks, "far")
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(16, 8, D, generator=g).to(dtype) for _ in range(2))
    slots = (nb - 1) * 16 + torch.arange(16)
    rot = gllm_amd.Rotary(D, device=DEV)
    zero = torch.zeros(16, dtype=torch.int64, device=DEV)
    paged.rotary_kv_write(k.to(DEV), v.to(DEV), zero, rot, kc, vc, slots.to(DEV))
    small_k, small_v = (torch.zeros(1, 8, rec, dtype=torch.uint8) for _ in range(2))
    kv4.write(small_k, torch.arange(16), k, 16)
    kv4.write(small_v, torch.arange(16), v, 16)
    n = 16 * (D // 32 * 17)                     # a record without its padding
    assert torch.equal(kc[-1:, :, :n].cpu(), small_k[..., :n]) and torch.equal(vc[-1:, :, :n].cpu(), small_v[..., :n])
    got = paged.kv4_values(kc, slots.to(DEV), D, torch.float32).cpu()
    assert torch.equal(got.double(), kv4.read(small_k, torch.arange(16), 16, D))


def test_graph_replays():
    """A mixed batch over a 4-bit cache and a decode with splits, captured on one
    stream and replayed with eager calls between, on another."""
    cases = []
    for ctx, ql in (([0, 37, 1000, 700], [150, 77, 1, 1]), ([2500, 40], [1, 1])):
        b = Batch(ctx, ql, D=128, kv="4", seed=12)
        q, kc, vc, bt = (x.to(DEV) for x in (b.q, b.kc, b.vc, b.bt))
        cases.append((_plan(b), q, kc, vc, bt, torch.empty_like(q)))
    for plan, q, kc, vc, bt, out in cases:
        paged.paged_attention(plan, q, kc, vc, bt, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for plan, q, kc, vc, bt, out in cases:
            paged.paged_attention(plan, q, kc, vc, bt, out=out)
    for i in range(3):
        want = []
        for plan, q, kc, vc, bt, out in cases:
            q.mul_(-0.5)
            want.append(paged.paged_attention(plan, q, kc, vc, bt))
            out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(c[-1], w) for c, w in zip(cases, want))


def test_refusals():
    b = Batch([10], [1], D=64, kv="4")
    q, kc, vc, bt = (x.to(DEV) for x in (b.q, b.kc, b.vc, b.bt))
    plan = _plan(b)
    with pytest.raises(ValueError):
        paged.paged_attention(plan, q, kc[..., :-16], vc[..., :-16], bt)
    with pytest.raises(NotImplementedError):
        paged.paged_attention(plan, q, kc, vc, bt, kv_new=(q[:, :2], q[:, :2]))
    plan = paged.AttentionPlan([1], [10], num_q_heads=8, num_kv_heads=2, head_dim=80, block_size=16, dtype=BF, device=DEV)
    with pytest.raises(ValueError):
        paged.paged_attention(plan, torch.zeros(1, 8, 80, dtype=BF, device=DEV), kc, vc, bt)


@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("ctx,ql", [([0, 40, 300], [1, 1, 1]), ([0, 200], [70, 40])])
def test_fp16_rows_up_to_the_largest(D, ctx, ql):
    """K and V rows of an fp16 model up to 65,504, written and attended to."""
    print(f"fp16 up to 65504 D={D} {ctx}", flush=True)
    b = Batch(ctx, ql, D=D, dtype=F16, kv="4", seed=D, scale_q=2.0 ** -13)
    g = torch.Generator().manual_seed(D)
    k, v = (((torch.rand(b.nb * b.bs, b.Hkv, D, generator=g) - 0.5) * 2 * 65504).to(F16) for _ in range(2))
    kc, vc = b.kc.to(DEV), b.vc.to(DEV)
    slots = torch.arange(b.nb * b.bs, device=DEV)
    paged.rotary_kv_write(k.to(DEV), v.to(DEV), torch.zeros_like(slots), gllm_amd.Rotary(D, device=DEV), kc, vc, slots)
    b.kc, b.vc = kc.cpu(), vc.cpu()
    assert b.rows(b.kc, 0).isfinite().all() and b.rows(b.vc, 0).isfinite().all()
    b.check(_run(b), None, 0, "fp16, large rows")
