"""Sliding-window attention with sinks against the 64-bit oracle: decode,
prompt chunks and mixed batches, every cache dtype, plans split and balanced,
windows and sinks at and beside the kernels' 16- and 64-key units."""
import pytest
import torch

from gllm_amd import paged
from oracle import rope as orope
from tests.window_helpers import BF, F8, F16, F32, Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _plan(b, window, sinks, **kw):
    return paged.AttentionPlan(b.ql, b.L, num_q_heads=b.Hq, num_kv_heads=b.Hkv, head_dim=b.D, block_size=b.bs,
                               dtype=b.dtype, device=DEV, q_seq_stride=b.stride, window=window, sinks=sinks, **kw)


def _run(b, window, sinks, bt=None, kc=None, vc=None, **kw):
    bt, kc, vc = (x.to(DEV) for x in (b.bt if bt is None else bt, b.kc if kc is None else kc, b.vc if vc is None else vc))
    out = paged.paged_attention(_plan(b, window, sinks, **kw), b.q.to(DEV), kc, vc, bt)
    torch.cuda.synchronize()
    return out


DECODE = dict(ctx=[0, 3, 15, 16, 40, 299, 1000, 2500], ql=[1] * 8)
EDGES = [(1, 0), (2, 1), (16, 0), (17, 4), (33, 16), (100, 1), (129, 20), (600, 64), (4096, 4)]


@pytest.mark.parametrize("window,sinks", EDGES)
@pytest.mark.parametrize("D", [64, 128])
def test_decode(D, window, sinks):
    print(f"decode D={D} window={window} sinks={sinks}", flush=True)
    b = Batch(**DECODE, D=D, seed=window + D)
    b.check(_run(b, window, sinks), window, sinks, "decode")


@pytest.mark.parametrize("dtype,kv", [(BF, F8), (F16, F16), (F16, F8)])
@pytest.mark.parametrize("split", [0, 64, paged.BALANCED])
def test_decode_types_and_plans(dtype, kv, split):
    for D, bs, (window, sinks) in ((64, 16, (50, 3)), (128, 24, (700, 40)), (64, 1, (300, 17)), (128, 7, (95, 5))):
        print(f"decode {dtype} {kv} split={split} D={D} bs={bs} window={window}", flush=True)
        b = Batch(**DECODE, D=D, dtype=dtype, kv=kv, bs=bs, seed=D + bs)
        b.check(_run(b, window, sinks, split_tokens=split), window, sinks, "decode")


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 1), (6, 3), (32, 8)])
def test_decode_rows_and_heads(Hq, Hkv):
    """Several query rows a sequence on the decode path, padded layout."""
    n = min(4, 16 // (Hq // Hkv))
    b = Batch([0, 14, 130, 777, 1500], [1, n, 1, n, n], Hq=Hq, Hkv=Hkv, D=64, stride=5, seed=Hq)
    for window, sinks in ((1, 0), (16, 2), (130, 33)):
        print(f"rows {Hq}/{Hkv} window={window}", flush=True)
        b.check(_run(b, window, sinks), window, sinks, "rows")


@pytest.mark.parametrize("window,sinks", EDGES)
@pytest.mark.parametrize("D", [64, 128])
def test_prefill(D, window, sinks):
    print(f"prefill D={D} window={window} sinks={sinks}", flush=True)
    b = Batch([0, 0, 37, 1000], [33, 200, 77, 130], D=D, seed=window + D)
    b.check(_run(b, window, sinks), window, sinks, "prefill")


@pytest.mark.parametrize("dtype,kv,bs", [(BF, F8, 16), (F16, F16, 24), (F16, F8, 1), (BF, BF, 7)])
def test_prefill_types(dtype, kv, bs):
    b = Batch([0, 600], [150, 70], D=128, dtype=dtype, kv=kv, bs=bs, stride=160, seed=bs)
    for window, sinks in ((40, 0), (64, 1), (200, 70)):
        print(f"prefill {dtype} {kv} bs={bs} window={window}", flush=True)
        b.check(_run(b, window, sinks), window, sinks, "prefill")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("split", [0, paged.BALANCED])
def test_mixed(D, split):
    b = Batch([300, 0, 57, 1000, 5, 2500], [1, 120, 64, 1, 1, 1], D=D, seed=D)
    for window, sinks in ((30, 4), (257, 0), (1024, 130)):
        print(f"mixed D={D} split={split} window={window}", flush=True)
        b.check(_run(b, window, sinks, split_tokens=split), window, sinks, "mixed")


def _many(kind, D, kv, seed):
    """Batches large enough for the plans that small ones never get."""
    if kind == "half prefill":                # 1,024 (head dim 128) / 768 items: half-size workgroups
        n = 128 if D == 128 else 96
        return Batch([40 * (i % 5) for i in range(n)], [33 + (7 * i) % 32 for i in range(n)], Hq=32, Hkv=8, D=D, kv=kv, seed=seed)
    if kind == "half mixed":                  # 200 decodes beside three chunks
        return Batch([150 + (37 * i) % 200 for i in range(200)] + [0, 70, 200], [1] * 200 + [40, 64, 33], Hq=32, Hkv=8, D=D,
                     kv=kv, seed=seed)
    return Batch([100 + (37 * i) % 300 for i in range(140)], [1] * 140, Hq=32, Hkv=8, D=D, kv=kv, seed=seed)


@pytest.mark.parametrize("kind", ["half prefill", "half mixed", "balanced"])
@pytest.mark.parametrize("D,kv", [(64, BF), (128, BF), (128, F8), (128, "4"), (64, "4")])
def test_plans_of_large_batches(kind, D, kv):
    print(f"{kind} D={D} kv={kv}", flush=True)
    b = _many(kind, D, kv, D)
    plan = _plan(b, 90, 3)
    assert plan.info["prefill_waves"] == 4 if kind == "half prefill" else plan.info["prefill_waves"] == 8
    assert (plan.info["decode_segments"] > 0) == (kind == "balanced" and D == 128)
    b.check(_run(b, 90, 3), 90, 3, kind)


@pytest.mark.parametrize("dtype,kv,D", [(F32, F32, 64), (F32, F8, 128), (F32, BF, 50), (BF, BF, 96), (F16, F16, 256),
                                        (BF, F32, 64), (F32, F32, 2)])
def test_generic(dtype, kv, D):
    """Model and cache dtypes and head dims of the generic kernel."""
    for window, sinks, bs in ((1, 0, 16), (17, 4, 16), (100, 33, 24)):
        print(f"generic {dtype} {kv} D={D} window={window}", flush=True)
        b = Batch([0, 20, 500, 0, 130], [1, 3, 1, 60, 40], D=D, dtype=dtype, kv=kv, bs=bs, seed=D)
        b.check(_run(b, window, sinks), window, sinks, "generic")


@pytest.mark.parametrize("dtype,D,bs", [(BF, 64, 16), (F16, 128, 4), (F32, 64, 16), (BF, 128, 100)])
def test_blocks_behind_the_window_may_be_gone(dtype, D, bs):
    """Keys that no row sees are not read: their blocks hold NaN and their
    table entries are other blocks' or no block at all; the output is the same."""
    b = Batch([900, 0, 301, 64], [1, 150, 1, 40], D=D, dtype=dtype, bs=bs, seed=3)
    for window, sinks in ((20, 0), (130, 1), (64, 70)):
        print(f"evicted {dtype} D={D} bs={bs} window={window}", flush=True)
        want = _run(b, window, sinks)
        got = _run(b, window, sinks, *b.evict(window, sinks))
        assert torch.equal(got, want)


@pytest.mark.parametrize("D", [64, 128])
def test_large_scores_and_low_first_tiles(D):
    """Scores far from 0 in the first visible tile, and far larger ones later."""
    b = Batch([0, 700], [160, 90], D=D, seed=9, scale_q=12.0)
    for window, sinks in ((70, 0), (90, 2)):
        b.check(_run(b, window, sinks), window, sinks, "scaled q")
    # the window's first keys score about -300, the later ones about 0
    b = Batch([500], [64], Hq=2, Hkv=1, D=D, seed=11)
    b.q[...] = 1.0
    t = torch.arange(b.L[0])
    slots = b.bt[0, t // b.bs].long() * b.bs + t % b.bs
    for key, x in ((slice(0, 500), -300.0), (slice(500, 564), 0.0)):
        b.kc[slots[key]] = x / D ** 0.5
    b.check(_run(b, 100, 0), 100, 0, "low first tiles")


def test_a_window_that_hides_nothing_is_none():
    b = Batch(**DECODE, D=64, seed=5)
    assert torch.equal(_run(b, 2501, 0), _run(b, None, 0))
    assert torch.equal(_run(b, 2400, 101), _run(b, None, 0))


@pytest.mark.parametrize("D,kv", [(64, BF), (128, F8)])
def test_kv_write_and_rope_in_the_launch(D, kv):
    """Decode step with the new tokens' K/V rotated and written by the launch."""
    b = Batch([0, 15, 16, 300, 1000], [1, 2, 1, 4, 1], D=D, kv=kv, seed=D)
    g = torch.Generator().manual_seed(1)
    rows = sum(b.ql)
    k, v = (torch.randn(rows, b.Hkv, D, generator=g).to(BF) for _ in range(2))
    cos, sin = orope.rope_cache(2048, D, 500000.0, BF)
    pos = torch.cat([torch.arange(c, c + n) for c, n in zip(b.ctx, b.ql)])
    kr = orope.apply_rope(k[None], cos[pos][None], sin[pos][None])[0]
    q, b.q = b.q, orope.apply_rope(b.q[None], cos[pos][None], sin[pos][None])[0]
    kc, vc = b.kc.to(DEV), b.vc.to(DEV)
    at = 0
    for i, (c, n) in enumerate(zip(b.ctx, b.ql)):
        t = torch.arange(c, c + n)
        slots = b.bt[i, t // b.bs].long() * b.bs + t % b.bs
        b.kc[slots], b.vc[slots] = kr[at:at + n].to(b.kv), v[at:at + n].to(b.kv)
        at += n
    for window, sinks in ((5, 0), (64, 18)):
        out = paged.paged_attention(_plan(b, window, sinks), q.to(DEV), kc, vc, b.bt.to(DEV),
                                    rope=(cos.to(DEV), sin.to(DEV), "position"), kv_new=(k.to(DEV), v.to(DEV)))
        torch.cuda.synchronize()
        b.check(out, window, sinks, "fused write")
        for a, x in ((kc, b.kc), (vc, b.vc)):
            assert torch.equal(a.cpu().view(torch.uint8), x.view(torch.uint8))


@pytest.mark.parametrize("kind,kv", [("balanced", BF), ("balanced", F8), ("split", BF), ("asked", F8)])
def test_kv_write_in_every_decode_plan(kind, kv):
    """The new keys are written once and seen, whichever part of a split or
    page-balanced sequence holds them."""
    if kind == "balanced":
        n = 140
        b = Batch([100 + (37 * i) % 300 for i in range(n)], [1 + i % 4 for i in range(n)], Hq=32, Hkv=8, D=128, kv=kv, seed=3)
    else:
        b = Batch([0, 15, 700, 2500, 31, 64], [1, 2, 4, 1, 3, 4], Hq=32, Hkv=8, D=128, kv=kv, seed=4)
    kw = {"balanced": {}, "split": dict(split_tokens=32), "asked": dict(split_tokens=paged.BALANCED)}[kind]
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(sum(b.ql), b.Hkv, b.D, generator=g).to(BF) for _ in range(2))
    at = 0
    for i, (c, n) in enumerate(zip(b.ctx, b.ql)):
        t = torch.arange(c, c + n)
        slots = b.bt[i, t // b.bs].long() * b.bs + t % b.bs
        b.kc[slots], b.vc[slots] = k[at:at + n].to(kv), v[at:at + n].to(kv)
        at += n
    for window, sinks in ((90, 3), (17, 0)):
        plan = _plan(b, window, sinks, **kw)
        assert paged.fused_kv_write_ok(plan, kv)
        assert (plan.info["decode_segments"] > 0) == (kind != "split")
        kc, vc = b.kc.to(DEV), b.vc.to(DEV)
        at = 0
        for i, (c, n) in enumerate(zip(b.ctx, b.ql)):        # what the slots held before
            t = torch.arange(c, c + n)
            slots = (b.bt[i, t // b.bs].long() * b.bs + t % b.bs).to(DEV)
            kc[slots], vc[slots] = float("nan"), float("nan")
        out = paged.paged_attention(plan, b.q.to(DEV), kc, vc, b.bt.to(DEV), kv_new=(k.to(DEV), v.to(DEV)))
        torch.cuda.synchronize()
        for a, x in ((kc, b.kc), (vc, b.vc)):
            assert torch.equal(a.cpu().view(torch.uint8), x.view(torch.uint8))
        b.check(out, window, sinks, f"write, {kind}")


def test_graph_replays():
    """Captured with one plan, replayed with new values between the replays."""
    b = Batch(**DECODE, D=128, seed=8)
    plan = _plan(b, 300, 4)
    q, kc, vc, bt = (x.to(DEV) for x in (b.q, b.kc, b.vc, b.bt))
    out = torch.empty_like(q)
    paged.paged_attention(plan, q, kc, vc, bt, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged.paged_attention(plan, q, kc, vc, bt, out=out)
    for i in range(3):
        q.mul_(-0.5)
        want = paged.paged_attention(plan, q, kc, vc, bt)
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_rows_of_other_sequences_stay():
    """Padded rows past a sequence's length are left as they were or not
    written at all beyond the last sequence."""
    b = Batch([100, 900], [1, 1], D=64, stride=1, seed=2)
    q = torch.cat([b.q, b.q, b.q])
    out = torch.full_like(q, 7.0).to(DEV)
    paged.paged_attention(_plan(b, 50, 2), q.to(DEV), b.kc.to(DEV), b.vc.to(DEV), b.bt.to(DEV), out=out)
    torch.cuda.synchronize()
    b.check(out[:2], 50, 2)
    assert (out[2:] == 7.0).all()


@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF, 96)])
def test_kv_write_in_the_launch_under_a_window_that_hides_nothing(dtype, D):
    """The generic kernel's write is lost to a window only where keys are hidden."""
    b = Batch([0, 15, 300], [1, 2, 1], D=D, dtype=dtype, seed=D)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(sum(b.ql), b.Hkv, D, generator=g).to(dtype) for _ in range(2))
    got = []
    for window, sinks in ((None, 0), (301, 0), (290, 11)):
        plan = _plan(b, window, sinks)
        assert paged.fused_kv_write_ok(plan, dtype)
        kc, vc = b.kc.to(DEV), b.vc.to(DEV)
        out = paged.paged_attention(plan, b.q.to(DEV), kc, vc, b.bt.to(DEV), kv_new=(k.to(DEV), v.to(DEV)))
        torch.cuda.synchronize()
        got.append((out, kc, vc))
    for x in got[1:]:
        assert all(torch.equal(s, t) for s, t in zip(x, got[0]))
    hiding = _plan(b, 290, 10)
    assert not paged.fused_kv_write_ok(hiding, dtype)
    with pytest.raises(NotImplementedError):
        paged.paged_attention(hiding, b.q.to(DEV), kc, vc, b.bt.to(DEV), kv_new=(k.to(DEV), v.to(DEV)))


@pytest.mark.parametrize("hw", [0, 1, 4, 8])
@pytest.mark.parametrize("D,kv", [(64, BF), (128, F8), (64, "4"), (128, "4")])
def test_half_size_mixed_workgroups(hw, D, kv):
    """Decodes, split and whole, beside many short chunks, two workgroups an item:
    each number of KV heads a workgroup, the larger ones with idle heads too."""
    for Hq, Hkv, window in ((32, 8, 1000), (24, 6, 900))[:1 + (hw > 2)]:
        ctx = [1000 + (37 * i) % 200 for i in range(16)] + [20 * (i % 5) for i in range(60)]
        b = Batch(ctx, [1] * 16 + [33] * 60, Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=D + Hkv)
        plan = _plan(b, window, 3, heads_per_wg=hw)
        info = plan.info
        print(f"half mixed hw={hw} D={D} kv={kv} heads {Hq}/{Hkv} {info}", flush=True)
        assert info["mixed_half"] == 1 and info["decode_segments"] == 0 and info["heads_per_wg"] == (hw or 2)
        assert info["partials"] > 0
        b.check(_run(b, window, 3, heads_per_wg=hw), window, 3, "half mixed")


@pytest.mark.parametrize("D", [64, 128])
def test_half_size_mixed_workgroups_of_one_head(D):
    """The planner's own choice of one KV head a workgroup (whole sequences)."""
    n = 70 if D == 64 else 40
    b = Batch([150 + (37 * i) % 200 for i in range(n)] + [20 * (i % 5) for i in range(60)], [1] * n + [33] * 60, Hq=32, Hkv=8,
              D=D, kv="4", seed=D)
    info = _plan(b, 90, 3).info
    print(f"half mixed, one head, D={D} {info}", flush=True)
    assert info["mixed_half"] == 1 and info["heads_per_wg"] == 1 and info["partials"] == 0
    for window, sinks in ((90, 3), (None, 0)):
        assert _plan(b, window, sinks).info["mixed_half"] == 1
        b.check(_run(b, window, sinks), window, sinks, "half mixed, one head")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kv", [BF, F8, "4"])
def test_the_half_mixed_batch_runs_in_half_size_workgroups(D, kv):
    assert _plan(_many("half mixed", D, kv, D), 90, 3).info["mixed_half"] == 1
