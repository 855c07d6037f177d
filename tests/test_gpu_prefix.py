"""Paged attention of batches that share prefixes against the 64-bit oracle, which
knows nothing of sharing (error bound of oracle/window.py)."""
import pytest
import torch

import gllm_amd
from gllm_amd import paged
from oracle import rope as orope
from tests.gpu_helpers import assert_close_bf16
from tests.window_helpers import BF, F8, F16, F32, Batch

pytestmark = pytest.mark.gpu


def share(b, groups):
    """Gives the groups' sequences their first keys in common: whole blocks once, a cut
    block copied."""
    for seqs, P in groups:
        seqs = list(seqs)
        first, w = seqs[0], P // b.bs
        for i in seqs[1:]:
            b.bt[i, :w] = b.bt[first, :w]
            if P % b.bs:
                src, dst, n = int(b.bt[first, w]), int(b.bt[i, w]), P % b.bs
                for c in (b.kc, b.vc):
                    if b.kv == "4":
                        # rows of codes, then rows of scales
                        h = b.bs * b.D // 2
                        c[dst, :, :n * b.D // 2] = c[src, :, :n * b.D // 2]
                        c[dst, :, h:h + n * b.D // 32] = c[src, :, h:h + n * b.D // 32]
                    else:
                        c[dst * b.bs:dst * b.bs + n] = c[src * b.bs:src * b.bs + n]
    return b


def plan_of(b, groups, **kw):
    return paged.AttentionPlan(b.ql, b.L, num_q_heads=b.Hq, num_kv_heads=b.Hkv, head_dim=b.D, block_size=b.bs, dtype=b.dtype,
                               device="cuda", q_seq_stride=b.stride, shared_prefixes=groups, **kw)


def run(b, groups, plan=None, **kw):
    plan = plan or plan_of(b, groups)
    return paged.paged_attention(plan, b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv,dtype,kv,bs", [(8, 2, BF, BF, 16), (32, 8, BF, BF, 16), (4, 4, F16, F16, 3), (16, 1, BF, F8, 24),
                                                (6, 2, F16, F8, 16), (8, 2, BF, "4", 16), (10, 2, F16, "4", 7)])
def test_groups(Hq, Hkv, dtype, kv, bs, D):
    """Two groups in no order, a sequence alone, prefixes that end inside a block or
    a sub-tile, one own key and many."""
    b = Batch([630, 711, 600, 55, 633, 900, 610], [1] * 7, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, kv=kv, bs=bs, seed=D + Hq)
    groups = [([4, 0, 2], 600), ([6, 1], 523)]
    share(b, groups)
    plan = plan_of(b, groups)
    assert plan.info["prefix_items"] > 0
    out = run(b, groups, plan)
    b.check(out, None, 0)
    assert torch.equal(out, run(b, groups, plan))


@pytest.mark.parametrize("P", [1, 255, 256, 273, 511, 512, 527, 575, 576, 577, 1000, 4097])
@pytest.mark.parametrize("D", [64, 128])
def test_prefix_lengths(P, D):
    b = share(Batch([P + 3, P, P + 40], [1, 1, 1], Hq=8, Hkv=2, D=D), [([0, 1, 2], P)])
    plan = plan_of(b, [([0, 1, 2], P)])
    assert (plan.info["prefix_items"] > 0) == (P >= (512 if D == 64 else 256))
    b.check(run(b, None, plan), None, 0)


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (12, 4), (8, 1)])
def test_more_columns_than_a_workgroup_takes(Hq, Hkv):
    n = 70
    b = Batch([530 + i for i in range(n)], [1] * n, Hq=Hq, Hkv=Hkv, D=64, seed=2)
    groups = [(range(n), 520)]
    plan = plan_of(share(b, groups), groups)
    assert plan.info["prefix_items"] > 0
    b.check(run(b, groups, plan), None, 0)


def test_several_query_rows_and_prompts():
    """Members with 1 to 4 query rows (speculative tokens), a prompt in the group and one
    beside it, packed and padded rows."""
    for stride in (0, 40):
        b = Batch([330, 300, 310, 305, 20, 300], [1, 4, 2, 33, 40, 3], Hq=8, Hkv=2, D=128, stride=stride)
        groups = [([5, 0, 1, 3, 2], 299)]
        plan = plan_of(share(b, groups), groups)
        assert plan.info["prefill_seqs"] == 2 and plan.info["prefix_items"] > 0
        b.check(run(b, groups, plan), None, 0, f"stride {stride}")


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("scale_q", [0.0, 8.0, 40.0])
def test_large_scores(dtype, scale_q):
    """Scores far apart: the rows' references move within the prefix and differ from their
    own keys'.  (All equal at 0.)"""
    b = Batch([1200, 1300, 1250], [1, 1, 1], Hq=8, Hkv=2, D=64, dtype=dtype, scale_q=scale_q, seed=5)
    groups = [([0, 1, 2], 1184)]
    b.check(run(share(b, groups), groups), None, 0)


def test_long_prefix_of_many_blocks():
    """More block ids than an item caches (1,024), of one key each."""
    P = 40000
    b = Batch([P + 5, P + 9], [1, 1], Hq=2, Hkv=1, D=64, bs=1)
    groups = [([0, 1], P)]
    plan = plan_of(share(b, groups), groups)
    b.check(run(b, groups, plan), None, 0)


@pytest.mark.parametrize("kv", [BF, F8])
@pytest.mark.parametrize("mode", ["position", "row"])
def test_rotation_and_the_write_inside_the_launch(mode, kv):
    """q rotated on load in both parts and the new keys written by the launch: bit for bit
    the cache, and the attention, of the calls apart."""
    groups = [([0, 1, 2], 528)]
    b = share(Batch([540, 570, 529], [1, 1, 2], Hq=8, Hkv=2, D=64, kv=kv, seed=3), groups)
    plan, plain = plan_of(b, groups), plan_of(b, ())
    assert plan.info["prefix_items"] > 0
    cos, sin = (x.cuda() for x in orope.rope_cache(600, 64, 10000.0, BF))
    pos = torch.tensor([540, 570, 529, 530]).cuda()
    rope = (cos, sin, mode) if mode == "position" else (cos[pos], sin[pos], mode)
    k, v = (torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(i)).to(BF).cuda() for i in (1, 2))
    kc, vc, bt, q = b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), b.q.cuda()
    assert paged.fused_kv_write_ok(plan, kv)
    out = paged.paged_attention(plan, q, kc, vc, bt, rope=rope, kv_new=(k, v))
    kc2, vc2 = b.kc.cuda(), b.vc.cuda()
    seq = torch.tensor([0, 1, 2, 2]).cuda()
    slots = bt[seq, pos // 16].long() * 16 + pos % 16
    paged.rope_kv_write(k, v, cos, sin, kc2, vc2, slots, rope_rows=pos)
    assert torch.equal(kc.view(torch.uint8), kc2.view(torch.uint8)) and torch.equal(vc.view(torch.uint8), vc2.view(torch.uint8))
    assert torch.equal(out, paged.paged_attention(plan, q, kc2, vc2, bt, rope=rope))
    # against the oracle, on rotated q
    b.q = paged.rope_rotate(q, cos, sin, rope_rows=pos).cpu()
    b.kc, b.vc = kc.cpu(), vc.cpu()
    b.check(out, None, 0)
    b.check(paged.paged_attention(plain, q, kc2, vc2, bt, rope=rope), None, 0)


@pytest.mark.parametrize("D,dtype,kv", [(64, F32, F32), (96, BF, BF), (64, BF, F32)])
def test_other_kernels_take_the_plan(D, dtype, kv):
    """fp32 models, other head dims, another cache dtype: the generic kernel, which reads
    the keys for each sequence."""
    b = Batch([330, 300, 310], [1, 1, 1], Hq=8, Hkv=2, D=D, dtype=dtype, kv=kv)
    groups = [([0, 1, 2], 299)]
    b.check(run(share(b, groups), groups), None, 0)


def test_shared_blocks_are_read_from_one_row():
    """The other members' entries for whole shared sub-tiles are not followed outside the
    pool; entries outside it are never addresses."""
    groups = [([0, 1], 528)]
    b = share(Batch([570, 540], [1, 1], Hq=8, Hkv=2, D=64), groups)
    want = run(b, groups)
    b.bt[1, :33] = 1 << 30
    assert torch.equal(want, run(b, groups))


def test_rows_past_the_batch_stay():
    b = share(Batch([330, 300], [1, 2], Hq=8, Hkv=2, D=128, stride=3), [([0, 1], 288)])
    out = torch.full((7, 8, 128), 7.0, dtype=BF, device="cuda")
    run(b, [([0, 1], 288)], out=out)
    b.check(out, None, 0)
    assert (out[[1, 2, 5, 6]] == 7.0).all()


def test_replays_of_a_captured_call():
    b = share(Batch([330, 300, 420], [1, 1, 1], Hq=8, Hkv=2, D=128), [([0, 1, 2], 288)])
    groups = [([0, 1, 2], 288)]
    plan = plan_of(b, groups)
    q, kc, vc, bt = b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda()
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.paged_attention(plan, q, kc, vc, bt, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.paged_attention(plan, q, kc, vc, bt, out=out)
    g = torch.Generator().manual_seed(8)
    for i in range(4):
        q.copy_(torch.randn(3, 8, 128, generator=g).to(BF))
        kc.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, paged.paged_attention(plan, q, kc, vc, bt)), f"replay {i}"


def test_pool_past_4_gib():
    bs, Hkv, D = 16, 8, 128
    nb = (1 << 32) // (bs * Hkv * D * 2) + 500
    b = share(Batch([330, 300], [1, 1], Hq=8, Hkv=Hkv, D=D), [([0, 1], 288)])
    kc = torch.zeros(nb * bs, Hkv, D, dtype=BF, device="cuda")
    vc = torch.zeros_like(kc)
    shift = nb - b.nb
    kc[shift * bs:], vc[shift * bs:] = b.kc.cuda(), b.vc.cuda()
    out = paged.paged_attention(plan_of(b, [([0, 1], 288)]), b.q.cuda(), kc, vc, (b.bt + shift).cuda())
    b.check(out, None, 0)


@pytest.mark.parametrize("kv", [BF, F8])
def test_attention_layer_shares_what_the_metadata_says(kv):
    """Attention.attention and forward with AttentionMetadata.shared_prefixes; a layer
    with a window takes no notice."""
    Hq, Hkv, D, hid = 8, 2, 128, 1024
    groups = [([0, 2, 1], 288)]
    b = share(Batch([330, 300, 420, 50], [1] * 4, Hq=Hq, Hkv=Hkv, D=D, kv=kv), groups)
    pos = torch.tensor(b.ctx)
    slots = b.bt[torch.arange(4), pos // 16].long() * 16 + pos % 16
    lens = torch.tensor(b.L, dtype=torch.int32, device="cuda")

    def meta(groups):
        return gllm_amd.AttentionMetadata(torch.ones(4, dtype=torch.int32, device="cuda"), lens, max(b.L), b.bt.cuda(), None,
                                          slots[:, None].cuda(), None, 16, groups)

    class Cfg:
        num_attn_heads, num_kv_heads, head_dim, hidden_size, dtype = Hq, Hkv, D, hid, BF

    g = torch.Generator().manual_seed(4)
    w = {f"model.layers.0.self_attn.{n}_proj.weight": (torch.randn(r, hid, generator=g) / 32).to(BF).cuda()
         for n, r in (("q", hid), ("k", Hkv * D), ("v", Hkv * D), ("o", hid))}
    att, win = gllm_amd.Attention(0, Cfg, w), gllm_amd.Attention(0, Cfg, w, window=64)
    cos, sin = (x[pos][:, None].cuda() for x in orope.rope_cache(500, D, 10000.0, BF))
    k, v = (torch.randn(4, 1, Hkv, D, generator=g).to(BF).cuda() for _ in range(2))
    pool = torch.stack([b.kc.view(torch.uint8) if kv == F8 else b.kc, b.vc.view(torch.uint8) if kv == F8 else b.vc]).cuda()
    pool = pool.view(F8) if kv == F8 else pool
    m = meta(groups)
    out = att.attention(b.q[:, None].cuda(), k, v, cos, sin, pool, m)
    assert m._gllm_plan.info["prefix_items"] > 0
    b.q = paged.rope_rotate(b.q.cuda(), cos[:, 0], sin[:, 0]).cpu()
    b.kc, b.vc = pool[0].cpu(), pool[1].cpu()
    b.check(out.view(4, Hq, D), None, 0)
    # the whole layer, on its fused route too: up to roundings of the 16-bit steps, whose
    # errors are those of the plan without groups
    x = torch.randn(4, 1, hid, generator=g).to(BF).cuda()
    m = meta(groups)
    got, want = att.forward(x, cos, sin, pool.clone(), m), att.forward(x, cos, sin, pool.clone(), meta(None))
    assert m._gllm_plan.info["prefix_items"] > 0
    assert_close_bf16(got, want, "forward")
    m = meta(groups)
    assert torch.equal(win.forward(x, cos, sin, pool.clone(), m), win.forward(x, cos, sin, pool.clone(), meta(None)))
