"""Sparse attention of prompts in several slabs, of tiles and of single rows."""
import pytest
import torch

from gllm_amd import sparse
from tests import test_gpu_sparse as gs
from tests.test_gpu_tile_runs import check_rows
from tests.window_helpers import BF, F8, Batch

pytestmark = pytest.mark.gpu


def lists(b, blocks, seed):
    """A random selection of every row's blocks, its own block among them; -1 behind shorter ones."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    sel = torch.full((sum(b.ql), b.Hkv, blocks), -1, dtype=torch.int32, device="cuda")
    for i, n in enumerate(b.ql):
        own = (torch.arange(b.ctx[i], b.L[i]) // b.bs).cuda()
        for r0 in range(0, n, 256):
            o = own[r0:min(n, r0 + 256), None, None]
            x = torch.rand(len(o), b.Hkv, -(-b.L[i] // b.bs), generator=g, device="cuda")
            at = torch.arange(x.shape[-1], device="cuda")
            x = torch.where(at > o, -1.0, torch.where(at == o, 2.0, x))
            k = min(blocks, x.shape[-1])
            v, at = x.topk(k)
            at = torch.where(v < 0, 1 << 30, at).sort().values
            sel[b.start[i] + r0:b.start[i] + r0 + len(o), :, :k] = torch.where(at == 1 << 30, -1, at).int()
    return sel


@pytest.mark.parametrize("kv", [BF, F8])
def test_slabs_of_tiles(kv):
    """Two slabs of one prompt's tiles, and a chunk, a single row and a short prompt around it;
    captured, and replayed with other lists."""
    b = Batch([900, 120000, 5000, 0], [40, 4096, 1, 70], Hq=16, Hkv=2, D=128, kv=kv, seed=1)
    plan = gs.plan_of(b, 600, 0)
    assert plan.info["tiles"] > 128 and plan.info["tile_slabs"] == 2
    q, kc, vc, bt = b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda()
    rows = [0, 39, 40, 41, 71, 72, 500, 1023, 2048, 2900, 3400, 3600, 3700, 3800, 3850, 3900, 3950, 4000, 4135, 4136, 4137, 4206]
    sel = lists(b, 600, 1)
    out = sparse.sparse_attention(plan, q, kc, vc, bt, sel)
    check_rows(b, out, sel.cpu(), rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = torch.empty_like(out)
    with torch.cuda.stream(side):
        sparse.sparse_attention(plan, q, kc, vc, bt, sel, out=got)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sparse.sparse_attention(plan, q, kc, vc, bt, sel, out=got)
    first = sel.clone()
    for seed in (2, 3, 1):
        sel.copy_(lists(b, 600, seed))
        graph.replay()
        torch.cuda.synchronize()
        replayed = got.clone()
        assert torch.equal(replayed, sparse.sparse_attention(plan, q, kc, vc, bt, sel)), f"lists {seed}"
    assert torch.equal(sel, first) and torch.equal(got, out)


def test_many_short_tiles_in_slabs():
    """Chunks of many sequences: each row as in a plan of its sequence alone, up to the runs
    that its keys fall in, so against the oracle."""
    n = 48
    b = Batch([26000 + 100 * i for i in range(n)], [256] * n, Hq=16, Hkv=2, D=128, seed=2)
    plan = gs.plan_of(b, 512, 0)
    assert plan.info["tiles"] == 8 * n and plan.info["tile_slabs"] >= 2
    sel = lists(b, 512, 4)
    out = sparse.sparse_attention(plan, b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel)
    assert torch.isfinite(out).all()
    check_rows(b, out, sel.cpu(), [256 * i + (37 * i) % 256 for i in range(n)] + [256 * n - 1])


def test_slabs_of_single_rows():
    """Rows in two splits, more than fit at a time: bit for bit those of plans of their own."""
    b = Batch([6000], [4100], Hq=16, Hkv=8, D=64, bs=8, seed=3)
    plan = gs.plan_of(b, 600, 0)
    assert plan.info["tiles"] == 0 and plan.info["splits"] == 2 and plan.info["row_slabs"] == 2
    sel = lists(b, 600, 5)
    sel[7] = -1
    sel[4000, 3, 5:] = -1
    args = (b.kc.cuda(), b.vc.cuda(), b.bt.cuda())
    q = b.q.cuda()
    out = sparse.sparse_attention(plan, q, *args, sel)
    for r0, r1 in ((0, 90), (3900, 4100)):
        part = sparse.SparsePlan([r1 - r0], [6000 + r1], num_q_heads=16, num_kv_heads=8, head_dim=64, block_size=8, dtype=BF,
                                 device="cuda", blocks=600, first_blocks=0)
        assert part.info["row_slabs"] == 1 and part.info["splits"] == 2
        assert torch.equal(out[r0:r1], sparse.sparse_attention(part, q[r0:r1], *args, sel[r0:r1].contiguous()))
    assert (out[7] == 0).all()
    check_rows(b, out, sel.cpu(), [0, 1, 3970, 3971, 3972, 4099])
