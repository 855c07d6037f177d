"""Joins of partial results whose references lie far from their rows' largest scores:
ranges of a shared prefix, and the parts of a tile of prompt rows.  Against the 64-bit
oracles of the two operators."""
import pytest
import torch

from gllm_amd import sparse
from tests import test_gpu_prefix as gp
from tests import test_gpu_sparse as gs
from tests.window_helpers import BF, F16, Batch

pytestmark = pytest.mark.gpu

# Scores in log2 units are 64 k_0 / 8 log2(e) = 11.54 k_0 with these queries.  A range of 256
# keys that starts at -129.1 and rises to -69.6 holds 224 x 2^-69.6 = 2^-61.8 of the row's
# weight; one whose first key is at -63.8 and the others far below, 2^-63.8.
RISING, SINGLE, FAR = (-11.1875, -6.03125), -5.53125, -26.0


def _far_scores(b, order):
    """Sets q and the first 1,024 keys of sequence 0: ranges of 256 keys."""
    b.q[:] = 0
    b.q[..., 0] = 64.0
    k = torch.full((b.L[0],), FAR)
    for r, kind in enumerate(order):
        if kind == "rising":
            k[256 * r:256 * r + 256] = RISING[1]
            k[256 * r:256 * r + 32] = RISING[0]
        if kind == "single":
            k[256 * r] = SINGLE
    for i in range(len(b.L)):
        for t in range(min(len(k), b.L[i])):
            b.kc[int(b.bt[i, t // b.bs]) * b.bs + t % b.bs, :, 0] = k[t]


ORDERS = [("rising", "single", "", ""), ("single", "rising", "", ""), ("", "single", "rising", "single"),
          ("rising", "", "", "rising")]


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("dtype", [BF, F16])
def test_prefix_ranges_far_from_their_references(dtype, order):
    P = 1024
    b = Batch([P + 40, P + 7], [1, 1], Hq=8, Hkv=2, D=64, dtype=dtype)
    groups = [([0, 1], P)]
    gp.share(b, groups)
    _far_scores(b, order)
    plan = gp.plan_of(b, groups)
    assert plan.info["prefix_items"] == 2 * P // 256         # ranges of 256 keys
    b.check(gp.run(b, groups, plan), None, 0)


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("dtype", [BF, F16])
def test_tile_parts_far_from_their_references(dtype, order):
    """17 tiles of 64 keys in four runs: of 256 keys but the last."""
    b = Batch([1024], [64], Hq=4, Hkv=1, D=64, dtype=dtype)
    _far_scores(b, order)
    plan = gs.plan_of(b, 68, 0)
    assert plan.info["tiles"] == 1
    sel = gs.random_lists(b, 68, 1, whole=True)
    out = sparse.sparse_attention(plan, b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    gs.check_attention(b, out, {(r, 0): sel[r, 0].tolist() for r in range(64)})


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("scale_q", [0.0, 8.0, 40.0])
def test_tiles_of_large_scores(dtype, scale_q):
    b = Batch([1500, 300], [70, 40], Hq=8, Hkv=2, D=64, dtype=dtype, scale_q=scale_q, seed=3)
    plan = gs.plan_of(b, 9, 0)
    assert plan.info["tiles"] >= 2
    sel = gs.random_lists(b, 9, 2, whole=True)
    out = sparse.sparse_attention(plan, b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    gs.check_attention(b, out, {(row, h): sel[row, h].tolist() for _, row, _ in gs.rows_of(b) for h in range(2)})
