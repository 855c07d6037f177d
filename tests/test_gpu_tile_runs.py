"""Sparse attention of prompt rows where a workgroup's run of keys is as long as it gets
(255 tiles of 64 keys, 1,020 block ids of 1,024), and where there are more runs than CUs."""
import math

import pytest
import torch

from gllm_amd import sparse
from oracle import sparse as osp
from oracle import window as ow
from tests import test_gpu_sparse as gs
from tests.window_helpers import BF, Batch

pytestmark = pytest.mark.gpu


def whole_lists(b, blocks):
    """Every block that a row sees."""
    sel = torch.full((sum(b.ql), b.Hkv, blocks), -1, dtype=torch.int32)
    for _, row, p in gs.rows_of(b):
        n = min(blocks, p // b.bs + 1)
        sel[row, :, :n] = torch.arange(n)
    return sel


def check_rows(b, out, sel, rows):
    """These rows against the 64-bit attention over their lists, on the GPU."""
    scale, G = 1 / math.sqrt(b.D), b.Hq // b.Hkv
    of = {row: (i, p) for i, row, p in gs.rows_of(b)}
    kv = {}
    for row in rows:
        i, p = of[row]
        if i not in kv:
            kv = {i: (b.rows(b.kc, i).cuda().double(), b.rows(b.vc, i).cuda().double())}
        for h in range(b.Hkv):
            t = osp.keys_of(osp.listed(sel[row, h].tolist(), p // b.bs), p, b.bs).cuda()
            ref, spread, mag = osp.attention(b.q[row, h * G:h * G + G].cuda(), kv[i][0][t, h], kv[i][1][t, h], scale)
            tol = ow.bound(ref, spread, mag, b.D, len(t), b.dtype, torch.finfo(b.dtype).eps / 2)
            worst = ((out[row, h * G:h * G + G].double() - ref).abs() / tol).max().item()
            assert worst <= 1, f"row {row} head {h}: {worst:.2f} of the bound"


@pytest.mark.parametrize("L,runs", [(130560, 256), (131328, 512)])
def test_full_runs(L, runs):
    """256 rows in four tiles a head, all keys selected: 65,232 tiles of 64 keys in 256 runs
    of 254 or 255, 65,616 in 512."""
    b = Batch([L - 256], [256], Hq=8, Hkv=8, D=64, seed=runs)
    plan = gs.plan_of(b, -(-L // 16), 0)
    assert plan.info["tiles"] == 4
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert plan.info["tile_workgroups"] == runs
    sel = whole_lists(b, -(-L // 16))
    args = (b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    out = sparse.sparse_attention(plan, *args)
    assert torch.isfinite(out).all()
    check_rows(b, out, sel, [0, 1, 31, 63, 64, 100, 127, 128, 160, 191, 192, 223, 254, 255])
    assert torch.equal(out, sparse.sparse_attention(plan, *args))
