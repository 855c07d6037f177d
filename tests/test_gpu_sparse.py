"""Key bounds, block selection and sparse attention on the GPU against the
64-bit oracle.  Bounds and selections are whole numbers and have to be equal;
attention keeps the error bound of oracle/window.py."""
import math

import pytest
import torch

import gllm_amd
from gllm_amd import paged, sparse
from oracle import kv4
from oracle import sparse as osp
from oracle import window as ow
from tests.window_helpers import BF, F8, F16, F32, Batch

pytestmark = pytest.mark.gpu


def plan_of(b, blocks, first=1, recent=1):
    return sparse.SparsePlan(b.ql, b.L, num_q_heads=b.Hq, num_kv_heads=b.Hkv, head_dim=b.D, block_size=b.bs, dtype=b.dtype,
                             device="cuda", q_seq_stride=b.stride, blocks=blocks, first_blocks=first, recent_blocks=recent)


def rows_of(b):
    """(sequence, row of q, position) of every query row."""
    return [(i, b.start[i] + r, c + r) for i, (c, n) in enumerate(zip(b.ctx, b.ql)) for r in range(n)]


def block_bounds(b, i, j):
    """The oracle's (codes, bytes) of block j of sequence i."""
    n = min(b.bs, b.L[i] - j * b.bs)
    return osp.key_bounds(b.rows(b.kc, i)[j * b.bs:j * b.bs + n])


def all_bounds(b, extra=0):
    """Records of every sequence's blocks as the oracle writes them; others are 0xAB."""
    rec = torch.full((b.nb, osp.record_bytes(b.Hkv, b.D) + extra), 0xAB, dtype=torch.uint8)
    out = {}
    for i, L in enumerate(b.L):
        for j in range(-(-L // b.bs)):
            out[i, j] = block_bounds(b, i, j)
            x = osp.record(*out[i, j])
            rec[int(b.bt[i, j]), :len(x)] = x
    return rec, out


def oracle_selection(b, bounds, blocks, first, recent):
    """{(row of q, KV head): selected blocks}"""
    sel = {}
    for i, row, p in rows_of(b):
        nb = p // b.bs + 1
        codes, byte = (torch.stack([bounds[i, j][x] for j in range(nb)]) for x in (0, 1))
        sc = osp.scores(b.q[row], codes, byte) if nb > blocks else torch.zeros(b.Hkv, nb)
        for h in range(b.Hkv):
            sel[row, h] = osp.select(sc[h], blocks, first, recent)
    return sel


def check_attention(b, out, sel, what=""):
    """out against the 64-bit attention over sel {(row, KV head): blocks}."""
    out = out.cpu().view(-1, b.Hq, b.D)
    scale, G = 1 / math.sqrt(b.D), b.Hq // b.Hkv
    p_bits = 2.0 ** -24 if b.dtype == F32 else 0.0
    mfma = b.dtype != F32 and b.D in (64, 128) and G <= 16 and b.kv in (b.dtype, F8, "4")
    if mfma:                                     # the weights enter P V in the model dtype
        p_bits = torch.finfo(b.dtype).eps / 2
    kv = [(b.rows(b.kc, i), b.rows(b.vc, i)) for i in range(len(b.L))]
    for i, row, p in rows_of(b):
        for h in range(b.Hkv):
            t = osp.keys_of(osp.listed(sel[row, h], p // b.bs), p, b.bs)
            heads = slice(h * G, (h + 1) * G)
            ref, spread, mag = osp.attention(b.q[row, heads], kv[i][0][t, h], kv[i][1][t, h], scale)
            got = out[row, heads].double()
            if not len(t):
                assert (got == 0).all(), f"{what}: row {row} head {h} without keys"
                continue
            tol = ow.bound(ref, spread, mag, b.D, len(t), b.dtype, p_bits)
            if mfma and b.dtype == F16:          # weights below 2^-14 of the largest are fp16 subnormals, 2^-25 off each
                tol = tol + len(t) * 2.0 ** -25 * 2 * kv[i][1][t, h].double().abs().max()
            assert torch.isfinite(got).all(), f"{what}: row {row} head {h} not finite"
            worst = ((got - ref).abs() / tol).max().item()
            assert worst <= 1, f"{what}: row {row} head {h}: {worst:.2f} of the bound"


# ---------------------------------------------------------------- key bounds
@pytest.mark.parametrize("Hkv,D,dtype,kv,bs", [
    (8, 128, BF, BF, 16), (8, 64, F16, F16, 16), (2, 128, F32, F32, 3), (2, 64, BF, F8, 24), (3, 96, F16, F8, 64),
    (1, 8, F32, F32, 1), (20, 128, BF, BF, 16), (5, 40, BF, F32, 7), (1, 256, F16, BF, 100), (2, 64, BF, "4", 16),
    (3, 96, F16, "4", 7), (2, 128, F32, "4", 24), (12, 256, F32, F16, 16)])
def test_bounds_are_the_oracles(Hkv, D, dtype, kv, bs):
    b = Batch([0, 99, 40, 15], [1, 1, 70, 1], Hq=Hkv, Hkv=Hkv, D=D, dtype=dtype, kv=kv, bs=bs, seed=D + bs)
    rec = torch.full((b.nb, osp.record_bytes(Hkv, D) + 32), 0xAB, dtype=torch.uint8).cuda()
    want = rec.cpu().clone()
    touched = {(i, j) for i, (c, n) in enumerate(zip(b.ctx, b.ql)) for j in range(c // bs, (c + n - 1) // bs + 1)}
    for i, j in touched:
        x = osp.record(*block_bounds(b, i, j))
        want[int(b.bt[i, j]), :len(x)] = x
    plan = plan_of(b, 4)
    sparse.write_key_bounds(plan, b.kc.cuda(), rec, b.bt.cuda())
    assert torch.equal(rec.cpu(), want)                       # neither padding nor other blocks are written
    # read back, also a block twice, in another order and outside the pool
    blocks = [int(b.bt[i, j]) for i, j in sorted(touched)][::-1]
    blocks += [blocks[0], -1, b.nb, 1 << 40]
    got = sparse.key_bounds_values(rec, torch.tensor(blocks).cuda(), Hkv, D).cpu()
    for x, blk in zip(got, blocks):
        if not 0 <= blk < b.nb:
            assert (x == 0).all()
            continue
        w = want[blk]
        codes = w[:Hkv * 2 * D].view(torch.int8).view(Hkv, 2, D)
        assert torch.equal(x.double(), osp.values(codes, w[Hkv * 2 * D:Hkv * 2 * D + Hkv].long()))


def test_bounds_of_special_values():
    """Infinities, NaN, the largest and least magnitudes, one sign only, zeros; and
    magnitudes at the border between two powers of two."""
    bs, Hkv, D = 16, 4, 64
    b = Batch([0], [bs * 8], Hq=Hkv, Hkv=Hkv, D=D, dtype=F32, bs=bs)
    blk = [int(b.bt[0, j]) * bs for j in range(8)]
    k = b.kc
    k[blk[0] + 3, 0, 5], k[blk[0] + 1, 1, 0], k[blk[0], 2, 1] = math.inf, math.nan, -math.inf
    k[blk[1]:blk[1] + bs, 0] = 0
    k[blk[1]:blk[1] + bs, 1] *= 1e-40
    k[blk[1]:blk[1] + bs, 2] = -k[blk[1]:blk[1] + bs, 2].abs()
    k[blk[2]:blk[2] + bs] = k[blk[2]:blk[2] + bs].clamp(-0.9, 0.9)
    for h, top in enumerate((127.0, math.nextafter(127.0, 128.0) + 1e-5, 63.5, 128.0)):
        k[blk[2] + h, h, 7] = -top
    k[blk[3], 0, 0], k[blk[3], 1, 0], k[blk[3], 2, 0], k[blk[3], 3, 0] = 127 * 2.0 ** 100, 128 * 2.0 ** 100, 3e38, -127 * 2.0 ** 100
    k[blk[4], 0, 0], k[blk[4], 0, 1], k[blk[4], 0, 2] = 2.0 ** 100, 2.0 ** -140, -2.0 ** -140   # beside a huge key
    k[blk[4] + 1:blk[4] + bs, 0, 1:3] = 0
    k[blk[4] + 1:blk[4] + bs, 0, 1], k[blk[4] + 1:blk[4] + bs, 0, 2] = 2.0 ** -145, -2.0 ** -145
    rec = sparse.new_key_bounds(b.nb, Hkv, D, "cuda")
    sparse.write_key_bounds(plan_of(b, 4), k.cuda(), rec, b.bt.cuda())
    for j in range(8):
        x = osp.record(*block_bounds(b, 0, j))
        assert torch.equal(rec[blk[j] // bs, :len(x)].cpu(), x), f"block {j}"


@pytest.mark.parametrize("dtype,kv", [(BF, BF), (F16, F16), (BF, F8), (F16, F32), (BF, "4")])
def test_one_nan_opens_its_block_and_head(dtype, kv):
    """In every type of cache: bounds of the other blocks and heads stay as they were.  F16
    over a float32 cache: a key that fp16 holds as infinity."""
    bs, Hkv, D = 16, 4, 64
    b = Batch([0, 5], [bs * 4, 40], Hq=Hkv, Hkv=Hkv, D=D, dtype=dtype, bs=bs, kv=kv)
    plan, kc, bt = plan_of(b, 4), b.kc.cuda(), b.bt.cuda()
    before, after = sparse.new_key_bounds(b.nb, Hkv, D, "cuda"), sparse.new_key_bounds(b.nb, Hkv, D, "cuda")
    sparse.write_key_bounds(plan, kc, before, bt)
    blk = int(b.bt[0, 2])
    if kv == "4":
        kc[blk, 1, bs * D // 2 + 7 * D // 32 + 1] = 255      # the scale of dims 32-63 of key 7
    elif kv == F8:
        kc.view(torch.uint8)[blk * bs + 7, 1, 33] = 0x7F
    else:
        kc[blk * bs + 7, 1, 33] = 1e6 if kv == F32 else math.nan
    sparse.write_key_bounds(plan, kc, after, bt)
    want = before.clone()
    want[blk, 1 * 2 * D:2 * 2 * D] = 0
    want[blk, Hkv * 2 * D + 1] = 255
    assert torch.equal(after, want)


# ---------------------------------------------------------------- selection
def check_selection(b, rec, bounds, blocks, first, recent, padded=True):
    plan = plan_of(b, blocks, first, recent)
    out = torch.full((plan.rows, b.Hkv, blocks), -7, dtype=torch.int32, device="cuda")
    got = sparse.select_blocks(plan, b.q.cuda(), rec.cuda(), b.bt.cuda(), out=out).cpu()
    want = oracle_selection(b, bounds, blocks, first, recent)
    for i, row, p in rows_of(b):
        for h in range(b.Hkv):
            w = want[row, h]
            assert got[row, h].tolist() == w + [-1] * (blocks - len(w)), f"row {row} (position {p}) head {h}"
    real = {row for _, row, _ in rows_of(b)}
    for row in range(plan.rows):
        if row not in real:
            assert (got[row] == -7).all()
    return plan, want


@pytest.mark.parametrize("Hq,Hkv,D,dtype,bs,blocks,first,recent", [
    (8, 2, 64, BF, 16, 6, 1, 1), (32, 8, 128, BF, 16, 9, 1, 2), (8, 8, 128, F16, 3, 20, 0, 1), (6, 2, 96, F32, 7, 5, 2, 3),
    (16, 2, 40, BF, 1, 33, 1, 1), (16, 1, 256, F16, 16, 2, 1, 1), (40, 2, 64, BF, 16, 4, 0, 4), (64, 2, 128, F32, 24, 3, 0, 1),
    (5, 1, 8, BF, 16, 7, 1, 1), (20, 4, 72, F32, 2, 50, 3, 2), (24, 2, 64, F16, 16, 600, 1, 1)])
def test_selection_is_the_oracles(Hq, Hkv, D, dtype, bs, blocks, first, recent):
    b = Batch([0, 400, 95, 777], [1, 1, 9, 3], Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, bs=bs, seed=Hq + D)
    check_selection(b, *all_bounds(b), blocks, first, recent)


@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(4, 4, 64, BF), (4, 2, 128, F16), (12, 4, 128, BF), (8, 2, 64, BF), (8, 1, 128, F32),
                                            (20, 2, 40, F16), (16, 1, 96, BF), (20, 1, 64, BF), (8, 2, 256, BF)])
def test_selection_of_prompt_rows_in_tiles(Hq, Hkv, D, dtype):
    """Prompts of every remainder of a tile's rows beside single rows, in one plan."""
    b = Batch([400, 300, 250, 500, 260, 333, 290], [1, 31, 5, 1, 17, 3, 66], Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, bs=4, seed=Hq + D)
    rec, bounds = all_bounds(b)
    check_selection(b, rec, bounds, 9, 1, 2)


def test_selection_of_padded_rows_and_strided_tensors():
    b = Batch([300, 0, 500], [2, 1, 4], Hq=8, Hkv=2, D=64, bs=16, stride=5)
    rec, bounds = all_bounds(b, extra=48)
    plan, want = check_selection(b, rec, bounds, 8, 1, 1)
    # rows of a wider tensor, a wider table
    wide = torch.randn(plan.rows, 12, 64).to(BF).cuda()
    wide[:, 2:10] = b.q.cuda()
    bt = torch.full((5, 60), -3, dtype=torch.int32).cuda()
    bt[:3, :b.bt.shape[1]] = b.bt.cuda()
    got = sparse.select_blocks(plan, wide[:, 2:10], rec.cuda(), bt[:3])
    for (row, h), w in want.items():
        assert got[row, h].tolist() == w + [-1] * (8 - len(w))


def test_equal_scores_go_to_the_lower_block():
    b = Batch([16 * 40 - 1], [1], Hq=4, Hkv=2, D=64, bs=16)
    g = torch.Generator().manual_seed(5)
    kinds = torch.randn(3, 16, 2, 64, generator=g).to(BF)
    for j in range(40):                               # three kinds of blocks
        blk = int(b.bt[0, j]) * 16
        b.kc[blk:blk + 16] = kinds[j * j % 3]
    rec, bounds = all_bounds(b)
    for blocks in (3, 7, 14, 20, 39):
        check_selection(b, rec, bounds, blocks, 1, 1)


def test_selection_with_open_blocks_and_odd_queries():
    b = Batch([16 * 30 - 1, 16 * 30 - 1, 16 * 30 - 1, 16 * 30 - 1], [1] * 4, Hq=8, Hkv=2, D=64, bs=16, dtype=F32)
    for i in range(4):
        for j, x in ((5, math.inf), (11, math.nan), (20, 3e38)):
            b.kc[int(b.bt[i, j]) * 16 + j % 16, i % 2, j] = x
    b.q[1, :4] = 0                                    # all scores 0: the lowest blocks
    b.q[2, 1, 3] = math.nan
    b.q[3, 5, 3], b.q[3, 0] = math.inf, b.q[3, 0] * 1e-42
    rec, bounds = all_bounds(b)
    for blocks in (4, 2, 3, 10):
        check_selection(b, rec, bounds, blocks, 0, 1)


@pytest.mark.parametrize("L,blocks", [(2048, 100), (2049, 1), (5000, 2000), (8192, 64), (8193, 64), (20001, 300)])
def test_selection_among_many_blocks(L, blocks):
    """Either side of the numbers of blocks that the kernel holds in registers;
    whole-number keys, so that many scores are equal."""
    g = torch.Generator().manual_seed(L)
    D = 64
    k = torch.randint(-2, 3, (L, 1, D), generator=g).float()
    k[:, :, 3:] = 0
    q = torch.randint(-9, 10, (1, 2, D), generator=g).float()
    plan = sparse.SparsePlan([1], [L], num_q_heads=2, num_kv_heads=1, head_dim=D, block_size=1, dtype=F32, device="cuda",
                             blocks=blocks, first_blocks=0)
    full = sparse.SparsePlan([L], [L], num_q_heads=2, num_kv_heads=1, head_dim=D, block_size=1, dtype=F32, device="cuda",
                             blocks=blocks, first_blocks=0)
    bt = torch.randperm(L, generator=g).to(torch.int32)[None]
    kc = torch.empty_like(k)
    kc[bt[0].long()] = k
    rec = sparse.new_key_bounds(L, 1, D, "cuda")
    sparse.write_key_bounds(full, kc.cuda(), rec, bt.cuda())
    got = sparse.select_blocks(plan, q.cuda(), rec, bt.cuda())[0, 0].tolist()
    # one key a block, lo = hi: codes k / 2^e, e = -6 for 1, -5 for 2; the dot product is exact
    c = osp.query_codes(q[0])
    sc = (c @ k[:, 0].double().t()).amax(0)
    assert got == osp.select(sc, blocks, 0, 1)


# ---------------------------------------------------------------- attention
def random_lists(b, blocks, seed, whole=False):
    """Lists of every kind: full, short, empty, without the own block, out of order,
    repeated, negative in the middle, behind the row."""
    g = torch.Generator().manual_seed(seed)
    rows = len(b.ql) * b.stride if b.stride else sum(b.ql)
    sel = torch.full((rows, b.Hkv, blocks), -1, dtype=torch.int32)
    k = 0
    for i, row, p in rows_of(b):
        own = p // b.bs
        for h in range(b.Hkv):
            n = min(blocks, own + 1)
            s = torch.randperm(own + 1, generator=g)[:n].sort().values.to(torch.int32)
            if whole or k % 8 == 0:
                s[-1] = own
            if not whole and k % 8 == 1:
                s = s[:n // 2]
            if not whole and k % 8 == 2:
                s = s[:0]
            if not whole and k % 8 == 3 and n > 2:
                s[n // 2] = s[n // 2 - 1]
            if not whole and k % 8 == 4 and n > 2:
                s[n // 2] = -1
            if not whole and k % 8 == 5 and n > 2:
                s[-1] = own + 1 + int(torch.randint(0, 1 << 20, (1,), generator=g))
            if not whole and k % 8 == 6 and n > 3:
                s = s.flip(0)
            sel[row, h, :len(s)] = s
            k += 1
    return sel


CASES = [
    (8, 2, 64, BF, BF, 16), (32, 8, 128, BF, BF, 16), (8, 1, 128, F16, F16, 3), (16, 2, 64, F16, F8, 24), (4, 4, 128, BF, F8, 64),
    (16, 1, 64, BF, BF, 1), (32, 2, 128, BF, "4", 16), (6, 2, 64, F16, "4", 7), (6, 3, 96, F32, F32, 16), (8, 2, 64, F32, F8, 5),
    (40, 2, 64, BF, BF, 16), (4, 2, 40, F16, F32, 16), (2, 1, 256, BF, F16, 8), (4, 2, 96, F32, "4", 16), (5, 1, 8, F32, F32, 2)]


@pytest.mark.parametrize("Hq,Hkv,D,dtype,kv,bs", CASES)
@pytest.mark.parametrize("blocks", [1, 5, 40])
def test_attention_over_any_lists(Hq, Hkv, D, dtype, kv, bs, blocks):
    b = Batch([0, 400, 95, 16, 777], [1, 1, 5, 2, 1], Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, kv=kv, bs=bs, seed=Hq + D + bs)
    sel = random_lists(b, blocks, blocks)
    out = sparse.sparse_attention(plan_of(b, blocks, 0), b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    check_attention(b, out, {(row, h): sel[row, h].tolist() for _, row, _ in rows_of(b) for h in range(Hkv)})


@pytest.mark.parametrize("Hq,Hkv,D,dtype,kv,bs", [
    (8, 2, 64, BF, BF, 16), (8, 2, 128, BF, BF, 32), (16, 2, 128, F16, F16, 16), (4, 1, 64, F16, F8, 48), (6, 2, 128, BF, F8, 16),
    (8, 1, 128, BF, "4", 16), (32, 2, 64, BF, "4", 32), (2, 2, 64, BF, BF, 16), (12, 1, 128, F16, F16, 112)])
def test_prompt_rows_in_tiles(Hq, Hkv, D, dtype, kv, bs):
    """Chunks whose rows attend in tiles, beside rows on their own: any lists, whole ones
    and rows that all miss some tiles of keys."""
    b = Batch([500, 0, 900, 333], [70, 40, 1, 3], Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, kv=kv, bs=bs, seed=Hq + bs)
    plan = plan_of(b, 9, 0)
    assert plan.info["tiles"] >= 2
    for seed, whole in ((1, False), (2, True)):
        sel = random_lists(b, 9, seed, whole)
        if whole:
            sel[5:40, 0] = torch.where(sel[5:40, 0] > 3, -1, sel[5:40, 0])     # only early blocks
            sel[45:60] = -1
        out = sparse.sparse_attention(plan, b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
        check_attention(b, out, {(row, h): sel[row, h].tolist() for _, row, _ in rows_of(b) for h in range(Hkv)}, f"seed {seed}")


@pytest.mark.parametrize("ctx,rows,blocks", [(40000, 64, 20), (70000, 20, 12), (3000, 200, 3)])
@pytest.mark.parametrize("kv", [BF, F8])
def test_tiles_of_many_blocks(ctx, rows, blocks, kv):
    """More blocks than a workgroup caches (the keys in parts) and than are marked at a
    time; no row of a tile left out of the parts' joining."""
    b = Batch([ctx], [rows], Hq=4, Hkv=1, D=64, kv=kv, bs=16, seed=ctx)
    plan = plan_of(b, blocks, 0)
    assert plan.info["tiles"] >= 1 and (ctx < 10000 or plan.info["tile_workgroups"] > 1)
    sel = random_lists(b, blocks, 7, whole=True)
    sel[rows // 2] = -1
    args = (b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    out = sparse.sparse_attention(plan, *args)
    check_attention(b, out, {(r, 0): sel[r, 0].tolist() for r in range(rows)})
    assert torch.equal(out, sparse.sparse_attention(plan, *args))


@pytest.mark.parametrize("ql,Hkv,blocks", [([300] * 3, 2, 8), ([64] * 70, 8, 6), ([20] * 160, 2, 8), ([100, 1, 1000], 4, 3)])
def test_runs_that_cut_and_span_tiles(ql, Hkv, blocks):
    """Fewer (tile, KV head) units than runs of keys and more; units without keys between
    others; rows of every part."""
    b = Batch([700 + 37 * (i % 5) for i in range(len(ql))], ql, Hq=2 * Hkv, Hkv=Hkv, D=64, bs=16, seed=sum(ql))
    plan = plan_of(b, blocks, 0)
    assert plan.info["tiles"] >= 2
    sel = random_lists(b, blocks, 3, whole=True)
    sel[b.start[1]:b.start[1] + b.ql[1], 0] = -1
    out = sparse.sparse_attention(plan, b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    check_attention(b, out, {(row, h): sel[row, h].tolist() for _, row, _ in rows_of(b) for h in range(Hkv)})


def test_tiles_do_not_read_behind_the_last_row():
    """NaN behind the sequence's end, and in every block that no row selected."""
    b = Batch([700], [50], Hq=8, Hkv=2, D=128, bs=32)
    plan = plan_of(b, 6, 0)
    assert plan.info["tiles"] >= 1
    sel = random_lists(b, 6, 1, whole=True) % 14
    sel = torch.where(sel < 0, -1, sel).sort(-1).values
    sel[..., -1] = torch.tensor([p // 32 for _, _, p in rows_of(b)], dtype=torch.int32)[:, None]
    args = (b.q.cuda(), b.bt.cuda(), sel.cuda())
    out = sparse.sparse_attention(plan, args[0], b.kc.cuda(), b.vc.cuda(), args[1], args[2])
    check_attention(b, out, {(r, h): sel[r, h].tolist() for r in range(50) for h in range(2)})
    kc, vc, bt = b.kc.clone(), b.vc.clone(), b.bt.clone()
    used = {int(x) for x in sel.flatten()} | {p // 32 for _, _, p in rows_of(b)}
    seen = torch.zeros(b.nb * 32, dtype=torch.bool)
    for j in range(-(-750 // 32)):
        if j in used:
            n = min(32, 750 - 32 * j)
            seen[int(bt[0, j]) * 32:int(bt[0, j]) * 32 + n] = True
        else:
            bt[0, j] = (-1, 1 << 30)[j % 2]
    assert not seen.all()
    kc[~seen], vc[~seen] = math.nan, math.nan
    assert torch.equal(out, sparse.sparse_attention(plan, args[0], kc.cuda(), vc.cuda(), bt.cuda(), args[2]))


@pytest.mark.parametrize("D,kv", [(64, BF), (128, BF), (64, F8), (128, "4")])
def test_attention_in_splits(D, kv):
    """One long row: its keys are split over workgroups; short and empty lists leave
    splits without keys."""
    b = Batch([5000, 9000], [1, 1], Hq=4, Hkv=2, D=D, kv=kv, bs=16)
    plan = plan_of(b, 300, 0)
    assert plan.info["splits"] > 1
    sel = random_lists(b, 300, 3, whole=True)
    sel[0, 1, 20:] = -1
    sel[1, 0] = -1
    args = (b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    out = sparse.sparse_attention(plan, *args)
    check_attention(b, out, {(r, h): sel[r, h].tolist() for r in range(2) for h in range(2)})
    assert torch.equal(out, sparse.sparse_attention(plan, *args))


@pytest.mark.parametrize("rows", [1, 40])
def test_lists_longer_than_a_task_caches(rows):
    """More than 512 entries a list: looked up part by part."""
    b = Batch([9000] * rows, [1] * rows, Hq=4, Hkv=2, D=64, bs=8, seed=rows)
    sel = random_lists(b, 700, 5, whole=True)
    sel[0, 1, 600:] = -1
    out = sparse.sparse_attention(plan_of(b, 700, 0), b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    part = Batch.__new__(Batch)
    part.__dict__.update(b.__dict__, ql=b.ql[:2], ctx=b.ctx[:2], L=b.L[:2])
    check_attention(part, out, {(r, h): sel[r, h].tolist() for r in range(rows) for h in range(2)})


def test_all_blocks_are_all_keys():
    """Where a row selects every block, the result is paged attention's."""
    b = Batch([200, 0, 77], [3, 1, 1], Hq=8, Hkv=2, D=64, bs=16)
    plan = plan_of(b, 20)
    args = (b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda())
    sel = sparse.select_blocks(plan, args[0], sparse.new_key_bounds(b.nb, 2, 64, "cuda"), args[3])
    b.check(sparse.sparse_attention(plan, *args, sel), None, 0)


def test_unselected_blocks_are_not_read():
    """NaN in every block that is not selected, ids outside the pool for them, and
    NaN behind the row's position in its own."""
    b = Batch([600, 333], [1, 1], Hq=8, Hkv=2, D=128, bs=16)
    sel = random_lists(b, 7, 1, whole=True)
    out = sparse.sparse_attention(plan_of(b, 7, 0), b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda(), sel.cuda())
    bt, kc, vc = b.bt.clone(), b.kc.clone(), b.vc.clone()
    seen = torch.zeros(b.nb * 16, 2, dtype=torch.bool)
    for i in range(2):
        used = {int(x) for x in sel[i].flatten()}
        for h in range(2):
            t = osp.keys_of(sel[i, h].tolist(), b.ctx[i], 16)
            seen[b.bt[i, t // 16].long() * 16 + t % 16, h] = True
        for j in range(-(-b.L[i] // 16)):
            if j not in used:
                bt[i, j] = (-1, 1 << 30)[j % 2]
    kc[~seen], vc[~seen] = math.nan, math.nan
    assert torch.equal(out, sparse.sparse_attention(plan_of(b, 7, 0), b.q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), sel.cuda()))


def test_rows_that_are_left_alone_and_strides():
    b = Batch([300, 0, 500], [2, 1, 4], Hq=8, Hkv=2, D=64, bs=16, stride=5)
    plan, sel = plan_of(b, 6, 0), random_lists(b, 6, 2)
    q = torch.zeros(plan.rows + 2, 9, 64, dtype=BF, device="cuda")
    q[:plan.rows, :8] = b.q.cuda()
    out = torch.full((plan.rows + 2, 10, 64), 7.0, dtype=BF, device="cuda")
    # caches of wider slots
    pool = torch.full((2, b.nb * 16, 3, 64), math.nan, dtype=BF, device="cuda")
    pool[0, :, :2], pool[1, :, :2] = b.kc.cuda(), b.vc.cuda()
    got = sparse.sparse_attention(plan, q[:, :8], pool[0, :, :2], pool[1, :, :2], b.bt.cuda(), sel.cuda(), out=out[:, 1:9])
    assert got.data_ptr() == out[:, 1:9].data_ptr()
    real = [row for _, row, _ in rows_of(b)]
    check_attention(b, out[:plan.rows, 1:9].contiguous(),
                    {(row, h): sel[row, h].tolist() for row in real for h in range(2)})
    out[real, 1:9] = 7.0
    assert (out == 7.0).all()


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype,kv,D", [(BF, BF, 128), (F16, F8, 64), (BF, "4", 64), (F32, F32, 64)])
def test_decode_steps_with_rotary_writes(dtype, kv, D):
    """Steps of a layer as an engine runs them: keys rotated and written, bounds,
    selection, attention; each step against the oracle on what the cache holds."""
    lens = [197, 25, 70]                             # their next three keys lie in blocks that they have
    b = Batch(lens, [1, 1, 1], Hq=8, Hkv=2, D=D, dtype=dtype, kv=kv, bs=16, seed=9)
    rotary = gllm_amd.Rotary(D, theta=10000.0, device="cuda")
    kc, vc, bt = b.kc.cuda(), b.vc.cuda(), b.bt.cuda()
    bounds = sparse.new_key_bounds(b.nb, 2, D, "cuda")
    g = torch.Generator().manual_seed(11)
    prompts = sparse.SparsePlan(lens, lens, num_q_heads=8, num_kv_heads=2, head_dim=D, block_size=16, dtype=dtype,
                                device="cuda", blocks=4)
    sparse.write_key_bounds(prompts, kc, bounds, bt)
    for step in range(3):
        c = [x + step for x in lens]
        q, k, v = (torch.randn(3, h, D, generator=g).to(dtype) for h in (8, 2, 2))
        pos = torch.tensor(c)
        slots = (b.bt[torch.arange(3), pos // 16].long() * 16 + pos % 16).cuda()
        qr = torch.empty_like(q, device="cuda")
        paged.rotary_kv_write(k.cuda(), v.cuda(), pos.cuda(), rotary, kc, vc, slots, q=q.cuda(), q_out=qr)
        now = Batch(c, [1, 1, 1], Hq=8, Hkv=2, D=D, dtype=dtype, kv=kv, bs=16)
        now.bt, now.q, now.kc, now.vc, now.nb = b.bt, qr.cpu(), kc.cpu(), vc.cpu(), b.nb
        plan = plan_of(now, 4)
        sparse.write_key_bounds(plan, kc, bounds, bt)
        sel = sparse.select_blocks(plan, qr, bounds, bt)
        out = sparse.sparse_attention(plan, qr, kc, vc, bt, sel)
        want = oracle_selection(now, all_bounds(now)[1], 4, 1, 1)
        assert {(r, h): [x for x in sel[r, h].tolist() if x >= 0] for r in range(3) for h in range(2)} == want, f"step {step}"
        check_attention(now, out, want, f"step {step}")


def test_replays_of_a_captured_step():
    """A step in a graph, replayed with new inputs and the caller's own work between."""
    b = Batch([900, 500], [1, 1], Hq=8, Hkv=2, D=64, bs=16)
    plan = plan_of(b, 12)
    q, kc, vc, bt = b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda()
    rec, _ = all_bounds(b)
    bounds = rec.cuda()
    sel = torch.empty(2, 2, 12, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def step(o):
        sparse.write_key_bounds(plan, kc, bounds, bt)
        sparse.select_blocks(plan, q, bounds, bt, out=sel)
        return sparse.sparse_attention(plan, q, kc, vc, bt, sel, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    gen = torch.Generator().manual_seed(3)
    for i in range(4):
        q.copy_(torch.randn(2, 8, 64, generator=gen).to(BF))
        for s, L in enumerate(b.L):                # the newest key
            kc[int(b.bt[s, (L - 1) // 16]) * 16 + (L - 1) % 16] = torch.randn(2, 64, generator=gen).to(BF).cuda() * (i + 1)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone(), sel.clone()
        want = step(torch.empty_like(q))
        assert torch.equal(replayed[0], want) and torch.equal(replayed[1], sel), f"replay {i}"


def test_replays_of_captured_prompt_tiles():
    """Lists that change between replays move the runs of keys and the tiles that they
    cut: each replay is the eager call's, bit for bit."""
    b = Batch([1500, 300, 700], [130, 1, 70], Hq=8, Hkv=2, D=128, bs=16)
    plan = plan_of(b, 8, 0)
    assert plan.info["tiles"] >= 3
    q, kc, vc, bt = b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda()
    lists = [random_lists(b, 8, seed, seed % 2 == 0).cuda() for seed in range(4)]
    lists += [torch.full_like(lists[0], -1), torch.where(lists[0] > 5, -1, lists[0])]
    sel, out = lists[0].clone(), torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sparse.sparse_attention(plan, q, kc, vc, bt, sel, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sparse.sparse_attention(plan, q, kc, vc, bt, sel, out=out)
    for k, x in enumerate(lists + lists[::-1]):
        sel.copy_(x)
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        want = sparse.sparse_attention(plan, q, kc, vc, bt, x)
        assert torch.equal(replayed, want), f"replay {k}"
        if k < len(lists):
            check_attention(b, want, {(row, h): x[row, h].tolist() for _, row, _ in rows_of(b) for h in range(2)}, f"lists {k}")


def test_calls_on_another_stream():
    b = Batch([900, 500], [1, 1], Hq=8, Hkv=2, D=64, bs=16)
    q, kc, vc, bt = b.q.cuda(), b.kc.cuda(), b.vc.cuda(), b.bt.cuda()
    rec, _ = all_bounds(b)
    bounds = rec.cuda()
    plans = [plan_of(b, 12), plan_of(b, 12)]
    want = sparse.sparse_attention(plans[0], q, kc, vc, bt, sparse.select_blocks(plans[0], q, bounds, bt))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i, stream in enumerate((torch.cuda.current_stream(), side)):       # a plan each: the workspaces differ
        with torch.cuda.stream(stream):
            outs.append(sparse.sparse_attention(plans[i], q, kc, vc, bt, sparse.select_blocks(plans[i], q, bounds, bt)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_slabs_of_rows():
    """More scores than fit at a time: rows are scored and selected in slabs, each
    as a plan of those rows alone would."""
    D, L, n = 8, 70000, 1100                          # bs 1: 70,000 blocks, 280 KB of scores a row
    g = torch.Generator().manual_seed(4)
    k = torch.randn(L, 1, D, generator=g).cuda()
    q = torch.randn(n, 1, D, generator=g).cuda()
    bt = torch.arange(L, dtype=torch.int32, device="cuda")[None]
    args = dict(num_q_heads=1, num_kv_heads=1, head_dim=D, block_size=1, dtype=F32, device="cuda", blocks=5)
    rec = sparse.new_key_bounds(L, 1, D, "cuda")
    sparse.write_key_bounds(sparse.SparsePlan([L], [L], **args), k, rec, bt)
    plan = sparse.SparsePlan([n], [L], **args)
    assert plan.info["slabs"] == 2
    got = sparse.select_blocks(plan, q, rec, bt)
    for r0, r1 in ((0, 3), (955, 962), (1097, 1100)):
        part = sparse.SparsePlan([r1 - r0], [L - n + r1], **args)
        assert part.info["slabs"] == 1
        assert torch.equal(sparse.select_blocks(part, q[r0:r1], rec, bt), got[r0:r1])


def test_many_blocks_a_wave():
    """So many rows of many blocks that a wave takes more than 16 groups of blocks: each
    row as in a plan of its own."""
    D, L, n, Hkv = 8, 2100, 80, 8
    g = torch.Generator().manual_seed(6)
    k = torch.randn(L, Hkv, D, generator=g).cuda()
    q = torch.randn(n, Hkv, D, generator=g).cuda()
    bt = torch.randperm(L, generator=g).to(torch.int32)[None].expand(n, -1).contiguous().cuda()
    args = dict(num_q_heads=Hkv, num_kv_heads=Hkv, head_dim=D, block_size=1, dtype=F32, device="cuda", blocks=40)
    rec = sparse.new_key_bounds(L, Hkv, D, "cuda")
    sparse.write_key_bounds(sparse.SparsePlan([L], [L], **args), k, rec, bt)
    lens = [L - i for i in range(n)]
    got = sparse.select_blocks(sparse.SparsePlan([1] * n, lens, **args), q, rec, bt)
    for r in (0, 1, 33, 79):
        assert torch.equal(sparse.select_blocks(sparse.SparsePlan([1], lens[r:r + 1], **args), q[r:r + 1], rec, bt)[0], got[r])
    # against the definition: one key a block, its codes the same at both ends
    c = osp.query_codes(q[5, 3:4].cpu())
    keys = k[bt[0, :lens[5]].long(), 3].cpu()
    sc = []
    for x in keys:
        codes, byte = osp.key_bounds(x[None, None])
        sc.append(torch.maximum(c * codes[0, 0], c * codes[0, 1]).sum() * 2.0 ** (int(byte) - 128))
    assert got[5, 3].tolist() == osp.select(torch.stack(sc), 40, 1, 1)


def test_blocks_past_4_gib():
    """Places past 2^32 bytes in the cache and in the bounds."""
    bs, Hkv, D = 16, 8, 128
    nb = (1 << 32) // (bs * Hkv * D * 2) + 2000
    kc = torch.zeros(nb * bs, Hkv, D, dtype=BF, device="cuda")
    vc = torch.zeros_like(kc)
    bounds = torch.zeros(nb, 1 << 15, dtype=torch.uint8, device="cuda")     # records 32 KB apart: past 2^32 too
    b = Batch([16 * 30 - 1], [1], Hq=8, Hkv=Hkv, D=D, bs=bs)
    far = (nb - 1 - torch.arange(30) * 60).to(torch.int32)
    for j in range(30):
        src, dst = int(b.bt[0, j]) * bs, int(far[j]) * bs
        kc[dst:dst + bs], vc[dst:dst + bs] = b.kc[src:src + bs].cuda(), b.vc[src:src + bs].cuda()
    bt, q = far[None].cuda(), b.q.cuda()
    whole = Batch([0], [16 * 30], Hq=8, Hkv=Hkv, D=D, bs=bs)
    sparse.write_key_bounds(plan_of(whole, 8), kc, bounds, bt)
    plan = plan_of(b, 8)
    sel = sparse.select_blocks(plan, q, bounds, bt)
    want = oracle_selection(b, all_bounds(b)[1], 8, 1, 1)
    assert {(0, h): sel[0, h].tolist() for h in range(Hkv)} == want
    check_attention(b, sparse.sparse_attention(plan, q, kc, vc, bt, sel), want)


def test_empty_batch():
    plan = sparse.SparsePlan([], [], num_q_heads=8, num_kv_heads=2, head_dim=64, block_size=16, dtype=BF, device="cuda", blocks=3)
    q = torch.zeros(0, 8, 64, dtype=BF, device="cuda")
    kc, bt = torch.zeros(32, 2, 64, dtype=BF, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    bounds = sparse.new_key_bounds(2, 2, 64, "cuda")
    sparse.write_key_bounds(plan, kc, bounds, bt)
    sel = sparse.select_blocks(plan, q, bounds, bt)
    assert sel.shape == (0, 2, 3) and sparse.sparse_attention(plan, q, kc, kc, bt, sel).shape == q.shape
    for none in (bt[:0], bt[:0, :0]):
        sparse.write_key_bounds(plan, kc, bounds, none)
        sel = sparse.select_blocks(plan, q, bounds, none)
        assert sel.shape == (0, 2, 3) and sparse.sparse_attention(plan, q, kc, kc, none, sel).shape == q.shape
    assert sparse.key_bounds_values(bounds, torch.zeros(0, dtype=torch.int64, device="cuda"), 2, 64).shape == (0, 2, 2, 64)
