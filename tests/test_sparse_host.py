"""Sparse attention and shared prefixes on the CPU: the oracle from its
definition, the planners, and what the entry points refuse."""
import ctypes
import math

import pytest
import torch

from gllm_amd import _lib, paged, sparse
from oracle import sparse as osp


def test_exponents_at_their_borders():
    assert osp.exponent(0.0) == -100 and osp.exponent(127 * 2.0 ** -100) == -100
    assert osp.exponent(127.0) == 0 and osp.exponent(math.nextafter(127.0, 200)) == 1 and osp.exponent(63.5) == -1
    assert osp.exponent(127 * 2.0 ** 100) == 100 and osp.exponent(127.01 * 2.0 ** 100) is None
    assert osp.exponent(math.inf) is None and osp.exponent(math.nan) is None


def test_bounds_hold_every_key():
    g = torch.Generator().manual_seed(0)
    k = torch.randn(9, 3, 16, generator=g) * torch.exp2(torch.randint(-20, 20, (1, 3, 1), generator=g).float())
    k[:, 1] = -k[:, 1].abs()                 # a head of negative keys only
    codes, byte = osp.key_bounds(k)
    box = osp.values(codes, byte)
    assert (box[:, 0] <= k.double().amin(0)).all() and (box[:, 1] >= k.double().amax(0)).all()
    assert codes.abs().max() <= 127 and codes.abs().amax((1, 2)).min() >= 64
    # off by less than one step of the code
    step = torch.exp2(byte.double() - 128)[:, None]
    assert (k.double().amin(0) - box[:, 0] < step).all() and (box[:, 1] - k.double().amax(0) < step).all()
    assert osp.record(codes, byte).numel() == 3 * 33 and osp.record_bytes(3, 16) == 112


def test_open_blocks():
    k = torch.ones(4, 3, 8)
    k[1, 0, 3], k[2, 1, 0] = math.nan, -math.inf
    codes, byte = osp.key_bounds(k)
    assert byte.tolist() == [255, 255, 128 - 6] and (codes[:2] == 0).all() and (codes[2] == 64).all()
    assert (osp.values(codes, byte)[0, 0] == -math.inf).all() and (osp.values(codes, byte)[1, 1] == math.inf).all()


def test_no_key_scores_above_its_block():
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(6, 32, generator=g) * 3, torch.randn(5, 8, 2, 32, generator=g)
    b = [osp.key_bounds(x) for x in k]
    codes, byte = torch.stack([x[0] for x in b]), torch.stack([x[1] for x in b])
    sc = osp.scores(q, codes, byte)
    for h in range(2):
        c = osp.query_codes(q.view(2, 3, 32)[h])
        assert c.abs().max() <= 127
        assert ((c @ k[:, :, h].double().reshape(-1, 32).t()).view(3, 5, 8).amax((0, 2)) <= sc[h]).all()


def test_selection():
    s = torch.tensor([5.0, 1, 7, 7, 7, -3, 2, 9])
    assert osp.select(s, 8, 1, 1) == list(range(8)) and osp.select(s[:3], 5, 1, 1) == [0, 1, 2]
    assert osp.select(s, 4, 1, 1) == [0, 2, 3, 7]          # of three equal ones the first two
    assert osp.select(s, 4, 0, 1) == [2, 3, 4, 7]
    assert osp.select(s, 3, 1, 2) == [0, 6, 7]
    s[5] = math.inf
    assert osp.select(s, 3, 1, 1) == [0, 5, 7]
    assert osp.listed([1, 4, 4, 6], 9) == [1, 4] and osp.listed([3, 2], 9) == [3] and osp.listed([-1, 2], 9) == []
    assert osp.listed([1, 10], 9) == [1] and osp.listed([0, 9], 9) == [0, 9]
    assert osp.keys_of([0, 2], 9, 4).tolist() == [0, 1, 2, 3, 8, 9] and osp.keys_of([], 9, 4).numel() == 0


def _info(ql, sl, Hq=32, Hkv=8, D=128, bs=16, dtype=_lib.DTYPE_BF16, stride=0, blocks=64, first=1, recent=1):
    lib, h, info = _lib.load(), ctypes.c_void_p(), (ctypes.c_int64 * 6)()
    n = len(ql)
    rc = lib.gllm_sparse_plan_create(ctypes.byref(h), (ctypes.c_int32 * n)(*ql), (ctypes.c_int32 * n)(*sl), n, stride, Hq, Hkv,
                                     D, bs, dtype, blocks, first, recent)
    if rc:
        assert not h.value
        return rc, lib.gllm_attn_last_error().decode()
    assert lib.gllm_sparse_plan_info(h, info, 6) == 0
    size = lib.gllm_sparse_plan_workspace_bytes(h)
    assert lib.gllm_sparse_plan_destroy(h) == 0
    return dict(zip(("rows", "query_rows", "blocks", "tiles", "slabs", "splits"), info)) | {"bytes": size}


def test_plan_facts():
    i = _info([1, 3, 40], [100, 5000, 4096])
    assert i["rows"] == i["query_rows"] == 44 and i["slabs"] == 1
    # the last key's block; keys 4997 .. 4999 (block 312); 4056 .. 4095 (blocks 253 .. 255)
    assert i["blocks"] == 1 + 1 + 3
    # 4 rows a tile at G = 4, twice as many where a sequence has more; the first has 7 blocks,
    # all selected
    assert i["tiles"] == 1 + 5
    assert _info([1, 3, 4], [100, 5000, 4096])["tiles"] == 1 + 1
    assert _info([1, 3, 40], [100, 5000, 4096], Hq=8)["tiles"] == 1 + 2       # 16 rows
    assert _info([1, 3, 40], [100, 5000, 4096], D=192)["tiles"] == 1 + 10
    assert _info([1, 3, 40], [100, 5000, 4096], Hq=256)["tiles"] == 3 + 40
    assert _info([1, 3, 40], [100, 5000, 4096], blocks=400)["tiles"] == 0
    assert _info([3, 1], [10, 20], stride=5) | {"bytes": 0} == dict(rows=10, query_rows=4, blocks=2, tiles=0, slabs=1, splits=1, bytes=0)
    assert _info([], [])["rows"] == 0
    # scores stay at 256 MiB: 8 heads x 8192 blocks x 4 bytes a row
    i = _info([4096], [131072], blocks=64)
    assert i["slabs"] == 4 and i["bytes"] < (256 << 20) + (2 << 20)


def _tiles(ql, sl, **kw):
    p = _plan(ql, sl, num_q_heads=32, num_kv_heads=8, head_dim=128, **kw)
    return p.info["tiles"], p.info["tile_workgroups"], p.workspace.numel()


def test_prompt_rows_go_in_tiles_where_that_reads_less():
    # 64 rows a tile at G = 4; decode rows and other block sizes go alone
    assert _tiles([386, 1], [12000, 12000], blocks=64, block_size=32)[0] == 7
    assert _tiles([386], [12000], blocks=64, block_size=24)[0] == 0
    assert _tiles([1] * 9, [12000] * 9, blocks=64, block_size=32)[0] == 0
    # choices spread over very many blocks have little in common
    assert _tiles([64], [1 << 20], blocks=64, block_size=16)[0] == 0
    # a run of keys per CU, of at most 1,022 blocks; partials stay below 1 GiB
    n, wgs, size = _tiles([512], [16384 * 4], blocks=256, block_size=16)
    assert n == 8 and wgs % 256 == 0 and wgs * 1022 * 16 >= 8 * 8 * 65536 and size < 1 << 30
    n, wgs, size = _tiles([2000], [16384 * 8], blocks=512, block_size=16)
    assert n == 32 and wgs * 1022 * 16 >= 32 * 8 * 16384 * 8 * 0.98 and wgs % 256 == 0 and size < 3 << 30
    assert _tiles([16384], [65536], blocks=256, block_size=16)[2] < 4 << 30


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bs", [1, 3, 16, 100])
@pytest.mark.parametrize("rows", [1, 3, 64, 600])
def test_split_keys_cache_their_blocks(rows, bs, D):
    """A split's block ids fit the 512 of a task, and few rows get a workgroup per CU at most."""
    for blocks in (2, 64, 511, 2000):
        keys = min(blocks * bs, 200000)
        s = _info([1] * rows, [200000] * rows, D=D, bs=bs, blocks=blocks)["splits"]
        length = -(-(-(-keys // s)) // 16) * 16
        assert (length - 1) // bs + 2 <= 512
        assert s == 1 or rows * 8 * s <= 256 * (2 if D == 64 else 1) or s == -(-keys // (510 * bs // 16 * 16 - 16))


@pytest.mark.parametrize("kw,rc", [
    (dict(blocks=0, first=0, recent=0), _lib.EINVAL), (dict(recent=0), _lib.EINVAL), (dict(first=-1), _lib.EINVAL),
    (dict(blocks=5, first=3, recent=3), _lib.EINVAL), (dict(D=60), _lib.EUNSUPPORTED), (dict(D=264), _lib.EUNSUPPORTED),
    (dict(Hq=12), _lib.EINVAL), (dict(bs=0), _lib.EINVAL), (dict(bs=65537), _lib.EINVAL), (dict(dtype=_lib.DTYPE_FP8_E4M3), _lib.EUNSUPPORTED),
    (dict(stride=-1), _lib.EINVAL), (dict(stride=1), _lib.EINVAL), (dict(blocks=1 << 28), _lib.EINVAL)])
def test_sparse_plan_refuses(kw, rc):
    assert _info([1, 2], [50, 60], **kw)[0] == rc


def test_sparse_plan_refuses_lengths():
    assert _info([0], [5])[0] == _info([6], [5])[0] == _info([1], [2 ** 31 - 1])[0] == _lib.EINVAL
    lib = _lib.load()
    assert lib.gllm_sparse_plan_create(None, None, None, 0, 0, 8, 2, 64, 16, 1, 4, 0, 1) == _lib.EINVAL
    h = ctypes.c_void_p()
    assert lib.gllm_sparse_plan_create(ctypes.byref(h), None, None, 1, 0, 8, 2, 64, 16, 1, 4, 0, 1) == _lib.EINVAL
    assert lib.gllm_sparse_plan_info(None, None, 0) == _lib.EINVAL
    assert lib.gllm_sparse_plan_upload(None, None, 0, None) == _lib.EINVAL
    assert lib.gllm_sparse_plan_destroy(None) == 0


def test_record_bytes():
    for Hkv, D in ((1, 8), (3, 16), (8, 128), (20, 96), (1, 256)):
        assert sparse.key_bounds_bytes(Hkv, D) == osp.record_bytes(Hkv, D) == _lib.load().gllm_key_bounds_record_bytes(Hkv, D)
    for Hkv, D in ((0, 64), (8, 60), (8, 264), (8, 0)):
        assert _lib.load().gllm_key_bounds_record_bytes(Hkv, D) == 0
        with pytest.raises(ValueError):
            sparse.key_bounds_bytes(Hkv, D)
    b = sparse.new_key_bounds(3, 2, 64, "cpu")
    assert b.shape == (3, 272) and b.dtype == torch.uint8 and not b.any()


def _plan(ql=(1, 2), sl=(50, 60), **kw):
    args = dict(num_q_heads=8, num_kv_heads=2, head_dim=64, block_size=16, dtype=torch.bfloat16, device="cpu", blocks=3)
    args.update(kw)
    return sparse.SparsePlan(ql, sl, **args)


def test_arguments_are_checked():
    p = _plan()
    assert p.rows == 3 and p.table_width == 4 and p.info["touched_blocks"] == 2
    bt = torch.zeros(2, 4, dtype=torch.int32)
    q, cache = torch.zeros(3, 8, 64, dtype=torch.bfloat16), torch.zeros(160, 2, 64, dtype=torch.bfloat16)
    bounds, sel = sparse.new_key_bounds(10, 2, 64, "cpu"), torch.zeros(3, 2, 3, dtype=torch.int32)
    bad = [
        lambda: sparse.write_key_bounds(p, cache, bounds, bt.long()),
        lambda: sparse.write_key_bounds(p, cache, bounds, bt[:1]),
        lambda: sparse.write_key_bounds(p, cache, bounds, bt[:, :3]),
        lambda: sparse.write_key_bounds(p, cache, bounds[:9], bt),
        lambda: sparse.write_key_bounds(p, cache, bounds[:, :256], bt),
        lambda: sparse.write_key_bounds(p, cache, bounds.to(torch.int8), bt),
        lambda: sparse.write_key_bounds(p, cache[:, :1], bounds, bt),
        lambda: sparse.select_blocks(p, q[:2], bounds, bt),
        lambda: sparse.select_blocks(p, q.float(), bounds, bt),
        lambda: sparse.select_blocks(p, q[:, :4], bounds, bt),
        lambda: sparse.select_blocks(p, q, bounds, bt, out=sel.long()),
        lambda: sparse.select_blocks(p, q, bounds, bt, out=sel[..., :2]),
        lambda: sparse.select_blocks(p, q, bounds, bt, out=sel[:2]),
        lambda: sparse.sparse_attention(p, q, cache, cache, bt, sel[:, :1]),
        lambda: sparse.sparse_attention(p, q, cache, cache[:100], bt, sel),
        lambda: sparse.sparse_attention(p, q, cache, cache.float(), bt, sel),
        lambda: sparse.sparse_attention(p, q, cache, cache, bt, sel, out=q[:2]),
        lambda: sparse.sparse_attention(p, q, cache, cache, bt, sel, out=q.half()),
        lambda: sparse.key_bounds_values(bounds, torch.zeros(2), 2, 64),
        lambda: sparse.key_bounds_values(bounds, torch.zeros(2, dtype=torch.int64), 4, 64),
        lambda: sparse.key_bounds_values(bounds, torch.zeros(2, dtype=torch.int64), 2, 64, out=torch.zeros(2, 2, 2, 32)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    # every other check passed
    for call in (lambda: sparse.write_key_bounds(p, cache, bounds, bt), lambda: sparse.select_blocks(p, q, bounds, bt),
                 lambda: sparse.sparse_attention(p, q, cache, cache, bt, sel)):
        with pytest.raises(ValueError, match="CPU"):
            call()


def test_plan_arguments_are_checked():
    for kw in (dict(blocks=-1), dict(blocks=2, first_blocks=2), dict(recent_blocks=0), dict(blocks=1 << 40)):
        with pytest.raises(ValueError):
            _plan(**kw)
    with pytest.raises(TypeError):
        _plan(blocks=2.5)
    with pytest.raises(ValueError):
        _plan(ql=[1])
    with pytest.raises(NotImplementedError):
        _plan(head_dim=60)


def test_c_calls_refuse():
    lib, p, h = _lib.load(), 1 << 20, ctypes.c_void_p()          # p is never dereferenced
    one, fifty = (ctypes.c_int32 * 1)(1), (ctypes.c_int32 * 1)(50)
    _lib.check(lib.gllm_sparse_plan_create(ctypes.byref(h), one, fifty, 1, 0, 8, 2, 64, 16, _lib.DTYPE_BF16, 3, 1, 1))
    assert lib.gllm_key_bounds_write(h, p, 128, 10, p, 4, p, 272, _lib.DTYPE_BF16, None) == _lib.EINVAL
    assert b"not uploaded" in lib.gllm_attn_last_error()
    assert lib.gllm_select_blocks(None, p, 512, p, 272, 10, p, 4, p, 1, None) == _lib.EINVAL
    assert lib.gllm_key_bounds_values(p, 270, 10, p, 1, 2, 64, p, None) == _lib.EINVAL          # stride
    assert lib.gllm_key_bounds_values(p + 8, 272, 10, p, 1, 2, 64, p, None) == _lib.EINVAL      # alignment
    assert lib.gllm_key_bounds_values(p, 272, 10, None, 1, 2, 64, p, None) == _lib.EINVAL
    assert lib.gllm_key_bounds_values(p, 272, 0, p, 1, 2, 64, p, None) == _lib.EINVAL
    assert lib.gllm_key_bounds_values(p, 272, 10, p, 1, 2, 60, p, None) == _lib.EUNSUPPORTED
    lib.gllm_sparse_plan_destroy(h)


# ---------------------------------------------------------------- shared prefixes
def _shared(lens, groups, Hq=32, Hkv=8, D=128, bs=16, split=0, dtype=_lib.DTYPE_BF16, heads=0):
    lib, h, info = _lib.load(), ctypes.c_void_p(), (ctypes.c_int64 * 13)()
    arr = [(ctypes.c_int32 * len(lens))(*x) for x in zip(*lens)]
    members, ptr = [i for s, _ in groups for i in s], [0]
    for s, _ in groups:
        ptr.append(ptr[-1] + len(s))
    rc = lib.gllm_attn_plan_create_shared(ctypes.byref(h), *arr, len(lens), 0, Hq, Hkv, D, bs, dtype, split, heads, len(groups),
                                          (ctypes.c_int32 * len(ptr))(*ptr), (ctypes.c_int32 * max(1, len(members)))(*members),
                                          (ctypes.c_int32 * max(1, len(groups)))(*[n for _, n in groups]))
    if rc:
        return rc, lib.gllm_attn_last_error().decode()
    _lib.check(lib.gllm_attn_plan_info(h, info, 13))
    lib.gllm_attn_plan_destroy(h)
    return dict(zip(("wgs", "split", "dec", "pre", "parts", "rows", "hw", "dw", "pw", "segs", "half", "ids", "prefix"), info))


def test_prefix_plans():
    i = _shared([(1, 9000)] * 64, [(range(64), 8192)])
    # 256 columns: one workgroup of columns, 8 heads, ranges of at least 256 keys
    assert i["prefix"] > 0 and i["prefix"] % 8 == 0 and i["prefix"] <= 8 * 32 and i["dec"] == 64 and i["ids"] <= 512
    # every (sequence, head) has a partial of each range and its own segments'
    assert i["parts"] >= 64 * 8 * (i["prefix"] // 8 + 1)
    # 65 sequences: a second workgroup of columns
    assert _shared([(1, 9000)] * 65, [(range(65), 8192)])["prefix"] % 16 == 0
    # a group of one, too few keys, no group: nothing shared
    for groups in ([([0], 8192)], [([0, 1], 15)], [([], 3)], [], [([0, 1], 0)], [([0, 1], 255)]):
        assert _shared([(1, 9000)] * 4, groups)["prefix"] == 0
    assert _shared([(1, 9000)] * 4, [([0, 1], 256)])["prefix"] > 0
    assert _shared([(1, 9000)] * 4, [([0, 1], 511)], D=64)["prefix"] == 0
    assert _shared([(1, 9000)] * 4, [([0, 1], 512)], D=64)["prefix"] > 0
    # prompts (query_len x G > 16) keep their keys; two decodes beside them share
    i = _shared([(1, 9000), (300, 9000), (4, 9000)], [(range(3), 4000)])
    assert i["pre"] == 1 and i["dec"] == 2 and i["prefix"] > 0
    assert _shared([(1, 9000), (300, 9000)], [(range(2), 4000)])["prefix"] == 0
    # another kernel's model: a plan without sharing
    assert _shared([(1, 900)] * 4, [(range(4), 512)], dtype=_lib.DTYPE_F32)["prefix"] == 0


@pytest.mark.parametrize("bs", [1, 3, 16, 100])
@pytest.mark.parametrize("own", [1, 40, 9000])
def test_prefix_segments_cache_their_blocks(own, bs):
    for P in (16, 257, 5000):
        i = _shared([(1, P + own)] * 5, [((3, 0, 4), P)], bs=bs)
        assert i["ids"] <= 512 and (i["prefix"] > 0) == (P > 16)


@pytest.mark.parametrize("groups", [[([0, 1], 49)], [([0, 2], 10)], [([0, -1], 10)], [([0, 1], 10), ([1], 5)], [([0, 0], 10)],
                                    [([0, 1], -1)]])
def test_prefix_plans_refuse(groups):
    assert _shared([(2, 50), (1, 60)], groups)[0] == _lib.EINVAL
    with pytest.raises(ValueError):
        paged.AttentionPlan([2, 1], [50, 60], num_q_heads=8, num_kv_heads=2, head_dim=64, block_size=16,
                            dtype=torch.bfloat16, device="cpu", shared_prefixes=groups)


def test_prefix_plans_refuse_splits_and_windows():
    assert _shared([(1, 50), (1, 60)], [([0, 1], 32)], split=64)[0] == _lib.EINVAL
    args = dict(num_q_heads=8, num_kv_heads=2, head_dim=64, block_size=16, dtype=torch.bfloat16, device="cpu")
    with pytest.raises(NotImplementedError):
        paged.AttentionPlan([1, 1], [50, 60], shared_prefixes=[([0, 1], 32)], window=20, **args)
    with pytest.raises(TypeError):
        paged.AttentionPlan([1, 1], [50, 60], shared_prefixes=[([0, 1], 32.0)], **args)
    with pytest.raises(ValueError):
        paged.AttentionPlan([1, 1], [50, 60], shared_prefixes=[([0, 1], 1 << 40)], **args)


def test_metadata_passes_prefixes_to_the_plan(monkeypatch):
    """plan_for: what the engine knows of prefixes reaches the plan, but not windowed ones;
    metadata without the field (the reference's own) shares nothing."""
    import types
    from gllm_amd import attention
    seen = []

    def plan(ql, sl, **kw):
        seen.append((kw["shared_prefixes"], kw["window"]))
        return types.SimpleNamespace()
    monkeypatch.setattr(attention.paged, "AttentionPlan", plan)

    def meta(**kw):
        return types.SimpleNamespace(query_lens=torch.tensor([1, 1]), seq_lens=torch.tensor([40, 50]), block_size=16,
                                     block_table=torch.tensor([[1, 2, 3, 0], [1, 2, 4, 5]]),
                                     query_slot_mapping=torch.tensor([[3 * 16 + 7], [5 * 16 + 1]]), **kw)
    args = dict(num_q_heads=8, num_kv_heads=2, head_dim=64, dtype=torch.bfloat16, device="cpu")
    groups = [([0, 1], 32)]
    attention.plan_for(meta(shared_prefixes=groups), **args)
    attention.plan_for(meta(shared_prefixes=groups), window=16, **args)
    attention.plan_for(meta(shared_prefixes=None), **args)
    attention.plan_for(meta(), **args)
    assert seen == [(groups, None), ((), 16), ((), None), ((), None)]
