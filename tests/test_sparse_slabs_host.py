"""Sparse plans of long prompts on the CPU: rows keep their tiles at any length and
beside any other sequence, and the workspace stays bounded."""
import ctypes

import pytest

from gllm_amd import _lib

MIB = 1 << 20
KEYS = ("rows", "query_rows", "touched_blocks", "score_tiles", "slabs", "splits", "tiles", "tile_workgroups", "tile_slabs",
        "row_slabs")


def info(ql, sl, Hq=32, Hkv=8, D=128, bs=16, blocks=128, dtype=_lib.DTYPE_BF16):
    lib, h, arr, n = _lib.load(), ctypes.c_void_p(), (ctypes.c_int64 * len(KEYS))(), len(ql)
    _lib.check(lib.gllm_sparse_plan_create(ctypes.byref(h), (ctypes.c_int32 * n)(*ql), (ctypes.c_int32 * n)(*sl), n, 0, Hq, Hkv,
                                           D, bs, dtype, blocks, 1, 1))
    _lib.check(lib.gllm_sparse_plan_info(h, arr, len(KEYS)))
    size = lib.gllm_sparse_plan_workspace_bytes(h)
    assert lib.gllm_sparse_plan_destroy(h) == 0
    return dict(zip(KEYS, arr)) | {"bytes": size}


def tables(i):
    """Room for the tables of rows, tiles, touched blocks and score items."""
    return 64 * i["query_rows"] + 64 * i["touched_blocks"] + 128 * i["score_tiles"] + 64 * i["tiles"] + 4 * MIB


@pytest.mark.parametrize("ql,sl", [([32000], [32000]), ([32768], [32768]), ([131072], [131072]), ([16384], [65536]),
                                   ([512] * 64, [32768] * 64), ([2048] * 8, [131072] * 8), ([65536, 1], [65536, 100000])])
def test_long_prompts_keep_their_tiles(ql, sl):
    # 256 of 8,192 blocks: rows near each other select most of them between them
    i = info(ql, sl, blocks=256 if max(sl) > 32768 else 128)
    assert i["tiles"] == sum(-(-n // 64) for n in ql if n > 1) and i["tile_slabs"] >= 1
    # scores, blocks of tiles, their partials
    assert i["bytes"] <= 3 * 256 * MIB + tables(i)
    # a run per CU and round, 1,022 blocks at most each
    assert i["tile_workgroups"] % 256 == 0


def test_tiles_beside_a_long_prompt():
    """One sequence decides nothing for another."""
    alone = [info([n], [L]) for n, L in ((512, 8192), (32768, 32768), (300, 12000))]
    both = info([512, 32768, 300, 1], [8192, 32768, 12000, 500])
    assert all(x["tiles"] > 0 for x in alone) and both["tiles"] == sum(x["tiles"] for x in alone)


def test_a_tile_too_large_for_a_slab_goes_by_rows():
    """Rows that select 300,000 blocks each of 134 million: that sequence alone."""
    i = info([64, 128], [(1 << 31) - 20000, 8192], Hkv=4, Hq=16, blocks=300000)
    assert i["tiles"] == 2 and i["row_slabs"] >= 1 and i["splits"] > 1


@pytest.mark.parametrize("rows,ctx,bs", [(8192, 65536, 8), (8192, 65536, 24), (32768, 65536, 8), (20000, 40000, 1)])
def test_partials_of_single_rows_stay_bounded(rows, ctx, bs):
    """Lists longer than a task caches are split whatever the number of rows."""
    i = info([rows], [ctx], bs=bs, blocks=600)
    assert i["tiles"] == 0 and i["splits"] == 2 and i["row_slabs"] == -(-rows // (256 * MIB // (8 * 2 * 16 * 130 * 4)))
    assert i["bytes"] <= 2 * 256 * MIB + tables(i)
    assert info([rows], [ctx], bs=bs, blocks=64)["row_slabs"] == 1
