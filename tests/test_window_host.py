"""Sliding windows and the 4-bit cache on the CPU: the oracle from its
definition, the planner, and what the entry points refuse."""
import math
import types

import pytest
import torch

from gllm_amd import _lib, paged
from oracle import attention as oa
from oracle import kv4
from oracle import window as ow


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (5, 2), (9, 30), (64, 1)])
def test_window_oracle_against_a_mask(window, sinks):
    g = torch.Generator().manual_seed(1)
    ctx, n, Hq, Hkv, D = 20, 13, 4, 2, 8
    q, k, v = torch.randn(n, Hq, D, generator=g), torch.randn(ctx + n, Hkv, D, generator=g), torch.randn(ctx + n, Hkv, D, generator=g)
    p, t = ctx + torch.arange(n)[:, None], torch.arange(ctx + n)[None]
    seen = t <= p
    if window is not None:
        seen &= (t > p - window) | (t < sinks)
    bias = torch.where(seen, 0.0, -math.inf)
    ref = oa.reference_attention(q[None], k[None], v[None], bias[None])[0]
    out, spread, mag = ow.attention(q, k, v, ctx, window, sinks, 1 / math.sqrt(D))
    assert (out - ref).abs().max() < 1e-5
    assert (spread >= 0).all() and spread.shape == out.shape and mag.shape == (n, Hq, 1)


def test_kv4_format():
    """Ties to the even code, the scale at its border, zeros, NaN and infinity."""
    x = torch.zeros(10, 32)
    x[0, :12] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -5, 0.26, 4.9])
    x[1, 0], x[2, 0], x[3, 0] = 6.99, 7.0, -7.0
    x[4, 0], x[5, 0] = math.nan, math.inf
    x[6, 0] = 2.0 ** -140
    x[7, 0], x[8, 0] = 3.4e38, 448.0
    code, byte = kv4.quantize(x)
    val = kv4.values(code, byte)
    assert val[0, :12].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -4, 0.5, 4]
    assert byte[:4, 0].tolist() == [127, 127, 128, 128] and val[1:4, 0].tolist() == [6, 8, -8]
    assert byte[4:6, 0].tolist() == [255, 255] and val[4:6].isnan().all()
    assert byte[6, 0] == 1 and val[6, 0] == 0 and byte[9, 0] == 1 and (val[9] == 0).all()
    assert byte[7, 0] == 253 and val[7, 0] == 2.0 ** 128 and val[8, 0] == 512


def test_kv4_is_off_by_half_a_step_at_most():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(64, 128, generator=g) * torch.exp2(torch.randint(-30, 30, (64, 1), generator=g).float())
    code, byte = kv4.quantize(x)
    d = (kv4.values(code, byte) - x.double()).abs()
    scale = torch.exp2(byte.double() - 127).repeat_interleave(32, -1)
    a = x.double().abs() / scale
    assert (a < 7).all() and (a.unflatten(-1, (-1, 32)).amax(-1) >= 3.5).all()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)) * scale
    assert (d <= step / 2).all()


@pytest.mark.parametrize("bs,D", [(16, 128), (16, 64), (1, 32), (7, 96), (24, 64)])
def test_kv4_write_read(bs, D):
    g = torch.Generator().manual_seed(3)
    cache = torch.full((5, 2, kv4.record_bytes(bs, D)), 170, dtype=torch.uint8)
    assert kv4.record_bytes(bs, D) == paged.kv4_record_bytes(bs, D)
    slots = torch.randperm(5 * bs, generator=g)[:3]
    x = torch.randn(3, 2, D, generator=g)
    kv4.write(cache, slots, x, bs)
    assert torch.equal(kv4.read(cache, slots, bs, D), kv4.values(*kv4.quantize(x)))


def _plan(lens=((1, 100),), **kw):
    args = dict(num_q_heads=8, num_kv_heads=2, head_dim=64, block_size=16, dtype=torch.bfloat16, device="cpu")
    args.update(kw)
    return paged.AttentionPlan([q for q, _ in lens], [s for _, s in lens], **args)


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(window=1 << 31), dict(sinks=2), dict(window=4, sinks=-1),
                                dict(window=4, sinks=1 << 31)])
def test_plan_refuses(kw):
    with pytest.raises(ValueError):
        _plan(**kw)


def test_c_plan_refuses():
    import ctypes
    lib = _lib.load()
    h = ctypes.c_void_p()
    one, long = (ctypes.c_int32 * 1)(1), (ctypes.c_int32 * 1)(2 ** 31 - 1)

    def create(lens, window, sinks):
        return lib.gllm_attn_plan_create_window(ctypes.byref(h), one, lens, 1, 0, 8, 2, 64, 16, _lib.DTYPE_BF16, 0, 0,
                                                window, sinks)
    assert create(one, -1, 0) == _lib.EINVAL and create(one, 0, 1) == _lib.EINVAL and create(one, 4, -1) == _lib.EINVAL
    assert create(long, 100, 0) == _lib.EINVAL and b"too long" in lib.gllm_attn_last_error()


@pytest.mark.parametrize("name", ["kv_dtype", "record", "heads", "strided", "blocks", "float"])
def test_kv4_cache_layout_is_checked(name):
    rec = paged.kv4_record_bytes(16, 64)
    k = v = torch.zeros(4, 2, rec, dtype=torch.uint8)
    if name == "record":
        k = v = torch.zeros(4, 2, rec + 16, dtype=torch.uint8)
    if name == "heads":
        k = v = torch.zeros(4, 1, rec, dtype=torch.uint8)
    if name == "strided":
        k = v = torch.zeros(4, 2, 2 * rec, dtype=torch.uint8)[..., ::2]
    if name == "blocks":
        v = torch.zeros(5, 2, rec, dtype=torch.uint8)
    if name == "float":
        v = torch.zeros(4, 2, rec)
    if name == "kv_dtype":
        paged._kv4_blocks(k, v, 2, 64, 16)
        return
    with pytest.raises(ValueError):
        paged._kv4_blocks(k, v, 2, 64, 16)


def _info(lens, D, window=0, sinks=0):
    import ctypes
    lib, h, info = _lib.load(), ctypes.c_void_p(), (ctypes.c_int64 * 10)()
    arr = [(ctypes.c_int32 * len(lens))(*x) for x in zip(*lens)]
    _lib.check(lib.gllm_attn_plan_create_window(ctypes.byref(h), arr[0], arr[1], len(lens), 0, 32, 8, D, 16, _lib.DTYPE_BF16,
                                                0, 0, window, sinks))
    _lib.check(lib.gllm_attn_plan_info(h, info, 10))
    lib.gllm_attn_plan_destroy(h)
    return list(info)


def test_planner_counts_the_window_only():
    """4,096 keys of 32,768 make as many splits as a sequence of 4,096."""
    short = _info([(1, 4096)] * 4, 128)
    assert _info([(1, 32768)] * 4, 128, 4096) == short
    assert _info([(1, 32768)] * 4, 128) != short
    # a window that reaches every first key changes nothing
    assert _info([(1, 4096)] * 4, 128, 4096) == short
    assert _info([(1, 4096)] * 4, 128, 4000, 96) == short


@pytest.mark.parametrize("bs", [1, 3, 16, 100])
@pytest.mark.parametrize("split", [0, 8192, -1])
def test_segments_cache_their_blocks(bs, split):
    """Plans over two runs of blocks (sinks, window) are made for every block
    size (a task's block ids have to fit its cache)."""
    import ctypes
    lib, h = _lib.load(), ctypes.c_void_p()
    ql, sl = (ctypes.c_int32 * 3)(1, 1, 4), (ctypes.c_int32 * 3)(70000, 9000, 40)
    _lib.check(lib.gllm_attn_plan_create_window(ctypes.byref(h), ql, sl, 3, 0, 8, 2, 64, bs, _lib.DTYPE_BF16, split, 0,
                                                60000, 333))
    lib.gllm_attn_plan_destroy(h)


def test_fused_kv_write_and_windows():
    def plan(dtype, window):
        return types.SimpleNamespace(max_query_len=1, dtype=dtype, head_dim=64, num_q_heads=8, num_kv_heads=2, window=window)
    assert paged.fused_kv_write_ok(plan(torch.bfloat16, 10), torch.bfloat16)
    assert not paged.fused_kv_write_ok(plan(torch.float32, 10), torch.float32)
    assert paged.fused_kv_write_ok(plan(torch.float32, None), torch.float32)
    assert not paged.fused_kv_write_ok(plan(torch.bfloat16, None), paged.KV4)


def test_windows_are_integers():
    for kw in (dict(window=4.0), dict(window="4"), dict(window=4, sinks=1.5)):
        with pytest.raises(TypeError):
            _plan(**kw)


def test_sinks_without_a_window_are_refused_with_a_kept_plan():
    """An earlier layer's plan on the metadata is no answer to other arguments."""
    from gllm_amd import attention
    meta = types.SimpleNamespace(_gllm_plan="plan", _gllm_window_plans={(4, 1): "windowed"})
    assert attention._kept_plan(meta, None, 0) == "plan" and attention._kept_plan(meta, 4, 1) == "windowed"
    assert attention._kept_plan(meta, None, 2) is None and attention._kept_plan(meta, 4, 0) is None


def test_projections_refuse_4_bit_caches():
    cache = torch.zeros(4, 2, paged.kv4_record_bytes(16, 64), dtype=torch.uint8)
    w, cs = torch.zeros(128, 64, dtype=torch.bfloat16), torch.zeros(3, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="4-bit"):
        paged.qkv_rope_kv_write(torch.zeros(3, 64, dtype=torch.bfloat16), w, w, w, cs, cs, cache, cache, torch.arange(3))


def test_sequences_too_long_for_a_4_bit_cache():
    import ctypes
    lib, p = _lib.load(), 1 << 20                    # never dereferenced
    for keys, why in ((2 ** 31 - 1, b"too long"), (2 ** 31 - 16384, b"not uploaded")):
        h = ctypes.c_void_p()
        one, long = (ctypes.c_int32 * 1)(1), (ctypes.c_int32 * 1)(keys)
        _lib.check(lib.gllm_attn_plan_create(ctypes.byref(h), one, long, 1, 0, 8, 2, 64, 4096, _lib.DTYPE_BF16, 0, 0))
        rc = lib.gllm_paged_attention(h, p, 512, p, 512, p, p, 1 << 20, 16, p, 8, None, None, 0, 0, 0.1, _lib.DTYPE_BF16,
                                      _lib.DTYPE_MXFP4, None)
        assert rc == _lib.EINVAL and why in lib.gllm_attn_last_error()
        lib.gllm_attn_plan_destroy(h)


def test_kv4_of_an_fp16_model_stays_finite():
    """57,344 and more would round to 65,536, past the largest fp16."""
    x = torch.zeros(6, 32)
    x[:, 0] = torch.tensor([49152.0, 57343.0, 57344.0, 65504.0, -65504.0, math.inf])
    x[:, 1] = 4096.0
    code, byte = kv4.quantize(x, torch.float16)
    val = kv4.values(code, byte)
    assert val[:5, 0].tolist() == [49152.0] * 4 + [-49152.0] and val[5].isnan().all()
    assert (val[:5, 1] == 4096).all() and byte[:5, 0].tolist() == [127 + 13] * 5
    assert kv4.values(*kv4.quantize(x))[2:4, 0].tolist() == [65536.0] * 2
    assert torch.equal(kv4.values(*kv4.quantize(x[:2], torch.float16)), kv4.values(*kv4.quantize(x[:2])))


def test_fused_kv_write_under_a_window_that_hides_nothing():
    plan = types.SimpleNamespace(max_query_len=1, dtype=torch.float32, head_dim=64, num_q_heads=8, num_kv_heads=2, window=10,
                                 hides_keys=False)
    assert paged.fused_kv_write_ok(plan, torch.float32) and not paged.fused_kv_write_ok(plan, paged.KV4)
    plan.hides_keys = True
    assert not paged.fused_kv_write_ok(plan, torch.float32)


def test_plan_says_where_mixed_launches_take_half_size_workgroups():
    import ctypes
    lib = _lib.load()

    def half(lens, D, window, hw=0):
        h, info = ctypes.c_void_p(), (ctypes.c_int64 * 11)(*[-1] * 11)
        arr = [(ctypes.c_int32 * len(lens))(*x) for x in zip(*lens)]
        _lib.check(lib.gllm_attn_plan_create_window(ctypes.byref(h), arr[0], arr[1], len(lens), 0, 32, 8, D, 16,
                                                    _lib.DTYPE_BF16, 0, hw, window, 0))
        _lib.check(lib.gllm_attn_plan_info(h, info, 11))
        lib.gllm_attn_plan_destroy(h)
        return info[10]
    # many short chunks beside the decodes; one long chunk ends last; one kind alone
    for hw in (0, 1, 2, 4, 8):
        assert half([(1, 1100)] * 16 + [(33, 33)] * 40, 64, 1000, hw) == 1
    assert half([(1, 1100)] * 4 + [(1024, 8000)], 128, 5000) == 0
    assert half([(1, 1100)] * 16, 64, 1000) == 0 and half([(33, 33)] * 40, 64, 20) == 0


@pytest.mark.parametrize("bs", [1, 3, 7, 8, 16, 17, 24, 100])
@pytest.mark.parametrize("split", [0, 32, 8192, -1])
def test_a_tasks_blocks_fit_its_cache(bs, split):
    """The decode kernels cache 512 block ids a task, of one or two runs of keys."""
    import ctypes
    lib = _lib.load()
    seen = set()
    for window, sinks in ((0, 0), (60000, 333), (60001, 1), (400, 70), (8200, 8100), (17, 30000), (30000, 8)):
        for lens in ([(1, 70000), (1, 9000), (4, 40)], [(1, 70007)] * 33, [(4, 31000 + 13 * i) for i in range(20)],
                     [(1, 33000), (64, 900)]):
            for D, hw in ((64, 0), (128, 8)):
                h, info = ctypes.c_void_p(), (ctypes.c_int64 * 12)()
                arr = [(ctypes.c_int32 * len(lens))(*x) for x in zip(*lens)]
                _lib.check(lib.gllm_attn_plan_create_window(ctypes.byref(h), arr[0], arr[1], len(lens), 0, 32, 8, D, bs,
                                                            _lib.DTYPE_BF16, split, hw, window, sinks))
                _lib.check(lib.gllm_attn_plan_info(h, info, 12))
                lib.gllm_attn_plan_destroy(h)
                assert 0 < info[11] <= 512, (window, sinks, lens[0], D, hw, list(info))
                seen.add(info[11])
    assert max(seen) > 400 or bs > 16 or split == 32      # tasks near the limit are among them


def test_counted_blocks_of_a_small_plan():
    """One sequence, whole: the sinks' blocks and the window's."""
    import ctypes
    lib = _lib.load()

    def most(keys, bs, window=0, sinks=0):
        h, info, one, sl = ctypes.c_void_p(), (ctypes.c_int64 * 12)(), (ctypes.c_int32 * 1)(1), (ctypes.c_int32 * 1)(keys)
        _lib.check(lib.gllm_attn_plan_create_window(ctypes.byref(h), one, sl, 1, 0, 8, 2, 64, bs, _lib.DTYPE_BF16, 8192, 0,
                                                    window, sinks))
        _lib.check(lib.gllm_attn_plan_info(h, info, 12))
        lib.gllm_attn_plan_destroy(h)
        return info[11]
    assert most(100, 16) == 7 and most(96, 16) == 6 and most(100, 1) == 100
    # keys 0..15 hold the sinks' unit, the window's starts at 256 (of 270)
    assert most(300, 16, 30, 2) == 1 + 3 and most(300, 10, 30, 2) == 2 + 5 and most(300, 16, 30, 0) == 3


def _fake_plan(rows=3, window=None):
    """What paged_attention reads of a plan before it launches anything."""
    return types.SimpleNamespace(num_q_heads=4, num_kv_heads=2, head_dim=64, dtype=torch.bfloat16, block_size=16,
                                 query_lens=[1] * rows, rows=rows, table_width=1, max_seq_len=16, window=window, _h=None, _lib=None)


@pytest.mark.parametrize("v", [torch.zeros(64, 2, 64), torch.zeros(64, 2, 64, dtype=torch.uint8),
                               torch.zeros(63, 2, 64, dtype=torch.bfloat16)])
def test_a_v_cache_unlike_the_k_cache_is_refused(v):
    """The kernels address V by K's slots and read it in K's dtype."""
    k = torch.zeros(64, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="v_cache"):
        paged.paged_attention(_fake_plan(), q, k, v, torch.zeros(3, 1, dtype=torch.int32))
    kv, cs = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="v_cache"):
        paged.rope_kv_write(kv, kv, cs, cs, k, v, torch.arange(3))


@pytest.mark.parametrize("window", [None, 8])
def test_an_out_with_too_few_rows_is_refused(window):
    k = torch.zeros(64, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="out has 2"):
        paged.paged_attention(_fake_plan(window=window), q, k, k, torch.zeros(3, 1, dtype=torch.int32), out=q[:2].clone())
    with pytest.raises(ValueError, match="q has 2"):
        paged.paged_attention(_fake_plan(window=window), q[:2], k, k, torch.zeros(3, 1, dtype=torch.int32), out=q.clone())
