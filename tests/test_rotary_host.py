"""Rotary positions on the CPU: the frequency schedules against the oracle's
loops, known values, and what the entry points refuse."""
import math

import pytest
import torch

import gllm_amd
from gllm_amd import _lib, paged
from oracle import rope as orope
from oracle import rotary as orot

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
SCALINGS = [None, {"rope_type": "linear", "factor": 2.5}, LLAMA3, YARN,
            dict(YARN, factor=40.0, beta_fast=16, beta_slow=2, attention_factor=0.7)]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("D,R,theta", [(128, 128, 500000.0), (64, 32, 10000.0), (96, 24, 1e6), (8, 2, 10000.0)])
def test_frequencies(scaling, D, R, theta):
    r = gllm_amd.Rotary(D, theta=theta, rotary_dim=R, scaling=scaling, device="cpu")
    f, m = orot.frequencies(R, theta, scaling)
    assert r.freq.dtype == torch.float64 and r.freq.shape == (R // 2,)
    assert torch.allclose(r.freq, f, rtol=1e-13, atol=0) and math.isclose(r.factor, m, rel_tol=1e-15)


def test_tables_are_the_unscaled_models():
    cos, sin = gllm_amd.Rotary(64, theta=500000.0, device="cpu").tables(100, torch.float32)
    c, s = orope.rope_cache(100, 64, 500000.0, torch.float32)
    # the fp32 table's angles are fp32 products: 100 * 2^-24
    assert (cos - c).abs().max() < 2e-5 and (sin - s).abs().max() < 2e-5
    for kw in (dict(interleaved=True), dict(rotary_dim=32)):
        with pytest.raises(ValueError):
            gllm_amd.Rotary(64, device="cpu", **kw).tables(4, torch.float32)


def test_oracle_rotates():
    x = torch.randn(3, 2, 8)
    f, m = orot.frequencies(8, 100.0, None)
    pos = torch.tensor([0, 1, 7])
    for inter in (False, True):
        y = orot.rotate(x, pos, f, m, 8, inter)
        assert torch.allclose(y[0], x[0].double())
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1))
    half, pairs = orot.rotate(x, pos, f, m, 8, False), orot.rotate(x[..., [0, 4, 1, 5, 2, 6, 3, 7]], pos, f, m, 8, True)
    assert torch.allclose(half[..., [0, 4, 1, 5, 2, 6, 3, 7]], pairs)
    assert torch.equal(orot.rotate(x, pos, f[:2], m, 4, False)[..., 4:], x[..., 4:].double())


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=130), dict(theta=0.0), dict(theta=math.inf),
                                dict(scaling={}), dict(scaling={"rope_type": "linear"}),
                                dict(scaling={"rope_type": "linear", "factor": 0}),
                                dict(scaling={"rope_type": "linear", "factor": "x"}),
                                dict(scaling=dict(LLAMA3, high_freq_factor=1.0)),
                                dict(scaling={"rope_type": "yarn", "factor": 2.0}),
                                dict(scaling=YARN, theta=1.0)])
def test_rotary_refuses(kw):
    with pytest.raises(ValueError):
        gllm_amd.Rotary(128, device="cpu", **kw)


def test_rotary_refuses_other_schedules():
    with pytest.raises(NotImplementedError):
        gllm_amd.Rotary(128, device="cpu", scaling={"rope_type": "dynamic", "factor": 2.0})


def test_rotary_refuses_what_it_would_ignore():
    """Keys of a configuration that change the rotation are taken or refused."""
    for kw in (dict(rope_theta=500.0), dict(partial_rotary_factor=0.5), dict(attention_factor=-1.0)):
        with pytest.raises(ValueError):
            gllm_amd.Rotary(128, device="cpu", scaling=dict(YARN, **kw))
    for kw in (dict(mscale=1.0), dict(mscale_all_dim=0.707), dict(truncate=False)):
        with pytest.raises(NotImplementedError):
            gllm_amd.Rotary(128, device="cpu", scaling=dict(YARN, **kw))
    same = gllm_amd.Rotary(128, theta=500.0, rotary_dim=32, device="cpu",
                           scaling=dict(LLAMA3, rope_theta=500.0, partial_rotary_factor=0.25))
    assert torch.equal(same.freq, gllm_amd.Rotary(128, theta=500.0, rotary_dim=32, device="cpu", scaling=LLAMA3).freq)


@pytest.mark.parametrize("kw", [dict(k=torch.zeros(6, 0, 64), v=torch.zeros(6, 0, 64)), dict(q=torch.zeros(64)),
                                dict(k=torch.zeros(64), v=torch.zeros(64))])
def test_rotary_kv_write_refuses_rows_without_heads(kw):
    with pytest.raises(ValueError):
        paged.rotary_kv_write(**_args(**kw))


def _args(**kw):
    n, Hq, Hkv, D = 6, 4, 2, 64
    a = dict(k=torch.zeros(n, Hkv, D), v=torch.zeros(n, Hkv, D), positions=torch.arange(n),
             rotary=gllm_amd.Rotary(D, device="cpu"), k_cache=torch.zeros(32, Hkv, D), v_cache=torch.zeros(32, Hkv, D),
             slot_mapping=torch.arange(n), q=torch.zeros(n, Hq, D), q_out=torch.zeros(n, Hq, D))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(v=None), dict(q=None), dict(k=None, v=None, q=None, q_out=None), dict(k_cache=None), dict(slot_mapping=None),
    dict(rotary=gllm_amd.Rotary(32, device="cpu")), dict(positions=torch.arange(5)), dict(positions=torch.zeros(6)),
    dict(v=torch.zeros(6, 2, 64, dtype=torch.bfloat16)), dict(v=torch.zeros(6, 1, 64)),
    dict(k_cache=torch.zeros(32, 1, 64)), dict(v_cache=torch.zeros(31, 2, 64)),
    dict(v_cache=torch.zeros(32, 2, 64, dtype=torch.bfloat16)), dict(slot_mapping=torch.arange(6, dtype=torch.int32)),
    dict(slot_mapping=torch.arange(12)[::2]), dict(q=torch.zeros(5, 4, 64)), dict(q_out=torch.zeros(6, 4, 64).bfloat16()),
    dict(query_lens=torch.zeros(4, dtype=torch.int32)), dict(query_lens=torch.zeros(0, dtype=torch.int32)),
    dict(k=torch.zeros(6, 64, 2).transpose(1, 2)), dict(k_cache=torch.zeros(4, 2, 100, dtype=torch.uint8))])
def test_rotary_kv_write_refuses(kw):
    with pytest.raises(ValueError):
        paged.rotary_kv_write(**_args(**kw))


def test_c_entries_refuse():
    """Null pointers, sizes and layouts are refused before anything is launched."""
    lib = _lib.load()
    p = 1 << 20                       # never dereferenced: every call is refused

    def rotary(R=64, D=64, Hkv=2, dtype=_lib.DTYPE_BF16, kv=_lib.DTYPE_BF16, stride=128, bs=16, slots=64, freq=p, pos=p, k=p,
               cache=p, factor=1.0, n=4, q_out=None):
        return lib.gllm_rotary_kv_write(None, q_out, k, k, cache, cache, p, None, 0, freq, factor, pos, R, 0, n, 4, Hkv, D,
                                        256, 128, 128, 256, stride, slots, bs, dtype, kv, None)
    bad = [dict(R=3), dict(R=66), dict(R=-2), dict(pos=None), dict(freq=None), dict(factor=math.inf), dict(n=-1), dict(Hkv=0),
           dict(stride=100), dict(slots=0), dict(cache=None), dict(k=None), dict(q_out=p),
           dict(kv=_lib.DTYPE_MXFP4, stride=1000), dict(kv=_lib.DTYPE_MXFP4, stride=1096), dict(kv=_lib.DTYPE_MXFP4, bs=0, stride=1088),
           dict(kv=_lib.DTYPE_MXFP4, stride=1088, cache=p + 8), dict(kv=_lib.DTYPE_MXFP4, stride=1 << 32)]
    for kw in bad:
        assert rotary(**kw) == _lib.EINVAL, kw
        assert lib.gllm_attn_last_error()
    for kw in (dict(D=60, R=4), dict(D=264), dict(dtype=_lib.DTYPE_FP8_E4M3), dict(kv=9)):
        assert rotary(**kw) == _lib.EUNSUPPORTED, kw
    def rope(k=p, cos=p, row=64):
        return lib.gllm_rope_kv_write_kv4(None, None, k, k, p, p, p, None, 0, cos, p, None, row, 4, 4, 2, 64, 256, 128, 128, 256,
                                          1000, 64, 16, _lib.DTYPE_BF16, None)
    assert rope() == _lib.EINVAL and rope(k=None) == _lib.EINVAL and rope(cos=None) == _lib.EINVAL and rope(row=31) == _lib.EINVAL

    def values(cache=p, stride=1088, n=4, dtype=_lib.DTYPE_BF16, D=64, out=128):
        return lib.gllm_kv4_values(cache, stride, 64, 16, p, n, 2, D, p, out, dtype, None)
    for kw in (dict(cache=None), dict(stride=16), dict(n=-1), dict(out=127)):
        assert values(**kw) == _lib.EINVAL, kw
    assert values(dtype=_lib.DTYPE_MXFP4) == _lib.EUNSUPPORTED and values(D=72) == _lib.EUNSUPPORTED
    assert lib.gllm_kv4_record_bytes(16, 128) == 1088 and lib.gllm_kv4_record_bytes(1, 64) == 48
    assert lib.gllm_kv4_record_bytes(0, 64) == 0 and lib.gllm_kv4_record_bytes(16, 40) == 0


def test_kv4_values_refuses():
    cache = torch.zeros(4, 2, paged.kv4_record_bytes(16, 64), dtype=torch.uint8)
    slots = torch.arange(3)
    for args in ((cache[..., :40], slots, 64, torch.float32), (cache, slots, 40, torch.float32),
                 (cache.float(), slots, 64, torch.float32)):
        with pytest.raises(ValueError):
            paged.kv4_values(*args)
    with pytest.raises(ValueError):
        paged.kv4_values(cache, slots, 64, torch.float32, out=torch.zeros(2, 2, 64))
    assert paged.kv4_values(cache, slots[:0], 64, torch.float32).shape == (0, 2, 64)


@pytest.mark.parametrize("scaling", [{"rope_type": "default"}, {"type": "default"}, {"rope_type": "linear", "factor": 2.0},
                                     LLAMA3, YARN])
@pytest.mark.parametrize("kw", [dict(rope_theta=500.0), dict(partial_rotary_factor=0.5)])
def test_every_schedule_refuses_another_theta_or_part(scaling, kw):
    """A configuration's dictionary that holds the theta or the part of the head
    that turns is not overruled in silence."""
    with pytest.raises(ValueError, match="not the theta"):
        gllm_amd.Rotary(128, device="cpu", scaling=dict(scaling, **kw))
    same = gllm_amd.Rotary(128, theta=500.0, rotary_dim=64, device="cpu", scaling=dict(scaling, rope_theta=500.0,
                                                                                       partial_rotary_factor=0.5))
    plain = gllm_amd.Rotary(128, theta=500.0, rotary_dim=64, device="cpu", scaling=scaling)
    assert torch.equal(same.freq, plain.freq) and same.factor == plain.factor


@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("kw", [
    dict(v=torch.zeros(6, 2, 64, dtype=torch.bfloat16)), dict(sin=torch.zeros(5, 32)), dict(query_lens=torch.ones(4)),
    dict(query_lens=torch.zeros(0)), dict(q_out=torch.zeros(6, 4, 64)), dict(q=torch.zeros(6, 4, 64).bfloat16(), q_out=torch.zeros(6, 4, 64)),
    dict(q=torch.zeros(6, 4, 64), q_out=torch.zeros(5, 4, 64)), dict(q=torch.zeros(5, 4, 64), q_out=torch.zeros(6, 4, 64)),
    dict(q=torch.zeros(6, 4, 64), q_out=torch.zeros(6, 4, 64).half()), dict(rope_rows=torch.arange(5))])
def test_rope_kv_write_refuses(kw, kv4):
    """Tensors that the kernels would read or write past their end, or in another dtype."""
    cache = torch.zeros(4, 2, paged.kv4_record_bytes(16, 64), dtype=torch.uint8) if kv4 else torch.zeros(64, 2, 64)
    a = dict(k=torch.zeros(6, 2, 64), v=torch.zeros(6, 2, 64), cos=torch.zeros(6, 32), sin=torch.zeros(6, 32), k_cache=cache,
             v_cache=cache, slot_mapping=torch.arange(6))
    a.update(kw)
    with pytest.raises(ValueError):
        paged.rope_kv_write(**a)
