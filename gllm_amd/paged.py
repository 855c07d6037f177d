"""Python entry points over the C ABI: fused RoPE + KV write, batch plans and
paged attention.  Tensors are torch device tensors; every call is enqueued on
torch's current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
import math
import operator

import torch
import torch.nn.functional as F

from . import _lib


def _rows(t: torch.Tensor, heads: int, head_dim: int, name: str) -> int:
    """Row stride (elements) of a [..., heads, head_dim] tensor whose leading
    dims flatten to rows without a copy."""
    if t.is_contiguous():                  # the common case, without a look at each dim
        shape, hd = t.shape, heads * head_dim
        if len(shape) >= 3 and shape[-1] == head_dim and shape[-2] == heads and t.stride()[-3] == hd:
            return hd
    if t.dim() < 2 or t.shape[-1] != head_dim or t.shape[-2] != heads:
        raise ValueError(f"{name}: expected [..., {heads}, {head_dim}], got {tuple(t.shape)}")
    if t.stride(-1) != 1 or t.stride(-2) != head_dim:
        raise ValueError(f"{name}: head dim and heads must be contiguous")
    lead = t.shape[:-2]
    stride = t.stride(-3) if t.dim() >= 3 else heads * head_dim
    # leading dims must flatten to one row axis of constant stride
    expect = stride
    for d in range(t.dim() - 3, -1, -1):
        if t.shape[d] > 1 and t.stride(d) != expect:
            raise ValueError(f"{name}: leading dims do not flatten to rows")
        expect *= t.shape[d]
    del lead
    return stride


def _flat(t: torch.Tensor) -> torch.Tensor:
    """The last dim as rows.  A single row goes through reshape too, which
    replaces the stride it has from a wider tensor."""
    return t if t.dim() == 2 and t.shape[0] != 1 else t.reshape(-1, t.shape[-1])


def _index_rows(t: torch.Tensor) -> torch.Tensor:
    """Row indices as one contiguous int64 vector."""
    if t.dim() == 1 and t.dtype == torch.int64 and t.is_contiguous():
        return t
    return t.reshape(-1).to(torch.int64).contiguous()


def _cache_rows(k_cache: torch.Tensor, v_cache: torch.Tensor, Hkv: int, D: int) -> None:
    """Checks that the caches are [num_slots, Hkv, D] with contiguous rows, of one
    dtype, and that V has K's slots (a call counts the slots, and reads the dtype, of K)."""
    shape, stride = k_cache.shape, k_cache.stride()
    if len(shape) == 3 and shape[1] == Hkv and shape[2] == D and stride[1] == D and stride[2] == 1 \
            and v_cache.shape == shape and v_cache.stride() == stride and v_cache.dtype == k_cache.dtype:
        return                             # the common case, without a look at each cache
    for t, nm in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        shape = t.shape
        if len(shape) != 3 or shape[1] != Hkv or shape[2] != D or t.stride()[1:] != (D, 1):
            raise ValueError(f"{nm}: expected [num_slots, {Hkv}, {D}] with contiguous rows")
    if v_cache.dtype != k_cache.dtype or v_cache.shape[0] < k_cache.shape[0]:
        raise ValueError(f"k_cache {k_cache.dtype} of {k_cache.shape[0]} slots, v_cache {v_cache.dtype} of {v_cache.shape[0]}")


# Storage type of a 4-bit KV cache (OCP MXFP4): uint8 ``[num_blocks, Hkv,
# kv4_record_bytes(block_size, D)]``.  A record holds, of one block and KV head,
# block_size rows of D / 2 code bytes (fp4 e2m1, the even dim in the low half),
# then block_size rows of D / 32 scale bytes (a block of 32 dims stands for code x
# 2^(byte - 127)), padded to 16 bytes.
KV4 = torch.uint8


def kv4_record_bytes(block_size: int, head_dim: int) -> int:
    """Bytes of one (block, KV head) of a 4-bit cache."""
    if head_dim <= 0 or head_dim % 32 or block_size <= 0:
        raise ValueError(f"4-bit cache: head_dim {head_dim} must be a multiple of 32, block_size {block_size} positive")
    return -(-block_size * (head_dim // 32 * 17) // 16) * 16


def _kv4_block_size(cache: torch.Tensor, Hkv: int, D: int, name: str = "cache") -> int:
    """The block size of a 4-bit cache of Hkv heads of D, after a check of its
    layout (a record's padding is shorter than a key's bytes)."""
    shape, unit = cache.shape, D // 32 * 17
    if cache.dtype == KV4 and len(shape) == 3 and shape[1] == Hkv and D > 0 and D % 32 == 0 and shape[2] >= unit:
        bs, rec = shape[2] // unit, shape[2]
        if -(-bs * unit // 16) * 16 == rec and cache.stride()[1:] == (rec, 1):
            return bs
    raise ValueError(f"{name}: expected a 4-bit cache of head_dim {D} (a multiple of 32), uint8 [num_blocks, {Hkv}, record "
                     f"bytes] with contiguous blocks, got {cache.dtype} {tuple(shape)}")


def _kv4_blocks(k_cache: torch.Tensor, v_cache: torch.Tensor, Hkv: int, D: int, block_size: int) -> int:
    """Blocks of a 4-bit cache pair of a plan's block size."""
    for t, nm in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if _kv4_block_size(t, Hkv, D, nm) != block_size:
            raise ValueError(f"{nm}: blocks of {t.shape[2] // (D // 32 * 17)} rows, the plan's have {block_size}")
    if k_cache.shape[0] != v_cache.shape[0]:
        raise ValueError("k_cache and v_cache must have the same shape")
    return k_cache.shape[0]


def _kv_code(cache: torch.Tensor) -> int:
    return _lib.DTYPE_MXFP4 if cache.dtype == KV4 else _lib.dtype_code(cache.dtype)


def rope_kv_write(k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                  query_lens: torch.Tensor | None = None, q: torch.Tensor | None = None,
                  q_out: torch.Tensor | None = None, rope_rows: torch.Tensor | None = None) -> None:
    """RoPE on k (and q -> q_out) plus the KV-cache write of
    ``gllm/model/layers/attention.py:151-161``.

    k/v ``[..., Hkv, D]`` (token rows), cos/sin ``[..., D/2]`` with one row per
    token (or ``rope_rows`` indexing a table), caches ``[num_slots, Hkv, D]``,
    ``slot_mapping`` int64 with one slot per token.  With ``query_lens``
    (padded ``[B, T_q]`` token layout) rows past each sequence's length are not
    written.  The caches may be 4-bit ones (:data:`KV4`; slots must differ there).
    """
    shape, dtype = k.shape, k.dtype
    Hkv, D = shape[-2], shape[-1]
    if v.shape != shape or v.dtype != dtype:
        raise ValueError("k and v shapes or dtypes differ")
    ks = _rows(k, Hkv, D, "k")
    vs = _rows(v, Hkv, D, "v")
    n = k.numel() // (Hkv * D)
    if k_cache.dtype == KV4:
        bs = _kv4_block_size(k_cache, Hkv, D, "k_cache")
        num_slots = _kv4_blocks(k_cache, v_cache, Hkv, D, bs) * bs
    else:
        _cache_rows(k_cache, v_cache, Hkv, D)
        num_slots = k_cache.shape[0]
    if k_cache.stride(0) != v_cache.stride(0) or k_cache.shape[0] != v_cache.shape[0]:
        raise ValueError("k_cache and v_cache must have the same shape and slot stride")
    sm = slot_mapping if slot_mapping.dim() == 1 else slot_mapping.reshape(-1)
    if sm.dtype != torch.int64 or sm.numel() != n or not sm.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int64 with one entry per token")
    cs, sn = _flat(cos), _flat(sin)
    if cs.stride(-1) != 1 or sn.stride(-1) != 1 or cs.stride(0) != sn.stride(0):
        raise ValueError("cos/sin must have contiguous rows of equal stride")
    if cs.dtype != dtype or sn.dtype != dtype:
        raise ValueError("cos/sin must be in the model dtype")
    for rows, width in {cs.shape, sn.shape}:
        if width < D // 2 or (rope_rows is None and rows < n):
            raise ValueError("cos/sin need one row of at least D/2 entries per token")
    tps = 0
    ql = None
    if query_lens is not None:
        ql = query_lens.to(torch.int32).contiguous()
        if ql.numel() == 0 or n % ql.numel():
            raise ValueError("query_lens: the tokens must be as many rows for each sequence")
        tps = n // ql.numel()
    qs = qos = 0
    Hq = 1
    if q_out is not None:
        if q is None or q.dtype != dtype or q_out.dtype != dtype:
            raise ValueError("q_out needs a q, both in the dtype of k")
        Hq = q.shape[-2]
        qs = _rows(q, Hq, D, "q")
        qos = _rows(q_out, Hq, D, "q_out")
        if min(q.numel(), q_out.numel()) < n * Hq * D:
            raise ValueError("q and q_out need one row per token")
    rr = None
    if rope_rows is not None:
        rr = _index_rows(rope_rows)
        if rr.numel() < n:
            raise ValueError("rope_rows needs one entry per token")
    dev = k.device
    lib = _lib.load()
    if k_cache.dtype == KV4:
        _lib.check(lib.gllm_rope_kv_write_kv4(
            _lib.ptr(q), _lib.ptr(q_out), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            sm.data_ptr(), _lib.ptr(ql), tps, cs.data_ptr(), sn.data_ptr(), _lib.ptr(rr), cs.stride(0), n,
            Hq, Hkv, D, qs, ks, vs, qos, k_cache.stride(0), num_slots, bs, _lib.dtype_code(k.dtype),
            _lib.stream_ptr(dev)))
        return
    _lib.check(lib.gllm_rope_kv_write(
        _lib.ptr(q), _lib.ptr(q_out), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        sm.data_ptr(), _lib.ptr(ql), tps, cs.data_ptr(), sn.data_ptr(), _lib.ptr(rr), cs.stride(0), n,
        Hq, Hkv, D, qs, ks, vs, qos, k_cache.stride(0), k_cache.shape[0],
        _lib.dtype_code(k.dtype), _lib.dtype_code(k_cache.dtype), _lib.stream_ptr(dev)))


def _same_device(index: int, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, the call on device {index}")


def _row_stride(t: torch.Tensor, shape, heads: int, head_dim: int, name: str) -> int:
    """:func:`_rows`, without its look at the strides of contiguous rows."""
    if len(shape) >= 3 and shape[-1] == head_dim and shape[-2] == heads and t.is_contiguous():
        return heads * head_dim
    return _rows(t, heads, head_dim, name)


def rotary_kv_write(k: torch.Tensor | None, v: torch.Tensor | None, positions: torch.Tensor, rotary,
                    k_cache: torch.Tensor | None, v_cache: torch.Tensor | None, slot_mapping: torch.Tensor | None,
                    query_lens: torch.Tensor | None = None, q: torch.Tensor | None = None,
                    q_out: torch.Tensor | None = None) -> None:
    """Rotary positions on k (and q -> q_out) plus the KV-cache write, in one
    launch and without a cos/sin table.

    ``rotary``: a :class:`gllm_amd.Rotary`; ``positions`` int64, one per token.
    k/v ``[..., Hkv, D]`` (token rows), caches ``[num_slots, Hkv, D]`` of any
    cache dtype or 4-bit ones (:data:`KV4`), ``slot_mapping`` int64 with one slot
    per token (outside the cache: not written; 4-bit: slots must differ),
    ``query_lens`` as in :func:`rope_kv_write`.  ``q_out`` may be q itself.  k is
    rounded once, to the cache dtype; q once, to the model dtype.
    """
    x = q if k is None else k
    if x is None or (k is None) != (v is None) or (q is None) != (q_out is None):
        raise ValueError("k and v, and q and q_out, go together; at least one pair is needed")
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    if len(shape) < 2 or q is not None and q.dim() < 2 or not shape[-2]:
        raise ValueError("expected [..., heads, head_dim] rows")
    if dev >= 0 and dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return rotary_kv_write(k, v, positions, rotary, k_cache, v_cache, slot_mapping, query_lens, q, q_out)
    D, H = shape[-1], shape[-2]
    if D != rotary.head_dim:
        raise ValueError(f"head_dim {D}, the rotary positions are for {rotary.head_dim}")
    n = x.numel() // (H * D)
    freq = rotary.freq
    pos, kind = positions, positions.dtype
    if kind != torch.int64 or not pos.is_contiguous():
        pos = _index_rows(pos)
    if pos.numel() != n or kind.is_floating_point:
        raise ValueError("positions must be integers, one per token")
    ks = vs = qs = qos = stride = num_slots = bs = 0
    Hq = Hkv = 1
    kp = vp = kcp = vcp = smp = qp = qop = qlp = None
    kv_code, tps = _lib.DTYPE_F32, 0
    same = pos.get_device() == dev and freq.get_device() == dev
    if k is not None:
        if k_cache is None or v_cache is None or slot_mapping is None:
            raise ValueError("k and v need caches and a slot mapping")
        Hkv = H
        if v.shape != shape or v.dtype != dtype:
            raise ValueError("k and v shapes or dtypes differ")
        ks = Hkv * D if k.is_contiguous() else _rows(k, Hkv, D, "k")     # k's and v's heads and dims are the shape's
        vs = Hkv * D if v.is_contiguous() else _rows(v, Hkv, D, "v")
        cdtype, cshape, cstride = k_cache.dtype, k_cache.shape, k_cache.stride()
        if v_cache.shape != cshape or v_cache.stride() != cstride or v_cache.dtype != cdtype:
            raise ValueError("k_cache and v_cache must have the same shape, dtype and strides")
        if cdtype == KV4:
            bs = _kv4_block_size(k_cache, Hkv, D, "k_cache")
            num_slots = cshape[0] * bs
            kv_code = _lib.DTYPE_MXFP4
        else:
            if len(cshape) != 3 or cshape[1] != Hkv or cshape[2] != D or cstride[1:] != (D, 1):
                raise ValueError(f"k_cache and v_cache: expected [num_slots, {Hkv}, {D}] with contiguous rows")
            num_slots = cshape[0]
            kv_code = _lib.dtype_code(cdtype)
        stride = cstride[0]
        sm = slot_mapping
        if not sm.is_contiguous() and sm.dim() != 1:
            sm = sm.reshape(-1)
        if sm.dtype != torch.int64 or sm.numel() != n or not sm.is_contiguous():
            raise ValueError("slot_mapping must be contiguous int64 with one entry per token")
        same = same and v.get_device() == dev and k_cache.get_device() == dev and v_cache.get_device() == dev \
            and sm.get_device() == dev
        kp, vp, kcp, vcp, smp = k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), sm.data_ptr()
    if q is not None:
        qshape, oshape = q.shape, q_out.shape
        Hq = qshape[-2]
        if q.dtype != dtype or q_out.dtype != dtype or q.numel() != n * Hq * D or q_out.numel() != n * Hq * D:
            raise ValueError("q and q_out need the model dtype and one row per token")
        qs, qos = _row_stride(q, qshape, Hq, D, "q"), _row_stride(q_out, oshape, Hq, D, "q_out")
        same = same and q.get_device() == dev and q_out.get_device() == dev
        qp, qop = q.data_ptr(), q_out.data_ptr()
    if query_lens is not None:
        ql = query_lens.to(torch.int32).contiguous()
        if ql.numel() == 0 or n % ql.numel():
            raise ValueError("query_lens: the tokens must be as many rows for each sequence")
        same = same and ql.get_device() == dev
        tps, qlp = n // ql.numel(), ql.data_ptr()
    if not same:
        _same_device(dev, v=v, q=q, q_out=q_out, positions=positions, freq=freq, k_cache=k_cache, v_cache=v_cache,
                     slot_mapping=slot_mapping, query_lens=query_lens)
    if n == 0:
        return
    _lib.check(_lib.load().gllm_rotary_kv_write(
        qp, qop, kp, vp, kcp, vcp, smp, qlp, tps, freq.data_ptr(), rotary.factor, pos.data_ptr(), rotary.rotary_dim,
        rotary.interleaved, n, Hq, Hkv, D, qs, ks, vs, qos, stride, num_slots, bs, _lib.dtype_code(dtype), kv_code,
        _lib.raw_stream(dev)))


def rotary_rotate(x: torch.Tensor, positions: torch.Tensor, rotary, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions of ``x [..., H, D]``, one position per row of heads;
    returns ``out`` (a new tensor by default, x itself rotates in place)."""
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    rotary_kv_write(None, None, positions, rotary, None, None, None, q=x, q_out=out)
    return out


def kv4_values(cache: torch.Tensor, slots: torch.Tensor, head_dim: int, dtype: torch.dtype,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows of a 4-bit cache (:data:`KV4`) as the values they stand for, in
    ``dtype``: ``[N, Hkv, head_dim]`` for int64 ``slots [N]`` (zeros for a slot
    outside the cache).  For moving rows to another cache or looking at them."""
    dev = cache.get_device()
    if dev >= 0 and dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return kv4_values(cache, slots, head_dim, dtype, out)
    shape = cache.shape
    nb, Hkv = shape[0], shape[1] if len(shape) == 3 else 0
    bs = _kv4_block_size(cache, Hkv, head_dim)
    sl = slots if slots.dtype == torch.int64 and slots.is_contiguous() else _index_rows(slots)
    if sl.get_device() != dev or out is not None and out.get_device() != dev:
        raise ValueError(f"slots and out must be on the cache's device {cache.device}")
    n, stride = sl.numel(), Hkv * head_dim
    if out is None:
        out = torch.empty((n, Hkv, head_dim), dtype=dtype, device=cache.device)
    elif out.dtype != dtype or out.numel() != n * stride:
        raise ValueError(f"out must be {dtype} with one row per slot")
    else:
        stride = _row_stride(out, out.shape, Hkv, head_dim, "out")
    if n == 0:
        return out
    _lib.check(_lib.load().gllm_kv4_values(cache.data_ptr(), cache.stride(0), nb * bs, bs, sl.data_ptr(), n, Hkv, head_dim,
                                           out.data_ptr(), stride, _lib.dtype_code(dtype), _lib.raw_stream(dev)))
    return out


# Token count from which qkv_rope_kv_write projects with hipBLASLt (three
# F.linear calls) and then runs the RoPE + KV write kernel, where the 256-column
# tiles do not take the batch or are behind (_tiles_ok).
QKV_UNFUSED_FROM = 3072


class _Default(int):
    """A threshold nobody asked for: the routing may set it aside."""


def qkv_fused_ok(x: torch.Tensor, w_q: torch.Tensor, w_k: torch.Tensor, w_v: torch.Tensor,
                 k_cache: torch.Tensor, v_cache: torch.Tensor) -> bool:
    """Whether the fused kernels of :func:`qkv_rope_kv_write` take these rows,
    weights and caches: bf16 rows of a hidden size that is a multiple of 32, 16-byte
    aligned and not overlapping, a bf16 or fp8 cache, head dim 64 or 128."""
    hidden = x.shape[-1]
    if x.dim() != 2 or hidden % 32 or k_cache.shape[2] not in (64, 128):
        return False
    if k_cache.dtype not in (torch.bfloat16, torch.float8_e4m3fn) or v_cache.dtype != k_cache.dtype:
        return False
    return all(t.dtype == torch.bfloat16 and t.dim() == 2 and t.shape[1] == hidden and t.stride(1) == 1
               and t.stride(0) >= hidden and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0 for t in (x, w_q, w_k, w_v))


def _tiles_ok(n: int, hidden: int, Hq: int, Hkv: int, D: int, k_cache, v_cache, cos, sin, q_out) -> bool:
    """Whether the projection's 256-column tiles take the call and are ahead of
    the library at prompt sizes: heads that fill 256 columns within q and within
    k / v, whole aligned 16-byte chunks, a token count whose tiles fill their
    rounds (``gllm_qkv_tiles_ahead``, with the measurements), and hidden up to
    4096: above it the two are level or alternate with the token count (3,072-19,679
    tokens, library / fused time: hidden 4608 0.93-1.24, 5120 1.00-1.30, 6144
    0.98-1.18, 7168 0.94-1.18, 8192 0.88-1.07).  Layers of few heads, which the
    launcher gives to smaller tiles or the split, are ahead too (768 columns 1.3-2.3,
    1,024 1.2-1.8)."""
    if hidden % 64 or hidden > 4096 or D not in (64, 128) or (Hkv * D) % 256 or (Hq * D) % 256:
        return False
    if k_cache.stride(0) % 16 or cos.stride(0) % 8 or (q_out is not None and not q_out.is_contiguous()):
        return False
    return all(t is None or t.data_ptr() % 16 == 0 for t in (k_cache, v_cache, cos, sin, q_out)) \
        and bool(_lib.load().gllm_qkv_tiles_ahead(n, Hq, Hkv, D))


def qkv_rope_kv_write(x: torch.Tensor, w_q: torch.Tensor | None, w_k: torch.Tensor, w_v: torch.Tensor,
                      cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_mapping: torch.Tensor, *, rotate_q: bool = True, q_out: torch.Tensor | None = None,
                      query_lens: torch.Tensor | None = None, rope_rows: torch.Tensor | None = None,
                      split_k: bool = True, unfused_from: int | None = _Default(QKV_UNFUSED_FROM)):
    """Fused ``linear_q/k/v`` + RoPE + KV-cache write of
    ``gllm/model/layers/attention.py:139-161`` (bf16 model).

    x ``[..., hidden]`` token rows; weights as the checkpoint stores them
    (``w_q [Hq*D, hidden]``, ``w_k``/``w_v [Hkv*D, hidden]``, ``F.linear``
    convention); caches ``[num_slots, Hkv, D]``; cos/sin / ``rope_rows`` /
    ``query_lens`` / ``slot_mapping`` as in :func:`rope_kv_write`.  Returns q
    ``[N, Hq, D]`` (rotated if ``rotate_q``) or None when ``w_q`` is None.
    ``split_k``: let batches of few tokens split the hidden dimension over
    more workgroups (a device workspace); False forces the tile kernel.
    ``unfused_from``: from this many tokens the projections run as three
    ``F.linear`` (hipBLASLt) followed by :func:`rope_kv_write`; by default from
    QKV_UNFUSED_FROM where the fused kernel's large tiles do not take the batch;
    None runs the fused kernel at any size.  Head dims other than 64
    and 128, and models that are not bf16 (the fused kernel's projection is
    bf16 MFMA), always take the unfused path.
    """
    hidden = x.shape[-1]
    xs = _flat(x)
    if xs.stride(-1) != 1:
        raise ValueError("x rows must be contiguous")
    n = xs.shape[0]
    for t, nm in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dtype == KV4:
            raise ValueError(f"{nm}: 4-bit caches are written by rope_kv_write and rotary_kv_write")
        if t.dim() != 3 or t.stride()[1:] != (t.shape[2], 1):
            raise ValueError(f"{nm}: expected [num_slots, Hkv, D] with contiguous rows")
    if k_cache.shape != v_cache.shape or k_cache.stride(0) != v_cache.stride(0):
        raise ValueError("k_cache and v_cache must have the same shape and slot stride")
    _, Hkv, D = k_cache.shape
    for w, nm in ((w_k, "w_k"), (w_v, "w_v"), (w_q, "w_q")):
        if w is None and nm == "w_q":
            continue
        shape = w.shape
        if len(shape) != 2 or shape[1] != hidden or w.stride(1) != 1 or w.dtype != x.dtype:
            raise ValueError(f"{nm}: expected [heads * D, {hidden}] with contiguous rows in the model dtype")
    if w_k.shape[0] != Hkv * D or w_v.shape[0] != Hkv * D:
        raise ValueError("w_k / w_v must have num_kv_heads * head_dim rows")
    Hq = 0
    if w_q is not None:
        if w_q.shape[0] % D:
            raise ValueError("w_q rows must be a multiple of head_dim")
        Hq = w_q.shape[0] // D
        if q_out is None:
            q_out = torch.empty(n, Hq, D, dtype=x.dtype, device=x.device)
        if not (q_out.is_contiguous() and q_out.numel() == n * Hq * D) and (
                q_out.reshape(-1, Hq * D).shape[0] != n or q_out.stride(-1) != 1):
            raise ValueError("q_out must hold one contiguous row of Hq * D per token")
    sm = slot_mapping if slot_mapping.dim() == 1 else slot_mapping.reshape(-1)
    if sm.dtype != torch.int64 or sm.numel() != n or not sm.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int64 with one entry per token")
    cs, sn = _flat(cos), _flat(sin)
    if cs.stride(-1) != 1 or sn.stride(-1) != 1 or cs.stride(0) != sn.stride(0):
        raise ValueError("cos/sin must have contiguous rows of equal stride")
    if cs.dtype != x.dtype or sn.dtype != x.dtype:
        raise ValueError("cos/sin must be in the model dtype")
    if cs.shape[-1] < D // 2 or (rope_rows is None and cs.shape[0] < n):
        raise ValueError("cos/sin need one row of at least D/2 entries per token")
    tps = 0
    ql = None
    if query_lens is not None:
        ql = query_lens.to(torch.int32).contiguous()
        tps = n // ql.numel()
    rr = None
    if rope_rows is not None:
        rr = _index_rows(rope_rows)
    if (D not in (64, 128) or x.dtype != torch.bfloat16 or unfused_from is not None and n >= unfused_from
            and not (isinstance(unfused_from, _Default)
                     and qkv_fused_ok(xs, w_k if w_q is None else w_q, w_k, w_v, k_cache, v_cache)
                     and _tiles_ok(n, hidden, Hq, Hkv, D, k_cache, v_cache, cs, sn, q_out))):
        k = F.linear(xs, w_k).view(n, Hkv, D)
        v = F.linear(xs, w_v).view(n, Hkv, D)
        q = F.linear(xs, w_q).view(n, Hq, D) if w_q is not None else None
        rotq = q is not None and rotate_q
        rope_kv_write(k, v, cos, sin, k_cache, v_cache, sm, query_lens=query_lens,
                      q=q if rotq else None, q_out=q_out.view(n, Hq, D) if rotq else None, rope_rows=rr)
        if q is not None and not rotate_q:
            q_out.view(n, Hq, D).copy_(q)
        return q_out
    lib = _lib.load()
    qrow = 0
    if q_out is not None:
        qrow = Hq * D if q_out.is_contiguous() else q_out.reshape(-1, Hq * D).stride(0)
    wsb = lib.gllm_qkv_workspace_bytes(n, hidden, max(Hq, 1), Hkv, D, int(w_q is not None)) if split_k else 0
    # per call, from the caching allocator: calls on other streams have their own
    ws = torch.empty(wsb, dtype=torch.uint8, device=x.device) if wsb else None
    _lib.check(lib.gllm_qkv_rope_kv_write(
        xs.data_ptr(), xs.stride(0), n, hidden, _lib.ptr(w_q), w_q.stride(0) if w_q is not None else 0,
        w_k.data_ptr(), w_k.stride(0), w_v.data_ptr(), w_v.stride(0), _lib.ptr(q_out), qrow, int(bool(rotate_q)),
        k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.shape[0], sm.data_ptr(), _lib.ptr(ql),
        tps, cs.data_ptr(), sn.data_ptr(), _lib.ptr(rr), cs.stride(0), max(Hq, 1), Hkv, D,
        _lib.dtype_code(x.dtype), _lib.dtype_code(k_cache.dtype), _lib.ptr(ws), wsb, _lib.stream_ptr(x.device)))
    return q_out


def rope_rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                rope_rows: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate-half RoPE of ``x [..., H, D]`` (``attention.py:91-118``),
    bit-identical to the reference's per-op rounding; returns a new tensor."""
    H, D = x.shape[-2], x.shape[-1]
    xs = _rows(x, H, D, "x")
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    n = x.numel() // (H * D)
    cs, sn = _flat(cos), _flat(sin)
    rr = None if rope_rows is None else rope_rows.reshape(-1).to(torch.int64).contiguous()
    if cs.shape[-1] < D // 2 or (rr is None and cs.shape[0] < n) or cs.stride(0) != sn.stride(0):
        raise ValueError("cos/sin need one row of at least D/2 entries per token")
    lib = _lib.load()
    _lib.check(lib.gllm_rope_kv_write(
        x.data_ptr(), out.data_ptr(), None, None, None, None, None, None, 0, cs.data_ptr(), sn.data_ptr(),
        _lib.ptr(rr), cs.stride(0), n, H, 1, D, xs, 0, 0, H * D, 0, 0,
        _lib.dtype_code(x.dtype), _lib.dtype_code(x.dtype), _lib.stream_ptr(x.device)))
    return out


def build_metadata(block_table: torch.Tensor, seq_lens: torch.Tensor, query_lens: torch.Tensor, block_size: int,
                   *, q_seq_stride: int = 0, num_rows: int | None = None):
    """Query-row slot mapping and positions on the device (``gllm/llm/llm.py:
    245-281`` without the per-row host loop or the dense bias).

    ``block_table`` int32 ``[B, W]`` (contiguous rows), ``seq_lens`` /
    ``query_lens`` int32 ``[B]`` on the same device.  ``q_seq_stride`` > 0:
    the reference's padded ``[B, T_q]`` rows (padded rows get slot 0);
    0: packed rows, and ``cu_seqlens`` (int32 ``[B+1]``) is returned too.
    ``num_rows`` (packed) is the total query rows; if omitted it is read back
    from the device (one synchronisation).  Returns
    ``(slot_mapping int64 [rows], positions int64 [rows], cu_seqlens or None)``.
    """
    B = int(seq_lens.shape[0])
    dev = block_table.device
    for t, nm in ((seq_lens, "seq_lens"), (query_lens, "query_lens"), (block_table, "block_table")):
        if t.dtype != torch.int32 or t.device != dev:
            raise ValueError(f"{nm} must be int32 on {dev}")
    if block_table.dim() != 2 or block_table.stride(1) != 1 or block_table.shape[0] < B or query_lens.shape[0] != B:
        raise ValueError("block_table must be [B, W] with contiguous rows and lengths [B]")
    if not seq_lens.is_contiguous() or not query_lens.is_contiguous():
        raise ValueError("lengths must be contiguous")
    if q_seq_stride > 0:
        rows = B * q_seq_stride
    else:
        rows = int(query_lens.sum().item()) if num_rows is None else int(num_rows)
    slots = torch.empty(rows, dtype=torch.int64, device=dev)
    pos = torch.empty(rows, dtype=torch.int64, device=dev)
    cu = torch.empty(B + 1, dtype=torch.int32, device=dev) if q_seq_stride == 0 else None
    lib = _lib.load()
    _lib.check(lib.gllm_build_metadata(block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                                       seq_lens.data_ptr(), query_lens.data_ptr(), B, q_seq_stride, block_size,
                                       slots.data_ptr(), pos.data_ptr(), _lib.ptr(cu), rows,
                                       _lib.stream_ptr(dev)))
    return slots, pos, cu


# split_tokens value that asks for a page-balanced decode plan (decode-only or mixed batches)
BALANCED = -1


class AttentionPlan:
    """Work plan for one batch (built once per engine step, reused by every
    layer).  Lengths are host ints, as ``gllm/llm/llm.py:233-241`` has them.

    ``q_seq_stride`` > 0: sequence i's rows start at ``i * q_seq_stride`` (the
    reference's padded ``[B, T_q]`` layout); 0: packed rows.  ``split_tokens``:
    0 lets the planner choose, a multiple of 32 fixes the decode split length,
    ``BALANCED`` deals the decode sequences' keys evenly to the workgroups (in
    a mixed batch: to part of the CUs, the prefill items run on the rest).

    ``window``: sliding window; the row at position p sees the ``window`` keys
    up to its own (t > p - window) and the sequence's first ``sinks`` keys
    (None: every earlier key).  Keys that no row of the batch sees are never
    read, so blocks that hold only such keys may have been given back.

    ``shared_prefixes``: ``[(sequences, tokens), ...]``, sequences of the batch (a
    sequence in one group at most) that have their first ``tokens`` keys in
    common: their block-table rows name blocks with the same contents there.  The
    MFMA kernels read those keys once for all decode sequences of the group
    (query_len x G <= 16; from 256 tokens on, at head dim 64 from 512); longer ones and
    the generic kernel read them for each.  Not with a window; the decode share is
    page-balanced (``split_tokens`` 0 or BALANCED).  In a batch that also holds prompts
    this pays from about a third of the decode sequences' keys on (fewer: up to 16% slower).
    """

    def __init__(self, query_lens, seq_lens, *, num_q_heads: int, num_kv_heads: int, head_dim: int,
                 block_size: int, dtype: torch.dtype, device, q_seq_stride: int = 0,
                 split_tokens: int = 0, heads_per_wg: int = 0, window: int | None = None, sinks: int = 0,
                 shared_prefixes=()):
        ql = [int(x) for x in query_lens]
        sl = [int(x) for x in seq_lens]
        if len(ql) != len(sl):
            raise ValueError("query_lens and seq_lens differ in length")
        window, sinks = None if window is None else operator.index(window), operator.index(sinks)
        if window is not None and not 1 <= window < 1 << 31:
            raise ValueError(f"window {window} must be at least 1 (None: no window)")
        if not 0 <= sinks < 1 << 31 or (sinks and window is None):
            raise ValueError(f"sinks {sinks} must be >= 0 and go with a window")
        lib = _lib.load()
        self._lib = lib
        self._h = ctypes.c_void_p()
        qa = (ctypes.c_int32 * max(len(ql), 1))(*ql)
        sa = (ctypes.c_int32 * max(len(sl), 1))(*sl)
        sizes = (ctypes.byref(self._h), qa, sa, len(ql), q_seq_stride, num_q_heads, num_kv_heads, head_dim, block_size,
                 _lib.dtype_code(dtype), split_tokens, heads_per_wg)
        groups = [([operator.index(i) for i in seqs], operator.index(n)) for seqs, n in shared_prefixes]
        if groups:
            if window is not None:
                raise NotImplementedError("shared prefixes with a window, which hides them")
            members, starts = [i for seqs, _ in groups for i in seqs], [0]
            for seqs, _ in groups:
                starts.append(starts[-1] + len(seqs))
            if not all(-(1 << 31) <= x < 1 << 31 for x in members + [n for _, n in groups]):
                raise ValueError("shared prefixes: sequence or token count out of range")
            arrays = [(ctypes.c_int32 * max(len(x), 1))(*x) for x in (starts, members, [n for _, n in groups])]
            _lib.check(lib.gllm_attn_plan_create_shared(*sizes, len(groups), *arrays))
        else:
            _lib.check(lib.gllm_attn_plan_create_window(*sizes, window or 0, sinks))
        self.shared_prefixes = groups
        self.window, self.sinks = window, sinks
        self.num_q_heads, self.num_kv_heads, self.head_dim = num_q_heads, num_kv_heads, head_dim
        self.block_size, self.dtype = block_size, dtype
        self.query_lens, self.seq_lens = ql, sl
        self.q_seq_stride = q_seq_stride
        self.device = torch.device(device)
        nbytes = lib.gllm_attn_plan_workspace_bytes(self._h)
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        _lib.check(lib.gllm_attn_plan_upload(self._h, self.workspace.data_ptr(), nbytes,
                                             _lib.stream_ptr(self.device)))
        keys = ("work_items", "split_tokens", "decode_seqs", "prefill_seqs", "partials", "rows", "heads_per_wg",
                "decode_waves", "prefill_waves", "decode_segments", "mixed_half")
        if groups:                         # two facts more, the first of which costs a count
            keys += ("most_task_blocks", "prefix_items")
        arr = (ctypes.c_int64 * len(keys))()
        _lib.check(lib.gllm_attn_plan_info(self._h, arr, len(keys)))
        self._info = dict(zip(keys, list(arr)))
        # facts every launch checks, computed once (a plan serves every layer of a step)
        self.rows = self._info["rows"]
        self.max_seq_len = max(sl, default=0)
        # a window that hides no key of the batch is none: the kernels are the plain ones
        self.hides_keys = window is not None and self.max_seq_len > window + sinks
        self.max_query_len = max(ql, default=0)
        self.table_width = -(-self.max_seq_len // block_size)

    @property
    def info(self) -> dict:
        return dict(self._info)

    def __del__(self):
        h = getattr(self, "_h", None)
        lib = getattr(self, "_lib", None)
        if h is not None and h.value and lib is not None:
            try:
                lib.gllm_attn_plan_destroy(h)
            except Exception:      # interpreter shutdown: ctypes may already be torn down
                return
            self._h = None


def fused_kv_write_ok(plan: AttentionPlan, kv_dtype: torch.dtype) -> bool:
    """Whether :func:`paged_attention` can take ``kv_new`` for this plan and
    cache dtype: every sequence on the decode path of the kernel that runs
    (MFMA kernels: query_len x G <= 16; generic kernel: query_len <= 16, no
    sliding window that hides a key), and no 4-bit cache."""
    if not plan.max_query_len or kv_dtype == KV4:   # no sequences; a 4-bit cache is written by a call of its own
        return False
    mfma = (plan.dtype in (torch.bfloat16, torch.float16) and plan.head_dim in (64, 128)
            and kv_dtype in (plan.dtype, torch.float8_e4m3fn))
    G = plan.num_q_heads // plan.num_kv_heads
    if mfma:
        return plan.max_query_len * G <= 16
    return plan.max_query_len <= 16 and not getattr(plan, "hides_keys", plan.window is not None)


def paged_attention(plan: AttentionPlan, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, out: torch.Tensor | None = None,
                    rope: tuple | None = None, scale: float | None = None,
                    kv_new: tuple | None = None) -> torch.Tensor:
    """Attention over the paged cache for every query row in ``plan``.

    q ``[rows, Hq, D]`` or ``[B, T_q, Hq, D]`` (rows flattened), caches
    ``[num_slots, Hkv, D]`` or 4-bit ones (:data:`KV4`), block_table int32 ``[B, W]``.  ``rope`` =
    ``(cos, sin, mode)`` with mode ``"position"`` (table rows ``c_i + r``) or
    ``"row"`` (one cos/sin row per query row, the reference's gathered
    ``cos_pos``) rotates q on load.  ``kv_new`` = ``(k, v)``, one row per
    query row in q's layout (``[..., Hkv, D]``): the new tokens' K/V, rotated
    (k) and written into the cache at their keys' slots by the same launch
    (``attention.py:151-161`` + this attention; the plan must pass
    :func:`fused_kv_write_ok`).  Returns ``out`` (same layout as q).
    """
    Hq, Hkv, D = plan.num_q_heads, plan.num_kv_heads, plan.head_dim
    qs = _rows(q, Hq, D, "q")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os_ = Hq * D
    else:
        os_ = _rows(out, Hq, D, "out")
        if out.numel() < plan.rows * Hq * D:
            raise ValueError(f"out has {out.numel() // (Hq * D)} rows, the plan addresses {plan.rows}")
    if q.dtype != plan.dtype or out.dtype != plan.dtype:
        raise ValueError("q/out dtype differs from the plan's")
    if k_cache.dtype == KV4:
        num_blocks = _kv4_blocks(k_cache, v_cache, Hkv, D, plan.block_size)
    else:
        _cache_rows(k_cache, v_cache, Hkv, D)
        num_blocks = k_cache.shape[0] // plan.block_size
    if k_cache.stride(0) != v_cache.stride(0):
        raise ValueError("k_cache and v_cache slot strides differ")
    bt_shape = block_table.shape
    if block_table.dtype != torch.int32 or len(bt_shape) != 2 or block_table.stride(1) != 1:
        raise ValueError("block_table must be int32 [B, W] with contiguous rows")
    if bt_shape[0] < len(plan.query_lens):
        raise ValueError("block_table has fewer rows than the plan's sequences")
    if bt_shape[1] < plan.table_width:
        raise ValueError(f"block_table width {bt_shape[1]} < {plan.table_width} blocks the longest "
                         "sequence needs")
    rows = q.numel() // (Hq * D)
    if rows < plan.rows:
        raise ValueError(f"q has {rows} rows, the plan addresses {plan.rows}")
    cos_p = sin_p = None
    rs = 0
    mode = _lib.ROPE_NONE
    if rope is not None:
        cos, sin, m = rope
        mode = {"position": _lib.ROPE_BY_POSITION, "row": _lib.ROPE_BY_ROW}[m]
        cos, sin = _flat(cos), _flat(sin)
        if cos.stride(-1) != 1 or sin.stride(-1) != 1 or cos.stride(0) != sin.stride(0):
            raise ValueError("cos/sin must have contiguous rows of equal stride")
        if cos.dtype != q.dtype:
            raise ValueError("cos/sin must be in the model dtype")
        need_rows = plan.max_seq_len if m == "position" else plan.rows
        if cos.shape[0] < need_rows or cos.shape[1] < D // 2:
            raise ValueError(f"cos/sin have {cos.shape[0]} rows, {need_rows} needed")
        cos_p, sin_p, rs = cos.data_ptr(), sin.data_ptr(), cos.stride(0)
    sc = 1.0 / math.sqrt(D) if scale is None else float(scale)
    lib = plan._lib
    if kv_new is not None:
        kn, vn = kv_new
        if kn.dtype != q.dtype or vn.dtype != q.dtype:
            raise ValueError("k_new / v_new must be in the model dtype")
        ks = _rows(kn, Hkv, D, "k_new")
        vs = _rows(vn, Hkv, D, "v_new")
        if kn.numel() // (Hkv * D) < plan.rows or vn.numel() // (Hkv * D) < plan.rows:
            raise ValueError("k_new / v_new need one row per query row of the plan")
        _lib.check(lib.gllm_paged_attention_write_kv(
            plan._h, q.data_ptr(), qs, out.data_ptr(), os_, k_cache.data_ptr(), v_cache.data_ptr(),
            k_cache.stride(0), num_blocks, block_table.data_ptr(), block_table.stride(0), kn.data_ptr(), ks,
            vn.data_ptr(), vs, cos_p, sin_p, rs, mode, sc, _lib.dtype_code(q.dtype), _kv_code(k_cache),
            _lib.stream_ptr(q.device)))
        return out
    _lib.check(lib.gllm_paged_attention(
        plan._h, q.data_ptr(), qs, out.data_ptr(), os_, k_cache.data_ptr(), v_cache.data_ptr(),
        k_cache.stride(0), num_blocks, block_table.data_ptr(), block_table.stride(0), cos_p, sin_p, rs, mode,
        sc, _lib.dtype_code(q.dtype), _kv_code(k_cache), _lib.stream_ptr(q.device)))
    return out
