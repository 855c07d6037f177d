"""Sparse attention over the paged cache: each query row and KV head attends to
the keys of a few blocks, chosen by a cheap score over the blocks' key bounds.

A layer of an engine step, after the step's keys are in the cache::

    plan = SparsePlan(query_lens, seq_lens, blocks=128, ...)      # once per step
    write_key_bounds(plan, k_cache, bounds, block_table)
    selected = select_blocks(plan, q, bounds, block_table)
    out = sparse_attention(plan, q, k_cache, v_cache, block_table, selected)

with one ``bounds`` pool per layer (:func:`new_key_bounds`), which lives as long
as the layer's cache.  q comes rotated.  Every call is enqueued on torch's current
stream of the tensors' device.  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math
import operator

import torch

from . import _lib
from .paged import KV4, _index_rows, _kv4_blocks, _row_stride, _same_device


def key_bounds_bytes(num_kv_heads: int, head_dim: int) -> int:
    """Bytes of one block's key bounds: for each KV head ``head_dim`` int8 codes of
    the least key values and ``head_dim`` of the largest, then one exponent byte
    per head (a code stands for code x 2^(byte - 128); 255: unbounded), padded to 16."""
    if num_kv_heads <= 0 or not 0 < head_dim <= 256 or head_dim % 8:
        raise ValueError(f"key bounds: {num_kv_heads} KV heads of head_dim {head_dim} (a multiple of 8, at most 256)")
    return -(-num_kv_heads * (2 * head_dim + 1) // 16) * 16


def new_key_bounds(num_blocks: int, num_kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """Key bounds of a layer's pool: uint8 ``[num_blocks, key_bounds_bytes]``, zeros."""
    return torch.zeros((num_blocks, key_bounds_bytes(num_kv_heads, head_dim)), dtype=torch.uint8, device=device)


class SparsePlan:
    """Work plan of one batch (built once per engine step, reused by every layer).

    Lengths are host ints, rows packed or padded as in
    :class:`gllm_amd.AttentionPlan`.  A row at position p selects ``blocks`` of the blocks
    0 .. p // block_size (all, if there are no more): the first ``first_blocks``, the last
    ``recent_blocks`` (at least 1: the row's own) and those of the highest scores.
    The calls of one plan share its workspace and follow each other on one stream.
    Beside tables of the rows the workspace holds four areas of at most 256 MiB each (or what
    one tile or row takes), through which longer batches go in slabs.
    """

    def __init__(self, query_lens, seq_lens, *, num_q_heads: int, num_kv_heads: int, head_dim: int, block_size: int,
                 dtype: torch.dtype, device, blocks: int, first_blocks: int = 1, recent_blocks: int = 1,
                 q_seq_stride: int = 0):
        ql, sl = [int(x) for x in query_lens], [int(x) for x in seq_lens]
        if len(ql) != len(sl):
            raise ValueError("query_lens and seq_lens differ in length")
        blocks, first_blocks, recent_blocks = (operator.index(x) for x in (blocks, first_blocks, recent_blocks))
        if not all(0 <= x < 1 << 31 for x in (blocks, first_blocks, recent_blocks)):
            raise ValueError("blocks, first_blocks and recent_blocks must be >= 0")
        lib = _lib.load()
        self._lib = lib
        self._h = ctypes.c_void_p()
        qa, sa = (ctypes.c_int32 * max(len(ql), 1))(*ql), (ctypes.c_int32 * max(len(sl), 1))(*sl)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        _lib.check(lib.gllm_sparse_plan_create(ctypes.byref(self._h), qa, sa, len(ql), q_seq_stride, num_q_heads,
                                               num_kv_heads, head_dim, block_size, _lib.dtype_code(dtype), blocks,
                                               first_blocks, recent_blocks))
        self.num_q_heads, self.num_kv_heads, self.head_dim = num_q_heads, num_kv_heads, head_dim
        self.block_size, self.dtype = block_size, dtype
        self.blocks, self.first_blocks, self.recent_blocks = blocks, first_blocks, recent_blocks
        self.query_lens, self.seq_lens, self.q_seq_stride = ql, sl, q_seq_stride
        self.table_width = -(-max(sl, default=0) // block_size)
        self.record_bytes = key_bounds_bytes(num_kv_heads, head_dim)
        keys = ("rows", "query_rows", "touched_blocks", "score_tiles", "slabs", "splits", "tiles", "tile_workgroups", "tile_slabs",
                "row_slabs")
        arr = (ctypes.c_int64 * len(keys))()
        _lib.check(lib.gllm_sparse_plan_info(self._h, arr, len(keys)))
        self._info = dict(zip(keys, list(arr)))
        # facts that every call looks at
        self.rows = self._info["rows"]
        self.row_elements = self.rows * num_q_heads * head_dim
        self.index = self.device.index if self.device.type == "cuda" else -1
        self.code, self.scale = _lib.dtype_code(dtype), 1.0 / math.sqrt(head_dim)
        nbytes = lib.gllm_sparse_plan_workspace_bytes(self._h)
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        if self.device.type == "cuda":
            with torch.cuda.device(self.device):
                _lib.check(lib.gllm_sparse_plan_upload(self._h, self.workspace.data_ptr(), nbytes,
                                                       _lib.stream_ptr(self.device)))

    @property
    def info(self) -> dict:
        return dict(self._info)

    def __del__(self):
        h, lib = getattr(self, "_h", None), getattr(self, "_lib", None)
        if h is not None and h.value and lib is not None:
            try:
                lib.gllm_sparse_plan_destroy(h)
            except Exception:      # interpreter shutdown: ctypes may already be torn down
                return
            self._h = None


# The calls look at each tensor's dtype, shape, strides and device once: on a decode
# step the host's part of a call is as long as the kernels'.
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _on_device(plan: SparsePlan, call, *args):
    """`call` with the plan's device as the current one."""
    with torch.cuda.device(plan.device):
        return call(*args)


def _elsewhere(plan: SparsePlan, **tensors) -> None:
    """Refuses tensors that are not all on the plan's GPU."""
    if plan.device.type != "cuda":
        raise ValueError("the plan is for the CPU: the kernels need a GPU")
    _same_device(plan.index, **tensors)


def _table(plan: SparsePlan, block_table: torch.Tensor) -> int:
    """The row stride of the block table, after a check of it."""
    shape, stride = block_table.shape, block_table.stride()
    if block_table.dtype != torch.int32 or len(shape) != 2 or stride[1] != 1:
        raise ValueError("block_table must be int32 [B, W] with contiguous rows")
    if shape[0] < len(plan.query_lens) or shape[1] < plan.table_width:
        raise ValueError(f"block_table {tuple(shape)}: {len(plan.query_lens)} rows of {plan.table_width} blocks needed")
    return stride[0]


def _bounds(bounds: torch.Tensor, record: int):
    """(blocks, bytes between records) of a bounds pool, after a check of it."""
    shape, stride = bounds.shape, bounds.stride()
    if bounds.dtype != torch.uint8 or len(shape) != 2 or shape[1] < record or stride[1] != 1:
        raise ValueError(f"bounds: expected uint8 [num_blocks, {record}] records, got {bounds.dtype} {tuple(shape)}")
    return shape[0], stride[0]


def _key_cache(plan: SparsePlan, k_cache: torch.Tensor):
    """(blocks, slot or block stride, dtype code) of a cache, after a check of it."""
    dtype, shape, stride = k_cache.dtype, k_cache.shape, k_cache.stride()
    Hkv, D = plan.num_kv_heads, plan.head_dim
    if dtype == KV4:
        return _kv4_blocks(k_cache, k_cache, Hkv, D, plan.block_size), stride[0], _lib.DTYPE_MXFP4
    if len(shape) != 3 or shape[1] != Hkv or shape[2] != D or stride[1] != D or stride[2] != 1:
        raise ValueError(f"k_cache: expected [num_slots, {Hkv}, {D}] with contiguous rows")
    return shape[0] // plan.block_size, stride[0], _lib.dtype_code(dtype)


def _query_rows(plan: SparsePlan, t: torch.Tensor, name: str) -> int:
    """Row stride of q or out, after a check of its rows."""
    if t.dtype != plan.dtype:
        raise ValueError(f"{name} is {t.dtype}, the plan's model dtype {plan.dtype}")
    stride = _row_stride(t, t.shape, plan.num_q_heads, plan.head_dim, name)
    if t.numel() < plan.row_elements:
        raise ValueError(f"{name} has {t.numel() // (plan.num_q_heads * plan.head_dim)} rows, the plan addresses {plan.rows}")
    return stride


def _selection(plan: SparsePlan, t: torch.Tensor, name: str) -> None:
    shape = t.shape
    if t.dtype != torch.int32 or len(shape) != 3 or shape[1] != plan.num_kv_heads or shape[2] != plan.blocks \
            or not t.is_contiguous():
        raise ValueError(f"{name}: expected contiguous int32 [rows, {plan.num_kv_heads}, {plan.blocks}], got {t.dtype} "
                         f"{tuple(shape)}")
    if shape[0] < plan.rows:
        raise ValueError(f"{name} has {shape[0]} rows, the plan addresses {plan.rows}")


def write_key_bounds(plan: SparsePlan, k_cache: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor) -> None:
    """The key bounds of every block that holds a new token of the step, from all
    the block's cached keys: call it after the step's KV write.

    ``k_cache`` ``[num_slots, Hkv, D]`` (or a 4-bit one), ``bounds`` uint8
    ``[num_blocks, >= key_bounds_bytes]``, block_table int32 ``[B, W]``.
    """
    index = plan.index
    if index >= 0 and _current_device() != index:
        return _on_device(plan, write_key_bounds, plan, k_cache, bounds, block_table)
    bt_stride = _table(plan, block_table)
    pool, stride = _bounds(bounds, plan.record_bytes)
    nb, slot, code = _key_cache(plan, k_cache)
    if pool < nb:
        raise ValueError(f"bounds of {pool} blocks for a cache of {nb}")
    if index < 0 or k_cache.get_device() != index or bounds.get_device() != index or block_table.get_device() != index:
        _elsewhere(plan, k_cache=k_cache, bounds=bounds, block_table=block_table)
    _lib.check(plan._lib.gllm_key_bounds_write(
        plan._h, k_cache.data_ptr(), slot, nb, block_table.data_ptr(), bt_stride, bounds.data_ptr(), stride, code,
        _lib.raw_stream(index)))


def key_bounds_values(bounds: torch.Tensor, blocks: torch.Tensor, num_kv_heads: int, head_dim: int,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Key bounds as the values they stand for, for other scores or a look at
    them: float32 ``[N, Hkv, 2, D]`` (least, largest; infinities where a block is
    unbounded) for int64 ``blocks [N]`` (zeros for a block outside the pool)."""
    index = bounds.get_device()
    if index >= 0 and _current_device() != index:
        with torch.cuda.device(index):
            return key_bounds_values(bounds, blocks, num_kv_heads, head_dim, out)
    pool, stride = _bounds(bounds, key_bounds_bytes(num_kv_heads, head_dim))
    b = blocks
    if b.dtype != torch.int64 or b.dim() != 1 or not b.is_contiguous():
        if b.dtype.is_floating_point or b.dtype == torch.bool:
            raise ValueError("blocks must be integers")
        b = _index_rows(b)
    n = b.shape[0]
    if out is None:
        out = torch.empty((n, num_kv_heads, 2, head_dim), dtype=torch.float32, device=bounds.device)
    elif out.dtype != torch.float32 or out.shape != (n, num_kv_heads, 2, head_dim) or not out.is_contiguous():
        raise ValueError(f"out must be contiguous float32 {(n, num_kv_heads, 2, head_dim)}")
    if b.get_device() != index or out.get_device() != index:
        _same_device(index, blocks=b, out=out)
    if index < 0:
        raise ValueError("tensors on the CPU: the kernels need a GPU")
    if n:
        lib = _lib._lib or _lib.load()
        _lib.check(lib.gllm_key_bounds_values(bounds.data_ptr(), stride, pool, b.data_ptr(), n, num_kv_heads, head_dim,
                                              out.data_ptr(), _lib.raw_stream(index)))
    return out


def select_blocks(plan: SparsePlan, q: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The blocks for each query row and KV head: int32 ``[rows, Hkv, blocks]``,
    block-table columns in ascending order, then -1 (padded rows: not written).

    q ``[rows, Hq, D]`` or ``[B, T_q, Hq, D]``, rotated.  A block's score is the
    largest, over the group's heads, of sum_d max(q_d least_d, q_d largest_d) with q
    rounded to int8 steps of one power of two, so no key of the block scores
    higher (but for q's rounding); equal scores go to the lower block.
    """
    index = plan.index
    if index >= 0 and _current_device() != index:
        return _on_device(plan, select_blocks, plan, q, bounds, block_table, out)
    q_stride = _query_rows(plan, q, "q")
    bt_stride = _table(plan, block_table)
    pool, stride = _bounds(bounds, plan.record_bytes)
    if out is not None:
        _selection(plan, out, "out")
    if index < 0 or q.get_device() != index or bounds.get_device() != index or block_table.get_device() != index \
            or (out is not None and out.get_device() != index):
        _elsewhere(plan, q=q, bounds=bounds, block_table=block_table, out=out)
    if out is None:
        out = torch.empty((plan.rows, plan.num_kv_heads, plan.blocks), dtype=torch.int32, device=plan.device)
    _lib.check(plan._lib.gllm_select_blocks(
        plan._h, q.data_ptr(), q_stride, bounds.data_ptr(), stride, pool, block_table.data_ptr(), bt_stride,
        out.data_ptr(), plan.code, _lib.raw_stream(index)))
    return out


def sparse_attention(plan: SparsePlan, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     block_table: torch.Tensor, selected: torch.Tensor, out: torch.Tensor | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """Attention of each query row over the keys, at or before its position, of the
    blocks selected for it and the KV head.

    q and out as in :func:`gllm_amd.paged_attention` (q rotated), ``selected`` int32
    ``[rows, Hkv, blocks]`` from :func:`select_blocks` or any other choice: a list ends
    at the first entry that is negative, not above the entry before it, or behind
    the row's own block.  A row without blocks gives zeros.  A selected block's keys
    and values up to the position of the sequence's last row must be finite, those that
    rows before it do not see too.  Returns ``out``.
    """
    index = plan.index
    if index >= 0 and _current_device() != index:
        return _on_device(plan, sparse_attention, plan, q, k_cache, v_cache, block_table, selected, out, scale)
    q_stride = _query_rows(plan, q, "q")
    out_stride = plan.num_q_heads * plan.head_dim if out is None else _query_rows(plan, out, "out")
    bt_stride = _table(plan, block_table)
    _selection(plan, selected, "selected")
    nb, slot, code = _key_cache(plan, k_cache)
    if v_cache.shape != k_cache.shape or v_cache.stride() != k_cache.stride() or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must have the same shape, strides and dtype")
    if index < 0 or q.get_device() != index or k_cache.get_device() != index or v_cache.get_device() != index \
            or block_table.get_device() != index or selected.get_device() != index \
            or (out is not None and out.get_device() != index):
        _elsewhere(plan, q=q, out=out, k_cache=k_cache, v_cache=v_cache, block_table=block_table, selected=selected)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _lib.check(plan._lib.gllm_sparse_attention(
        plan._h, q.data_ptr(), q_stride, out.data_ptr(), out_stride, k_cache.data_ptr(), v_cache.data_ptr(), slot, nb,
        block_table.data_ptr(), bt_stride, selected.data_ptr(), plan.scale if scale is None else float(scale), plan.code,
        code, _lib.raw_stream(index)))
    return out
