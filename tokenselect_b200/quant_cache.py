"""A KV cache held in 4 bits: pool rows quantised as they are written, read back, and attended to by decode steps.

A pool row keeps one token's K and V of every KV head in ``9 * head_dim / 8`` bytes a head (144 at head_dim 128, where
bf16 takes 512): 4-bit floats (E2M1) with one 8-bit scale (E4M3) per sixteen elements; ``include/tokenselect_b200.h``
states the layout and the rounding.  Keys are kept un-rotated, and page size is 1, as in the bf16 pools: the same
``req_to_token`` tables, and the row lists that a selection leaves, index them.

``k_scale`` and ``v_scale`` are the pool's scales, powers of two, the same in every call on a pool: blocks whose largest
magnitude lies between ``0.006 * scale`` and ``2688 * scale`` are held (an element a 24th of its block's largest
rounds to zero; a smaller block becomes zeros, a larger one is clamped).  What is read back and written again keeps its
bytes where a block's largest magnitude was above ``0.02 * scale``.

The functions keep nothing between calls and enqueue on the current stream; they may be captured into CUDA graphs.
``status`` (optional, a CUDA int32 tensor) is set to a ``TS_ERR_*`` code when a kernel finds a row outside the pool or
a length that makes no sense; it is never cleared here.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import TsQuantAttendArgs, TsQuantRowsArgs, check
from .engine import _raw_stream

_ROWS_ARGS_SIZE, _ATTEND_ARGS_SIZE = C.sizeof(TsQuantRowsArgs), C.sizeof(TsQuantAttendArgs)
_DTYPES = {torch.bfloat16: _lib.TS_DTYPE_BF16, torch.float32: _lib.TS_DTYPE_F32}
_workspace_bytes = {}            # (device, batch, heads, head_dim) -> bytes


def kv4_row_bytes(head_dim: int) -> int:
    """Bytes of one token's K and V of one KV head."""
    return head_dim * 9 // 8


def kv4_pool(rows: int, num_kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """A pool of ``rows`` tokens of one layer, all zeros: ``[rows, num_kv_heads, 9 * head_dim / 8]`` bytes."""
    return torch.zeros((rows, num_kv_heads, kv4_row_bytes(head_dim)), dtype=torch.uint8, device=device)


_HEAD_DIMS = {kv4_row_bytes(d): d for d in (64, 128)}
_lib_ = _lib.load                # the library, loaded at the first call


def _check_pool(pool: torch.Tensor) -> int:
    """The pool's head_dim."""
    shape = pool.shape
    if len(shape) != 3 or pool.dtype != torch.uint8 or not pool.is_cuda or not pool.is_contiguous() or shape[0] == 0:
        raise ValueError("pool must be a contiguous CUDA uint8 tensor [rows, num_kv_heads, 9*head_dim/8]")
    d = _HEAD_DIMS.get(shape[2])
    if d is None:
        raise ValueError("pool rows are 72 bytes a head (head_dim 64) or 144 (head_dim 128)")
    return d


def _check_ints(device: int, named) -> None:
    i32 = torch.int32
    for name, t in named:
        if t is not None and (t.dtype != i32 or t.get_device() != device or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous int32 tensor on the pool's device")


def _row_stride(name: str, t: torch.Tensor, n: int, heads: int, d: int, dtype: torch.dtype, dev: int) -> int:
    """Elements between the rows of ``[n, heads, d]``; raises unless the heads of a row are packed."""
    if t.dtype != dtype or dtype not in _DTYPES or t.get_device() != dev or t.shape != (n, heads, d):
        raise ValueError(f"{name} must be [rows, num_kv_heads, head_dim] in bf16 or fp32 on the pool's device, k and v alike")
    s0, s1, s2 = t.stride()
    if n > 1 and s2 == 1 and s1 == d and s0 >= heads * d:
        return s0
    if n > 0 and (s2 != 1 or (heads > 1 and s1 != d) or (n > 1 and s0 < heads * d)):
        raise ValueError(f"{name}: the heads of a row must follow each other without gaps, and rows not overlap")
    return s0 if n > 1 else heads * d


def _row_args(pool, d, k, v, rows, k_scale, v_scale, status) -> TsQuantRowsArgs:
    # A decode step's rows cost the device less than a generous host path costs Python: one look at each property.
    dev, (pool_rows, heads, _) = pool.get_device(), pool.shape
    n, dtype = rows.numel(), k.dtype
    ks, vs = _row_stride("k", k, n, heads, d, dtype, dev), _row_stride("v", v, n, heads, d, dtype, dev)
    _check_ints(dev, (("rows", rows), ("status", status)))
    return TsQuantRowsArgs(_ROWS_ARGS_SIZE, dev, _DTYPES[dtype], heads, d, n, k.data_ptr(), v.data_ptr(), ks, vs,
                           rows.data_ptr(), pool.data_ptr(), pool_rows, k_scale, v_scale,
                           None if status is None else status.data_ptr(), _raw_stream(dev))


def kv4_write(pool: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor, k_scale: float = 1.0,
              v_scale: float = 1.0, status: Optional[torch.Tensor] = None) -> None:
    """Quantise ``k, v [n, num_kv_heads, head_dim]`` (bf16 or fp32, rows may be strided) into the pool rows
    ``rows [n]`` (``out_cache_loc`` of the serving stack).  A row outside the pool is skipped and reported; a row that
    is listed twice is left with a mixture of the two."""
    a = _row_args(pool, _check_pool(pool), k, v, rows, k_scale, v_scale, status)
    check(_lib_().ts_quant_write(C.byref(a)), "ts_quant_write")


def kv4_read(pool: torch.Tensor, rows: torch.Tensor, dtype: Optional[torch.dtype] = None, k_scale: float = 1.0,
             v_scale: float = 1.0, k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None,
             status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(k, v) [n, num_kv_heads, head_dim]`` of the pool rows ``rows [n]``: the values their codes stand for, exact in
    bf16 and in fp32 (``dtype``; bf16 by default).  ``k`` and ``v`` may be given (rows of a bf16 pool's slice, say), apart
    from each other and from the pool; the results then have their type.  A row outside the pool gives zeros and is
    reported."""
    d = _check_pool(pool)
    for t in (k, v):
        if t is not None and dtype is not None and t.dtype != dtype:
            raise ValueError("dtype must be that of the given k and v")
    shape = (rows.numel(), pool.shape[1], d)
    if k is None:
        k = pool.new_empty(shape, dtype=dtype or torch.bfloat16 if v is None else v.dtype)
    if v is None:
        v = torch.empty_like(k, memory_format=torch.contiguous_format)
    a = _row_args(pool, d, k, v, rows, k_scale, v_scale, status)
    check(_lib_().ts_quant_read(C.byref(a)), "ts_quant_read")
    return k, v


def kv4_attend_workspace(batch: int, num_q_heads: int, head_dim: int, device: int = 0) -> int:
    """Bytes of workspace one :func:`kv4_attend` call needs."""
    key = (device, batch, num_q_heads, head_dim)
    if key not in _workspace_bytes:
        n = C.c_size_t()
        check(_lib_().ts_quant_attend_workspace(device, batch, num_q_heads, head_dim, C.byref(n)), "ts_quant_attend_workspace")
        _workspace_bytes[key] = n.value
    return _workspace_bytes[key]


def kv4_attend(q: torch.Tensor, pool: torch.Tensor, req_to_token: torch.Tensor, req_pool_indices: torch.Tensor,
               seq_lens: torch.Tensor, sm_scale: float, rope_base: float, rope_scale: float = 1.0, logit_cap: float = 0.0,
               k_scale: float = 1.0, v_scale: float = 1.0, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention of a ragged batch over a 4-bit pool: request ``b`` attends to the pool rows
    ``req_to_token[req_pool_indices[b], :seq_lens[b]]``, entry ``j`` at position ``j``, its query at position
    ``seq_lens[b] - 1``; ``q [batch, heads * head_dim]`` and the pool's keys are un-rotated.  Query head ``h`` reads KV
    head ``h // group``, at most eight query heads share one.  With a selection's row lists for ``req_to_token``,
    ``arange(batch)`` for ``req_pool_indices`` and their counts for ``seq_lens`` it is the sparse attention of
    ``decode_layer``.  A request of length 0 (a padded slot of a captured batch) gets zeros.

    ``workspace``: uint8, at least :func:`kv4_attend_workspace` bytes, for callers that must not allocate; calls that
    may run at the same time need one each.  By default every call takes its own from PyTorch's allocator.
    ``out`` may be ``q``."""
    d, dev, (pool_rows, hkv, _) = _check_pool(pool), pool.get_device(), pool.shape
    i32, dtype, batch, total = torch.int32, q.dtype, q.shape[0], q.numel()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    hq = total // (batch * d) if batch > 0 else hkv
    if not (q.get_device() == out.get_device() == dev and dtype == out.dtype and dtype in _DTYPES
            and q.is_contiguous() and out.is_contiguous() and total == out.numel() == batch * hq * d and hq % hkv == 0):
        raise ValueError("q/out must be contiguous [batch, num_q_heads*head_dim] in bf16 or fp32 on the pool's device")
    table = req_to_token.stride()
    if len(table) != 2 or table[1] != 1 or req_to_token.dtype != i32 or req_to_token.get_device() != dev:
        raise ValueError("req_to_token must be int32 [max_reqs, max_ctx] with unit inner stride on the pool's device")
    if req_pool_indices.numel() != batch or seq_lens.numel() != batch:
        raise ValueError("req_pool_indices and seq_lens must have one entry per request")
    _check_ints(dev, (("req_pool_indices", req_pool_indices), ("seq_lens", seq_lens), ("status", status)))
    if batch == 0:
        return out
    nbytes = _workspace_bytes.get((dev, batch, hq, d)) or kv4_attend_workspace(batch, hq, d, dev)
    if workspace is None:
        workspace = pool.new_empty(nbytes)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous on the pool's device")
    max_reqs, max_ctx = req_to_token.shape
    a = TsQuantAttendArgs(_ATTEND_ARGS_SIZE, dev, _DTYPES[dtype], batch, hq, hkv, d, max_reqs, q.data_ptr(), pool.data_ptr(),
                          pool_rows, req_to_token.data_ptr(), table[0], max_ctx, req_pool_indices.data_ptr(),
                          seq_lens.data_ptr(), out.data_ptr(), sm_scale, logit_cap, rope_base, rope_scale, k_scale, v_scale,
                          workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                          None if status is None else status.data_ptr(), _raw_stream(dev))
    check(_lib_().ts_quant_attend(C.byref(a)), "ts_quant_attend")
    return out
