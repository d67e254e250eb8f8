"""A KV cache held in 4 bits: pool rows quantised as they are written, read back, and attended to by decode steps.

A pool row keeps one token's K and V of every KV head in ``9 * head_dim / 8`` bytes a head (144 at head_dim 128, where
bf16 takes 512): 4-bit floats (E2M1) with one 8-bit scale (E4M3) per sixteen elements; ``include/tokenselect_b200.h``
states the layout and the rounding.  Keys are kept un-rotated, and page size is 1, as in the bf16 pools: the same
``req_to_token`` tables, and the row lists that a selection leaves, index them.

``k_scale`` and ``v_scale`` are the pool's scales, powers of two, the same in every call on a pool: values between
``2**-10 * scale`` and ``2688 * scale`` are held (those of a block together: an element a 24th of its block's
largest rounds to zero).

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


def _check_pool(pool: torch.Tensor) -> int:
    """The pool's head_dim."""
    if pool.dim() != 3 or pool.dtype != torch.uint8 or not pool.is_cuda or not pool.is_contiguous() or pool.shape[0] == 0:
        raise ValueError("pool must be a contiguous CUDA uint8 tensor [rows, num_kv_heads, 9*head_dim/8]")
    d = pool.shape[2] * 8 // 9
    if d not in (64, 128) or pool.shape[2] * 8 != d * 9:
        raise ValueError("pool rows are 72 bytes a head (head_dim 64) or 144 (head_dim 128)")
    return d


def _check_ints(device: int, named) -> None:
    for name, t in named:
        if t is not None and (t.dtype != torch.int32 or t.get_device() != device or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous int32 tensor on the pool's device")


def _row_args(pool, k, v, rows, k_scale, v_scale, status) -> TsQuantRowsArgs:
    d, dev, (pool_rows, heads, _) = _check_pool(pool), pool.get_device(), pool.shape
    n = rows.numel()
    for name, t in (("k", k), ("v", v)):
        if t.get_device() != dev or t.dtype != k.dtype or t.dtype not in _DTYPES or t.shape != (n, heads, d):
            raise ValueError(f"{name} must be [rows, num_kv_heads, head_dim] in bf16 or fp32 on the pool's device, k and v alike")
        if n > 0 and (t.stride(2) != 1 or (heads > 1 and t.stride(1) != d) or (n > 1 and t.stride(0) < heads * d)):
            raise ValueError(f"{name}: the heads of a row must follow each other without gaps, and rows not overlap")
    _check_ints(dev, (("rows", rows), ("status", status)))
    ks, vs = (k.stride(0), v.stride(0)) if n > 1 else (heads * d, heads * d)
    return TsQuantRowsArgs(_ROWS_ARGS_SIZE, dev, _DTYPES[k.dtype], heads, d, n, k.data_ptr(), v.data_ptr(), ks, vs,
                           rows.data_ptr(), pool.data_ptr(), pool_rows, k_scale, v_scale,
                           None if status is None else status.data_ptr(), _raw_stream(dev))


def kv4_write(pool: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor, k_scale: float = 1.0,
              v_scale: float = 1.0, status: Optional[torch.Tensor] = None) -> None:
    """Quantise ``k, v [n, num_kv_heads, head_dim]`` (bf16 or fp32, rows may be strided) into the pool rows
    ``rows [n]`` (``out_cache_loc`` of the serving stack).  A row outside the pool is skipped and reported; a row that
    is listed twice is left with a mixture of the two."""
    a = _row_args(pool, k, v, rows, k_scale, v_scale, status)
    check(_lib.load().ts_quant_write(C.byref(a)), "ts_quant_write")


def kv4_read(pool: torch.Tensor, rows: torch.Tensor, dtype: torch.dtype = torch.bfloat16, k_scale: float = 1.0,
             v_scale: float = 1.0, k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None,
             status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(k, v) [n, num_kv_heads, head_dim]`` of the pool rows ``rows [n]``: the values their codes stand for, exact in
    bf16 and in fp32.  ``k`` and ``v`` may be given (rows of a bf16 pool's slice, say).  A row outside the pool gives
    zeros and is reported."""
    d = _check_pool(pool)
    shape = (rows.numel(), pool.shape[1], d)
    if k is None:
        k = torch.empty(shape, dtype=dtype, device=pool.device)
    if v is None:
        v = torch.empty(shape, dtype=dtype, device=pool.device)
    a = _row_args(pool, k, v, rows, k_scale, v_scale, status)
    check(_lib.load().ts_quant_read(C.byref(a)), "ts_quant_read")
    return k, v


def kv4_attend_workspace(batch: int, num_q_heads: int, head_dim: int, device: int = 0) -> int:
    """Bytes of workspace one :func:`kv4_attend` call needs."""
    key = (device, batch, num_q_heads, head_dim)
    if key not in _workspace_bytes:
        n = C.c_size_t()
        check(_lib.load().ts_quant_attend_workspace(device, batch, num_q_heads, head_dim, C.byref(n)), "ts_quant_attend_workspace")
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
    may run at the same time need one each.  By default every call takes its own from PyTorch's allocator."""
    d, dev, (pool_rows, hkv, _) = _check_pool(pool), pool.get_device(), pool.shape
    batch = q.shape[0]
    hq = q.numel() // (batch * d) if batch > 0 else hkv
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if not (q.get_device() == out.get_device() == dev and q.dtype == out.dtype and q.dtype in _DTYPES
            and q.is_contiguous() and out.is_contiguous() and q.numel() == out.numel() == batch * hq * d and hq % hkv == 0):
        raise ValueError("q/out must be contiguous [batch, num_q_heads*head_dim] in bf16 or fp32 on the pool's device")
    if req_to_token.dim() != 2 or req_to_token.stride(1) != 1 or req_to_token.dtype != torch.int32 or req_to_token.get_device() != dev:
        raise ValueError("req_to_token must be int32 [max_reqs, max_ctx] with unit inner stride on the pool's device")
    if req_pool_indices.numel() != batch or seq_lens.numel() != batch:
        raise ValueError("req_pool_indices and seq_lens must have one entry per request")
    _check_ints(dev, (("req_pool_indices", req_pool_indices), ("seq_lens", seq_lens), ("status", status)))
    if batch == 0:
        return out
    nbytes = kv4_attend_workspace(batch, hq, d, dev)
    if workspace is None:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=pool.device)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous on the pool's device")
    a = TsQuantAttendArgs(_ATTEND_ARGS_SIZE, dev, _DTYPES[q.dtype], batch, hq, hkv, d, req_to_token.shape[0], q.data_ptr(),
                          pool.data_ptr(), pool_rows, req_to_token.data_ptr(), req_to_token.stride(0), req_to_token.shape[1],
                          req_pool_indices.data_ptr(), seq_lens.data_ptr(), out.data_ptr(), sm_scale, logit_cap, rope_base,
                          rope_scale, k_scale, v_scale, workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                          None if status is None else status.data_ptr(), _raw_stream(dev))
    check(_lib.load().ts_quant_attend(C.byref(a)), "ts_quant_attend")
    return out
