"""Whole prompts: head norms with the position rotation, and causal attention of packed sequences.

``norm_rotate`` turns what a layer's projections leave into the rotated queries and keys that ``prompt_attend`` takes, and
the un-rotated keys that a pool keeps.  Both keep nothing between calls and enqueue on the current stream; they may be
captured into CUDA graphs.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import TsNormRotateArgs, TsPromptArgs, check
from .engine import _raw_stream

_NORM_ARGS_SIZE, _PROMPT_ARGS_SIZE = C.sizeof(TsNormRotateArgs), C.sizeof(TsPromptArgs)
_lib_ = _lib.load                # the library, loaded at the first call
_DTYPES = {torch.bfloat16: _lib.TS_DTYPE_BF16, torch.float32: _lib.TS_DTYPE_F32}


def _token_stride(name: str, t: torch.Tensor, n: int, d: int, dtype: torch.dtype, device: int) -> int:
    """Elements between the tokens of ``[n, heads, d]``; raises unless the heads of a token are packed."""
    shape = t.shape
    if len(shape) != 3 or t.get_device() != device or device < 0 or t.dtype != dtype or dtype not in _DTYPES or shape[0] != n \
            or shape[2] != d:
        raise ValueError(f"{name} must be a CUDA tensor [tokens, heads, head_dim] in bf16 or fp32, all of one type and device")
    s0, s1, s2 = t.stride()
    row = shape[1] * d
    if n > 1 and s2 == 1 and s1 == d and s0 >= row:
        return s0
    if n > 0 and (s2 != 1 or (shape[1] > 1 and s1 != d) or (n > 1 and s0 < row)):
        raise ValueError(f"{name}: the heads of a token must follow each other without gaps, and tokens not overlap")
    return s0 if n > 1 else row


def _check_out(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if t.shape != like.shape or t.dtype != like.dtype or t.get_device() != like.get_device() or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, of its input's shape, type and device")
    if t.data_ptr() == like.data_ptr() and not like.is_contiguous():
        raise ValueError(f"{name} may be its input only where that is contiguous")


def norm_rotate(q: torch.Tensor, k: torch.Tensor, positions: Optional[torch.Tensor], rope_base: float = 1e6,
                rope_scale: float = 1.0, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                eps: float = 1e-6, with_plain_k: bool = False, q_out: Optional[torch.Tensor] = None,
                k_out: Optional[torch.Tensor] = None, k_plain: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, ...]:
    """RMS norm of every head of ``q [tokens, heads, head_dim]`` and ``k [tokens, kv_heads, head_dim]`` with the weights
    ``[head_dim]`` (None: no norm) and rotation of the pairs ``(i, i + head_dim/2)`` by ``position * rope_base **
    (-2 i / head_dim) / rope_scale`` (``positions`` int32 ``[tokens]``; None: no rotation), in one pass, in fp32,
    rounded once.  Returns ``(q, k)``, and behind them the normed keys before the rotation, for the cache, when
    ``with_plain_k`` or ``k_plain`` asks for them.  Inputs may be slices of a fused projection's output; outputs are
    contiguous, and may be the input that they are made of where that is; otherwise they share no memory with the call's
    other tensors."""
    # One token costs the device less than a generous host path costs Python: one look at each property.
    dev, dtype, shape = q.get_device(), q.dtype, q.shape
    if len(shape) != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    n, hq, d = shape
    qs, ks = _token_stride("q", q, n, d, dtype, dev), _token_stride("k", k, n, d, dtype, dev)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.dtype != dtype or w.get_device() != dev or w.numel() != d or not w.is_contiguous()):
            raise ValueError(f"{name} must be [head_dim] of q's type on q's device")
    if positions is not None and (positions.dtype != torch.int32 or positions.get_device() != dev or positions.numel() != n
                                  or not positions.is_contiguous()):
        raise ValueError("positions must be a contiguous int32 tensor [tokens] on q's device")
    packed = torch.contiguous_format
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=packed)
    else:
        _check_out("q_out", q_out, q)
    if k_out is None:
        k_out = torch.empty_like(k, memory_format=packed)
    else:
        _check_out("k_out", k_out, k)
    if k_plain is None:
        k_plain = torch.empty_like(k, memory_format=packed) if with_plain_k else None
    else:
        _check_out("k_plain", k_plain, k)
        if k_plain.data_ptr() == k_out.data_ptr() and n > 0:
            raise ValueError("k_plain and k_out hold different results")
    a = TsNormRotateArgs(_NORM_ARGS_SIZE, dev, _DTYPES[dtype], n, hq, k.shape[1], d, eps, q.data_ptr(), k.data_ptr(), qs, ks,
                         None if positions is None else positions.data_ptr(), None if q_weight is None else q_weight.data_ptr(),
                         None if k_weight is None else k_weight.data_ptr(), rope_base, rope_scale, q_out.data_ptr(),
                         k_out.data_ptr(), None if k_plain is None else k_plain.data_ptr(), _raw_stream(dev))
    check(_lib_().ts_norm_rotate(C.byref(a)), "ts_norm_rotate")
    return (q_out, k_out) if k_plain is None else (q_out, k_out, k_plain)


def prompt_attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, sm_scale: float,
                  logit_cap: float = 0.0, out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed prompts: ``q [tokens, heads, head_dim]``, ``k, v [tokens, kv_heads, head_dim]``, q and
    k rotated; sequence ``b`` is the tokens ``cu_seqlens[b] .. cu_seqlens[b+1] - 1`` (int32 ``[sequences + 1]`` on the
    device, lengths of zero allowed).  Query head ``h`` reads KV head ``h // group``.  Returns ``[tokens, heads,
    head_dim]`` (``out`` shares no memory with the inputs); rows behind the last sequence are left as they were in ``out``.
    The tensors start on 16 bytes and their tokens lie a multiple of 16 bytes apart (slices of a fused projection do).
    ``status`` (optional, int32) is set when a bound of ``cu_seqlens`` makes no sense; the sequence then ends where it
    still does, and the next one starts behind all before it."""
    dev, dtype, shape = q.get_device(), q.dtype, q.shape
    if len(shape) != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    n, hq, d = shape
    qs, ks, vs = (_token_stride(name, t, n, d, dtype, dev) for name, t in (("q", q), ("k", k), ("v", v)))
    hkv = k.shape[1]
    if v.shape[1] != hkv or hkv == 0 or hq % hkv != 0:
        raise ValueError("k and v must have the same heads, a divisor of q's")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.get_device() != dev or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 \
            or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous int32 tensor [sequences + 1] on q's device")
    if status is not None and (status.dtype != torch.int32 or status.get_device() != dev):
        raise ValueError("status must be an int32 tensor on q's device")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_out("out", out, q)
        if n > 0 and out.data_ptr() in (q.data_ptr(), k.data_ptr(), v.data_ptr()):
            raise ValueError("out must not be one of the inputs")
    a = TsPromptArgs(_PROMPT_ARGS_SIZE, dev, _DTYPES[dtype], n, cu_seqlens.numel() - 1, hq, hkv, d, sm_scale, logit_cap,
                     q.data_ptr(), k.data_ptr(), v.data_ptr(), qs, ks, vs, cu_seqlens.data_ptr(), out.data_ptr(),
                     None if status is None else status.data_ptr(), _raw_stream(dev))
    check(_lib_().ts_prompt_attend(C.byref(a)), "ts_prompt_attend")
    return out
