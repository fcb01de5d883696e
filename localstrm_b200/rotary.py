"""Norms of queries and keys for each head and the position rotation, between the projection and the cache.

LocalStrm's counterpart is the eager torch code of its models (``q_norm``, ``k_norm`` and the rotary
embedding applied one after the other).  CUDA tensors only; the native library does the work.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .head import _CODES, _on, _stream
from .sampling import _require_cuda

__all__ = ["norm_rotate"]


_I32, _F32, _DENSE = torch.int32, torch.float32, torch.contiguous_format


def _out(name: str, out: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    if out.shape != x.shape or out.dtype is not x.dtype or out.get_device() != x.get_device() or out.stride(2) != 1:
        raise ValueError(f"{name}: expected {x.dtype} {list(x.shape)} on {x.device} with rows of stride 1")
    return out


def norm_rotate(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor,
                q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q, k)`` with each head normed and turned to its position.

    ``q [T, q_heads, dim]``, ``k [T, heads, dim]`` (f32, bf16 or f16; dim even, at most 512; any token and head
    strides): ``x / sqrt(mean(x ** 2) + eps) * weight`` for each head where there is a weight (``[dim]``, f32, bf16 or
    f16, both of one type), then the first ``2 * len(freqs)`` values are turned in pairs by ``positions[t] * freqs[i]``
    (``positions`` int32 ``[T]``, ``StepPlan.positions`` or ``TreePlan.positions``; ``freqs`` float32): value i with value
    ``i + len(freqs)``, or value 2 i with 2 i + 1 where ``interleaved``.  Computed in f32 (the angle is reduced in f64: far positions keep
    their fraction), rounded once; squares of the values have to lie within f32.  ``q_out`` / ``k_out`` may be ``q`` and ``k`` themselves; results that overlap the inputs
    in another way, or each other, are refused."""
    _require_cuda(q)
    dev, dtype, shape, k_shape = q.get_device(), q.dtype, q.shape, k.shape
    if len(shape) != 3 or len(k_shape) != 3 or k_shape[0] != shape[0] or k_shape[2] != shape[2] or k.get_device() != dev:
        raise ValueError(f"q, k: expected [T, heads, dim] of the same T and dim on cuda:{dev}")
    if dtype not in _CODES or k.dtype is not dtype:
        raise TypeError(f"unsupported dtypes {dtype}, {k.dtype}")
    T, heads, dim = shape
    if positions.dtype is not _I32 or positions.dim() != 1 or positions.numel() != T or positions.get_device() != dev \
            or not positions.is_contiguous():
        raise ValueError(f"positions: expected a contiguous int32 tensor of {T} entries on cuda:{dev}")
    half = freqs.numel()
    if freqs.dtype is not _F32 or freqs.dim() != 1 or freqs.get_device() != dev or not freqs.is_contiguous() or 2 * half > dim:
        raise ValueError(f"freqs: expected a contiguous float32 tensor of at most {dim // 2} entries on cuda:{dev}")
    code = 0
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if w.dim() != 1 or w.numel() != dim or w.get_device() != dev or not w.is_contiguous() or w.dtype not in _CODES:
            raise ValueError(f"{name}: expected a contiguous float32, bfloat16 or float16 tensor of {dim} entries on cuda:{dev}")
        code = _CODES[w.dtype]
    if q_weight is not None and k_weight is not None and q_weight.dtype is not k_weight.dtype:
        raise TypeError(f"weights of two types: {q_weight.dtype}, {k_weight.dtype}")
    qs, ks = q.stride(), k.stride()
    if qs[2] != 1:
        q = q.contiguous()
        qs = q.stride()
    if ks[2] != 1:
        k = k.contiguous()
        ks = k.stride()
    q_out = torch.empty_like(q, memory_format=_DENSE) if q_out is None else _out("q_out", q_out, q)
    k_out = torch.empty_like(k, memory_format=_DENSE) if k_out is None else _out("k_out", k_out, k)
    qo, ko = q_out.stride(), k_out.stride()
    lib = _lib.load()
    with _on(dev):
        status = lib.lss_norm_rotate(
            q.data_ptr(), qs[0], qs[1], q_out.data_ptr(), qo[0], qo[1], heads, k.data_ptr(), ks[0], ks[1], k_out.data_ptr(), ko[0],
            ko[1], k_shape[1], _CODES[dtype], T, dim, positions.data_ptr(), freqs.data_ptr(), 2 * half, interleaved,
            None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), code, eps, _stream(dev))
    if status:
        _lib.check("lss_norm_rotate", status)
    return q_out, k_out
