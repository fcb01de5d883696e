"""The 4-bit vocabulary projection in front of the sampler.

``int4_matvec`` multiplies the few rows of a decode step with a matrix held in 4 bits
(``Int4Weight``), ``sample_hidden`` goes from the last hidden states straight to token ids.
LocalStrm's counterpart is the eager W4A16 linear of ``src/kernels/quantization.py``.
CUDA tensors only; the native library does the work.
"""
from __future__ import annotations

import contextlib
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .sampling import _DT, _require_cuda, sample_batch

__all__ = ["Int4Weight", "int4_matvec", "sample_hidden"]

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


_HERE = contextlib.nullcontext()


def _on(dev: torch.device):
    """The device that the library launches on, where it is not the current one."""
    return _HERE if dev.index == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _stream(dev: torch.device) -> int:
    """torch's current stream on ``dev`` as a cudaStream_t."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


@dataclass
class Int4Weight:
    """A matrix ``[N, K]`` in 4 bits: ``W[n, k] = (code[n, k] - 8) * scales[n, k // group]``.

    ``packed``: uint8 ``[N, K / 2]``, column ``2 i`` in the low four bits of byte ``i`` and column
    ``2 i + 1`` in the high ones.  ``scales``: float16 or bfloat16 ``[N, K / group]``; groups of 32,
    64 or a multiple of 128 columns that divides K.
    """
    packed: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.packed.shape[0], 2 * self.packed.shape[1]

    @property
    def group(self) -> int:
        return 2 * self.packed.shape[1] // max(1, self.scales.shape[1])

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 128, scale_dtype: torch.dtype = torch.float16) -> "Int4Weight":
        """The nearest codes -7 .. 7 for the scale ``max |w| / 7`` of each group (done once, where
        the weights lie)."""
        if weight.dim() != 2 or weight.shape[1] % 32 or group < 32 or weight.shape[1] % group:
            raise ValueError(f"weight: expected [N, K] with K a multiple of 32 and of the group {group}")
        n, k = weight.shape
        w = weight.float().view(n, k // group, group)
        scales = (w.abs().amax(-1) / 7.0).to(scale_dtype)
        step = scales.float().clamp(min=torch.finfo(torch.float32).tiny)[..., None]
        codes = (torch.round(w / step).clamp(-7, 7) + 8).to(torch.uint8).view(n, k)
        return cls((codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scales.contiguous())

    def dequantize(self) -> torch.Tensor:
        """The matrix in float32."""
        codes = torch.stack([self.packed & 15, self.packed >> 4], -1).view(self.shape[0], -1)
        return ((codes.float() - 8.0).view(*self.scales.shape, -1) * self.scales.float()[..., None]).view(codes.shape)


def int4_matvec(x: torch.Tensor, weight: Int4Weight, out_dtype: Optional[torch.dtype] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ W.T`` for ``x [rows, K]`` or ``[K]`` (f32, bf16 or f16), sums in f32, one rounding to
    ``out_dtype`` (default: x's).  One pass over the matrix serves eight rows."""
    _require_cuda(x)
    packed, scales = weight.packed, weight.scales
    if x.dim() not in (1, 2):
        raise ValueError("x must be [K] or [rows, K]")
    dev = x.device
    if packed.device != dev or scales.device != dev:
        raise ValueError(f"weight on {packed.device} / {scales.device}, x on {dev}")
    if packed.dtype != torch.uint8 or packed.dim() != 2 or not packed.is_contiguous():
        raise ValueError("packed: expected a contiguous uint8 tensor [N, K / 2]")
    if scales.dtype not in (torch.float16, torch.bfloat16) or scales.dim() != 2 or not scales.is_contiguous() \
            or scales.shape[0] != packed.shape[0]:
        raise ValueError("scales: expected a contiguous float16 or bfloat16 tensor [N, K / group]")
    n, k, groups = packed.shape[0], 2 * packed.shape[1], scales.shape[1]
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {k}")
    if n < 1 or groups < 1 or k % groups:
        raise ValueError(f"{groups} groups do not divide {k} columns")
    out_dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if x.dtype not in _DT or out_dtype not in _DT:
        raise TypeError(f"unsupported dtypes {x.dtype} -> {out_dtype}")
    x2 = x if x.dim() == 2 else x.unsqueeze(0)
    rows = x2.shape[0]
    if x2.stride(1) != 1 or (rows > 1 and x2.stride(0) < k):
        x2 = x2.contiguous()
    want = (n,) if x.dim() == 1 else (rows, n)
    if out is None:
        out = torch.empty(want, dtype=out_dtype, device=dev)
    elif tuple(out.shape) != want or out.dtype != out_dtype or out.device != dev or out.stride(-1) != 1 \
            or (out.dim() == 2 and rows > 1 and out.stride(0) < n):
        raise ValueError(f"out: expected {out_dtype} {list(want)} on {dev} with rows of stride 1")
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_int4_matvec", lib.lss_int4_matvec(
            x2.data_ptr(), _CODES[x.dtype], rows, k, max(x2.stride(0), k), packed.data_ptr(), scales.data_ptr(),
            _CODES[scales.dtype], n, k // groups, out.data_ptr(), _CODES[out_dtype],
            max(out.stride(0), n) if out.dim() == 2 else n, _stream(dev)))
    return out


def sample_hidden(hidden: torch.Tensor, head: Int4Weight, params, past_token_ids=None,
                  uniforms: Optional[torch.Tensor] = None, return_kept: bool = False):
    """Tokens for the hidden states ``[B, K]`` of a decode step: the 4-bit vocabulary projection to
    f32 logits, then ``sample_batch`` (whose arguments these are)."""
    _require_cuda(hidden)
    if hidden.dim() != 2:
        raise ValueError("hidden must be [B, K]")
    logits = int4_matvec(hidden, head, out_dtype=torch.float32)
    return sample_batch(logits, params, past_token_ids, uniforms, return_kept)
