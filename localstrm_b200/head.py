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
from .sampling import _require_cuda, sample_batch

__all__ = ["Int4Weight", "int4_matvec", "sample_hidden"]

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


_HERE = contextlib.nullcontext()


def _on(device: int):
    """The device that the library launches on, where it is not the current one."""
    return _HERE if device == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _stream(device: int) -> int:
    """torch's current stream on a device as a cudaStream_t."""
    return torch._C._cuda_getCurrentRawStream(device)


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
        if weight.dim() != 2 or (group not in (32, 64) and (group < 128 or group % 128)) or weight.shape[1] % group:
            raise ValueError(f"weight: expected [N, K], K a multiple of the group {group}: 32, 64 or a multiple of 128")
        n, k = weight.shape
        w = weight.float().view(n, k // group, group)
        scales = (w.abs().amax(-1) / 7.0).to(scale_dtype)
        if not bool(scales.isfinite().all()):  # an infinite scale times the code 0 of a small weight is NaN
            raise ValueError(f"weight: not finite, or a group's largest magnitude / 7 is beyond {scale_dtype}")
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
    ``out_dtype`` (default: x's).  One pass over the matrix serves 64 rows.  ``out`` shares no memory with x.
    A group is summed before its scale is applied: these sums, up to 8 times those of ``|x|``, have to lie within f32."""
    _require_cuda(x)
    packed, scales = weight.packed, weight.scales
    shape, dev = x.shape, x.get_device()
    if len(shape) not in (1, 2):
        raise ValueError("x must be [K] or [rows, K]")
    if packed.get_device() != dev or scales.get_device() != dev:
        raise ValueError(f"weight on {packed.device} / {scales.device}, x on {x.device}")
    if packed.dtype is not torch.uint8 or packed.dim() != 2 or not packed.is_contiguous():
        raise ValueError("packed: expected a contiguous uint8 tensor [N, K / 2]")
    n, half = packed.shape
    k, scale_code = 2 * half, _CODES.get(scales.dtype, 0)
    if scale_code == 0 or scales.dim() != 2 or not scales.is_contiguous() or scales.shape[0] != n:
        raise ValueError("scales: expected a contiguous float16 or bfloat16 tensor [N, K / group]")
    groups = scales.shape[1]
    if shape[-1] != k:
        raise ValueError(f"x has {shape[-1]} columns, the weight {k}")
    if n < 1 or groups < 1 or k % groups:
        raise ValueError(f"{groups} groups do not divide {k} columns")
    if out_dtype is None:
        out_dtype = x.dtype if out is None else out.dtype
    if x.dtype not in _CODES or out_dtype not in _CODES:
        raise TypeError(f"unsupported dtypes {x.dtype} -> {out_dtype}")
    if len(shape) == 1:
        rows, x_stride, want = 1, k, (n,)
        if x.stride(0) != 1:
            x = x.contiguous()
    else:
        rows, want = shape[0], (shape[0], n)
        x_stride, inner = x.stride()
        if inner != 1 or (rows > 1 and x_stride < k):
            x = x.contiguous()
            x_stride = k
        x_stride = max(x_stride, k)  # one row: its stride says nothing
    y_stride = n
    if out is None:
        out = torch.empty(want, dtype=out_dtype, device=x.device)
    else:
        if tuple(out.shape) != want or out.dtype is not out_dtype or out.get_device() != dev or out.stride(-1) != 1 \
                or (rows > 1 and out.stride(0) < n):
            raise ValueError(f"out: expected {out_dtype} {list(want)} on {x.device} with rows of stride 1")
        if len(want) == 2:
            y_stride = max(out.stride(0), n)
    lib = _lib.load()
    with _on(dev):
        ws, size = None, 0
        # Few and short rows fit the shared memory of any SM.
        if rows > 8 or k > 16384 or rows * k * (6 if x.dtype is torch.float32 else 2) > 96000:
            size = lib.lss_int4_workspace_one_pass_bytes(rows, k, _CODES[x.dtype], n)
            # From torch's allocator for every call: other streams and captured calls have their own.
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        _lib.check("lss_int4_matvec", lib.lss_int4_matvec(
            x.data_ptr(), _CODES[x.dtype], rows, k, x_stride, packed.data_ptr(), scales.data_ptr(), scale_code, n, k // groups,
            out.data_ptr(), _CODES[out_dtype], y_stride, None if ws is None else ws.data_ptr(), size, _stream(dev)))
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
