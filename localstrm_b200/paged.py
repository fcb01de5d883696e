"""Block tables, the 8-bit key/value cache and its attention: the decode step's memory side.

A step runs ``plan_blocks`` (a place for every request's new tokens), ``append_kv`` (their keys and
values, in 8 bits with one scale per block and head) and ``attend`` per layer; after sampling,
``release_blocks`` takes the codes of ``check_stop_batch`` and returns the blocks of the requests
that stopped.  Everything stays on the device: no call reads a length back, so a step can be
captured in a CUDA graph.  LocalStrm's counterparts are the host-side ``BlockManager``
(``src/memory/block_manager.py``) and the gather + SDPA of ``src/kernels/paged_attention.py``.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .head import _CODES, _on, _stream

__all__ = ["StepPlan", "KVCache8", "plan_blocks", "release_blocks", "append_kv", "attend"]


@dataclass
class StepPlan:
    """Where the tokens of one step lie (all int32 on the device, ``slots`` int64).

    ``starts [B + 1]``: first token of each row in the step's token order; ``granted [B]``: tokens that
    the row may write (0: refused or idle); ``lens [B]``: its length with them; ``slots`` and
    ``positions [capacity]``: block * block_size + offset and position of each token (-1 and 0 where there
    is none); ``n_free [1]``: blocks left.  ``append_kv`` and ``attend`` read the first three.
    """
    starts: torch.Tensor
    granted: torch.Tensor
    lens: torch.Tensor
    slots: Optional[torch.Tensor] = None
    positions: Optional[torch.Tensor] = None
    n_free: Optional[torch.Tensor] = None


@dataclass
class KVCache8:
    """Keys and values in 8 bits: ``k``, ``v`` float8_e4m3fn ``[num_blocks, heads, block_size, dim]``,
    ``k_scale``, ``v_scale`` float32 ``[num_blocks, heads]``; a value is ``code * scale``."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, num_blocks: int, heads: int, block_size: int, dim: int, device="cuda") -> "KVCache8":
        """A zeroed cache."""
        values = lambda: torch.zeros(num_blocks, heads, block_size, dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        scales = lambda: torch.ones(num_blocks, heads, dtype=torch.float32, device=device)
        return cls(values(), values(), scales(), scales())

    def check(self, device: torch.device) -> Tuple[int, int, int, int]:
        """(num_blocks, heads, block_size, dim); raises where a tensor is not what the kernels read."""
        shape = self.k.shape
        if self.k.dim() != 4:
            raise ValueError("cache: k must be [num_blocks, heads, block_size, dim]")
        for name, t in (("k", self.k), ("v", self.v)):
            if t.shape != shape or t.dtype != torch.float8_e4m3fn or t.device != device or not t.is_contiguous():
                raise ValueError(f"cache: {name} must be a contiguous float8_e4m3fn {list(shape)} on {device}")
        for name, t in (("k_scale", self.k_scale), ("v_scale", self.v_scale)):
            if t.shape != shape[:2] or t.dtype != torch.float32 or t.device != device or not t.is_contiguous():
                raise ValueError(f"cache: {name} must be a contiguous float32 {list(shape[:2])} on {device}")
        return tuple(shape)


def _cuda(name: str, t: torch.Tensor) -> torch.device:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name}: a CUDA tensor is needed (no CPU fallback)")
    return t.device


def _ints(name: str, t: torch.Tensor, n: int, dev: torch.device) -> None:
    if t.dtype != torch.int32 or t.numel() != n or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 tensor of {n} entries on {dev}")


def _table(table: torch.Tensor) -> Tuple[torch.device, int, int]:
    dev = _cuda("block_table", table)
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[1] < 1 or table.stride(1) != 1 \
            or (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
        raise ValueError("block_table: expected int32 [B, width >= 1] with rows of stride 1")
    return dev, table.shape[0], table.shape[1]


def _stride0(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])  # one row: its stride says nothing


def _out(name: str, t: Optional[torch.Tensor], new: torch.Tensor, n: int, dev: torch.device) -> torch.Tensor:
    if t is None:
        return new
    _ints(name, t, n, dev)
    return t


def plan_blocks(block_table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor, free_blocks: torch.Tensor,
                n_free: torch.Tensor, block_size: int, capacity: int, lens_out: Optional[torch.Tensor] = None,
                n_free_out: Optional[torch.Tensor] = None) -> StepPlan:
    """A place for ``new_lens[b]`` more tokens of every row of ``block_table [B, width]``.

    ``lens [B]``: tokens that the rows hold; ``free_blocks [num_blocks]`` with ``n_free [1]``: a stack of
    free block ids, its top taken first; ``capacity``: tokens that the step has room for.  Rows are
    served in order, each with all of its tokens or none: none if they end behind the capacity or the
    table's width, or if the free list does not hold the blocks for it and the rows before it.  New
    blocks are written into the table.  ``lens_out`` / ``n_free_out`` may be ``lens`` / ``n_free``
    (state updated in place, as a captured step needs it); otherwise both inputs are left as they are.
    """
    dev, B, width = _table(block_table)
    _ints("lens", lens, B, dev)
    _ints("new_lens", new_lens, B, dev)
    _ints("free_blocks", free_blocks, free_blocks.numel(), dev)
    _ints("n_free", n_free, 1, dev)
    if capacity < 0 or free_blocks.numel() < 1:
        raise ValueError("capacity must not be negative, free_blocks not empty")
    # One allocation for the int32 results.
    positions, granted, starts, new_state, new_free = torch.empty(capacity + 3 * B + 2, dtype=torch.int32, device=dev).split_with_sizes(
        (capacity, B, B + 1, B, 1))
    lens_out, n_free_out = _out("lens_out", lens_out, new_state, B, dev), _out("n_free_out", n_free_out, new_free, 1, dev)
    slots = torch.empty(capacity, dtype=torch.int64, device=dev)
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_block_plan", lib.lss_block_plan(
            block_table.data_ptr(), _stride0(block_table), width, lens.data_ptr(), new_lens.data_ptr(), B, block_size,
            free_blocks.data_ptr(), free_blocks.numel(), n_free.data_ptr(), capacity, slots.data_ptr(), positions.data_ptr(),
            starts.data_ptr(), granted.data_ptr(), lens_out.data_ptr(), n_free_out.data_ptr(),
            _stream(dev)))
    return StepPlan(starts, granted, lens_out, slots, positions, n_free_out)


def release_blocks(block_table: torch.Tensor, lens: torch.Tensor, codes: torch.Tensor, free_blocks: torch.Tensor,
                   n_free: torch.Tensor, block_size: int, lens_out: Optional[torch.Tensor] = None,
                   n_free_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Returns the blocks of the rows with a non-zero code (``check_stop_batch``'s) to ``free_blocks``, in
    row and block order; their lengths become 0.  Gives ``(lens, n_free)`` afterwards; ``lens_out`` and
    ``n_free_out`` as for ``plan_blocks``.  Blocks that rows share must be released once."""
    dev, B, width = _table(block_table)
    _ints("lens", lens, B, dev)
    _ints("codes", codes, B, dev)
    _ints("free_blocks", free_blocks, free_blocks.numel(), dev)
    _ints("n_free", n_free, 1, dev)
    if free_blocks.numel() < 1:
        raise ValueError("free_blocks must not be empty")
    new_state, new_free = torch.empty(B + 1, dtype=torch.int32, device=dev).split_with_sizes((B, 1))
    lens_out, n_free_out = _out("lens_out", lens_out, new_state, B, dev), _out("n_free_out", n_free_out, new_free, 1, dev)
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_block_release", lib.lss_block_release(
            block_table.data_ptr(), _stride0(block_table), width, lens.data_ptr(), codes.data_ptr(), B, block_size,
            free_blocks.data_ptr(), free_blocks.numel(), n_free.data_ptr(), lens_out.data_ptr(), n_free_out.data_ptr(),
            _stream(dev)))
    return lens_out, n_free_out


def _plan(plan: StepPlan, B: int, dev: torch.device) -> None:
    _ints("plan.starts", plan.starts, B + 1, dev)
    _ints("plan.granted", plan.granted, B, dev)
    _ints("plan.lens", plan.lens, B, dev)


def append_kv(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, plan: StepPlan) -> None:
    """Writes the step's keys and values ``[T, heads, dim]`` (f32, bf16 or f16; any token and head
    strides) into the cache, at the places that ``plan`` gave them.

    A block's scale is the smallest power of two with which its finite values fit e4m3; where tokens
    of this step make it grow, the tokens that the block already holds are rounded again.  Tokens of
    refused rows are passed over.  A block that is written must belong to one row."""
    dev, B, width = _table(block_table)
    blocks, heads, bs, dim = cache.check(dev)
    _plan(plan, B, dev)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (heads, dim) or k.dtype != v.dtype or k.device != dev or v.device != dev:
        raise ValueError(f"k, v: expected [T, {heads}, {dim}] of one dtype on {dev}")
    if k.dtype not in _CODES:
        raise TypeError(f"unsupported dtype {k.dtype}")
    k = k if k.stride(2) == 1 else k.contiguous()
    v = v if v.stride(2) == 1 else v.contiguous()
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_kv_append", lib.lss_kv_append(
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _CODES[k.dtype], k.shape[0], heads,
            dim, cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), blocks, bs,
            block_table.data_ptr(), _stride0(block_table), width, plan.starts.data_ptr(), plan.granted.data_ptr(),
            plan.lens.data_ptr(), B, _stream(dev)))


def attend(q: torch.Tensor, cache: KVCache8, block_table: torch.Tensor, plan: StepPlan, scale: Optional[float] = None,
           out: Optional[torch.Tensor] = None, lse_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal softmax attention of the step's queries ``[T, q_heads, dim]`` (bf16 or f16; dim 64, 128 or
    256) over the cache, one token per row or many; query head h reads key head ``h // (q_heads / heads)``.

    The queries of row b see its positions up to their own, the step's own tokens among them (append
    first).  ``scale`` defaults to ``dim ** -0.5``; ``lse_out`` (float32 ``[T, q_heads]``) receives the natural
    log of the softmax sums.  Tokens of refused rows, and those behind the last row, are left as they
    are in ``out`` and ``lse_out`` (in a fresh ``out``: undefined)."""
    dev, B, width = _table(block_table)
    blocks, heads, bs, dim = cache.check(dev)
    _plan(plan, B, dev)
    if q.dim() != 3 or q.shape[2] != dim or q.shape[1] < heads or q.shape[1] % heads or q.device != dev:
        raise ValueError(f"q: expected [T, a multiple of {heads}, {dim}] on {dev}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"unsupported dtype {q.dtype}")
    q = q if q.stride(2) == 1 else q.contiguous()
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1 \
            or out.stride(1) < dim or out.stride(0) < out.stride(1):
        raise ValueError(f"out: expected {q.dtype} {list(q.shape)} on {dev}, rows of stride 1 that do not overlap")
    if lse_out is not None and (lse_out.dtype != torch.float32 or lse_out.shape != q.shape[:2] or lse_out.device != dev
                                or not lse_out.is_contiguous()):
        raise ValueError(f"lse_out: expected a contiguous float32 {list(q.shape[:2])} on {dev}")
    lib = _lib.load()
    with _on(dev):
        # From torch's allocator for every call: calls on other streams, and captured ones, have their own.
        ws = torch.empty(int(lib.lss_attend_workspace_bytes(dim)), dtype=torch.uint8, device=dev)
        _lib.check("lss_attend", lib.lss_attend(
            q.data_ptr(), q.stride(0), q.stride(1), _CODES[q.dtype], q.shape[0], q.shape[1], heads, dim, cache.k.data_ptr(),
            cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), blocks, bs, block_table.data_ptr(),
            _stride0(block_table), width, plan.starts.data_ptr(), plan.granted.data_ptr(), plan.lens.data_ptr(), B,
            float(scale if scale is not None else dim ** -0.5), out.data_ptr(), out.stride(0), out.stride(1),
            lse_out.data_ptr() if lse_out is not None else None, ws.data_ptr(), ws.numel(),
            _stream(dev)))
    return out
