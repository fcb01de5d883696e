"""Block tables, the 8-bit key/value cache and its attention: the decode step's memory side.

A step runs ``plan_blocks`` (a place for every request's new tokens), ``append_kv`` (their keys and
values, in 8 bits with one scale per block and head) and ``attend`` per layer; after sampling,
``release_blocks`` takes the codes of ``check_stop_batch`` (those of the rows that had a token of their own:
``StepPlan.stops``) and returns the blocks of the requests that stopped.  Everything stays on the device: no call reads a length back, so a step can be
captured in a CUDA graph.  LocalStrm's counterparts are the host-side block manager
(``src/memory/``) and the gather + SDPA of ``src/kernels/paged_attention.py``.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .head import _CODES, _on, _stream

__all__ = ["StepPlan", "TreePlan", "Forks", "KVCache8", "plan_blocks", "release_blocks", "fork_blocks", "copy_blocks", "append_kv", "attend"]


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

    def stops(self, codes: torch.Tensor, prompt_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The codes (``check_stop_batch``'s) of the rows that sampled a token of their own in this step,
        0 for the others: what ``release_blocks`` may be given.

        A row without tokens in the step (idle or refused) has no last token: ``starts[b + 1] - 1`` is
        another row's, or one that ``attend`` passed over, and a code for it would free a live request.
        With ``prompt_lens [B]`` rows that do not hold their whole prompt yet are left out too.  The
        tokens of all rows left out mean nothing.  To be called before ``lens`` changes again."""
        own = self.granted > 0
        for name, t in (("codes", codes), ("prompt_lens", prompt_lens)):
            if t is not None and (t.dtype is not _I32 or t.shape != own.shape or t.device != own.device):
                raise ValueError(f"{name}: expected int32 {list(own.shape)} on {own.device}")
        if prompt_lens is not None:
            own = own & (self.lens >= prompt_lens)
        return torch.where(own, codes, 0)


@dataclass
class TreePlan:
    """The trees of a step's new tokens, as ``plan_tree`` makes them (int32 on the device).

    ``span [T, 2]``: a token's place in the pre-order of its row's tree and the number of tokens of its branch (token j is
    i or an ancestor of it where ``0 <= span[i, 0] - span[j, 0] < span[j, 1]``); ``positions [T]``: context and depth,
    for the rotation; ``parents [T]``: what ``plan_tree`` was given.
    """
    span: torch.Tensor
    positions: torch.Tensor
    parents: torch.Tensor


@dataclass
class Forks:
    """What ``fork_blocks`` did (int32 on the device): ``lens [B]`` and ``n_free [1]`` afterwards; ``granted [n]``: tokens
    that a fork took (0: refused); ``copies [n, 2]``: the block to copy for it and the one it is copied to (-1, -1: none),
    for ``copy_blocks`` on every layer's cache."""
    lens: torch.Tensor
    n_free: torch.Tensor
    granted: torch.Tensor
    copies: torch.Tensor


@dataclass
class KVCache8:
    """Keys and values in 8 bits: ``k``, ``v`` float8_e4m3fn ``[num_blocks, heads, block_size, dim]``,
    ``k_scale``, ``v_scale`` float32 ``[num_blocks, heads]``, positive and finite; a value is ``code * scale``."""
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

    def check(self, device: int) -> torch.Size:
        """[num_blocks, heads, block_size, dim]; raises where a tensor is not what the kernels read on
        this CUDA device."""
        k, v, ks, vs = self.k, self.v, self.k_scale, self.v_scale
        shape = k.shape
        if len(shape) != 4:
            raise ValueError("cache: k must be [num_blocks, heads, block_size, dim]")
        if not (k.dtype is _E4M3 and v.dtype is _E4M3 and k.get_device() == device and v.get_device() == device and k.is_contiguous()
                and v.is_contiguous() and v.shape == shape):
            raise ValueError(f"cache: k and v must be contiguous float8_e4m3fn {list(shape)} on cuda:{device}")
        if not (ks.dtype is _F32 and vs.dtype is _F32 and ks.get_device() == device and vs.get_device() == device and ks.is_contiguous()
                and vs.is_contiguous() and ks.shape == shape[:2] and vs.shape == shape[:2]):
            raise ValueError(f"cache: k_scale and v_scale must be contiguous float32 {list(shape[:2])} on cuda:{device}")
        return shape


_I32, _F32, _E4M3 = torch.int32, torch.float32, torch.float8_e4m3fn


def _ints(name: str, t: torch.Tensor, n: int, device: int) -> int:
    """The address of a contiguous int32 tensor of n entries on this device; raises for any other."""
    if t.dtype is not _I32 or t.numel() != n or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 tensor of {n} entries on cuda:{device}")
    return t.data_ptr()


def _table(table: torch.Tensor) -> Tuple[int, int, int, int]:
    """(device, rows, width, row stride) of a block table."""
    if not isinstance(table, torch.Tensor) or not table.is_cuda:
        raise RuntimeError("block_table: a CUDA tensor is needed (no CPU fallback)")
    if table.dtype is not _I32 or table.dim() != 2:
        raise ValueError("block_table: expected int32 [B, width]")
    B, width = table.shape
    stride, inner = table.stride()
    if width < 1 or inner != 1 or (B > 1 and stride < width):
        raise ValueError("block_table: expected int32 [B, width >= 1] with rows of stride 1")
    return table.get_device(), B, width, max(stride, width)  # one row: its stride says nothing


def plan_blocks(block_table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor, free_blocks: torch.Tensor,
                n_free: torch.Tensor, block_size: int, capacity: int, lens_out: Optional[torch.Tensor] = None,
                n_free_out: Optional[torch.Tensor] = None) -> StepPlan:
    """A place for ``new_lens[b]`` more tokens of every row of ``block_table [B, width]``.

    ``lens [B]``: tokens that the rows hold; ``free_blocks [num_blocks]`` with ``n_free [1]``: a stack of
    free block ids, its top taken first; ``capacity``: tokens that the step has room for.  Rows are
    served in order, each with all of its tokens or none: none if they end behind the capacity or the
    table's width, or if the free list does not hold the blocks for it and the rows before it (those
    refused for this reason among them: once one is, no later row gets a new block; one that needs none is
    granted all the same).  New blocks are written into the table.  ``lens_out`` / ``n_free_out`` may be ``lens`` / ``n_free``
    (state updated in place, as a captured step needs it); otherwise both inputs are left as they are.
    """
    dev, B, width, stride = _table(block_table)
    lens_at, new_at = _ints("lens", lens, B, dev), _ints("new_lens", new_lens, B, dev)
    blocks = free_blocks.numel()
    free_at, n_free_at = _ints("free_blocks", free_blocks, blocks, dev), _ints("n_free", n_free, 1, dev)
    if capacity < 0 or blocks < 1:
        raise ValueError("capacity must not be negative, free_blocks not empty")
    # One allocation for the int32 results.
    positions, granted, starts, new_state, new_free = torch.empty(
        capacity + 3 * B + 2, dtype=_I32, device=block_table.device).split_with_sizes((capacity, B, B + 1, B, 1))
    lens_out, n_free_out = new_state if lens_out is None else lens_out, new_free if n_free_out is None else n_free_out
    slots = torch.empty(capacity, dtype=torch.int64, device=block_table.device)
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_block_plan", lib.lss_block_plan(
            block_table.data_ptr(), stride, width, lens_at, new_at, B, block_size, free_at, blocks, n_free_at, capacity,
            slots.data_ptr(), positions.data_ptr(), starts.data_ptr(), granted.data_ptr(), _ints("lens_out", lens_out, B, dev),
            _ints("n_free_out", n_free_out, 1, dev), _stream(dev)))
    return StepPlan(starts, granted, lens_out, slots, positions, n_free_out)


def release_blocks(block_table: torch.Tensor, lens: torch.Tensor, codes: torch.Tensor, free_blocks: torch.Tensor,
                   n_free: torch.Tensor, block_size: int, lens_out: Optional[torch.Tensor] = None,
                   n_free_out: Optional[torch.Tensor] = None, keep: Optional[torch.Tensor] = None,
                   shares: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Returns the blocks of the rows with a non-zero code (``check_stop_batch``'s, through
    ``StepPlan.stops``) to ``free_blocks``, in row and block order; their lengths become 0.  Gives ``(lens, n_free)`` afterwards; ``lens_out`` and
    ``n_free_out`` as for ``plan_blocks``.

    With ``keep [B]`` the other rows give back what lies behind their first ``keep[b]`` tokens, which become their length
    (``Accepted.lens``).  With ``shares [num_blocks]`` (as ``fork_blocks`` keeps them) a block goes back with the last of its
    holders, in the order of these; without, blocks that rows share must be released once.  ``keep`` must not end inside a block
    that another row holds, which nothing here can tell (``Accepted.lens`` never does): the row's next tokens would be written
    over the other's.  To cut a row there, fork it onto an idle row with ``upto`` and release it."""
    dev, B, width, stride = _table(block_table)
    lens_at, codes_at = _ints("lens", lens, B, dev), _ints("codes", codes, B, dev)
    blocks = free_blocks.numel()
    free_at, n_free_at = _ints("free_blocks", free_blocks, blocks, dev), _ints("n_free", n_free, 1, dev)
    if blocks < 1:
        raise ValueError("free_blocks must not be empty")
    if lens_out is None:
        lens_out = lens.new_empty((B,))
    if n_free_out is None:
        n_free_out = lens.new_empty((1,))
    lens_out_at, n_free_out_at = _ints("lens_out", lens_out, B, dev), _ints("n_free_out", n_free_out, 1, dev)
    lib = _lib.load()
    with _on(dev):
        if keep is None and shares is None:
            _lib.check("lss_block_release", lib.lss_block_release(
                block_table.data_ptr(), stride, width, lens_at, codes_at, B, block_size, free_at, blocks, n_free_at,
                lens_out_at, n_free_out_at, _stream(dev)))
        else:
            _lib.check("lss_block_give", lib.lss_block_give(
                block_table.data_ptr(), stride, width, lens_at, codes_at, None if keep is None else _ints("keep", keep, B, dev), B,
                block_size, None if shares is None else _ints("shares", shares, blocks, dev), free_at, blocks, n_free_at,
                lens_out_at, n_free_out_at, _stream(dev)))
    return lens_out, n_free_out


def fork_blocks(block_table: torch.Tensor, lens: torch.Tensor, src_rows: torch.Tensor, dst_rows: torch.Tensor,
                shares: torch.Tensor, free_blocks: torch.Tensor, n_free: torch.Tensor, block_size: int,
                upto: Optional[torch.Tensor] = None, lens_out: Optional[torch.Tensor] = None,
                n_free_out: Optional[torch.Tensor] = None) -> Forks:
    """Lets the idle rows ``dst_rows [n]`` go on from the tokens of the rows ``src_rows [n]``, from the first ``upto [n]`` of
    them where given: more samples of a prompt, or a prompt whose beginning another row holds.

    Their full blocks are shared: ``shares [num_blocks]`` (int32, zeros at first) counts the holders beyond the first, in
    place; the tokens behind these get a block of their own from the free list, to be filled by ``copy_blocks`` on every layer's
    cache.  Forks are served in order, as the rows of ``plan_blocks`` are; one is refused where its rows are outside the
    table, the destination is not idle or an earlier fork's, or there is nothing to take.  Lengths are those before the call.
    ``lens_out`` / ``n_free_out`` as for ``plan_blocks``.  Blocks so shared are given back with ``release_blocks(shares=)``."""
    dev, B, width, stride = _table(block_table)
    n, blocks = src_rows.numel(), free_blocks.numel()
    if blocks < 1:
        raise ValueError("free_blocks must not be empty")
    lens_at = _ints("lens", lens, B, dev)
    free_at, n_free_at = _ints("free_blocks", free_blocks, blocks, dev), _ints("n_free", n_free, 1, dev)
    # One allocation for the results.
    copies, granted, new_state, new_free = lens.new_empty((3 * n + B + 1,)).split_with_sizes((2 * n, n, B, 1))
    lens_out, n_free_out = new_state if lens_out is None else lens_out, new_free if n_free_out is None else n_free_out
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_block_fork", lib.lss_block_fork(
            block_table.data_ptr(), stride, width, lens_at, B, block_size, _ints("src_rows", src_rows, n, dev),
            _ints("dst_rows", dst_rows, n, dev), None if upto is None else _ints("upto", upto, n, dev), n,
            _ints("shares", shares, blocks, dev), free_at, blocks, n_free_at, granted.data_ptr(), copies.data_ptr(),
            _ints("lens_out", lens_out, B, dev), _ints("n_free_out", n_free_out, 1, dev), _stream(dev)))
    return Forks(lens_out, n_free_out, granted, copies.view(n, 2))


def copy_blocks(cache: "KVCache8", copies: torch.Tensor) -> None:
    """Copies whole blocks of one layer's cache, with their scales: ``copies`` int32 ``[n, 2]``, from and to (``Forks.copies``).
    Pairs that are not two blocks of the cache are passed over.  No block may be copied to twice, or both copied from and
    to, in one call."""
    if not isinstance(copies, torch.Tensor) or not copies.is_cuda:
        raise RuntimeError("copies: a CUDA tensor is needed (no CPU fallback)")
    dev = copies.get_device()
    blocks, heads, bs, dim = cache.check(dev)
    if copies.dim() != 2 or copies.shape[1] != 2:
        raise ValueError("copies: expected int32 [n, 2]")
    n = copies.shape[0]
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_kv_copy", lib.lss_kv_copy(
            cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), blocks, heads, bs, dim,
            _ints("copies", copies, 2 * n, dev), n, _stream(dev)))


def append_kv(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, plan: StepPlan) -> None:
    """Writes the step's keys and values ``[T, heads, dim]`` (f32, bf16 or f16; any token and head
    strides) into the cache, at the places that ``plan`` gave them.

    A block's scale is the smallest power of two with which its finite values fit e4m3; where tokens
    of this step make it grow, the tokens that the block already holds are rounded again.  Tokens of
    refused rows are passed over.  A block that is written must belong to one row."""
    dev, B, width, stride = _table(block_table)
    blocks, heads, bs, dim = cache.check(dev)
    shape, dtype = k.shape, k.dtype
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or shape != v.shape or dtype is not v.dtype \
            or k.get_device() != dev or v.get_device() != dev:
        raise ValueError(f"k, v: expected [T, {heads}, {dim}] of one dtype on cuda:{dev}")
    if dtype not in _CODES:
        raise TypeError(f"unsupported dtype {dtype}")
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[2] != 1:
        v = v.contiguous()
        vs = v.stride()
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_kv_append", lib.lss_kv_append(
            k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], _CODES[dtype], shape[0], heads, dim, cache.k.data_ptr(),
            cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), blocks, bs, block_table.data_ptr(), stride,
            width, _ints("plan.starts", plan.starts, B + 1, dev), _ints("plan.granted", plan.granted, B, dev),
            _ints("plan.lens", plan.lens, B, dev), B, _stream(dev)))


def attend(q: torch.Tensor, cache: KVCache8, block_table: torch.Tensor, plan: StepPlan, scale: Optional[float] = None,
           out: Optional[torch.Tensor] = None, lse_out: Optional[torch.Tensor] = None,
           tree: Optional[TreePlan] = None) -> torch.Tensor:
    """Causal softmax attention of the step's queries ``[T, q_heads, dim]`` (bf16 or f16; dim 64, 128 or
    256) over the cache, one token per row or many; query head h reads key head ``h // (q_heads / heads)``.

    The queries of row b see its positions up to their own, the step's own tokens among them (append
    first).  With a ``tree`` (``plan_tree``'s) the step's tokens lie in the cache in their order, and a query sees the tokens before
    them, itself and its ancestors.  A step of no more tokens than rows is taken for one of single tokens; a chunk among many idle rows
    runs faster where only the rows with tokens are passed.  ``scale`` defaults to ``dim ** -0.5``; ``lse_out`` (float32 ``[T, q_heads]``) receives the natural
    log of the softmax sums.  ``out`` may be ``q`` itself; where it overlaps q in any other way the call is
    refused.  Tokens of refused rows, and those behind the last row, are left as they
    are in ``out`` and ``lse_out`` (in a fresh ``out``: undefined)."""
    dev, B, width, stride = _table(block_table)
    blocks, heads, bs, dim = cache.check(dev)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3 or shape[2] != dim or shape[1] < heads or shape[1] % heads or q.get_device() != dev:
        raise ValueError(f"q: expected [T, a multiple of {heads}, {dim}] on cuda:{dev}")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"unsupported dtype {dtype}")
    qs = q.stride()
    if qs[2] != 1:
        q = q.contiguous()
        qs = q.stride()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os = out.stride()
    else:
        os = out.stride()
        if out.shape != shape or out.dtype is not dtype or out.get_device() != dev or os[2] != 1 \
                or (shape[1] > 1 and os[1] < dim) or (shape[0] > 1 and os[0] < dim) \
                or (shape[0] > 1 and os[0] < (shape[1] - 1) * os[1] + dim and os[1] < (shape[0] - 1) * os[0] + dim):
            raise ValueError(f"out: expected {dtype} {list(shape)} on cuda:{dev}, rows of stride 1 that do not overlap")
    if lse_out is not None and (lse_out.dtype is not _F32 or lse_out.shape != shape[:2] or lse_out.get_device() != dev
                                or not lse_out.is_contiguous()):
        raise ValueError(f"lse_out: expected a contiguous float32 {list(shape[:2])} on cuda:{dev}")
    extra = ()
    if tree is not None:
        span = tree.span
        if span.dim() != 2 or span.shape[0] != shape[0]:
            raise ValueError(f"tree.span: expected int32 [{shape[0]}, 2]")
        extra = (_ints("tree.span", span, 2 * shape[0], dev),)
    lib = _lib.load()
    with _on(dev):
        # From torch's allocator for every call: calls on other streams, and captured ones, have their own.
        size = _WORKSPACE.get(dim)
        if size is None:
            size = _WORKSPACE[dim] = int(lib.lss_attend_workspace_bytes(dim))
        ws = block_table.new_empty((size // 4,))
        name = "lss_attend" if tree is None else "lss_attend_tree"
        _lib.check(name, getattr(lib, name)(
            q.data_ptr(), qs[0], qs[1], _CODES[dtype], shape[0], shape[1], heads, dim, cache.k.data_ptr(), cache.v.data_ptr(),
            cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), blocks, bs, block_table.data_ptr(), stride, width,
            _ints("plan.starts", plan.starts, B + 1, dev), _ints("plan.granted", plan.granted, B, dev),
            _ints("plan.lens", plan.lens, B, dev), B, dim ** -0.5 if scale is None else scale, out.data_ptr(), os[0], max(os[1], dim),
            None if lse_out is None else lse_out.data_ptr(), ws.data_ptr(), size, *extra, _stream(dev)))
    return out


_WORKSPACE = {}  # bytes that the attention needs, by head dimension
