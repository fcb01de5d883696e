"""Several tokens per request and step, drafted as a tree: which of them see each other, and which are kept.

A step with drafts runs ``plan_blocks`` for all drafted tokens, ``plan_tree`` once, and per layer ``norm_rotate`` (at
``TreePlan.positions``), ``append_kv`` and ``attend`` (with ``tree=``).  After sampling a token behind every drafted one,
``accept_drafts`` follows the sampled tokens through the trees, ``compact_kv`` moves the accepted tokens' keys and
values up in each layer's cache, and ``release_blocks`` (with ``keep=``) takes the rejected tokens' blocks back.  As
with the other operators everything stays on the device; what the sampler takes as Python lists (histories of penalties, stop
ids) does not, see ``accept_drafts``.  LocalStrm decodes token by token and has no counterpart.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .head import _on, _stream
from .paged import KVCache8, StepPlan, TreePlan, _ints, _table

__all__ = ["Accepted", "plan_tree", "accept_drafts", "compact_kv"]

_I32 = torch.int32


@dataclass
class Accepted:
    """What the sampled tokens confirm (all int32 on the device).

    ``path [T]``: in each row's part of the step, the accepted tokens (counted from the row's first one), -1 behind them;
    ``tokens [T]``: likewise the request's new tokens; ``counts [B]``: accepted tokens; ``lens [B]``: lengths with
    these alone; ``last [B]``: the newest token, the next step's first (-1: none); ``codes [B]``: its stop code.
    """
    path: torch.Tensor
    tokens: torch.Tensor
    counts: torch.Tensor
    lens: torch.Tensor
    last: torch.Tensor
    codes: torch.Tensor


def _device(plan: StepPlan) -> int:
    if not isinstance(plan.starts, torch.Tensor) or not plan.starts.is_cuda:
        raise RuntimeError("plan: CUDA tensors are needed (no CPU fallback)")
    return plan.starts.get_device()


def plan_tree(plan: StepPlan, parents: torch.Tensor) -> TreePlan:
    """The trees of a step's new tokens.

    ``parents`` int32 ``[T]``, in the step's token order: the token that each one goes on from, counted from its row's
    first new token; parents come before their children, and -1 (or anything that is no earlier token) goes on from
    the context.  A row of more than 1,024 new tokens is a prompt chunk, whose tokens follow one another whatever their
    parents say."""
    dev = _device(plan)
    B, T = plan.granted.numel(), parents.numel()
    at = _ints("parents", parents, T, dev)
    span, positions = parents.new_empty((T, 2)), parents.new_empty((T,))
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_tree_plan", lib.lss_tree_plan(
            _ints("plan.starts", plan.starts, B + 1, dev), _ints("plan.granted", plan.granted, B, dev),
            _ints("plan.lens", plan.lens, B, dev), B, at, T, span.data_ptr(), positions.data_ptr(), _stream(dev)))
    return TreePlan(span, positions, parents)


def accept_drafts(plan: StepPlan, tree: TreePlan, tokens: torch.Tensor, targets: torch.Tensor,
                  codes: Optional[torch.Tensor] = None, given: Optional[torch.Tensor] = None,
                  lens_out: Optional[torch.Tensor] = None) -> Accepted:
    """Follows the sampled tokens through the trees of drafted ones.

    ``tokens`` int32 ``[T]``: the step's tokens; ``targets`` int32 ``[T]``: the token sampled behind each of them;
    ``codes`` int32 ``[T]``: ``check_stop_batch``'s of the targets.  The first ``given[b]`` tokens of row b (default 1: the
    one sampled last) are accepted as they are; from the last of them the walk goes to the first child that is the sampled
    token, until there is none or the sampled token has a code.  So the request's new tokens are those that
    sampling one by one gives with the same logits, whatever was drafted.  A row with a prompt chunk has all of it given; where the
    prompt goes on its new token means nothing (``plan.stops(accepted.codes, prompt_lens)`` drops its code).

    Each target is sampled as if its token were the request's last: with penalties its history holds the drafted tokens
    from the row's first to it, its ancestors, and not the other branches.  The logits are those of the 8-bit cache as the step left it:
    a drafted token of large values in the context's last block widens that block's scale, the context's values in it are
    rounded again to the larger step (below 2^-6 of the scale they lose bits), and stay so when the token is rejected.  Where two
    logits are nearly equal that can decide otherwise than a run without drafts.

    ``lens_out`` may be ``plan.lens``, which ``compact_kv``, ``plan.stops`` and ``release_blocks(keep=)`` still need as it is."""
    dev = _device(plan)
    B, T = plan.granted.numel(), tree.parents.numel()
    starts_at = _ints("plan.starts", plan.starts, B + 1, dev)
    new = plan.starts.new_empty((2 * T + 4 * B,))  # one allocation for the results
    path, said, counts, lens, last, stop = new.split_with_sizes((T, T, B, B, B, B))
    lens = lens if lens_out is None else lens_out
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_tree_accept", lib.lss_tree_accept(
            starts_at, _ints("plan.granted", plan.granted, B, dev),
            _ints("plan.lens", plan.lens, B, dev), B, _ints("tree.parents", tree.parents, T, dev), _ints("tokens", tokens, T, dev),
            _ints("targets", targets, T, dev), None if codes is None else _ints("codes", codes, T, dev),
            None if given is None else _ints("given", given, B, dev), T, path.data_ptr(), said.data_ptr(), counts.data_ptr(),
            _ints("lens_out", lens, B, dev), last.data_ptr(), stop.data_ptr(), _stream(dev)))
    return Accepted(path, said, counts, lens, last, stop)


def compact_kv(cache: KVCache8, block_table: torch.Tensor, plan: StepPlan, path: torch.Tensor, counts: torch.Tensor) -> None:
    """Moves the keys and values of the accepted tokens (``Accepted.path``, ``Accepted.counts``) to the places
    behind the context, in one layer's cache.  ``plan.lens`` are the lengths with all new tokens.

    A block that takes in tokens gets the largest of the scales that they, and the tokens that stay in it, had; codes of
    a smaller scale are rounded again.  A scale that a rejected token widened stays.  What lies behind the accepted tokens is
    left as it was."""
    dev, B, width, stride = _table(block_table)
    blocks, heads, bs, dim = cache.check(dev)
    T = path.numel()
    lib = _lib.load()
    with _on(dev):
        _lib.check("lss_kv_compact", lib.lss_kv_compact(
            cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), blocks, heads, bs, dim,
            block_table.data_ptr(), stride, width, _ints("plan.starts", plan.starts, B + 1, dev),
            _ints("plan.granted", plan.granted, B, dev), _ints("plan.lens", plan.lens, B, dev), B, _ints("path", path, T, dev),
            _ints("counts", counts, B, dev), T, _stream(dev)))
