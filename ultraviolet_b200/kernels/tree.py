"""Trees of drafted tokens over the int8 cache: attention of every node, the accepted path into the caches, and rows forked to a group.

A tree is ``parents`` (B, T) or, one for all rows, (T,): integers, at most 64 nodes.  -1 marks the root -- the last token drawn,
not in the cache yet --, a value in [0, i) the parent of node i; a node with any other parent is absent (padding), and so is everything
below it.  Node i of row b stands at position ``pos[b]`` + its depth.

Each function goes to its kernel through the native host path; where something watches the call (a dispatch mode, a tracer, a
transform, a gradient that is wanted) it goes through a torch operator of the ``uvb200`` namespace.  The kernels have no backward.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch import Tensor

from .. import _lib


@torch.library.custom_op("uvb200::tree_positions", mutates_args=())
def _positions_op(parents: Tensor, pos: Tensor) -> Tensor:
    return _lib.host().tree_positions(parents, pos, True)


@_positions_op.register_fake
def _(parents, pos):
    return pos.new_empty((pos.size(0), parents.size(-1)), dtype=torch.int64)


def tree_positions(parents: Tensor, pos: Tensor) -> Tensor:
    """(B, T) int64: pos[b] + depth of every node (absent nodes: pos[b]), as the step's rotary embedding takes them."""
    if not torch.compiler.is_compiling():
        out = _lib.host().tree_positions(parents, pos, False)
        if out is not None:
            return out
    return _positions_op(parents, pos)


@torch.library.custom_op("uvb200::tree_attn", mutates_args=())
def _tree_attn_op(q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, pos: Tensor, starts: Tensor, parents: Tensor,
                  scale: float, k_scale: Tensor, v_scale: Tensor, window: int, ring: bool, row_map: Optional[Tensor],
                  num_splits: int) -> Tensor:
    return _lib.host().tree_attention(q, k, v, k_cache, v_cache, pos, starts, parents, scale, k_scale, v_scale, window, int(ring),
                                      row_map, num_splits, None, 0.0, None, None, None, True)


@_tree_attn_op.register_fake
def _(q, k, v, k_cache, v_cache, pos, starts, parents, scale, k_scale, v_scale, window, ring, row_map, num_splits):
    return torch.empty_like(q, memory_format=torch.contiguous_format)


def tree_attention(q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, pos: Tensor, starts: Tensor, parents: Tensor,
                   scale: float, *, k_scale: Tensor, v_scale: Tensor, window: int = 0, ring: bool | None = None,
                   row_map: Tensor | None = None, num_splits: int | None = None) -> Tensor:
    """Attention of every node of the trees to the cached keys of its row and to its own ancestors: (B, T, H, hd) like q.

    q (B, T, H, hd), k and v (B, T, K, hd) fp16 / bf16: the nodes' projections (slices of a packed projection are taken as they are);
    k_cache, v_cache (rows, K, S, hd) int8 with k_scale / v_scale (rows, K, S) fp16; pos (B,) the first position that is not cached,
    starts (B,) the first valid one.  A node at position p sees the cached positions max(starts, p - window + 1, 0) .. pos - 1
    (window 0: no limit; ring, default window > 0: the newest S of them, position t in slot t % S) and its ancestors within the
    window, itself included.  The nodes' keys and values pass through the cache's quantiser first: a step of a tree reads what
    the same tokens would read one at a time.  row_map (B,): cache row of batch row b.  An absent node gets zeros; a present one sees
    itself at least, and gets NaN where its query is not finite or a scale that it sees is no number.  num_splits: parts into which a row's
    keys are cut (None: chosen by the library)."""
    scale, window, splits = float(scale), int(window), int(num_splits or 0)
    if not torch.compiler.is_compiling():
        out = _lib.host().tree_attention(q, k, v, k_cache, v_cache, pos, starts, parents, scale, k_scale, v_scale, window,
                                         -1 if ring is None else int(bool(ring)), row_map, splits, None, 0.0, None, None, None,
                                         False)
        if out is not None:
            return out
    return _tree_attn_op(q, k, v, k_cache, v_cache, pos, starts, parents, scale, k_scale, v_scale, window,
                         window > 0 if ring is None else bool(ring), row_map, splits)


@torch.library.custom_op("uvb200::tree_advance", mutates_args=("k_caches", "v_caches", "k_scales", "v_scales", "pos_out", "oob"))
def _advance_op(k: Sequence[Tensor], v: Sequence[Tensor], k_caches: Sequence[Tensor], v_caches: Sequence[Tensor],
                k_scales: Sequence[Tensor], v_scales: Sequence[Tensor], rings: Sequence[bool], parents: Tensor, tokens: Tensor,
                target: Tensor, pos: Tensor, row_map: Optional[Tensor], pos_out: Tensor,
                oob: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor]:
    return _lib.host().tree_advance(k, v, k_caches, v_caches, k_scales, v_scales, list(rings), parents, tokens, target, pos, row_map,
                                    pos_out, oob, True)


@_advance_op.register_fake
def _(k, v, k_caches, v_caches, k_scales, v_scales, rings, parents, tokens, target, pos, row_map, pos_out, oob):
    B, T = tokens.shape
    return (pos.new_empty((B, T), dtype=torch.int32), pos.new_empty((B,), dtype=torch.int32), pos.new_empty((B, T), dtype=torch.int64))


def tree_advance(k, v, k_caches, v_caches, k_scales, v_scales, rings, parents: Tensor, tokens: Tensor, target: Tensor, pos: Tensor, *,
                 row_map: Tensor | None = None, pos_out: Tensor | None = None, oob: Tensor | None = None):
    """The accepted path of every tree, with its keys and values appended to the caches of all layers, in one launch.

    tokens (B, T) the drafted tokens, target (B, T) the token that the model drew behind each of them.  The walk starts at the root and
    goes from node i to its first child whose token is target[i].  Returns (path, count, drawn): the accepted nodes in order and -1
    behind them (B, T) int32, their number (B,) int32, and the tokens drawn behind them, then -1, (B, T) int64: the row's new
    tokens, the last of which is not cached yet.

    k, v: per layer (B, T, K, hd), the projections that tree_attention took; k_caches .. v_scales: per layer the tensors of a decode
    state; rings: per layer whether its cache is a ring.  The j-th accepted node is quantised and written at position pos + j; what
    falls outside a linear cache is skipped (and counted in oob, an int32 word).  pos_out (B,) becomes pos + count; by default
    pos itself does."""
    pos_out = pos if pos_out is None else pos_out
    if not torch.compiler.is_compiling():
        got = _lib.host().tree_advance(k, v, k_caches, v_caches, k_scales, v_scales, rings, parents, tokens, target, pos, row_map, pos_out,
                                       oob, False)
        if got is not None:
            return got
    if pos_out is pos:      # (an operator may not be told of one tensor as read and as written)
        new = torch.empty_like(pos)
        got = _advance_op(k, v, k_caches, v_caches, k_scales, v_scales, rings, parents, tokens, target, pos, row_map, new, oob)
        pos.copy_(new)
        return got
    return _advance_op(k, v, k_caches, v_caches, k_scales, v_scales, rings, parents, tokens, target, pos, row_map, pos_out, oob)


@torch.library.custom_op("uvb200::kv_fork", mutates_args=("k_caches", "v_caches", "k_scales", "v_scales", "pos", "starts", "oob"))
def _fork_op(k_caches: Sequence[Tensor], v_caches: Sequence[Tensor], k_scales: Sequence[Tensor], v_scales: Sequence[Tensor],
             rings: Sequence[bool], src: Tensor, dst: Tensor, pos: Tensor, starts: Tensor, oob: Optional[Tensor]) -> None:
    _lib.host().kv_fork(k_caches, v_caches, k_scales, v_scales, list(rings), src, dst, pos, starts, oob, True)


@_fork_op.register_fake
def _(k_caches, v_caches, k_scales, v_scales, rings, src, dst, pos, starts, oob):
    return None


def kv_fork(k_caches, v_caches, k_scales, v_scales, rings, src: Tensor, dst: Tensor, pos: Tensor, starts: Tensor, *,
            oob: Tensor | None = None) -> None:
    """Copies the cached positions starts[s] .. pos[s] - 1 of cache row s = src[i] to row dst[i] in every layer, and pos and starts with
    them, in one launch.  A row may be the source of many; a destination must not be the source or the destination of another
    pair.  src[i] == dst[i] does nothing; rows outside the cache are skipped (and counted in oob, an int32 word)."""
    if not torch.compiler.is_compiling() and _lib.host().kv_fork(k_caches, v_caches, k_scales, v_scales, rings, src, dst, pos, starts,
                                                                 oob, False):
        return
    _fork_op(k_caches, v_caches, k_scales, v_scales, rings, src, dst, pos, starts, oob)
