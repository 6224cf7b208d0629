"""Drafted tokens that form a tree, over a paged cache.

A draft proposes several continuations of each sequence at once: node t has a token and a
parent, one of the nodes before it (-1: a root).  One pass through the model takes all nodes
together, each at the position of its depth, with their keys and values appended behind the
sequence's own, node by node.

    masks, depths = tree.ancestors(parents)            # once a step
    out = tree.attention(q, k_pool, v_pool, table, lengths, masks)     # in every layer
    path, accepted, nxt = tree.accept(tokens, parents, picks)          # after the head
    lengths = cache.keep(lengths, path, accepted)      # pages.Pages: the path's positions

Node t attends to the sequence's cached positions and to the nodes its mask names.  The
kernels and their exact definitions are declared in ``include/tf_search.h``.

Every call runs on its tensors' device and that device's current stream, allocates its outputs
like any torch operation (so calls can be captured into a HIP graph and made from several
streams) and computes no gradients.  What memory is indexed with is checked on the device: a
bad value raises a bit (``_lib.ERR_*``) in *err*, an int32 tensor of one element, where one
is given, and its access is left out.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import lib, ptr
from .mx4 import BF16, INT32, check_device, check_input, launch

MAX_NODES = _lib.TREE_MAX_NODES
MAX_ROWS = 65535
HEAD_DIMS = (64, 128, 256)
INT64 = (torch.int64,)


def _err(err, device) -> None:
    if err is not None:
        check_input(err, "err", INT32)
        if err.numel() != 1:
            raise ValueError(f"err: one element, got {tuple(err.shape)}")
        check_device(device, err)


def _rows_of_nodes(x, what: str, like=None) -> tuple[int, int]:
    check_input(x, what, INT32)
    if x.dim() != 2 or (like is not None and x.shape != like.shape):
        raise ValueError(f"{what} must be [rows, nodes]"
                         f"{'' if like is None else f' like {tuple(like.shape)}'}, got "
                         f"{tuple(x.shape)}")
    rows, nodes = x.shape
    if not 1 <= nodes <= MAX_NODES or rows > MAX_ROWS:
        raise ValueError(f"{what}: 1 to {MAX_NODES} nodes of up to {MAX_ROWS} rows, got "
                         f"{tuple(x.shape)}")
    return rows, nodes


def _counts(counts, rows: int, device):
    if counts is None:
        return None
    check_input(counts, "counts", INT32)
    if counts.shape != (rows,):
        raise ValueError(f"counts must be [{rows}], got {tuple(counts.shape)}")
    check_device(device, counts)
    return counts.contiguous()


def ancestors(parents: torch.Tensor, counts: torch.Tensor | None = None,
              err: torch.Tensor | None = None):
    """Parents int32 ``[rows, nodes]`` (and how many of a row's nodes are there, int32
    ``[rows]``) -> masks int64 ``[rows, nodes, ceil(nodes / 64)]``, whose bit n is set where
    node n is the node itself or one of its ancestors, and depths int32 ``[rows, nodes]``."""
    rows, nodes = _rows_of_nodes(parents, "parents")
    check_device(parents.device)
    counts = _counts(counts, rows, parents.device)
    _err(err, parents.device)
    parents = parents.contiguous()
    masks = parents.new_empty((rows, nodes, -(-nodes // 64)), dtype=torch.int64)
    depths = torch.empty_like(parents)
    launch(parents.get_device(), lib().tfd_tree_masks, ptr(parents), ptr(counts), rows, nodes,
           ptr(masks), ptr(depths), ptr(err))
    return masks, depths


def accept(tokens: torch.Tensor, parents: torch.Tensor, picks: torch.Tensor,
           counts: torch.Tensor | None = None):
    """The path along which the model's picks agree with the draft: from node 0 (whose token
    is the sequence's last one) to the lowest child whose token is its parent's pick, and so
    on.  Tokens, parents and picks int32 ``[rows, nodes]`` -> path int32 ``[rows, nodes]`` (the
    nodes in order, -1 behind them), accepted int32 ``[rows]`` (how many) and next int32
    ``[rows]`` (the last one's pick, a token that is not in the cache yet)."""
    rows, nodes = _rows_of_nodes(tokens, "tokens")
    for x, what in ((parents, "parents"), (picks, "picks")):
        _rows_of_nodes(x, what, tokens)
    check_device(tokens.device, parents, picks)
    counts = _counts(counts, rows, tokens.device)
    tokens, parents, picks = tokens.contiguous(), parents.contiguous(), picks.contiguous()
    path = torch.empty_like(tokens)
    accepted, after = tokens.new_empty((2, rows)).unbind(0)
    launch(tokens.get_device(), lib().tfd_tree_accept, ptr(tokens), ptr(parents), ptr(picks),
           ptr(counts), rows, nodes, ptr(path), ptr(accepted), ptr(after))
    return path, accepted, after


def attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, table: torch.Tensor,
              lengths: torch.Tensor, masks: torch.Tensor, counts: torch.Tensor | None = None, *,
              scale: float | None = None, err: torch.Tensor | None = None,
              rounded: bool = False) -> torch.Tensor:
    """Attention of drafted nodes over a paged cache, bf16 ``[rows, nodes, heads, dim]``.

    q: bf16 of that shape, any strides.  Pools: bf16 ``[pages, kv_heads, 16, dim]``; table: int32
    ``[rows, max_pages]``; lengths: int32 ``[rows]``, the cached positions of each sequence.
    Row b's nodes have their keys and values at positions ``lengths[b] + t``.  Node t attends to
    the positions below ``lengths[b]`` and to the nodes of ``masks[b, t]`` (``ancestors``, or any
    other bits); one that sees nothing gets zeros.  Of a row with ``counts[b]`` nodes the others
    are not there and their outputs are not written.  Scale: dim^-1/2 unless given.

    Probabilities are held to 2^-16 in the product with the values.  *rounded* lets them be bf16
    (2^-8) where many nodes and heads share a kv head, which is up to a quarter faster there."""
    check_input(q, "q", BF16)
    check_input(k_pool, "k_pool", BF16)
    check_input(v_pool, "v_pool", BF16)
    check_input(table, "table", INT32)
    check_input(lengths, "lengths", INT32)
    check_input(masks, "masks", INT64)
    if q.dim() != 4:
        raise ValueError(f"q must be [rows, nodes, heads, dim], got {tuple(q.shape)}")
    rows, nodes, heads, dim = q.shape
    pool = k_pool.shape
    if len(pool) != 4 or pool != v_pool.shape or pool[2] != _lib.PAGE_SIZE or pool[3] != dim:
        raise ValueError(f"pools must be [pages, kv_heads, {_lib.PAGE_SIZE}, {dim}], got "
                         f"{tuple(k_pool.shape)} and {tuple(v_pool.shape)}")
    pages, kv_heads = pool[0], pool[1]
    if dim not in HEAD_DIMS:
        raise ValueError(f"head dimension {dim} is none of {', '.join(map(str, HEAD_DIMS))}")
    if not 1 <= nodes <= MAX_NODES or rows > MAX_ROWS:
        raise ValueError(f"1 to {MAX_NODES} nodes of up to {MAX_ROWS} rows, got {nodes} of {rows}")
    if not 1 <= kv_heads <= heads <= 65535 or heads % kv_heads or pages < 1:
        raise ValueError(f"{heads} heads over {kv_heads} kv heads in {pages} pages")
    width = table.shape[1] if table.dim() == 2 else 0
    if not 1 <= width <= 1 << 22 or table.shape[0] != rows:
        raise ValueError(f"table must be [{rows}, 1..2^22], got {tuple(table.shape)}")
    if lengths.shape != (rows,):
        raise ValueError(f"lengths must be [{rows}], got {tuple(lengths.shape)}")
    if masks.shape != (rows, nodes, -(-nodes // 64)):
        raise ValueError(f"masks must be [{rows}, {nodes}, {-(-nodes // 64)}], got "
                         f"{tuple(masks.shape)}")
    if rows * nodes * heads > 1 << 25 or pages > (1 << 31) - 1:
        raise ValueError(f"up to 2^25 queries a call, got {rows} x {nodes} x {heads}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale < 3.4e38:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if not k_pool.is_contiguous() or not v_pool.is_contiguous() or \
            k_pool.data_ptr() % 16 or v_pool.data_ptr() % 16:
        raise ValueError("pools must be contiguous and 16-byte aligned")
    check_device(q.device, k_pool, v_pool, table, lengths, masks)
    if counts is not None:
        counts = _counts(counts, rows, q.device)
    if err is not None:
        _err(err, q.device)
    of_row, of_node, of_head, of_dim = q.stride()
    if of_dim != 1 or q.data_ptr() % 16 or (of_row | of_node | of_head) % 8:
        q = q.clone(memory_format=torch.contiguous_format)
        of_row, of_node, of_head, of_dim = q.stride()
    table, lengths, masks = table.contiguous(), lengths.contiguous(), masks.contiguous()
    out = q.new_empty((rows, nodes, heads, dim))
    L = lib()
    need = L.tfd_tree_attn_work_bytes(rows, nodes, heads, kv_heads, dim, width)
    # of the stream that uses it, like the output: calls on several streams and captured
    # graphs share nothing
    work = q.new_empty(need, dtype=torch.uint8) if need else None
    a = _lib.TfdTreeAttnArgs(ptr(q), of_row, of_node, of_head, ptr(k_pool), ptr(v_pool), ptr(table),
                             ptr(lengths), ptr(counts), ptr(masks), rows, nodes, heads, kv_heads,
                             dim, width, pages, scale, ptr(out), 0, ptr(work), need, ptr(err),
                             1 if rounded else 0)
    launch(q.get_device(), L.tfd_tree_attn, ctypes.addressof(a))
    return out
