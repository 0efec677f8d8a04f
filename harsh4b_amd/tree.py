"""Steps over trees of drafted tokens on a paged cache (harsh4b_amd/paged.py):
the operators of include/hq.h's drafted trees.

A draft proposes a tree of tokens for each sequence, the model runs all of them
at once, and the longest path that its own choices follow is kept.  A tree's
first node is the sequence's last sure token, whose keys are not in the cache
yet; parents come before their children.  A sequence's n nodes take its last n
slots in the cache (`lengths` count them), base .. base + n - 1; a node's
position, for rotation and windows, is base + its depth.

    cache.resize(lengths_with_the_trees)
    tree = cache.plan_tree(parents, starts)              # once a step
    for layer in range(layers):
        q = cache.append_tree(layer, qkv, ..., tree)     # K/V of the nodes
        x = cache.attend_tree(layer, q, tree)            # each sees its ancestors
    kept, path, after = cache.accept(tree, drafted, logits=logits)
    cache.resize(kept)                                   # or on to the next trees' lengths

Everything lives on the device: a captured step is valid for every tree of as
many rows.  No reference counterpart.  There is no host fallback.
"""
from __future__ import annotations

import functools
import struct
from typing import NamedTuple

import torch

from . import _native
from .paged import MAX_GROUPS, _F32, _I32, _apart, _cache, _index, _launch, _refuse, _span, _starts

MAX_NODES = _native.HQ_TREE_NODES
ANCESTOR_WORDS = MAX_NODES // 32
MAX_VOCAB = 1 << 30

_pack = struct.Struct("2i4P").pack


class DraftTree(NamedTuple):
    """The trees of a batch.  parents: int32 [tokens], the place of a node's
    parent among its sequence's nodes, or -1; starts: int32 [sequences + 1], a
    sequence's rows; and the plan (tree_plan) of them: depths, int32 [tokens],
    and ancestors, int32 [tokens, 8], a node's 256 bits."""
    parents: torch.Tensor
    starts: torch.Tensor
    depths: torch.Tensor
    ancestors: torch.Tensor


def _nodes(t, name: str, tokens: int, index: int) -> int:
    if t.shape != (tokens,) or t.dtype is not _I32 or t.get_device() != index or not t.is_contiguous():
        _refuse(name, t, _I32, index, "[tokens]")
    return t.data_ptr()


def _tree(tree: DraftTree, tokens: int, sequences: int, index: int) -> bytes:
    parents, starts, depths, ancestors = tree
    if starts is None:
        raise ValueError("a tree needs starts")
    first = _starts(starts, sequences, tokens, index)
    if (ancestors.shape != (tokens, ANCESTOR_WORDS) or ancestors.dtype is not _I32 or ancestors.get_device() != index or
            not ancestors.is_contiguous()):
        _refuse("ancestors", ancestors, _I32, index, f"[tokens, {ANCESTOR_WORDS}]")
    return _pack(tokens, 0, first, _nodes(parents, "parents", tokens, index), _nodes(depths, "depths", tokens, index),
                 ancestors.data_ptr())


def tree_plan(parents: torch.Tensor, starts: torch.Tensor, status: torch.Tensor, depths: torch.Tensor | None = None,
              ancestors: torch.Tensor | None = None, stream=None) -> DraftTree:
    """Depths and ancestors of a batch's trees (hq_tree_plan), once for all
    layers of a step.  parents: int32 [tokens] (-1: none; else before the node);
    starts: int32 [sequences + 1].  A sequence with a parent outside its range
    or more than 256 nodes gets depths of -1 and sets HQ_PAGES_BAD in `status`."""
    if not isinstance(parents, torch.Tensor) or not parents.is_cuda or parents.dim() != 1:
        raise ValueError("parents must be a contiguous int32 device tensor [tokens]")
    index = parents.get_device()
    tokens = parents.shape[0]
    if starts is None or starts.dim() != 1 or starts.shape[0] < 2:
        raise ValueError("starts must be a contiguous int32 device tensor [sequences + 1]")
    if status is None or status.numel() != 1 or status.dtype is not _I32 or status.get_device() != index:
        _refuse("status", status, _I32, index, "[1]")
    given = depths is not None or ancestors is not None
    if depths is None:
        depths = torch.empty_like(parents)
    if ancestors is None:
        ancestors = torch.empty((tokens, ANCESTOR_WORDS), dtype=_I32, device=parents.device)
    tree = DraftTree(parents, starts, depths, ancestors)
    sequences = starts.shape[0] - 1
    packed = _tree(tree, tokens, sequences, index)
    if given:
        _apart(((depths.data_ptr(), 4 * tokens), (ancestors.data_ptr(), 4 * ANCESTOR_WORDS * tokens)),
               ((parents.data_ptr(), 4 * tokens), (starts.data_ptr(), 4 * sequences + 4), (status.data_ptr(), 4)))
    if tokens:
        _launch(_native.lib().hq_tree_plan, (packed, sequences, status.data_ptr()), None, index, stream,
                stream and (*tree, status), "hq_tree_plan")
    return tree


def paged_append_tree(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, rope_cos: torch.Tensor,
                      rope_sin: torch.Tensor, eps: float, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor,
                      lengths: torch.Tensor, status: torch.Tensor, tree: DraftTree, out: torch.Tensor | None = None,
                      stream=None) -> torch.Tensor:
    """paged_append of a batch's nodes (hq_paged_append_tree): K and V to the
    nodes' slots, the rotation by their positions; returns the queries, float32
    [tokens, heads, head_dim]."""
    if status is None or lengths is None:
        raise ValueError("paged_append_tree needs the cache's lengths and status")
    index = _index(table)
    cache, sequences, kv, d = _cache(index, keys, values, table, lengths, None, status, 4)
    shape = qkv.shape
    if len(shape) != 2 or qkv.dtype is not _F32 or qkv.get_device() != index or not qkv.is_contiguous():
        _refuse("qkv", qkv, _F32, index, "[tokens, (heads + 2 kv_heads) * head_dim]")
    tokens, width = shape
    heads = width // d - 2 * kv
    if width % d or heads < 1 or heads % kv or heads // kv > MAX_GROUPS:
        raise ValueError("qkv must be [tokens, (heads + 2 kv_heads) * head_dim] with 1 to 8 heads a kv head")
    if (q_norm.shape != (d,) or q_norm.dtype is not _F32 or q_norm.get_device() != index or
            not q_norm.is_contiguous()):
        _refuse("q_norm", q_norm, _F32, index, "[head_dim]")
    if (k_norm.shape != (d,) or k_norm.dtype is not _F32 or k_norm.get_device() != index or
            not k_norm.is_contiguous()):
        _refuse("k_norm", k_norm, _F32, index, "[head_dim]")
    shape = rope_cos.shape
    if rope_cos.dtype is not _F32 or rope_cos.get_device() != index or not rope_cos.is_contiguous():
        _refuse("rope_cos", rope_cos, _F32, index, "[positions, head_dim / 2]")
    if (rope_sin.shape != shape or rope_sin.dtype is not _F32 or rope_sin.get_device() != index or
            not rope_sin.is_contiguous()):
        _refuse("rope_sin", rope_sin, _F32, index, "[positions, head_dim / 2]")
    if len(shape) != 2 or 2 * shape[1] != d or shape[0] < 1:
        raise ValueError("rope_cos and rope_sin must be [positions, head_dim / 2]")
    packed = _tree(tree, tokens, sequences, index)
    if out is None:
        out = torch.empty((tokens, heads, d), dtype=_F32, device=qkv.device)
    elif (out.shape != (tokens, heads, d) or out.dtype is not _F32 or out.get_device() != index or
          not out.is_contiguous()):
        _refuse("out", out, _F32, index, "[tokens, heads, head_dim]")
    elif -4 * out.numel() < out.data_ptr() - qkv.data_ptr() < 4 * qkv.numel():
        raise ValueError("out must not overlap qkv")
    if tokens:
        _launch(_native.lib().hq_paged_append_tree,
                (cache, qkv.data_ptr(), packed, heads, q_norm.data_ptr(), k_norm.data_ptr(), eps, rope_cos.data_ptr(),
                 rope_sin.data_ptr(), shape[0], out.data_ptr()), None, index, stream,
                stream and (qkv, q_norm, k_norm, rope_cos, rope_sin, keys, values, table, lengths, status, *tree, out),
                "hq_paged_append_tree")
    return out


@functools.lru_cache(maxsize=1024)
def _attention_workspace_bytes(tokens: int, heads: int, kv_heads: int, head_dim: int) -> int:
    return _native.lib().hq_paged_attention_tree_workspace_bytes(tokens, heads, kv_heads, head_dim)


def paged_attention_tree(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor,
                         lengths: torch.Tensor, tree: DraftTree, window: int = 0, sinks: int = 0,
                         out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Grouped-query attention of a batch's nodes, float32 [tokens, heads,
    head_dim], over one layer's pages (hq_paged_attention_tree): a node sees the
    slots before its tree that have a page, its ancestors and itself; with
    `window` > 0 only positions above its own - window, or below `sinks`.  A node
    of a tree that is none gets zeros; rows past the last sequence's are not
    touched."""
    if lengths is None:
        raise ValueError("paged_attention_tree needs the cache's lengths")
    index = _index(table)
    cache, sequences, kv, d = _cache(index, keys, values, table, lengths, None, None, 4)
    shape = query.shape
    if len(shape) != 3 or query.dtype is not _F32 or query.get_device() != index or not query.is_contiguous():
        _refuse("query", query, _F32, index, "[tokens, heads, head_dim]")
    tokens, heads, width = shape
    if width != d or heads < 1 or heads % kv or heads // kv > MAX_GROUPS:
        raise ValueError("query must be [tokens, heads, head_dim] with 1 to 8 heads a kv head")
    if not 0 <= window <= 0x7FFFFFFF or not 0 <= sinks <= 0x7FFFFFFF:
        raise ValueError("window and sinks must not be negative")
    packed = _tree(tree, tokens, sequences, index)
    if out is None:
        out = torch.empty_like(query)
    elif out.shape != shape or out.dtype is not _F32 or out.get_device() != index or not out.is_contiguous():
        _refuse("out", out, _F32, index, "like query")
    elif abs(out.data_ptr() - query.data_ptr()) < 4 * tokens * heads * d:
        raise ValueError("out must not overlap query")
    if tokens:
        _launch(_native.lib().hq_paged_attention_tree,
                (cache, query.data_ptr(), packed, heads, window, sinks, out.data_ptr()),
                _attention_workspace_bytes(tokens, heads, kv, d), index, stream,
                stream and (query, keys, values, table, lengths, *tree, out), "hq_paged_attention_tree")
    return out


@functools.lru_cache(maxsize=1024)
def _accept_workspace_bytes(tokens: int, sequences: int, vocab: int, levels: int) -> int:
    return _native.lib().hq_pages_accept_workspace_bytes(tokens, sequences, vocab, levels)


def pages_accept(keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                 status: torch.Tensor, tree: DraftTree, drafted: torch.Tensor, choices: torch.Tensor | None = None,
                 logits: torch.Tensor | None = None, levels: int = MAX_NODES, out: tuple | None = None, stream=None):
    """Keep the path that the model's choices follow (hq_pages_accept): from
    each sequence's root the child whose drafted token (int32 [tokens]) is the
    choice at its parent, and so on, at most `levels` nodes (a tree's depth + 1
    where the caller knows it: by logits fewer blocks, of which up to 16 levels
    side by side have some each).  The choices are given (int32
    [tokens], e.g. a sampler's), or the largest of `logits` (float32 [tokens,
    vocab], ties to the lowest index).  The path's K and V, in every layer of
    keys/values [layers, pages, kv_heads, page_size, head_dim], move to the
    slots behind the base.  Returns int32 (kept [sequences], path [tokens],
    next [sequences]): the lengths to resize to, the path's nodes in a
    sequence's first rows (then -1), and the choice at the path's end (before a
    fork, and before growth under a window, resize to kept itself); a
    sequence without nodes, or all while status says that the cache refused to
    grow, have kept -1 (a resize leaves them) and next -1."""
    if status is None or lengths is None:
        raise ValueError("pages_accept needs the cache's lengths and status")
    index = _index(table)
    cache, sequences, _, _ = _cache(index, keys, values, table, lengths, None, status, 5)
    if not isinstance(drafted, torch.Tensor) or drafted.dim() != 1:
        _refuse("drafted", drafted, _I32, index, "[tokens]")
    tokens = drafted.shape[0]
    ids = _nodes(drafted, "drafted", tokens, index)
    packed = _tree(tree, tokens, sequences, index)
    if (choices is None) == (logits is None):
        raise ValueError("pages_accept takes either choices or logits")
    if not 1 <= levels <= MAX_NODES:
        raise ValueError(f"levels must be from 1 to {MAX_NODES}")
    vocab = 0
    if logits is not None:
        if (logits.dim() != 2 or logits.shape[0] != tokens or logits.shape[1] < 1 or logits.dtype is not _F32 or
                logits.get_device() != index or not logits.is_contiguous()):
            _refuse("logits", logits, _F32, index, "[tokens, vocab]")
        vocab = logits.shape[1]
        if vocab > MAX_VOCAB:
            raise ValueError("logits must have a vocabulary of at most 2^30")
        chosen, rows = None, logits.data_ptr()
    else:
        chosen, rows = _nodes(choices, "choices", tokens, index), None
    if out is None:
        kept, path, after = torch.empty_like(lengths), torch.empty_like(drafted), torch.empty_like(lengths)
    else:
        kept, path, after = out
        _nodes(path, "path", tokens, index)
        for t, name in ((kept, "kept"), (after, "next")):
            if t.shape != (sequences,) or t.dtype is not _I32 or t.get_device() != index or not t.is_contiguous():
                _refuse(name, t, _I32, index, "[sequences]")
        given = keys, values, table, lengths, status, *tree, drafted, choices, logits
        _apart([_span(t) for t in (kept, path, after)], [_span(t) for t in given if t is not None])
    if tokens == 0:
        vocab, rows = 0, None                  # (nothing is read)
    _launch(_native.lib().hq_pages_accept,
            (cache, packed, ids, chosen, rows, vocab, levels, kept.data_ptr(), path.data_ptr(), after.data_ptr()),
            _accept_workspace_bytes(tokens, sequences, vocab, levels), index, stream,
            stream and (keys, values, table, lengths, status, *tree, drafted, choices, logits, kept, path, after),
            "hq_pages_accept")
    return kept, path, after
