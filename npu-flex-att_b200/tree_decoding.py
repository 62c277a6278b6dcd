"""Decoding with a tree of drafted tokens over a paged K/V cache, on
hand-written sm_100a kernels (include/bfa.h; no CPU path).

One step of a decoder that drafts several tokens at once:

    q, k = rotary_embedding(q, k, cos, sin, depths, cache.lens)   # rotary.py
    o = tree_attention(q, k, v, cache, parents)                   # every layer
    path, count, token = verify_tree(p, tokens, parents, u, noise, draft_probs)
    lens = cache_append(cache, k, v, take=path, count=count)      # every layer
    cache = cache._replace(lens=lens)                             # once, at the end

A tree of N <= 64 nodes per sequence is the int32 tensor ``parents`` [N] or
[B, N]: node 0 is the root (the last decided token, whose K/V is not in the
cache yet), 0 <= parents[n] < n for the others, and -1 marks an absent node
(with everything under it). None is a chain; N = 1 is ordinary decoding of one
token. Node n stands at position lens[b] + its depth. No counterpart in the
reference, whose attention takes contiguous K/V.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

import bfa_lib as _bfa
from npu_flash_attention import _CHECK_STATUS, check_device_status

__all__ = ["PagedKVCache", "tree_attention", "verify_tree", "cache_append", "tree_depths"]

class PagedKVCache(NamedTuple):
    """K/V of cached tokens in pages: k_pages and v_pages [num_pages, Hkv,
    page_size, D], page_table int32 [B, max_pages], lens int32 [B]. Token t of
    sequence b lies in page page_table[b, t // page_size], slot t % page_size;
    table entries past a sequence's length are not read, nor, with a sliding
    window W, those of pages wholly before token lens[b] - W: they may be given
    back. The caller owns the tensors and hands out the pages."""
    k_pages: torch.Tensor
    v_pages: torch.Tensor
    page_table: torch.Tensor
    lens: torch.Tensor


_module = None


def _binding():
    global _module
    if _module is None:
        _module = _bfa.binding()
    return _module


def tree_depths(parents):
    """Edges from the root to each node, int32 of the shape of ``parents`` (0 at
    the root and at absent nodes, those under one among them): with the cached
    lengths as offsets, the rotary positions of the nodes. A parent outside
    -1 <= parents[n] < n makes its node absent, as in tree_attention, which
    reports it. Works on host tensors too; a fixed tree's depths are computed
    once."""
    n = parents.shape[-1]
    node = torch.arange(n, device=parents.device)
    # Node n is "no parent", above itself like the root.
    up = torch.where((parents >= 0) & (parents < node), parents, n).long()
    up = torch.nn.functional.pad(up, (0, 1), value=n)
    up[..., 0] = 0
    depth = torch.ones_like(up)
    depth[..., 0] = depth[..., n] = 0
    for _ in range((n - 1).bit_length()):  # each round doubles the climbed distance
        depth = depth + depth.gather(-1, up)
        up = up.gather(-1, up)
    return torch.where(up == 0, depth, 0)[..., :n].to(torch.int32)


def tree_attention(query, key, value, cache, parents=None, *, scale=None, sliding_window=0, soft_cap=0.0,
                   alibi_slope=None, return_lse=False):
    """Attention of a tree of drafted tokens: node n sees its sequence's cached
    tokens, itself and the nodes above it.

    query [B, Hq, N, D]; key, value [B, Hkv, N, D], the nodes' own K/V (not in
    the cache yet); cache: a PagedKVCache; parents: the tree (module docstring).
    ``scale``, ``sliding_window``, ``soft_cap`` and ``alibi_slope`` as in
    npu_flash_attention_forward, on absolute positions: with a window W, keys
    with position i - j <= W. N is 1 to 64, D up to 256, fp32 / fp16 / bf16; the
    probabilities are rounded to the input type for the product with V, as in
    the other forwards. Returns O like query (and the fp32 natural-log LSE [B,
    Hq, N]); rows of absent nodes give O = 0 and LSE = -inf. Not
    differentiable: a serving operator. Indices outside their tables are
    reported by ``check_device_status``.
    """
    if alibi_slope is not None and not isinstance(alibi_slope, torch.Tensor):
        alibi_slope = torch.as_tensor(alibi_slope, dtype=torch.float32)
    o, lse = _binding().tree_attention(query, key, value, cache[0], cache[1], cache[2], cache[3], parents, scale,
                                       sliding_window, soft_cap, alibi_slope, return_lse)
    if _CHECK_STATUS:
        check_device_status(query.device)
    return (o, lse) if return_lse else o


def verify_tree(target_probs, draft_tokens, parents, uniforms, noise, *, draft_probs=None):
    """Which drafted tokens stay, and the token after them, so that what is
    kept is distributed as the target's own tokens.

    target_probs [B, N, V]: row n is the target's distribution after node n
    (fp32 / fp16 / bf16, each row summing to 1). draft_tokens int32/int64
    [B, N]: the token of each node (the root's is not read). parents: the tree.
    uniforms fp32 [B, N] in [0, 1), noise fp32 [B, V] standard exponential draws
    (> 0): all randomness comes in here, so equal inputs give equal outputs.
    draft_probs [B, N, V] of the target's dtype: row n is the distribution from
    which the children of node n were drawn independently; None for candidates
    that are no draws (a draft's best tokens).

    From the root down, the children of the current node are tested in index
    order; the first accepted one becomes the current node, and where none is
    the next token is drawn from what the rejections left of the target's
    distribution (include/bfa.h has the formulas). Returns int32 tensors:
    path [B, N] (accepted nodes from the root, then -1), count [B] (the root
    among them) and next_token [B].
    """
    out = _binding().verify_tree(target_probs, draft_tokens, parents, uniforms, noise, draft_probs)
    if _CHECK_STATUS:
        check_device_status(target_probs.device)
    return out


def cache_append(cache, key, value, *, take=None, count=None):
    """Writes new tokens into the cache's pages, in place, and returns the new
    lengths (int32 [B]) in a tensor of their own: ``cache.lens`` keeps the old
    ones, so that every layer of a model appends at the same place.

    key, value [B, Hkv, S, D]. Sequence b appends its first count[b] tokens
    (``count`` int32 [B]; None: all S), or with ``take`` (int32 [B, S], a path of
    verify_tree) the tokens take[b, :count[b]] in that order. The page table
    must hold pages for them; a token past it, or with an index outside its
    table, is not written and is reported by ``check_device_status``. Not
    differentiable: inputs that require a gradient are refused.
    """
    out = _binding().cache_append(cache[0], cache[1], cache[2], cache[3], key, value, take, count)
    if _CHECK_STATUS:
        check_device_status(key.device)
    return out
