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

import math
from typing import NamedTuple

import torch

import bfa_lib as _bfa

__all__ = ["PagedKVCache", "tree_attention", "verify_tree", "cache_append", "tree_depths"]

MAX_NODES = 64


class PagedKVCache(NamedTuple):
    """K/V of cached tokens in pages: k_pages and v_pages [num_pages, Hkv,
    page_size, D], page_table int32 [B, max_pages], lens int32 [B]. Token t of
    sequence b lies in page page_table[b, t // page_size], slot t % page_size;
    table entries past a sequence's length are not read. The caller owns the
    tensors and hands out the pages."""
    k_pages: torch.Tensor
    v_pages: torch.Tensor
    page_table: torch.Tensor
    lens: torch.Tensor


def _check_cache(cache, B, Hkv, D, dtype, dev, what):
    kp, vp, table, lens = cache
    if kp.dim() != 4 or vp.shape != kp.shape or kp.shape[1] != Hkv or kp.shape[3] != D:
        raise ValueError(f"{what}: pages must be two [num_pages, {Hkv}, page_size, {D}] tensors, got {tuple(kp.shape)} "
                         f"and {tuple(vp.shape)}")
    if kp.dtype != dtype or vp.dtype != dtype:
        raise RuntimeError(f"{what}: pages must have the dtype of the new tokens, {dtype}")
    if kp.stride(3) != 1 or vp.stride(3) != 1:
        raise ValueError(f"{what}: pages need a unit innermost stride")
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != B or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"{what}: page_table must be int32 [{B}, max_pages] with unit inner stride")
    if lens.dtype != torch.int32 or tuple(lens.shape) != (B,) or (B > 1 and lens.stride(0) != 1):
        raise ValueError(f"{what}: lens must be a contiguous int32 [{B}]")
    _bfa.require_cuda(what, (kp, vp, table, lens), dev)


def _check_parents(parents, B, N, dev, what):
    """(pointer, row stride) of the tree; None is a chain."""
    if parents is None:
        return 0, 0
    if parents.dtype != torch.int32 or tuple(parents.shape) not in ((N,), (1, N), (B, N)) or (N > 1 and parents.stride(-1) != 1):
        raise ValueError(f"{what}: parents must be int32 [{N}] or [{B}, {N}] with unit inner stride, got "
                         f"{parents.dtype} {tuple(parents.shape)}")
    _bfa.require_cuda(what, (parents,), dev)
    return parents.data_ptr(), parents.stride(0) if parents.dim() == 2 and parents.shape[0] > 1 else 0


def _rows(t):
    """The kernels read rows of head_dim elements in place; other layouts are copied."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def tree_depths(parents):
    """Edges from the root to each node, int32 of the shape of ``parents`` (0 at
    the root and at absent nodes): with the cached lengths as offsets, the
    rotary positions of the nodes. Works on host tensors too; a fixed tree's
    depths are computed once."""
    n = parents.shape[-1]
    up = parents.long().clone()
    up[..., 0] = -1
    depth = torch.zeros_like(up)
    here = up
    for _ in range(n - 1):
        depth += here >= 0
        here = torch.where(here >= 0, up.gather(-1, here.clamp(min=0)), here)
    return depth.to(torch.int32)


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
    assert query.dim() == 4 and key.dim() == 4 and value.dim() == 4, "query, key and value are [B, H, N, D]"
    B, Hq, N, D = query.shape
    Hkv = key.shape[1]
    assert tuple(key.shape) == (B, Hkv, N, D) and value.shape == key.shape, "key and value must be [B, Hkv, N, D] of the query's B, N, D"
    assert Hkv > 0 and Hq % Hkv == 0, "Hq must be divisible by Hkv"
    if not 1 <= N <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {N}")
    if sliding_window < 0 or soft_cap < 0:
        raise ValueError("sliding_window and soft_cap must be >= 0")
    dt, dev = query.dtype, query.device
    if key.dtype != dt or value.dtype != dt:
        raise RuntimeError("query, key and value must have one dtype")
    _bfa.require_cuda("tree_attention", (query, key, value), dev)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        raise RuntimeError("tree_attention has no backward; call it under torch.no_grad()")
    _check_cache(cache, B, Hkv, D, dt, dev, "tree_attention")
    kp, vp, table, lens = cache
    up, up_stride = _check_parents(parents, B, N, dev, "tree_attention")
    slopes = None
    if alibi_slope is not None:
        slopes = torch.as_tensor(alibi_slope, dtype=torch.float32, device=dev).reshape(-1).contiguous()
        if slopes.numel() != Hq:
            raise RuntimeError(f"alibi_slope must have one slope per query head ({Hq}), got {slopes.numel()}")
    q, k, v = _rows(query), _rows(key), _rows(value)
    o = torch.empty((B, Hq, N, D), dtype=dt, device=dev)
    lse = torch.empty((B, Hq, N), dtype=torch.float32, device=dev) if return_lse else None
    sizes = (B, Hq, Hkv, N, D, _bfa.bfa_dtype(dt), kp.shape[0], kp.shape[2], table.shape[1], int(sliding_window),
             float(scale) if scale is not None else 1.0 / math.sqrt(D), float(soft_cap))
    # Scratch of the partial results, from torch's caching allocator: the library allocates nothing.
    nbytes = _bfa.tree_workspace_bytes(dev.index, *sizes)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _bfa.launch("bfa_tree_fwd", _bfa.pack_tree(
        *sizes, slopes.data_ptr() if slopes is not None else 0,
        *_bfa.flat(q), *_bfa.flat(k), *_bfa.flat(v), *_bfa.flat(o), lse.data_ptr() if return_lse else 0,
        *_bfa.flat(kp), *_bfa.flat(vp), table.data_ptr(), table.stride(0), lens.data_ptr(), up, up_stride,
        _bfa.status_ptr(dev), ws.data_ptr(), nbytes), dev)
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
    assert target_probs.dim() == 3, "target_probs is [B, N, V]"
    B, N, V = target_probs.shape
    dev = target_probs.device
    if not 1 <= N <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {N}")
    if V < 1:
        raise ValueError("the vocabulary is empty")
    if tuple(draft_tokens.shape) != (B, N):
        raise ValueError(f"draft_tokens must be [{B}, {N}], got {tuple(draft_tokens.shape)}")
    if draft_tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError("draft_tokens must be int32 or int64")
    if uniforms.dtype != torch.float32 or tuple(uniforms.shape) != (B, N) or noise.dtype != torch.float32 or tuple(noise.shape) != (B, V):
        raise ValueError(f"uniforms must be fp32 [{B}, {N}] and noise fp32 [{B}, {V}]")
    if draft_probs is not None and (draft_probs.shape != target_probs.shape or draft_probs.dtype != target_probs.dtype):
        raise ValueError("draft_probs must match target_probs in shape and dtype")
    _bfa.require_cuda("verify_tree", (target_probs, draft_tokens, uniforms, noise), dev)
    p = target_probs if target_probs.stride(2) == 1 or V == 1 else target_probs.contiguous()
    law = law_b = law_n = 0
    if draft_probs is not None:
        _bfa.require_cuda("verify_tree", (draft_probs,), dev)
        q = draft_probs if draft_probs.stride(2) == 1 or V == 1 else draft_probs.contiguous()
        law, law_b, law_n = q.data_ptr(), q.stride(0), q.stride(1)
    tokens, u, e = (t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous() for t in (draft_tokens, uniforms, noise))
    up, up_stride = _check_parents(parents, B, N, dev, "verify_tree")
    out = torch.empty(B * (N + 2), dtype=torch.int32, device=dev)
    path, count, token = out[:B * N].view(B, N), out[B * N:B * N + B], out[B * N + B:]
    at = out.data_ptr()
    packed = _bfa.pack_verify(
        B, N, V, _bfa.bfa_dtype(p.dtype), p.data_ptr(), p.stride(0), p.stride(1), law, law_b, law_n,
        tokens.data_ptr(), tokens.element_size(), tokens.stride(0), up, up_stride, u.data_ptr(), u.stride(0),
        e.data_ptr(), e.stride(0), at, at + 4 * B * N, at + 4 * B * (N + 1), _bfa.status_ptr(dev))
    _bfa.launch("bfa_verify_tree", packed, dev)
    return path, count, token


def cache_append(cache, key, value, *, take=None, count=None):
    """Writes new tokens into the cache's pages, in place, and returns the new
    lengths (int32 [B]) in a tensor of their own: ``cache.lens`` keeps the old
    ones, so that every layer of a model appends at the same place.

    key, value [B, Hkv, S, D]. Sequence b appends its first count[b] tokens
    (``count`` int32 [B]; None: all S), or with ``take`` (int32 [B, S], a path of
    verify_tree) the tokens take[b, :count[b]] in that order. The page table
    must hold pages for them; a token past it, or with an index outside its
    table, is not written and is reported by ``check_device_status``.
    """
    assert key.dim() == 4 and value.shape == key.shape, "key and value are [B, Hkv, S, D]"
    B, Hkv, S, D = key.shape
    dt, dev = key.dtype, key.device
    if value.dtype != dt:
        raise RuntimeError("key and value must have one dtype")
    _bfa.require_cuda("cache_append", (key, value), dev)
    _check_cache(cache, B, Hkv, D, dt, dev, "cache_append")
    kp, vp, table, lens = cache
    if take is not None:
        if take.dtype != torch.int32 or tuple(take.shape) != (B, S) or (S > 1 and take.stride(1) != 1):
            raise ValueError(f"take must be int32 [{B}, {S}] with unit inner stride")
        _bfa.require_cuda("cache_append", (take,), dev)
    if count is not None:
        if count.dtype != torch.int32 or tuple(count.shape) != (B,) or (B > 1 and count.stride(0) != 1):
            raise ValueError(f"count must be a contiguous int32 [{B}]")
        _bfa.require_cuda("cache_append", (count,), dev)
    out = torch.empty(B, dtype=torch.int32, device=dev)
    packed = _bfa.pack_append(
        B, Hkv, S, D, _bfa.bfa_dtype(dt), kp.shape[0], kp.shape[2], table.shape[1], *_bfa.flat(key.detach()),
        *_bfa.flat(value.detach()), *_bfa.flat(kp), *_bfa.flat(vp), table.data_ptr(), table.stride(0), lens.data_ptr(),
        take.data_ptr() if take is not None else 0, take.stride(0) if take is not None else 0,
        count.data_ptr() if count is not None else 0, out.data_ptr(), _bfa.status_ptr(dev))
    _bfa.launch("bfa_cache_append", packed, dev)
    return out
