"""Tree attention where keys or values are not finite, against a 64-bit
restatement: they reach the rows that see them and no other. Tolerances as in
test_tree_decoding_gpu.py."""
import math

import pytest
import torch

import npu_flash_attention as nfa
import tree_decoding as td
from test_tree_decoding_gpu import BF, DEV, FP, HF, compare, gen, kernel, tree  # noqa: F401 (kernel: both 16-bit kernels)
from tree_reference import attention, climb, page_cache

BAD = [float("nan"), float("inf"), -float("inf")]


def problem(lens, N, Hq, D, dtype, kind, seed, page=16):
    """(q, k, v, cache, parents as lists, parents on the device), one KV head."""
    g = gen(seed)
    cache = td.PagedKVCache(*page_cache(lens, max(lens), page, 1, D, dtype, DEV, g))
    q, k, v = (torch.randn(len(lens), h, N, D, generator=g, device=DEV).to(dtype) for h in (Hq, 1, 1))
    parents = tree(kind, N, len(lens))
    return q, k, v, cache, parents, torch.tensor(parents, dtype=torch.int32, device=DEV)


def slot(cache, b, t):
    """Index of sequence b's cached token t in the pages."""
    page = cache.k_pages.shape[2]
    return int(cache.page_table[b, t // page]), slice(None), t % page


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("N,Hq,D", [(12, 2, 64), (12, 2, 128), (40, 2, 64), (40, 3, 128), (20, 4, 256), (64, 4, 128)])
def test_bad_nodes_after_whole_chunks(dtype, bad, N, Hq, D):
    """O is added to by hand for such a node while the products of the chunks
    before it are only just formed: no key of theirs is lost, in a node's row
    or in its siblings'."""
    lens = [1100, 640, 3000]
    q, k, v, cache, parents, up = problem(lens, N, Hq, D, dtype, "star", 21)
    ref = attention(q, k, v, cache, parents)
    for b in range(len(lens)):
        k[b, :, 3 + b], v[b, :, 3 + b], v[b, :, N - 1] = bad, bad, bad
    keep = torch.ones(N, dtype=torch.bool, device=DEV).repeat(len(lens), Hq, 1)
    for b in range(len(lens)):
        keep[b, :, 3 + b] = keep[b, :, N - 1] = False
    for _ in range(3):
        o, lse = td.tree_attention(q, k, v, cache, up, return_lse=True)
        compare(o[keep], lse[keep], ref[0][keep], ref[1][keep], ref[2][keep])
    nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("N,Hq,D", [(20, 1, 64), (20, 1, 128), (40, 3, 128), (20, 4, 256), (64, 4, 64)])
@pytest.mark.parametrize("window", [150, 301, 700])
def test_bad_cached_values_at_the_windows_edge(dtype, bad, N, Hq, D, window):
    """A cached token that the root sees and deeper nodes do not, with whole
    chunks, or one, or none between it and the tree."""
    lens = [1111, 333]
    q, k, v, cache, parents, up = problem(lens, N, Hq, D, dtype, "chain", 22)
    ref = attention(q, k, v, cache, parents, window=window)
    keep = torch.ones(len(lens), Hq, N, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        at = n - window + 7
        if at < 0:
            continue
        cache.k_pages[slot(cache, b, at)] = bad
        cache.v_pages[slot(cache, b, at)] = bad
        depth = torch.tensor([len(w) - 1 for w in climb(parents[b])], device=DEV)
        keep[b] &= (n + depth - at > window)[None]
    for _ in range(3):
        o, lse = td.tree_attention(q, k, v, cache, up, sliding_window=window, return_lse=True)
        compare(o[keep], lse[keep], ref[0][keep], ref[1][keep], ref[2][keep])
    nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N,Hq,D,window", [(20, 1, 64, 200), (20, 1, 128, 200), (40, 3, 128, 200), (64, 4, 128, 200), (20, 4, 256, 100)])
def test_bad_values_two_chunks_apart(dtype, N, Hq, D, window):
    """The window's edge and the tree hold them, the whole chunk between does
    not: each chunk's own are found, none left over from the other."""
    n = 1152  # whole chunks: the window's first one, one that every row sees, the tree
    q, k, v, cache, parents, up = problem([n] * 3, N, Hq, D, dtype, "chain", 23)
    ref = attention(q, k, v, cache, parents, window=window)
    keep = torch.ones(3, Hq, N, dtype=torch.bool, device=DEV)
    depth = torch.arange(N, device=DEV)
    for b in range(3):
        at = n - window + 3 + b
        if b != 1:
            cache.v_pages[slot(cache, b, at)] = math.nan
            keep[b] &= (n + depth - at > window)[None]
        if b != 2:
            v[b, :, N - 2 + b] = math.inf
            keep[b] &= (depth < N - 2 + b)[None]
    for _ in range(3):
        o, lse = td.tree_attention(q, k, v, cache, up, sliding_window=window, return_lse=True)
        compare(o[keep], lse[keep], ref[0][keep], ref[1][keep], ref[2][keep])
    nfa.check_device_status(DEV)
