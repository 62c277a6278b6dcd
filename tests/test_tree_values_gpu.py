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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("lens", [[3000], [20] * 170, [500, 0, 90]], ids=["split", "whole", "mixed"])
@pytest.mark.parametrize("N,Hq,D", [(5, 2, 64), (40, 2, 128), (64, 4, 128), (6, 2, 256)])
def test_logits_that_are_no_numbers_are_passed_on(dtype, bad, lens, N, Hq, D):
    """A query or a visible key that is not finite gives NaN in O and LSE of
    every row that sees it, whole or split over blocks, and leaves the others."""
    q, k, v, cache, parents, up = problem(lens, N, Hq, D, dtype, "binary", 24)
    ref = attention(q, k, v, cache, parents) if len(lens) < 10 else None
    clean = td.tree_attention(q, k, v, cache, up, return_lse=True)
    sees = torch.zeros(len(lens), Hq, N, dtype=torch.bool, device=DEV)
    q[0, 1, 3] = bad                                                   # one row
    sees[0, 1, 3] = True
    below = [n for n, way in enumerate(climb(parents[0])) if 2 in way]  # a node and those under it
    last = len(lens) - 1
    k[last, :, 2] = bad
    sees[last][:, below] = True
    if lens[0] > 100:                                                  # a cached key: all of a sequence's rows
        cache.k_pages[slot(cache, 0, lens[0] // 2)] = bad
        sees[0] = True
    o, lse = td.tree_attention(q, k, v, cache, up, return_lse=True)
    assert o[sees].isnan().all() and lse[sees].isnan().all()
    assert torch.equal(o[~sees], clean[0][~sees]) and torch.equal(lse[~sees], clean[1][~sees])
    if ref is not None:
        compare(o[~sees], lse[~sees], ref[0][~sees], ref[1][~sees], ref[2][~sees])
    nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("kw", [dict(soft_cap=20.0), dict(alibi=-0.1), dict(sliding_window=100)])
def test_logits_that_are_no_numbers_in_the_other_forms(dtype, kw):
    q, k, v, cache, parents, up = problem([1500, 30], 9, 2, 128, dtype, "binary", 25)
    kw = dict(kw)
    if "alibi" in kw:
        kw["alibi_slope"] = torch.tensor([1.0, 0.5], device=DEV) * kw.pop("alibi")
    clean = td.tree_attention(q, k, v, cache, up, return_lse=True, **kw)
    q[1, 0, 4] = math.nan
    cache.k_pages[slot(cache, 0, 1450)] = math.nan
    sees = torch.zeros(2, 2, 9, dtype=torch.bool, device=DEV)
    sees[1, 0, 4] = sees[0] = True
    o, lse = td.tree_attention(q, k, v, cache, up, return_lse=True, **kw)
    assert o[sees].isnan().all() and lse[sees].isnan().all()
    assert torch.equal(o[~sees], clean[0][~sees]) and torch.equal(lse[~sees], clean[1][~sees])


def same_values(o, ref):
    """NaN and the infinities lie where the definition has them."""
    for which in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(which(o), which(ref)), which.__name__


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("lens", [[1500], [20] * 170, [300, 70]], ids=["split", "whole", "mixed"])
@pytest.mark.parametrize("N,Hq,D,window", [(5, 2, 64, 0), (8, 4, 128, 0), (8, 4, 128, 60), (40, 2, 128, 0), (64, 4, 64, 0), (6, 2, 256, 0),
                                           (1, 1, 128, 0)])
def test_values_that_all_rows_see_are_summed(dtype, lens, N, Hq, D, window):
    """Infinite values of V give infinities of their sign in their own columns,
    NaN where both signs meet or V is NaN; the other columns keep their values."""
    q, k, v, cache, parents, up = problem(lens, N, Hq, D, dtype, "binary", 26)
    B = len(lens)
    some = list(range(B)) if B < 10 else [0, B - 1]
    clean = td.tree_attention(q, k, v, cache, up, sliding_window=window, return_lse=True)
    bad = [(11, math.inf), (13, -math.inf), (3, math.nan), (7, math.inf), (7, -math.inf), (20, math.inf), (20, math.inf)]
    for b in some:
        for i, (col, x) in enumerate(bad):
            page, every, at = slot(cache, b, lens[b] - 1 - (i * 37) % min(lens[b], window // 2 or lens[b]))
            cache.v_pages[page, every, at, col] = x
        v[b, :, 0, 30] = -math.inf
    sub = td.PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table[some], cache.lens[some])
    ref = attention(q[some], k[some], v[some], sub, [parents[b] for b in some], window=window)
    o, lse = td.tree_attention(q, k, v, cache, up, sliding_window=window, return_lse=True)
    same_values(o[some], ref[0])
    touched = torch.zeros(D, dtype=torch.bool, device=DEV)
    touched[[c for c, _ in bad] + [30]] = True
    compare(o[some][..., ~touched], lse[some], ref[0][..., ~touched], ref[1], ref[2][..., ~touched])
    others = [b for b in range(B) if b not in some]
    assert torch.equal(o[others], clean[0][others]) and torch.equal(lse, clean[1])
    nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
def test_infinite_values_with_a_cap_at_head_dim_256(dtype):
    q, k, v, cache, parents, up = problem([700, 90], 6, 2, 256, dtype, "binary", 27)
    cache.v_pages[slot(cache, 0, 400)] = math.inf
    v[1, :, 1, 200] = -math.inf
    ref = attention(q, k, v, cache, parents, cap=20.0)
    same_values(td.tree_attention(q, k, v, cache, up, soft_cap=20.0), ref[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("N,Hq,D,window", [(5, 2, 64, 40), (20, 1, 128, 200), (40, 2, 80, 33), (64, 4, 128, 1), (6, 2, 256, 300)])
def test_values_behind_the_window_do_not_spread(dtype, bad, N, Hq, D, window):
    """Cached tokens before the window, and inside it for the root alone, whose
    values are not finite: rows that do not see them keep theirs."""
    lens = [511, 200, 1]
    q, k, v, cache, parents, up = problem(lens, N, Hq, D, dtype, "chain", 28)
    ref = attention(q, k, v, cache, parents, window=window)
    keep = torch.ones(3, Hq, N, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        for at in (n - window - 1, n - window - 2, n - window - 20, n - window - 150, n - window):
            if 0 <= at < n:
                cache.v_pages[slot(cache, b, at)] = bad
        if n >= window:
            keep[b, :, 0] = False  # the root sees the last one of them
    o, lse = td.tree_attention(q, k, v, cache, up, sliding_window=window, return_lse=True)
    compare(o[keep], lse[keep], ref[0][keep], ref[1][keep], ref[2][keep])
    nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("N,window", [(1, 0), (2, 0), (2, 9)])
def test_infinite_values_in_many_short_sequences(dtype, N, window):
    """Several items to a block, each with columns of its own that are infinite."""
    B = 700
    lens = [20 + b % 3 for b in range(B)]
    q, k, v, cache, parents, up = problem(lens, N, 1, 64, dtype, "chain", 29)
    for b in range(0, B, 3 if N == 1 else 1):
        cache.v_pages[slot(cache, b, lens[b] - 3)[:3] + (b % 64,)] = math.inf if b % 2 else -math.inf
    ref = attention(q, k, v, cache, parents, window=window)
    o, lse = td.tree_attention(q, k, v, cache, up, sliding_window=window, return_lse=True)
    same_values(o, ref[0])
    fine = ref[0].isfinite()
    u = 2.0 ** -24 if dtype == FP else 2.0 ** -8
    tol = 1.5 * u * ref[2] + u * ref[0].abs() + 1e-4 * (ref[2] + 1)
    assert ((o.double() - ref[0]).abs() <= tol)[fine].all()
    assert ((lse.double() - ref[1]).abs() <= 1e-4 * (1 + ref[1].abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D", [64, 136])
@pytest.mark.parametrize("N,Hq", [(5, 1), (12, 2), (31, 4), (64, 4)])
def test_absent_rows_stay_empty_over_infinite_logits(dtype, D, N, Hq):
    """One infinite entry of an absent node's query makes its logits infinite,
    not NaN, over whole chunks of cached keys: the row is empty all the same."""
    q, k, v, cache, parents, up = problem([900, 22], N, Hq, D, dtype, "star", 30)
    up[:, 2:4] = -1
    for h, bad in enumerate([math.inf, -math.inf, math.inf, math.nan][:Hq]):
        q[:, h, 2, h], q[:, h, 3, D - 1] = bad, -bad
    ref = attention(q, k, v, cache, up.tolist())
    compare(*td.tree_attention(q, k, v, cache, up, return_lse=True), *ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("cap", [0.5, 5.0, 100.0])
@pytest.mark.parametrize("N,Hq,D", [(9, 2, 64), (40, 2, 128), (64, 4, 128), (6, 2, 256)])
def test_a_cap_passes_nan_on_and_bounds_infinities(dtype, cap, N, Hq, D):
    """NaN under the cap stays NaN, whichever form of tanh the logits beside it
    take; an infinite logit is a finite one there, plus or minus the cap."""
    q, k, v, cache, parents, up = problem([300, 50], N, Hq, D, dtype, "binary", 31)
    q.mul_(3)
    q[0, 0, 2] = math.nan
    k[1, :, 1] = math.nan
    q[1, 1, 3, 5] = math.inf                   # infinite logits of both signs
    cache.k_pages[slot(cache, 0, 77)][:, 0] = -math.inf
    ref = attention(q, k, v, cache, parents, cap=cap)
    o, lse = td.tree_attention(q, k, v, cache, up, soft_cap=cap, return_lse=True)
    bad = ref[1].isnan()
    assert bad[0, 0, 2] and bad[1, :, 1].all() and not bad[0, 1].any()
    assert o[bad].isnan().all() and lse[bad].isnan().all()
    # Of the cap of 100 an fp32 tanh keeps 1e-7·100 in the logits.
    compare(o[~bad], lse[~bad], ref[0][~bad], ref[1][~bad], ref[2][~bad])
