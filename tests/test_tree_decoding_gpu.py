"""Tree attention over a paged cache, draft verification and cache append on
the GPU against 64-bit restatements.

Attention tolerance, from the arithmetic: probabilities rounded to the input
type for the product with V (u·sum p|v|, u the type's unit roundoff), the
result rounded once (u·|o|), and the fp32 logits: a dot product of D <= 256
terms of size ~1 carries at most D·2^-24·sum|q||k|·scale, typically below 2e-5,
which moves p by as much, relatively. Together 1.5·u·S + u·|o| + 1e-4·(S + 1)
with S = sum p|v|; the LSE 1e-4·(1 + |lse|)."""
import math

import pytest
import torch

import npu_flash_attention as nfa
import tree_decoding as td
from tree_reference import attention, dense, page_cache, verify

DEV = "cuda:0"


@pytest.fixture(params=["", "0"], ids=["tcgen05", "mma"], autouse=True)
def kernel(request, monkeypatch):
    """Attention tests run on the kernel that the library chooses (tcgen05
    wherever TMA can read the layouts) and on the mma.sync kernel."""
    name = request.node.name
    if request.param and ("verify" in name or "append" in name or "refusals" in name):
        pytest.skip("one kernel")
    if request.param:
        monkeypatch.setenv("BFA_TREE_TCGEN05", request.param)


U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def tree(kind, N, B=1):
    row = {"chain": [-1] + list(range(N - 1)), "binary": [-1] + [(n - 1) // 2 for n in range(1, N)],
           "star": [-1] + [0] * (N - 1)}[kind]
    return [list(row) for _ in range(B)]


def check(lens, N, Hq, Hkv, D, dtype, page, parents, capacity=None, seed=0, peak=1.0, poison=float("nan"), **kw):
    g = gen(seed)
    B = len(lens)
    cache = td.PagedKVCache(*page_cache(lens, capacity or max(lens), page, Hkv, D, dtype, DEV, g, poison=poison))
    q = (torch.randn(B, Hq, N, D, generator=g, device=DEV) * peak).to(dtype)
    k, v = (torch.randn(B, Hkv, N, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    up = torch.tensor(parents, dtype=torch.int32, device=DEV) if parents is not None else None
    o, lse = td.tree_attention(q, k, v, cache, up, return_lse=True, **kw)
    ref_kw = dict(scale=kw.get("scale"), window=kw.get("sliding_window", 0), cap=kw.get("soft_cap", 0.0), slopes=kw.get("alibi_slope"))
    ro, rl, size = attention(q, k, v, cache, parents if parents is not None else tree("chain", N, B), **ref_kw)
    compare(o, lse, ro, rl, size)
    nfa.check_device_status(DEV)
    return o


def compare(o, lse, ro, rl, size):
    u = U[o.dtype]
    tol = 1.5 * u * size + u * ro.abs() + 1e-4 * (size + 1)
    err = (o.double() - ro).abs()
    assert (err <= tol).all(), f"O off by {err.max().item():.3g} (tolerance there {tol.flatten()[err.argmax()].item():.3g})"
    empty = rl == -math.inf
    assert (lse[empty] == -math.inf).all() and (o[empty] == 0).all()
    assert ((lse.double() - rl).abs()[~empty] <= 1e-4 * (1 + rl.abs()[~empty])).all()


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("lens,N,Hq,Hkv,D,page,kind", [
    ([1], 1, 1, 1, 64, 16, "chain"), ([0], 1, 2, 1, 128, 16, "chain"), ([0, 5, 0], 7, 4, 2, 64, 8, "binary"),
    ([63, 64, 65, 128], 5, 8, 2, 128, 16, "binary"), ([300, 1, 1000], 16, 8, 8, 128, 64, "star"),
    ([777], 64, 2, 1, 64, 48, "chain"), ([500, 130], 33, 16, 2, 128, 128, "binary"), ([257, 31], 64, 8, 1, 128, 1, "binary"),
    ([200, 90], 9, 4, 4, 256, 32, "binary"), ([600], 24, 8, 1, 256, 64, "star"), ([100, 333], 6, 6, 3, 80, 24, "binary"),
    ([100, 40], 3, 2, 2, 33, 7, "binary"), ([50], 2, 3, 1, 1, 4, "chain"), ([2100], 40, 10, 1, 64, 256, "binary")])
def test_sizes(dtype, lens, N, Hq, Hkv, D, page, kind):
    check(lens, N, Hq, Hkv, D, dtype, page, tree(kind, N, len(lens)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("kw", [dict(sliding_window=1), dict(sliding_window=40), dict(sliding_window=5000), dict(soft_cap=5.0),
                                dict(scale=0.3), dict(alibi=-0.1), dict(alibi=0.05), dict(alibi=0.2, sliding_window=70, soft_cap=20.0),
                                dict(alibi=-1.0, sliding_window=3)])
@pytest.mark.parametrize("D,N,Hq", [(128, 13, 4), (64, 40, 8), (256, 5, 4)])
def test_masks_and_logits(dtype, kw, D, N, Hq):
    kw = dict(kw)
    if "alibi" in kw:
        kw["alibi_slope"] = torch.linspace(0.25, 1.0, Hq, device=DEV) * kw.pop("alibi")
    check([300, 20, 0], N, Hq, 2, D, dtype, 16, tree("binary", N, 3), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("N", [9, 40, 64])
def test_absent_nodes_give_empty_rows(dtype, N):
    """Absent nodes, and nodes under them, give O = 0 and LSE = -inf; their own
    K/V (NaN here) reach no other row."""
    g = gen(5)
    lens = [130, 0, 64]
    parents = tree("binary", N, 3)
    parents[0][3] = -1               # with its subtree
    parents[1][1:] = [-1] * (N - 1)  # the root alone, over an empty cache
    parents[2][N // 2:] = [-1] * (N - N // 2)
    cache = td.PagedKVCache(*page_cache(lens, 200, 16, 2, 64, dtype, DEV, g))
    q, k, v = (torch.randn(3, h, N, 64, generator=g, device=DEV).to(dtype) for h in (4, 2, 2))
    ref = attention(q, k, v, cache, parents)
    gone = ref[1] == -math.inf
    assert gone[0, 0, 3] and gone[0, 0, 7] and gone[1, 0, 1:].all()
    up = torch.tensor(parents, dtype=torch.int32, device=DEV)
    compare(*td.tree_attention(q, k, v, cache, up, return_lse=True), *ref)
    for t in (k, v):
        t.masked_fill_(gone[:, :1, :, None], float("nan"))
    q.masked_fill_(gone[:, :, :, None], float("inf"))
    o, lse = td.tree_attention(q, k, v, cache, torch.tensor(parents, dtype=torch.int32, device=DEV), return_lse=True)
    compare(o, lse, *ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("N,Hq", [(12, 2), (40, 2), (64, 8)])
def test_values_of_unseen_nodes_do_not_spread(dtype, bad, N, Hq):
    """A node whose K/V is not finite spoils itself and the nodes under it, and
    no row that does not see it."""
    g = gen(8)
    parents = tree("star", N, 2)
    parents[1] = tree("binary", N)[0]
    cache = td.PagedKVCache(*page_cache([70, 200], 200, 16, 1, 128, dtype, DEV, g))
    q, k, v = (torch.randn(2, h, N, 128, generator=g, device=DEV).to(dtype) for h in (Hq, 1, 1))
    ref = attention(q, k, v, cache, parents)
    hit = [5, 2]
    for b in range(2):
        k[b, :, hit[b]], v[b, :, hit[b]] = bad, bad
    sees = torch.tensor([[hit[b] in way for way in __import__("tree_reference").climb(parents[b])] for b in range(2)], device=DEV)
    o, lse = td.tree_attention(q, k, v, cache, torch.tensor(parents, dtype=torch.int32, device=DEV), return_lse=True)
    keep = ~sees[:, None, :].expand(-1, Hq, -1)
    compare(o[keep], lse[keep], ref[0][keep], ref[1][keep], ref[2][keep])


@pytest.mark.gpu
def test_chain_is_the_causal_forward():
    """None and [-1, 0, 1, ...] are a chain: the last rows of a causal forward."""
    g = gen(2)
    L, N = 150, 6
    q, k, v = (torch.randn(1, h, L + N, 128, generator=g, device=DEV).to(BF) for h in (8, 2, 2))
    want = nfa.npu_flash_attention_forward(q[:, :, L:], k, v, causal=True, q_pos_offset=L)
    kp, vp = (torch.nn.functional.pad(x[0], (0, 0, 0, 4)).reshape(2, 10, 16, 128).transpose(0, 1).contiguous() for x in (k, v))
    cache = td.PagedKVCache(kp, vp, torch.arange(10, dtype=torch.int32, device=DEV)[None], torch.tensor([L], dtype=torch.int32, device=DEV))
    for parents in (None, torch.tensor([-1, 0, 1, 2, 3, 4], dtype=torch.int32, device=DEV)):
        o = td.tree_attention(q[:, :, L:], k[:, :, L:], v[:, :, L:], cache, parents)
        # Two roundings of P and of O apart.
        assert (o.float() - want.float()).abs().max() < 4 * 2 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("N,Hq", [(5, 4), (64, 8)])
def test_layouts(dtype, N, Hq):
    """q/k/v as transposed views and with a strided innermost dim, pages inside a
    larger allocation (every second head of a wider one, odd element offsets),
    a table with a row stride."""
    g = gen(4)
    lens = [100, 37]
    kp, vp, table, ln = page_cache(lens, 128, 16, 2, 64, dtype, DEV, g)
    q, k, v = (torch.randn(2, N, h, 64, generator=g, device=DEV).to(dtype).transpose(1, 2) for h in (Hq, 2, 2))
    parents = tree("binary", N, 2)
    up = torch.tensor(parents, dtype=torch.int32, device=DEV)
    ref = attention(q, k, v, (kp, vp, table, ln), parents)

    def run(kp, vp, table, q=q, k=k, v=v, up=up):
        compare(*td.tree_attention(q, k, v, td.PagedKVCache(kp, vp, table, ln), up, return_lse=True), *ref)
    run(kp, vp, table)
    wide = torch.full((kp.shape[0], 4, 16, 64), float("nan"), dtype=dtype, device=DEV)
    wide[:, ::2] = kp
    run(wide[:, ::2], vp, table)
    flat = torch.empty(kp.numel() + 3, dtype=dtype, device=DEV)  # rows off the 16-byte grid
    odd = flat[3:].view(kp.shape)
    odd.copy_(vp)
    run(kp, odd, table)
    seq_major = kp.transpose(1, 2).contiguous().transpose(1, 2)  # [pages, slot, head, D] in memory
    run(seq_major, vp, table)
    wt = torch.full((2, 2 * table.shape[1]), -7, dtype=torch.int32, device=DEV)
    wt[:, :table.shape[1]] = table
    run(kp, vp, wt[:, :table.shape[1]])
    strided = torch.empty(2, Hq, N, 128, dtype=dtype, device=DEV)[..., ::2]
    run(kp, vp, table, q=strided.copy_(q))
    run(kp, vp, table, up=up[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_mixed_lengths_and_many_sequences(dtype):
    """More sequences than a warp has lanes, lengths from 0 on; grids larger and
    smaller than the work."""
    lens = [(37 * i) % 211 for i in range(70)]
    check(lens, 3, 2, 1, 64, dtype, 16, tree("binary", 3, 70), capacity=4000)
    check([3], 1, 1, 1, 64, dtype, 16, None, capacity=100000)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [8, 24, 40, 64, 192, 256])
@pytest.mark.parametrize("D,N,Hq", [(128, 4, 4), (64, 20, 8), (256, 6, 2)])
def test_page_sizes_and_windows(page, D, N, Hq):
    """Pages smaller and larger than a chunk of keys, that divide it and that do
    not, windows that begin inside a page, lengths that end inside one."""
    check([1300, 257, 40], N, Hq, 1, D, BF, page, tree("binary", N, 3))
    check([1300, 257, 40], N, Hq, 1, D, BF, page, tree("chain", N, 3), sliding_window=301)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kw", [dict(), dict(soft_cap=20.0)])
def test_row_counts_around_the_tiles(D, kw):
    """Rows per KV head at and around 32, 128 and 256, where the tile changes."""
    for N, G in ((32, 1), (33, 1), (31, 4), (32, 4), (43, 3), (64, 4), (52, 5)):
        check([400, 70], N, G, 1, D, BF, 16, tree("binary", N, 2), seed=N * G, **kw)


@pytest.mark.gpu
def test_values_at_the_types_ends():
    """Keys and queries whose logits reach +-10^4, an fp16 cache near its
    largest value, and a soft-cap over them."""
    g = gen(12)
    for dtype, size in ((BF, 30.0), (HF, 30.0)):
        cache = td.PagedKVCache(*page_cache([300], 320, 16, 1, 128, dtype, DEV, g))
        cache.k_pages.mul_(size)
        q = (torch.randn(1, 4, 5, 128, generator=g, device=DEV) * size).to(dtype)
        k, v = (torch.randn(1, 1, 5, 128, generator=g, device=DEV).to(dtype) for _ in range(2))
        parents = tree("binary", 5)
        up = torch.tensor(parents, dtype=torch.int32, device=DEV)
        for cap in (0.0, 50.0):
            ro, rl, size_ = attention(q, k, v, cache, parents, cap=cap)
            o, lse = td.tree_attention(q, k, v, cache, up, soft_cap=cap, return_lse=True)
            # Logits near 10^4 carry an fp32 error of a few 2^-10, which moves
            # probabilities by as much; with the cap at most 50 * 1e-5.
            tol = 1.5 * U[dtype] * size_ + U[dtype] * ro.abs() + (2e-2 if cap == 0.0 else 1e-3) * (size_ + 1)
            assert ((o.double() - ro).abs() <= tol).all()
            assert ((lse.double() - rl).abs() <= 1e-5 * (1 + rl.abs()) + 1e-3).all()


@pytest.mark.gpu
def test_long_cache_and_peaked_rows():
    check([20011], 17, 4, 1, 128, BF, 64, tree("binary", 17), peak=3.0)
    check([9001], 64, 4, 1, 128, HF, 64, tree("binary", 64), peak=3.0)
    check([5003], 9, 4, 1, 64, FP, 64, tree("binary", 9), peak=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("N,Hq", [(4, 4), (64, 4)])
def test_offsets_past_32_bits(N, Hq):
    """Pages whose element offsets pass 2^31."""
    pages, page, H, D = 66000, 64, 4, 128
    big = torch.empty(pages, H, page, D, dtype=BF, device=DEV)  # 2.2e9 elements
    g = gen(11)
    ids = torch.tensor([[65999, 3, 65536, 65990]], dtype=torch.int32, device=DEV)
    big[ids[0].long()] = torch.randn(4, H, page, D, generator=g, device=DEV).to(BF)
    ln = torch.tensor([250], dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(1, h, N, D, generator=g, device=DEV).to(BF) for h in (Hq, H, H))
    parents = tree("binary", N)
    cache = td.PagedKVCache(big, big, ids, ln)
    up = torch.tensor(parents, dtype=torch.int32, device=DEV)
    compare(*td.tree_attention(q, k, v, cache, up, return_lse=True), *attention(q, k, v, cache, parents))
    out = td.cache_append(cache, k[:, :, :3], v[:, :, :3])
    assert out.tolist() == [253] and torch.equal(big[65990, :, 58:61], v[0, :, :3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N,Hq,D", [(BF, 7, 8, 128), (BF, 48, 8, 128), (HF, 9, 4, 256), (FP, 7, 8, 128)])
def test_repeats_bitwise_and_on_another_stream(dtype, N, Hq, D):
    g = gen(6)
    lens = [1500, 20, 333]
    cache = td.PagedKVCache(*page_cache(lens, 1600, 16, 2, D, dtype, DEV, g))
    q, k, v = (torch.randn(3, h, N, D, generator=g, device=DEV).to(dtype) for h in (Hq, 2, 2))
    up = torch.tensor(tree("binary", N, 3), dtype=torch.int32, device=DEV)
    first = td.tree_attention(q, k, v, cache, up, return_lse=True)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for _ in range(5):
            again = td.tree_attention(q, k, v, cache, up, return_lse=True)
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.gpu
def test_bad_indices_are_reported():
    g = gen(7)
    kp, vp, table, ln = page_cache([100, 40], 112, 16, 1, 64, BF, DEV, g, poison=0.0)
    q, k, v = (torch.randn(2, 1, 4, 64, generator=g, device=DEV).to(BF) for _ in range(3))
    good = torch.tensor(tree("chain", 4, 2), dtype=torch.int32, device=DEV)
    nfa.check_device_status(DEV)

    def bad(cache, up=good):
        td.tree_attention(q, k, v, cache, up)
        with pytest.raises(RuntimeError, match="outside its table"):
            nfa.check_device_status(DEV)
    for page in (-1, kp.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 2] = page
        bad(td.PagedKVCache(kp, vp, t, ln))
    for n in (-1, 113, 2 ** 31 - 1):
        bad(td.PagedKVCache(kp, vp, table, torch.tensor([100, n], dtype=torch.int32, device=DEV)))
    for up in (3, 2, -2):  # not below its own index (node 2), or under -1
        t = good.clone()
        t[1, 2] = up
        bad(td.PagedKVCache(kp, vp, table, ln), t)
    td.tree_attention(q, k, v, td.PagedKVCache(kp, vp, table, ln), good)
    nfa.check_device_status(DEV)


@pytest.mark.gpu
def test_attention_refusals():
    g = gen(1)
    cache = td.PagedKVCache(*page_cache([10], 16, 16, 2, 64, BF, DEV, g))
    q, k, v = (torch.randn(1, h, 3, 64, generator=g, device=DEV).to(BF) for h in (4, 2, 2))
    td.tree_attention(q, k, v, cache)
    with pytest.raises(AssertionError, match="Hq"):
        td.tree_attention(q[:, :3], k, v, cache)
    with pytest.raises(AssertionError):
        td.tree_attention(q, k[:, :, :2], v, cache)
    with pytest.raises(ValueError, match="nodes"):
        td.tree_attention(q[:, :, :0], k[:, :, :0], v[:, :, :0], cache)
    big = [torch.zeros(1, h, 65, 64, device=DEV, dtype=BF) for h in (4, 2, 2)]
    with pytest.raises(ValueError, match="nodes"):
        td.tree_attention(*big, cache)
    with pytest.raises(RuntimeError, match="dtype"):
        td.tree_attention(q.half(), k.half(), v.half(), cache)
    with pytest.raises(ValueError, match="pages"):
        td.tree_attention(q, k, v, cache._replace(v_pages=cache.v_pages[..., :32]))
    with pytest.raises(ValueError, match="page_table"):
        td.tree_attention(q, k, v, cache._replace(page_table=cache.page_table.long()))
    with pytest.raises(ValueError, match="lens"):
        td.tree_attention(q, k, v, cache._replace(lens=cache.lens.long()))
    with pytest.raises(ValueError, match="parents"):
        td.tree_attention(q, k, v, cache, torch.zeros(4, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="share a device|CUDA"):
        td.tree_attention(q, k, v, cache, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="slope"):
        td.tree_attention(q, k, v, cache, alibi_slope=torch.ones(3, device=DEV))
    with pytest.raises(ValueError):
        td.tree_attention(q, k, v, cache, sliding_window=-1)
    with pytest.raises(RuntimeError, match="no backward"):
        td.tree_attention(q.clone().requires_grad_(True), k, v, cache)
    zero = [torch.zeros(0, h, 3, 64, device=DEV, dtype=BF) for h in (4, 2, 2)]
    none = td.PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table[:0], cache.lens[:0])
    assert td.tree_attention(*zero, none).shape == (0, 4, 3, 64)


# ------------------------------------------------------------------ verify
def draws(B, N, V, dtype, parents, drafted, seed, sharp=3.0, near=0.7):
    g = gen(seed)
    logits = torch.randn(B, N, V, generator=g, device=DEV) * sharp
    p = torch.softmax(logits, -1).to(dtype)
    q = torch.softmax(logits + near * torch.randn(B, N, V, generator=g, device=DEV), -1).to(dtype)
    up = torch.tensor(parents, device=DEV).clamp(min=0)
    rows = torch.arange(B, device=DEV)[:, None]
    if drafted:
        e = torch.empty(B, N, V, device=DEV).exponential_(generator=g).clamp_(min=1e-20)
        tokens = (q.float()[rows, up] / e).argmax(-1)
    else:
        best = q.float().topk(min(V, N), -1).indices
        rank = torch.tensor([[sum(1 for m in range(1, n) if row[m] == row[n]) for n in range(N)] for row in parents], device=DEV)
        tokens = best[rows, up, rank.clamp(max=best.shape[-1] - 1)]
    u = torch.rand(B, N, generator=g, device=DEV)
    noise = torch.empty(B, V, device=DEV).exponential_(generator=g).clamp_(min=1e-20)
    return p, q if drafted else None, tokens, u, noise


def check_verify(p, q, tokens, u, noise, parents, up=None):
    B, N = tokens.shape
    if up is None:
        up = torch.tensor(parents, dtype=torch.int32, device=DEV)
    path, count, token = td.verify_tree(p, tokens, up, u, noise, draft_probs=q)
    for b in range(B):
        want, nxt = verify(p[b], tokens[b].tolist(), parents[b], u[b], noise[b], q[b] if q is not None else None)
        assert path[b].tolist() == want + [-1] * (N - len(want)) and int(count[b]) == len(want), b
        assert int(token[b]) == nxt, b
    return count


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("B,N,V,kind", [(1, 1, 5, "chain"), (3, 2, 1, "chain"), (2, 5, 1001, "chain"), (5, 64, 4096, "chain"),
                                        (7, 31, 2000, "binary"), (4, 64, 333, "star"), (3, 9, 40000, "binary"),
                                        (200, 6, 5000, "star"), (1, 12, 100003, "star")])
def test_verify(dtype, drafted, B, N, V, kind):
    parents = tree(kind, N, B)
    for b in range(0, B, 3):
        for n in range(max(1, (2 * N) // 3), N):
            parents[b][n] = -1
    counts = check_verify(*draws(B, N, V, dtype, parents, drafted, seed=B * 1000 + N), parents)
    nfa.check_device_status(DEV)
    if B == 200:
        assert counts.float().std() > 0  # some are accepted, some are not


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
def test_verify_many_rejections(drafted):
    """Stars of unlikely candidates: many rejections at one node, repeated tokens among them."""
    B, N, V = 12, 24, 5001
    parents = tree("star", N, B)
    p, q, tokens, u, noise = draws(B, N, V, FP, parents, drafted, 3, sharp=1.0, near=3.0)
    if not drafted:
        tokens = p[:, 0].topk(N, -1, largest=False).indices
        tokens[:, N // 2:] = tokens[:, :N - N // 2]
    counts = check_verify(p, q, tokens, u, noise, parents)
    assert (counts == 1).any()


@pytest.mark.gpu
def test_verify_edges():
    V = 4096
    parents = tree("chain", 4)
    g = gen(3)
    p = torch.softmax(torch.randn(1, 4, V, generator=g, device=DEV), -1)
    tokens = torch.tensor([[0, 5, 6, 7]], device=DEV)
    noise = torch.ones(1, V, device=DEV)
    half = torch.full((1, 4), 0.5, device=DEV)
    # The draft equals the target: everything is accepted.
    assert check_verify(p, p, tokens, half, noise, parents).item() == 4
    # A one-hot target (greedy decoding) keeps exactly the matching prefix.
    hot = torch.zeros(1, 4, V, device=DEV)
    for n, x in enumerate((5, 6, 9, 1)):
        hot[0, n, x] = 1.0
    assert check_verify(hot, None, tokens, half, noise, parents).item() == 3
    # A rejection by rounding alone leaves an empty residual: drawn from p.
    same = torch.zeros(1, 4, V, device=DEV)
    same[..., 11] = 1.0
    path, count, token = td.verify_tree(same, torch.full((1, 4), 11, device=DEV), torch.tensor(parents, dtype=torch.int32, device=DEV),
                                        torch.ones(1, 4, device=DEV), noise, draft_probs=same)
    assert count.item() == 1 and token.item() == 11
    # Ties go to the lowest index.
    flat = torch.full((1, 4, V), 1.0 / V, device=DEV)
    assert td.verify_tree(flat, tokens, None, torch.ones(1, 4, device=DEV), noise)[2].item() == 0
    # int32 tokens, a broadcast tree, strided rows.
    wide = torch.zeros(1, 8, V, device=DEV)
    wide[:, ::2] = p
    up = torch.tensor(parents[0], dtype=torch.int32, device=DEV)
    check_verify(wide[:, ::2], None, tokens.to(torch.int32), half, noise, parents, up)


@pytest.mark.gpu
def test_verify_draws_follow_the_target():
    """Kept tokens follow the target's law: over 20000 sequences that share p
    and q, the first token after the root (accepted child or next token) has
    frequencies within 5 standard deviations of p."""
    B, V = 20000, 8
    g = gen(1)
    p1 = torch.softmax(torch.randn(V, generator=g, device=DEV) * 1.5, -1)
    q1 = torch.softmax(torch.randn(V, generator=g, device=DEV) * 1.5, -1)
    p, q = (x.expand(B, 4, V).contiguous() for x in (p1, q1))
    u = torch.rand(B, 4, generator=g, device=DEV)
    noise = torch.empty(B, V, device=DEV).exponential_(generator=g).clamp_(min=1e-20)
    up = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=DEV)
    drawn = torch.multinomial(q1.expand(B, V), 4, replacement=True, generator=g)
    fixed = torch.tensor([0, 3, 1, 6], device=DEV).expand(B, 4).contiguous()
    for tokens, law in ((drawn, q), (fixed, None)):
        path, count, token = td.verify_tree(p, tokens, up, u, noise, draft_probs=law)
        first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token.long())
        freq = torch.bincount(first, minlength=V).double() / B
        pd = p1.double()
        assert ((freq - pd).abs() <= 5 * (pd * (1 - pd) / B).sqrt()).all()


@pytest.mark.gpu
def test_verify_refusals_and_bad_tokens():
    p = torch.full((2, 3, 10), 0.1, device=DEV)
    tokens, u, noise = torch.zeros(2, 3, dtype=torch.int64, device=DEV), torch.rand(2, 3, device=DEV), torch.ones(2, 10, device=DEV)
    nfa.check_device_status(DEV)
    for bad in (-1, 10, 2 ** 40):
        t = tokens.clone()
        t[1, 1] = bad
        _, count, _ = td.verify_tree(p, t, None, u, noise)
        assert count[1].item() == 1
        with pytest.raises(RuntimeError, match="outside its table"):
            nfa.check_device_status(DEV)
    for args in ((p, tokens[:, :2], None, u, noise), (p, tokens.float(), None, u, noise), (p, tokens, None, u.double(), noise),
                 (p, tokens, None, u, noise[:, :9]), (torch.zeros(2, 65, 4, device=DEV), tokens, None, u, noise),
                 (p, tokens, torch.zeros(2, dtype=torch.int32, device=DEV), u, noise)):
        with pytest.raises(ValueError):
            td.verify_tree(*args)
    with pytest.raises(ValueError):
        td.verify_tree(p, tokens, None, u, noise, draft_probs=p.half())
    with pytest.raises(RuntimeError):
        td.verify_tree(p, tokens.cpu(), None, u, noise)
    assert td.verify_tree(p[:0], tokens[:0], None, u[:0], noise[:0])[0].shape == (0, 3)


# ------------------------------------------------------------------ append
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,S,H,D,page,take", [([0], 1, 1, 64, 16, False), ([0, 5, 15, 16], 40, 2, 128, 16, False),
                                                  ([3, 100], 7, 8, 80, 24, True), ([60, 1, 0], 64, 3, 33, 7, True),
                                                  ([0, 10], 3000, 8, 128, 64, False)])
def test_append(dtype, lens, S, H, D, page, take):
    g = gen(2)
    B = len(lens)
    cap = max(lens) + S
    kp, vp, table, ln = page_cache(lens, cap, page, H, D, dtype, DEV, g, extra_pages=B * (S // page + 2))
    used = set(table[table >= 0].tolist())
    free = [i for i in range(kp.shape[0]) if i not in used]
    for b in range(B):
        for i in range(table.shape[1]):
            if table[b, i] < 0 and i * page < lens[b] + S:
                table[b, i] = free.pop()
    k, v = (torch.randn(B, S, H, D, generator=g, device=DEV).to(dtype).transpose(1, 2) for _ in range(2))
    counts = [(S * (b + 1)) // B for b in range(B)]
    if S > 2:
        counts[0] = 0 if B > 1 else S
    count = torch.tensor(counts, dtype=torch.int32, device=DEV)
    path = torch.stack([torch.randperm(S, generator=g, device=DEV) for _ in range(B)]).to(torch.int32) if take else None
    want = []
    cache = td.PagedKVCache(kp, vp, table, ln)
    for b in range(B):
        nodes = path[b, :counts[b]].long() if take else torch.arange(counts[b], device=DEV)
        want.append([torch.cat((x, y[b][:, nodes].double()), 1) for x, y in zip(dense(cache, b), (k, v))])
    before = kp.clone(), vp.clone()
    out = td.cache_append(cache, k, v, take=path, count=count)
    assert out.tolist() == [n + c for n, c in zip(lens, counts)] and ln.tolist() == lens
    for b in range(B):
        for got, ref in zip(dense((kp, vp, table, out), b), want[b]):
            assert torch.equal(got, ref)
    # Nothing else moved.
    changed = ((kp != before[0]) & ~(kp.isnan() & before[0].isnan())).any(-1).any(1)
    assert int(changed.sum()) <= sum(counts)
    if count is not None and counts == [S] * B:
        assert torch.equal(td.cache_append(cache, k, v), out)
    nfa.check_device_status(DEV)


@pytest.mark.gpu
def test_append_refusals_and_bad_indices():
    g = gen(2)
    kp, vp, table, ln = page_cache([10, 20], 32, 16, 2, 64, BF, DEV, g, extra_pages=0, poison=0.0)
    cache = td.PagedKVCache(kp, vp, table, ln)
    k, v = (torch.randn(2, 2, 4, 64, generator=g, device=DEV).to(BF) for _ in range(2))
    nfa.check_device_status(DEV)
    td.cache_append(cache, k, v)
    nfa.check_device_status(DEV)
    before = kp.clone()
    cases = [dict(count=torch.tensor([5, 1], dtype=torch.int32, device=DEV)), dict(count=torch.tensor([-1, 0], dtype=torch.int32, device=DEV)),
             dict(take=torch.tensor([[0, 1, 4, 3], [0, -1, 2, 3]], dtype=torch.int32, device=DEV))]
    for kw in cases:
        td.cache_append(cache, k, v, **kw)
        with pytest.raises(RuntimeError, match="outside its table"):
            nfa.check_device_status(DEV)
    kp.copy_(before)
    for lens in ([30, 20], [-1, 0], [33, 0]):  # past the table, or no length of this table
        out = td.cache_append(cache._replace(lens=torch.tensor(lens, dtype=torch.int32, device=DEV)), k, v)
        assert (out <= 32).all()
        with pytest.raises(RuntimeError, match="outside its table"):
            nfa.check_device_status(DEV)
    t = table.clone()
    t[0, 0], t[1, 1] = kp.shape[0], -1
    kp.copy_(before)
    td.cache_append(cache._replace(page_table=t), k, v)
    with pytest.raises(RuntimeError, match="outside its table"):
        nfa.check_device_status(DEV)
    assert torch.equal(kp, before)
    with pytest.raises(ValueError):
        td.cache_append(cache, k, v, take=torch.zeros(2, 3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        td.cache_append(cache, k, v, count=torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(AssertionError):
        td.cache_append(cache, k, v[:, :, :3])
    with pytest.raises(RuntimeError):
        td.cache_append(cache, k.float(), v.float())
    assert td.cache_append(cache, k[:, :, :0], v[:, :, :0]).tolist() == ln.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D,N,Hq", [(64, 5, 4), (128, 3, 8), (256, 20, 4), (80, 9, 2)])
def test_queries_off_the_grid(dtype, D, N, Hq):
    """Only q lies off the 16-byte grid (odd element offsets): K, V and the pages
    are still read in vectors, with missing rows in nearly every chunk."""
    g = gen(14)
    lens = [100, 37, 0]
    cache = td.PagedKVCache(*page_cache(lens, 128, 16, 2, D, dtype, DEV, g))
    k, v = (torch.randn(3, 2, N, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    parents = tree("binary", N, 3)
    up = torch.tensor(parents, dtype=torch.int32, device=DEV)
    for offset in (1, 3, 6):
        flat = torch.randn(3 * Hq * N * D + offset, generator=g, device=DEV).to(dtype)
        q = flat[offset:].view(3, Hq, N, D)
        compare(*td.tree_attention(q, k, v, cache, up, return_lse=True), *attention(q, k, v, cache, parents))
    nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_windows_without_end(dtype):
    a, *more = (check([300, 20, 0], 9, 4, 2, 64, dtype, 16, tree("binary", 9, 3), sliding_window=w)
                for w in (0, 400, 2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1))
    for b in more:
        # The same chunks and products: a window that ends nowhere masks nothing.
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("page", [8, 16, 24, 7, 64, 128])
@pytest.mark.parametrize("D,N,Hq,window", [(128, 4, 4, 200), (64, 20, 8, 37), (256, 6, 2, 301), (128, 64, 4, 1)])
def test_pages_behind_the_window_may_be_given_back(dtype, page, D, N, Hq, window):
    """Table entries of pages whose last token no row sees hold no page: the call
    is valid, reports nothing and gives the same bits."""
    g = gen(15)
    lens = [1300, 257, 40, 0]
    kp, vp, table, ln = page_cache(lens, 1312, page, 1, D, dtype, DEV, g)
    q, k, v = (torch.randn(4, h, N, D, generator=g, device=DEV).to(dtype) for h in (Hq, 1, 1))
    up = torch.tensor(tree("binary", N, 4), dtype=torch.int32, device=DEV)
    want = td.tree_attention(q, k, v, td.PagedKVCache(kp, vp, table, ln), up, sliding_window=window, return_lse=True)
    gone = table.clone()
    for b, n in enumerate(lens):
        for i in range(max(0, n - window) // page):  # the pages of tokens before n - window only
            gone[b, i] = (-1, 2 ** 31 - 1, kp.shape[0])[i % 3]
    assert (gone != table).any()
    got = td.tree_attention(q, k, v, td.PagedKVCache(kp, vp, gone, ln), up, sliding_window=window, return_lse=True)
    nfa.check_device_status(DEV)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    compare(*got, *attention(q, k, v, (kp, vp, table, ln), tree("binary", N, 4), window=window))
    # A page that a row does see is still reported.
    seen = gone.clone()
    seen[0, (lens[0] - 1) // page] = -1
    td.tree_attention(q, k, v, td.PagedKVCache(kp, vp, seen, ln), up, sliding_window=window)
    with pytest.raises(RuntimeError, match="outside its table"):
        nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_bad_lengths_are_reported_wherever_they_stand(dtype):
    """Many short sequences, several to a block: a length outside the table is
    reported for each of them, not for a block's first alone."""
    g = gen(16)
    B = 900
    kp, vp = (torch.randn(4, 1, 16, 64, generator=g, device=DEV).to(dtype) for _ in range(2))
    table = torch.randint(0, 4, (B, 1), generator=g, device=DEV, dtype=torch.int32)
    q, k, v = (torch.randn(B, 1, 1, 64, generator=g, device=DEV).to(dtype) for _ in range(3))
    nfa.check_device_status(DEV)
    for at in (0, 1, 2, 3, 17, 450, 451, 452, 897, 898, 899):
        for n in (-1, 17):
            ln = torch.full((B,), 5, dtype=torch.int32, device=DEV)
            ln[at] = n
            td.tree_attention(q, k, v, td.PagedKVCache(kp, vp, table, ln))
            with pytest.raises(RuntimeError, match="outside its table"):
                nfa.check_device_status(DEV)
    td.tree_attention(q, k, v, td.PagedKVCache(kp, vp, table, torch.full((B,), 16, dtype=torch.int32, device=DEV)))
    nfa.check_device_status(DEV)


@pytest.mark.gpu
def test_append_is_written_in_place_for_autograd():
    """Pages that autograd has saved and an append overwrites: the backward raises."""
    g = gen(2)
    cache = td.PagedKVCache(*page_cache([10, 4], 32, 16, 2, 64, FP, DEV, g, extra_pages=4, poison=0.0))
    cache.page_table[:, 1] = torch.tensor([2, 3], device=DEV)
    k, v = (torch.randn(2, 2, 4, 64, generator=g, device=DEV) for _ in range(2))
    for pages in (cache.k_pages, cache.v_pages):
        w = torch.ones_like(pages, requires_grad=True)
        before = pages._version
        y = (w * pages).sum()
        td.cache_append(cache, k, v)
        assert pages._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        other = td.PagedKVCache(*(t.clone() for t in cache))
    td.cache_append(other, k, v)
    nfa.check_device_status(DEV)


@pytest.mark.gpu
def test_gradients_are_refusals():
    """No operator of the cache drops a gradient that one of its inputs wants."""
    g = gen(2)
    cache = td.PagedKVCache(*page_cache([10], 16, 16, 2, 64, FP, DEV, g, poison=0.0))
    q, k, v = (torch.randn(1, h, 3, 64, generator=g, device=DEV) for h in (4, 2, 2))
    slopes = torch.ones(4, device=DEV)

    def grad(t):
        return t.clone().requires_grad_(True)
    for call in (lambda: td.tree_attention(grad(q), k, v, cache), lambda: td.tree_attention(q, k, grad(v), cache),
                 lambda: td.tree_attention(q, k, v, cache._replace(k_pages=grad(cache.k_pages))),
                 lambda: td.tree_attention(q, k, v, cache, alibi_slope=grad(slopes)),
                 lambda: td.cache_append(cache, grad(k), v), lambda: td.cache_append(cache, k, grad(v)),
                 lambda: td.cache_append(cache._replace(v_pages=grad(cache.v_pages)), k, v)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()
    nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N,Hq,D", [(BF, 6, 8, 128), (HF, 40, 8, 64), (BF, 9, 4, 256), (FP, 5, 4, 64)])
def test_a_step_inside_a_cuda_graph(dtype, N, Hq, D):
    """A captured step (rotary at the nodes' positions, attention, verification,
    append) gives on other inputs what the calls give outside the graph."""
    import rotary
    g = gen(17)
    B, Hkv, V, page = 3, 2, 1000, 16
    lens = [300, 41, 0]
    cos, sin = rotary.rotary_table(D, 500, device=DEV)
    kp, vp, table, ln = page_cache([n + N for n in lens], 352, page, Hkv, D, dtype, DEV, g, poison=0.0)
    ln.copy_(torch.tensor(lens, device=DEV))
    up = torch.tensor(tree("binary", N, B), dtype=torch.int32, device=DEV)

    def fresh(seed):
        h = gen(seed)
        q, k, v = (torch.randn(B, n, N, D, generator=h, device=DEV).to(dtype) for n in (Hq, Hkv, Hkv))
        p = torch.softmax(torch.randn(B, N, V, generator=h, device=DEV) * 3, -1).to(dtype)
        tokens = p.float().topk(2, -1).indices.flatten(1)[:, :N].contiguous()
        noise = torch.empty(B, V, device=DEV).exponential_(generator=h).clamp_(min=1e-20)
        return [q, k, v, p, tokens, torch.rand(B, N, generator=h, device=DEV), noise, kp.clone(), vp.clone(), ln + seed % 3 * (ln > 0).int(), up.clone()]

    def step(q, k, v, p, tokens, u, noise, kp, vp, ln, up):
        cache = td.PagedKVCache(kp, vp, table, ln)
        q, k = rotary.rotary_embedding(q, k, cos, sin, td.tree_depths(up), ln)
        o, lse = td.tree_attention(q, k, v, cache, up, return_lse=True)
        path, count, token = td.verify_tree(p, tokens, up, u, noise)
        return [q, k, o, lse, path, count, token, td.cache_append(cache, k, v, take=path, count=count), kp, vp]
    held = fresh(0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*(t.clone() for t in held))  # first calls set the kernels up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step(*held)
    for seed in (1, 2, 5):
        for t, x in zip(held, fresh(seed)):
            t.copy_(x)
        graph.replay()
        for a, b in zip(got, step(*fresh(seed))):
            assert torch.equal(a, b)
    nfa.check_device_status(DEV)
