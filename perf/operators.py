"""Timed cases of the operators around attention that a decoder with a tree of drafted tokens needs:

  rope    rotary positions on q and k (half and interleaved layouts, part of the head, scaled tables), with gradients
  tree    attention of a tree of drafted tokens over a paged K/V cache
  verify  which drafted tokens stay, from the target's probabilities and given random numbers, and the next token
  append  a prompt's tokens, or a tree's accepted path, into the paged cache

Where ``own`` is false, ``run`` computes them in elementary torch operations in 32 bits; where it is true, it calls the
library's kernels through their public Python entry points.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _rope(name, **kw):
    case = dict(op="rope", batch=1, seq=1, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, dtype="bf16",
                grad=False, seq_major=True, scaling="none", table=32768)
    return dict(case, name=name, **kw) if name else dict(case, **kw)


def _tree(name, **kw):
    case = dict(op="tree", batch=1, nodes=1, branch=1, ctx=4096, ragged=False, page=64, heads=32, kv_heads=8, dim=128,
                dtype="bf16", window=0, cap=0.0, alibi=False, absent=False)
    return dict(case, name=name, **kw) if name else dict(case, **kw)


def _verify(name, **kw):
    case = dict(op="verify", batch=1, nodes=5, branch=1, vocab=32768, drafted=True, dtype="fp32", absent=False)
    return dict(case, name=name, **kw) if name else dict(case, **kw)


def _append(name, **kw):
    case = dict(op="append", batch=1, tokens=8, take=False, ragged=False, ctx=0, page=64, kv_heads=8, dim=128, dtype="bf16")
    return dict(case, name=name, **kw) if name else dict(case, **kw)


def listed():
    return [
        # One new token for each of 8 sequences: every decoding step of every layer does this, and latency is all it costs.
        _rope("rope-step", batch=8, seq=1, table=65536),
        # A prompt of odd length, half of the head rotated in the interleaved layout, positions compressed linearly.
        _rope("rope-prompt-partial", batch=2, seq=2047, dim=128, rotary=64, interleaved=True, dtype="fp16",
              seq_major=False, scaling="linear"),
        # A training layer of the grouped-query configuration (B=4, S=4096, 32/8 heads), forward and backward.
        _rope("rope-train", batch=4, seq=4096, grad=True),
        # One sequence, one token: plain paged decoding, the smallest call of the tree operator.
        _tree("tree-token", batch=1, nodes=1, ctx=4095, page=16),
        # Eight sequences of different lengths with a short chain of drafted tokens each.
        _tree("tree-chain", batch=8, nodes=6, branch=1, ctx=3001, ragged=True, page=16, heads=16, kv_heads=8, dim=64,
              dtype="fp16"),
        # The windowed, soft-capped head-dim-256 configuration with a binary tree.
        _tree("tree-window-cap", batch=8, nodes=15, branch=2, ctx=8190, ragged=True, page=128, heads=16, kv_heads=8,
              dim=256, window=4096, cap=50.0),
        # Wide trees over long caches of a 64/8-head model: the largest call.
        _tree("tree-wide", batch=16, nodes=64, branch=3, ctx=16384, ragged=True, page=64, heads=64, kv_heads=8,
              absent=True),
        # One user, a chain of four drafted tokens.
        _verify("verify-chain", batch=1, nodes=5, branch=1, vocab=32768),
        # Sixteen users, a fixed tree of the draft's best tokens, an odd vocabulary, 16-bit probabilities.
        _verify("verify-best", batch=16, nodes=25, branch=3, vocab=50021, drafted=False, dtype="bf16", absent=True),
        # A full batch with sampled drafts, two per node, and a large vocabulary.
        _verify("verify-sampled", batch=64, nodes=15, branch=2, vocab=131072),
        # The accepted path of a step: a few tokens of each sequence.
        _append("append-path", batch=16, tokens=24, take=True, ragged=True, ctx=1000),
        # Prompts of different lengths into fresh pages.
        _append("append-prompt", batch=8, tokens=8192, ragged=True, page=64),
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "rope", "tree", "tree", "tree", "verify", "verify", "append"])
    if op == "rope":
        group, kv = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 128, 128, 256])
        most = 4 * 4096 * 40 * 128 // (kv * (group + 1) * dim)
        batch = _spread(rng, 1, 16)
        seq = _spread(rng, 1, max(1, min(16384, most // batch)))
        return _rope(None, batch=batch, seq=seq, heads=group * kv, kv_heads=kv, dim=dim,
                     rotary=rng.choice([dim, dim, dim // 2, dim // 4 + 2]), interleaved=rng.random() < 0.5,
                     dtype=rng.choice(["bf16", "bf16", "fp16"]) if rng.random() < 0.8 or most < 2 * batch * seq else "fp32",
                     grad=rng.random() < 0.5, seq_major=rng.random() < 0.6,
                     scaling=rng.choice(["none", "linear", "ntk", "yarn"]), table=rng.choice([32768, 65536]))
    if op == "tree":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
        kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128, 128, 256])
        group = rng.choice([1, 2, 4, 8]) if dtype != "fp32" else rng.choice([1, 2, 4])
        nodes = _spread(rng, 1, 64 if dtype != "fp32" else 16)
        batch = _spread(rng, 1, 32)
        # At most the largest listed case's products, and in fp32 a sixteenth of them.
        most = 16 * 64 * 64 * 16384 * 128 // (16 if dtype == "fp32" else 1) // (batch * group * kv * nodes * dim)
        most = min(most, 16 * 16384 * 8 * 128 // (batch * kv * dim), 60000)
        return _tree(None, batch=batch, nodes=nodes, branch=rng.choice([1, 2, 3, 4]), ctx=_spread(rng, 1, max(1, most)),
                     ragged=rng.random() < 0.7, page=rng.choice([8, 16, 48, 64, 64, 128, 256]), heads=group * kv,
                     kv_heads=kv, dim=dim, dtype=dtype, window=rng.choice([0, 0, 0, 100, 1024, 4096]),
                     cap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.25, absent=rng.random() < 0.3)
    if op == "verify":
        nodes, vocab = _spread(rng, 1, 64), _spread(rng, 1000, 160000)
        batch = _spread(rng, 1, max(1, min(128, 64 * 15 * 131072 // (nodes * vocab))))
        return _verify(None, batch=batch, nodes=nodes, branch=rng.choice([1, 2, 3, 4]), vocab=vocab,
                       drafted=rng.random() < 0.6, dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                       absent=rng.random() < 0.4)
    kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128, 256])
    batch, take = _spread(rng, 1, 32), rng.random() < 0.5
    tokens = _spread(rng, 1, 64) if take else _spread(rng, 1, max(1, min(16384, 8 * 8192 * 8 * 128 // (batch * kv * dim))))
    return _append(None, batch=batch, tokens=tokens, take=take, ragged=rng.random() < 0.7, ctx=rng.choice([0, 1, 37, 500, 1500]),
                   page=rng.choice([8, 16, 48, 64, 128]), kv_heads=kv, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


# ---------------------------------------------------------------- inputs
def _lens(case):
    """Cached tokens of each sequence, known from the case alone (prepare() shuffles them)."""
    n, b = case["ctx"], case["batch"]
    return [n - (n * 3 * i) // (4 * b) for i in range(b)] if case["ragged"] else [n] * b


def _counts(case):
    """Tokens that each sequence appends."""
    s, b = case["tokens"], case["batch"]
    if case["take"]:
        return [1 + (5 * i) % min(s, 8) for i in range(b)]
    return [s - (s * i) // (2 * b) for i in range(b)] if case["ragged"] else [s] * b


def _parents(case):
    """The tree: node n > 0 hangs under (n - 1) // branch. With "absent", every second sequence has fewer nodes."""
    n, b = case["nodes"], case["batch"]
    row = torch.tensor([-1] + [(i - 1) // case["branch"] for i in range(1, n)], dtype=torch.int32)
    parents = row.repeat(b, 1)
    if case["absent"]:
        for i in range(1, b, 2):
            parents[i, max(1, (2 * n) // 3):] = -1
    return parents


def _pages(lens, page, spare, gen, device):
    """A page table in random order over as many pages as the lengths need; unused entries are -1."""
    need = [-(-(n + spare) // page) for n in lens]
    order = torch.randperm(sum(need), generator=gen, device=device).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32, device=device)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, max(1, sum(need))


def _table(rotary, rows, scaling, device):
    """cos and sin of position * frequency, formed in 64 bits; the scaled forms are those for long contexts."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64, device=device)
    base, factor, m = 10000.0, 4.0, 1.0
    if scaling == "ntk":
        base *= factor ** (rotary / max(1, rotary - 2))
    freq = base ** (-i / rotary)
    if scaling == "linear":
        freq = freq / factor
    if scaling == "yarn":
        turns = 4096 * freq / (2 * math.pi)  # over the original length
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        m = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * freq
    return (angle.cos() * m).float().contiguous(), (angle.sin() * m).float().contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    s = {"case": dict(case)}
    if case["op"] == "rope":
        b, n, d = case["batch"], case["seq"], case["dim"]

        def heads(h):  # a projection's output [B, S, H, D] seen as [B, H, S, D], or that layout itself
            return randn(b, n, h, d).transpose(1, 2) if case["seq_major"] else randn(b, h, n, d)

        s["q"], s["k"] = heads(case["heads"]), heads(case["kv_heads"])
        if case["grad"]:
            s["dq"], s["dk"] = heads(case["heads"]), heads(case["kv_heads"])
            s["q"].requires_grad_(True), s["k"].requires_grad_(True)
        s["cos"], s["sin"] = _table(case["rotary"], case["table"], case["scaling"], dev)
        s["offsets"] = torch.randint(0, case["table"] - n + 1, (b,), generator=gen, device=dev, dtype=torch.int32)
        return s
    if case["op"] == "verify":
        b, n, v = case["batch"], case["nodes"], case["vocab"]
        s["parents"] = _parents(case).to(dev)
        logits = randn(b, n, v, dtype=torch.float32).mul_(4.0)
        s["p"] = torch.softmax(logits, -1).to(dt)
        draft = logits.add_(randn(b, n, v, dtype=torch.float32), alpha=0.8)
        up = s["parents"].clamp(min=0).long()
        rank = torch.tensor([0] + [(i - 1) % case["branch"] for i in range(1, n)], device=dev)
        rows = torch.arange(b, device=dev)[:, None]
        if case["drafted"]:  # children drawn from the draft's law of their parent
            s["q"] = torch.softmax(draft, -1).to(dt)
            race = torch.empty(b, n, v, device=dev).exponential_(generator=gen).clamp_(min=1e-20)
            race = torch.div(s["q"].float()[rows, up], race, out=race)
            s["tokens"] = race.argmax(-1)
        else:  # the draft's best tokens
            best = draft.topk(case["branch"], -1).indices
            s["q"], s["tokens"] = None, best[rows, up, rank.expand(b, n)]
        s["u"] = torch.rand(b, n, generator=gen, device=dev)
        s["noise"] = torch.empty(b, v, device=dev).exponential_(generator=gen).clamp_(min=1e-20)
        return s
    b, h, d = case["batch"], case["kv_heads"], case["dim"]
    lens = _lens(case)
    shuffled = torch.randperm(b, generator=gen, device=dev).tolist()
    lens = [lens[i] for i in shuffled]
    spare = case["nodes"] if case["op"] == "tree" else case["tokens"]
    s["table"], pages = _pages(lens, case["page"], spare, gen, dev)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["k_pages"], s["v_pages"] = randn(pages, h, case["page"], d), randn(pages, h, case["page"], d)
    if case["op"] == "tree":
        n = case["nodes"]
        # Heads from diffuse to peaked.
        peak = torch.linspace(0.5, 4.0, case["heads"], device=dev)[:, None, None]
        s["q"] = (randn(b, case["heads"], n, d, dtype=torch.float32) * peak).to(dt)
        s["k"], s["v"] = randn(b, h, n, d), randn(b, h, n, d)
        s["parents"] = _parents(case).to(dev)
        s["slopes"] = None
        if case["alibi"]:  # the slope multiplies (query position - key position): negative ones fade with distance
            s["slopes"] = -(2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device=dev, dtype=torch.float32) / case["heads"]))
        return s
    counts = _counts(case)
    s["count"] = torch.tensor([counts[i] for i in shuffled], dtype=torch.int32, device=dev)
    s["k"], s["v"] = randn(b, h, case["tokens"], d), randn(b, h, case["tokens"], d)
    s["take"] = None
    if case["take"]:  # a path through the tree's nodes, root first
        keys = torch.rand(b, case["tokens"], generator=gen, device=dev)
        keys[:, 0] = -1.0
        path = keys.argsort(-1)
        here = torch.arange(case["tokens"], device=dev) < s["count"][:, None]
        path = torch.where(here, path, case["tokens"]).sort(-1).values
        s["take"] = torch.where(here, path, -1).to(torch.int32)
    return s


# ---------------------------------------------------------------- one pass
def _modules():
    pkg = os.path.join(_ROOT, "npu-flex-att_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import rotary
    import tree_decoding
    return rotary, tree_decoding


_loaded = None


def run(state):
    global _loaded
    case = state["case"]
    if not own:
        return {"rope": _plain_rope, "tree": _plain_tree, "verify": _plain_verify, "append": _plain_append}[case["op"]](state, case)
    if _loaded is None:
        _loaded = _modules()
    rotary, td = _loaded
    if case["op"] == "rope":
        q, k = rotary.rotary_embedding(state["q"], state["k"], state["cos"], state["sin"], offsets=state["offsets"],
                                       interleaved=case["interleaved"])
        if not case["grad"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))
        return q, k, dq, dk
    if case["op"] == "verify":
        return td.verify_tree(state["p"], state["tokens"], state["parents"], state["u"], state["noise"], draft_probs=state["q"])
    cache = td.PagedKVCache(state["k_pages"], state["v_pages"], state["table"], state["lens"])
    if case["op"] == "tree":
        return td.tree_attention(state["q"], state["k"], state["v"], cache, state["parents"], sliding_window=case["window"],
                                 soft_cap=case["cap"], alibi_slope=state["slopes"], return_lse=True)
    lens = td.cache_append(cache, state["k"], state["v"], take=state["take"], count=state["count"])
    return state["k_pages"], state["v_pages"], lens


def _rotate(x, c, s, interleaved):
    r = 2 * c.shape[-1]
    x = x.float()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((turned, x[..., r:]), -1)


@torch.no_grad()
def _plain_rope(state, case):
    at = state["offsets"][:, None].long() + torch.arange(case["seq"], device=state["q"].device)
    c, s = state["cos"][at][:, None], state["sin"][at][:, None]
    dt, il = state["q"].dtype, case["interleaved"]
    out = tuple(_rotate(state[x], c, s, il).to(dt) for x in ("q", "k"))
    if case["grad"]:  # the transposed rotation of the gradients
        out += tuple(_rotate(state[x], c, -s, il).to(dt) for x in ("dq", "dk"))
    return out


def _ancestors(parents):
    """[B, N, N]: whether m is n or above n, and whether n hangs under the root at all."""
    n = parents.shape[1]
    up = parents.clone()
    up[:, 0] = -1
    step = (up[:, :, None] == torch.arange(n, device=parents.device)).float() + torch.eye(n, device=parents.device)
    over = torch.linalg.matrix_power(step, max(1, n - 1)) > 0
    return over, over[:, :, 0]


@torch.no_grad()
def _plain_tree(state, case):
    b, h, d, n = case["batch"], case["kv_heads"], case["dim"], case["nodes"]
    g = case["heads"] // h
    table, lens = state["table"], state["lens"].long()

    def gathered(pages):
        x = pages[table.clamp(min=0).long()]  # [B, pages, H, page, D]
        return x.transpose(1, 2).reshape(b, h, -1, d).float()

    over, there = _ancestors(state["parents"])
    pos = lens[:, None] + over.sum(-1) - 1  # [B, N]
    q = state["q"].float().view(b, h, g, n, d)
    k = gathered(state["k_pages"])
    at = torch.arange(k.shape[2], device=q.device)
    away = pos[:, :, None] - at  # [B, N, L]
    keep = (at < lens[:, None])[:, None] & there[:, :, None]
    away_t = pos[:, :, None] - pos[:, None, :]
    keep_t = over & there[:, :, None]
    if case["window"]:
        keep, keep_t = keep & (away <= case["window"]), keep_t & (away_t <= case["window"])
    slopes = state["slopes"].view(h, g, 1, 1) if case["alibi"] else None

    def logits(keys, away, keep):
        x = torch.matmul(q.view(b, h, g * n, d), keys.transpose(2, 3)).view(b, h, g, n, -1).mul_(1.0 / math.sqrt(d))
        if case["cap"]:
            x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
        if slopes is not None:
            x = x + slopes * away[:, None, None]
        return x.masked_fill_(~keep[:, None, None], -math.inf)

    x, y = logits(k, away, keep), logits(state["k"].float(), away_t, keep_t)
    del k
    top = torch.maximum(x.amax(-1, True), y.amax(-1, True))
    base = torch.where(top == -math.inf, 0.0, top)
    x, y = x.sub_(base).exp_(), y.sub_(base).exp_()
    total = x.sum(-1, True) + y.sum(-1, True)
    o = torch.matmul(x.view(b, h, g * n, -1), gathered(state["v_pages"])) + torch.matmul(y.view(b, h, g * n, -1), state["v"].float())
    o = o.view(b, h, g, n, d) / torch.where(total > 0, total, 1.0)
    lse = (base + total.log()).view(b, h * g, n)
    return o.view(b, h * g, n, d).to(state["q"].dtype), lse


@torch.no_grad()
def _plain_verify(state, case):
    p, tokens, u = state["p"].float(), state["tokens"], state["u"]
    b, n, v = p.shape
    dev = p.device
    parents = state["parents"].long()
    over, there = _ancestors(parents)
    up, rows, node = parents.clamp(min=0), torch.arange(b, device=dev)[:, None], torch.arange(n, device=dev)
    drawn = there & (node > 0)
    # Siblings before n, in the order in which they are tried.
    before = (parents[:, :, None] == parents[:, None, :]) & (node[None, :] < node[:, None]) & drawn[:, :, None] & drawn[:, None, :]
    rank = before.sum(-1)
    px = p[rows, up, tokens]
    a = torch.zeros(b, n, device=dev)
    if state["q"] is not None:
        q = state["q"].float()
        qx, w = q[rows, up, tokens], torch.ones(b, n, device=dev)
        yes = torch.zeros(b, n, dtype=torch.bool, device=dev)
        children = ((parents[:, None, :] == node[:, None]) & drawn[:, None, :]).sum(-1)  # of each node
        for c in range(case["branch"]):
            an, wn = a[rows, up], w[rows, up]
            yes |= drawn & (rank == c) & (u * (wn * qx) < (px - an * qx).clamp(min=0))
            a = torch.where(children > c, a + w, a)  # as if child c of every node were rejected
            w = (p - a[..., None] * q).clamp_(min=0).sum(-1)
    else:
        again = (before & (tokens[:, :, None] == tokens[:, None, :])).any(-1)
        gone = (before.float() * (px * ~again)[:, None, :]).sum(-1)
        yes = drawn & ~again & (u * (1.0 - gone) < px)
    first = yes & ~(before & yes[:, None, :]).any(-1)
    first[:, 0] = True
    kept = there & ~(over & ~first[:, None, :]).any(-1)
    count = kept.sum(-1)
    path = torch.where(kept, node, n).sort(-1).values
    path = torch.where(node < count[:, None], path, -1)
    last = torch.where(kept, node, 0).amax(-1, True)
    whole = p[rows, last][:, 0]
    if state["q"] is not None:
        rest = (whole - a.gather(1, last) * q[rows, last][:, 0]).clamp_(min=0)
    else:
        dropped = torch.zeros(b, v, device=dev).scatter_add_(1, tokens, (drawn & (up == last)).float())
        rest = whole * (dropped == 0)
    rest = torch.where(rest.amax(-1, True) > 0, rest, whole)
    token = (rest / state["noise"]).argmax(-1)
    return path.int(), count.int(), token.int()


@torch.no_grad()
def _plain_append(state, case):
    b, page = case["batch"], case["page"]
    rows = torch.arange(b, device=state["k"].device)[:, None]
    # Past its count a sequence writes its last token again.
    i = torch.minimum(torch.arange(case["tokens"], device=rows.device), state["count"][:, None].long() - 1)
    source = i if state["take"] is None else state["take"].long().gather(1, i)
    at = state["lens"][:, None].long() + i
    where, slot = state["table"].gather(1, at // page).long(), at % page
    state["k_pages"][where, :, slot] = state["k"][rows, :, source]
    state["v_pages"][where, :, slot] = state["v"][rows, :, source]
    return state["k_pages"], state["v_pages"], state["lens"] + state["count"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = _BYTES[case["dtype"]]
    b = case["batch"]
    if case["op"] == "rope":
        n = b * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        turned = n * case["rotary"] / case["dim"]
        table = b * case["seq"] * case["rotary"] * 4
        times = 2 if case["grad"] else 1
        return {"bytes": times * (2 * n * e + table), "flops": times * 3 * turned}
    if case["op"] == "tree":
        w = case["window"]
        seen = sum(min(n, w) if w else n for n in _lens(case))
        hq, h, n, d = case["heads"], case["kv_heads"], case["nodes"], case["dim"]
        new = b * n * d * e * 2 * (hq + h) + 4 * b * hq * n
        there = (b - b // 2) * n + (b // 2) * max(1, 2 * n // 3) if case["absent"] else b * n  # of the nodes
        return {"bytes": 2 * seen * h * d * e + new, "flops": 4 * d * hq * there / b * seen + 2 * d * there * hq * n}
    if case["op"] == "verify":
        v = case["vocab"]
        return {"bytes": b * v * ((2 if case["drafted"] else 1) * e + 4), "flops": 3 * b * v}
    tokens = sum(_counts(case))
    return {"bytes": 4 * tokens * case["kv_heads"] * case["dim"] * e, "flops": 0}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "tree": _exact_tree, "verify": _exact_verify, "append": _exact_append}[case["op"]](s, case)


@torch.no_grad()
def _exact_rope(s, case):
    r, n, out = case["rotary"], case["seq"], []
    for name in ("q", "k") + (("dq", "dk") if case["grad"] else ()):
        y = s[name].double().contiguous()
        for i, start in enumerate(s["offsets"].tolist()):  # pairs as complex numbers, times m e^(i theta)
            turn = torch.complex(s["cos"][start:start + n].double(), s["sin"][start:start + n].double())
            turn = turn.conj() if name in ("dq", "dk") else turn
            part = y[i, :, :, :r]
            if case["interleaved"]:
                z = torch.view_as_complex(part.reshape(*part.shape[:-1], r // 2, 2).contiguous()) * turn
                y[i, :, :, :r] = torch.view_as_real(z).reshape(part.shape)
            else:
                z = torch.complex(part[..., :r // 2].contiguous(), part[..., r // 2:].contiguous()) * turn
                y[i, :, :, :r] = torch.cat((z.real, z.imag), -1)
        out.append(y)
    return tuple(out)


def _climb(parents):
    """For each node the nodes from it up to the root, or [] where it does not hang under the root."""
    paths = []
    for n, up in enumerate(parents):
        if n == 0:
            paths.append([0])
        else:
            paths.append([n] + paths[up] if 0 <= up < n and paths[up] else [])
    return paths


@torch.no_grad()
def _exact_tree(s, case):
    b, hq, h, n, d = case["batch"], case["heads"], case["kv_heads"], case["nodes"], case["dim"]
    g, page = hq // h, case["page"]
    out = torch.zeros(b, hq, n, d, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((b, hq, n), -math.inf, dtype=torch.float64, device=out.device)
    for i in range(b):
        size, paths = int(s["lens"][i]), _climb(s["parents"][i].tolist())
        pages = s["table"][i, :-(-size // page)].long()
        low = max(0, size - case["window"]) if case["window"] else 0
        low = low // page * page
        pages = pages[low // page:]
        keys, vals = (torch.cat((c[pages].transpose(0, 1).reshape(h, -1, d)[:, :size - low], new[i]), 1).double()
                      for c, new in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])))
        here = torch.tensor([size + len(x) - 1 for x in paths], device=out.device)
        at = torch.cat((torch.arange(low, size, device=out.device), here))
        keep = torch.zeros(n, size - low + n, dtype=torch.bool)
        for m, x in enumerate(paths):
            if x:
                keep[m, :size - low] = True
                keep[m, [size - low + y for y in x]] = True
        keep = keep.to(out.device)
        away = here[:, None] - at
        if case["window"]:
            keep &= away <= case["window"]
        x = torch.einsum("hgnd,hld->hgnl", s["q"][i].double().view(h, g, n, d), keys) / math.sqrt(d)
        if case["cap"]:
            x = case["cap"] * torch.tanh(x / case["cap"])
        if case["alibi"]:
            x += s["slopes"].double().view(h, g, 1, 1) * away
        x = torch.where(keep, x, -math.inf)
        total = torch.logsumexp(x, -1)
        weight = torch.where(keep, torch.exp(x - total[..., None]), 0.0)
        out[i] = torch.einsum("hgnl,hld->hgnd", weight, vals).reshape(hq, n, d)
        lse[i] = total.reshape(hq, n)
    return out, lse


@torch.no_grad()
def _exact_verify(s, case):
    b, n = case["batch"], case["nodes"]
    paths, counts, nexts = [], [], []
    for i in range(b):
        parents, tokens, u = s["parents"][i].tolist(), s["tokens"][i].tolist(), s["u"][i].double().tolist()
        at, path = 0, [0]
        while True:
            rest = s["p"][i, at].double()
            law = None if s["q"] is None else s["q"][i, at].double()
            moved, whole = False, rest
            if law is None:
                rest = rest.clone()
            mass = 1.0
            for c in range(at + 1, n):
                if parents[c] != at:
                    continue
                x = tokens[c]
                chance = float(rest[x]) if law is None else float(rest[x] / law[x])
                if u[c] * mass < chance:
                    at, moved = c, True
                    path.append(c)
                    break
                if law is None:  # the token itself is taken out
                    mass -= float(rest[x])
                    rest[x] = 0.0
                else:
                    rest = (rest / mass - law).clamp(min=0)
                    mass = float(rest.sum())
            if not moved:
                break
        rest = rest if float(rest.max()) > 0 else whole
        nexts.append(int((rest / s["noise"][i].double()).argmax()))
        counts.append(len(path))
        paths.append(path + [-1] * (n - len(path)))
    return tuple(torch.tensor(x, dtype=torch.int32, device=s["p"].device) for x in (paths, counts, nexts))


@torch.no_grad()
def _exact_append(s, case):
    page, k_pages, v_pages = case["page"], s["k_pages"].double(), s["v_pages"].double()
    for i in range(case["batch"]):
        size, count = int(s["lens"][i]), int(s["count"][i])
        at = torch.arange(size, size + count, device=k_pages.device)
        nodes = s["take"][i, :count].long() if s["take"] is not None else slice(0, count)
        where = s["table"][i].long()[at // page]
        for pages, new in ((k_pages, s["k"]), (v_pages, s["v"])):
            pages[where, :, at % page] = new[i, :, nodes].transpose(0, 1).double()
    return k_pages, v_pages, s["lens"] + s["count"]
