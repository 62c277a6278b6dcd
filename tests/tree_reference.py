"""Plain 64-bit restatements of the tree-decoding operators for the tests."""
import math

import torch


def climb(parents):
    """For each node the list of nodes from it up to the root, [] where it is absent."""
    paths = []
    for n, up in enumerate(parents):
        paths.append([0] if n == 0 else [n] + paths[up] if 0 <= up < n and paths[up] else [])
    return paths


def page_cache(lens, capacity, page, Hkv, D, dtype, device, gen, extra_pages=2, poison=float("nan")):
    """(k_pages, v_pages, table, lens): pages in random order; every slot that
    holds no token, and every page that no sequence owns, is `poison`."""
    B = len(lens)
    maxp = max(1, -(-capacity // page))
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra_pages
    order = torch.randperm(total, generator=gen, device=device).to(torch.int32)
    table = torch.full((B, maxp), -1, dtype=torch.int32, device=device)
    pages = [torch.full((total, Hkv, page, D), poison, device=device, dtype=dtype) for _ in range(2)]
    at = 0
    for b, n in enumerate(lens):
        ids = order[at:at + need[b]].long()
        table[b, :need[b]] = ids.int()
        at += need[b]
        for t in range(0, n, page):
            m = min(page, n - t)
            for x in pages:
                x[ids[t // page], :, :m] = torch.randn(Hkv, m, D, generator=gen, device=device).to(dtype)
    return pages[0], pages[1], table, torch.tensor(lens, dtype=torch.int32, device=device)


def dense(cache, b):
    """Sequence b's cached K and V, [Hkv, len, D] in 64 bits."""
    kp, vp, table, lens = cache
    n, page = int(lens[b]), kp.shape[2]
    ids = table[b, :-(-n // page)].long()
    return [x[ids].transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n].double() for x in (kp, vp)]


def attention(q, k, v, cache, parents, scale=None, window=0, cap=0.0, slopes=None):
    """(O, LSE, sum of p·|v|) in 64 bits. parents: list per sequence."""
    B, Hq, N, D = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, N, D, dtype=torch.float64, device=q.device)
    size, lse = torch.zeros_like(out), torch.full((B, Hq, N), -math.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        K, V = dense(cache, b)
        L = K.shape[1]
        for n, way in enumerate(climb(parents[b])):
            if not way:
                continue
            i = L + len(way) - 1
            spots = torch.cat((torch.arange(L, device=q.device), torch.tensor([L + len(way) - 1 - x for x in range(len(way))], device=q.device)))
            keys, vals = (torch.cat((a, x[b][:, way].double()), 1) for a, x in ((K, k), (V, v)))
            if window:
                sel = (i - spots <= window).nonzero()[:, 0]
                spots, keys, vals = spots[sel], keys[:, sel], vals[:, sel]
            for h in range(Hq):
                s = keys[h // G] @ q[b, h, n].double() * scale
                if cap:
                    s = cap * torch.tanh(s / cap)
                if slopes is not None:
                    s = s + float(slopes[h]) * (i - spots)
                lse[b, h, n] = torch.logsumexp(s, 0)
                w = torch.exp(s - lse[b, h, n])
                out[b, h, n], size[b, h, n] = w @ vals[h // G], w @ vals[h // G].abs()
    return out, lse, size


def verify(p, tokens, parents, u, noise, q=None):
    """(path, next token) of one sequence, walking down with explicit residuals."""
    at, path = 0, [0]
    N = len(tokens)
    while True:
        whole = p[at].double()
        rest, mass, moved = whole.clone(), 1.0, False
        for c in range(at + 1, N):
            if parents[c] != at:
                continue
            x = int(tokens[c])
            if not 0 <= x < p.shape[1]:
                continue
            if q is not None:
                ok = float(u[c]) * mass * float(q[at, x]) < float(rest[x])
            else:
                ok = float(u[c]) * mass < float(rest[x])
            if ok:
                at, moved = c, True
                path.append(c)
                break
            if q is not None:
                rest = (rest / mass - q[at].double()).clamp(min=0)
                mass = float(rest.sum())
            else:
                mass -= float(rest[x])
                rest[x] = 0.0
        if not moved:
            rest = rest if float(rest.max()) > 0 else whole
            return path, int((rest / noise.double()).argmax())
