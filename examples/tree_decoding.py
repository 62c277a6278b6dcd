"""Greedy decoding with a tree of drafted tokens, end to end on the library's
kernels: rotary positions, attention of the tree over a paged cache, verification
and the append of the accepted path.

    python examples/tree_decoding.py [--steps 40] [--dtype bf16]

The model is a small decoder with random weights (there is no checkpoint to
load); the draft looks the current token up in what has been decoded so far and
proposes what followed it there, the two latest occurrences as two branches.
Whatever the draft proposes, the tokens are those of decoding one by one, which
the example does as well and compares with.
"""
import argparse
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "npu-flex-att_b200")
if PKG not in sys.path:
    sys.path.insert(0, PKG)

import npu_flash_attention as nfa  # noqa: E402
from rotary import rotary_embedding, rotary_table  # noqa: E402
from tree_decoding import PagedKVCache, cache_append, tree_attention, tree_depths, verify_tree  # noqa: E402

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


class Decoder:
    """Pre-norm decoder: `layers` blocks of grouped-query attention and a ReLU
    feed-forward, a paged K/V cache per layer, one page table for all."""

    def __init__(self, vocab=512, width=256, layers=2, heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16,
                 max_tokens=1024, page=16, batch=2, seed=0, device="cuda:0"):
        g = torch.Generator(device=device).manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=device) / math.sqrt(shape[0])).to(dtype)
        self.heads, self.kv_heads, self.head_dim, self.batch = heads, kv_heads, head_dim, batch
        self.embed = torch.randn(vocab, width, generator=g, device=device).to(dtype)
        self.out = w(width, vocab)
        self.layers = [dict(qkv=w(width, (heads + 2 * kv_heads) * head_dim), o=w(heads * head_dim, width),
                            up=w(width, 4 * width), down=w(4 * width, width)) for _ in range(layers)]
        self.cos, self.sin = rotary_table(head_dim, max_tokens, device=device)
        pages = -(-max_tokens // page)
        # Every sequence has its pages from the start, in mixed order.
        table = torch.randperm(batch * pages, generator=g, device=device).to(torch.int32).view(batch, pages)
        lens = torch.zeros(batch, dtype=torch.int32, device=device)
        shape = (batch * pages, kv_heads, page, head_dim)
        self.caches = [PagedKVCache(*(torch.empty(shape, dtype=dtype, device=device) for _ in range(2)), table, lens)
                       for _ in range(layers)]

    @property
    def lens(self):
        return self.caches[0].lens

    def advance(self, lens):
        self.caches = [c._replace(lens=lens) for c in self.caches]

    @torch.no_grad()
    def run(self, tokens, depths=None, parents=None, prompt=False):
        """Logits [B, N, vocab] of a prompt's tokens (causal), or of a tree's
        nodes; and the new K/V of every layer."""
        B, N = tokens.shape
        x = self.embed[tokens]
        new = []
        for layer, cache in zip(self.layers, self.caches):
            h = torch.nn.functional.rms_norm(x, (x.shape[-1],))
            q, k, v = (h @ layer["qkv"]).view(B, N, -1, self.head_dim).split(
                [self.heads, self.kv_heads, self.kv_heads], 2)
            q, k, v = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
            q, k = rotary_embedding(q, k, self.cos, self.sin, positions=depths, offsets=cache.lens)
            if prompt:
                o = nfa.npu_flash_attention_forward(q, k, v, causal=True)
            else:
                o = tree_attention(q, k, v, cache, parents)
            x = x + o.transpose(1, 2).reshape(B, N, -1) @ layer["o"]
            h = torch.nn.functional.rms_norm(x, (x.shape[-1],))
            x = x + torch.relu(h @ layer["up"]) @ layer["down"]
            new.append((k, v))
        return torch.nn.functional.rms_norm(x, (x.shape[-1],)) @ self.out, new

    def append(self, new, take=None, count=None):
        """K/V of a pass into every layer's cache: the prompt, or a path."""
        for cache, (k, v) in zip(self.caches, new):
            lens = cache_append(cache, k, v, take=take, count=count)
        self.advance(lens)


def lookup_tree(history, branch=3, width=2):
    """(tokens, parents) of one sequence's tree: the last token as the root, and
    for each of its latest earlier occurrences what followed, up to `branch`."""
    n = 1 + branch * width
    tokens, parents = [history[-1]] + [0] * (n - 1), [-1] * n
    at = 1
    places = [i for i in range(len(history) - 1) if history[i] == history[-1]][-width:]
    for i in places:
        up = 0
        for t in history[i + 1:i + 1 + branch]:
            tokens[at], parents[at], up, at = t, up, at, at + 1
    return tokens, parents


def decode(model, prompt, steps, drafted=True):
    """(tokens per sequence, passes): at least `steps` tokens after the prompt."""
    dev = prompt.device
    logits, new = model.run(prompt, prompt=True)
    model.append(new)
    history = [row + [t] for row, t in zip(prompt.tolist(), logits[:, -1].argmax(-1).tolist())]
    passes = 0
    while min(map(len, history)) < prompt.shape[1] + steps:
        trees = [lookup_tree(h) if drafted else ([h[-1]], [-1]) for h in history]
        tokens = torch.tensor([t for t, _ in trees], device=dev)
        parents = torch.tensor([p for _, p in trees], dtype=torch.int32, device=dev)
        logits, new = model.run(tokens, tree_depths(parents), parents)
        B, N, V = logits.shape
        # Greedy: all of the target's mass on its best token, so that the random
        # numbers have nothing to decide.
        best = torch.zeros(B, N, V, device=dev).scatter_(2, logits.argmax(-1, keepdim=True), 1.0)
        path, count, token = verify_tree(best, tokens, parents, torch.full((B, N), 0.5, device=dev),
                                         torch.ones(B, V, device=dev))
        model.append(new, take=path, count=count)
        for h, tree, row, c, t in zip(history, trees, path.tolist(), count.tolist(), token.tolist()):
            h += [tree[0][i] for i in row[1:c]] + [t]
        passes += 1
    nfa.check_device_status(dev)
    return history, passes


def main(steps=40, dtype="fp32", batch=2, seed=0):
    prompt = torch.randint(0, 512, (batch, 24), generator=torch.Generator().manual_seed(seed)).to("cuda:0")
    tree, passes = decode(Decoder(dtype=DTYPES[dtype], batch=batch, seed=seed), prompt, steps)
    plain, single = decode(Decoder(dtype=DTYPES[dtype], batch=batch, seed=seed), prompt, steps, drafted=False)
    end = prompt.shape[1] + steps
    same = [a[:end] == b[:end] for a, b in zip(tree, plain)]
    print(f"{dtype}: {steps} tokens in {passes} passes with a tree, {single} one by one; same tokens: {same}")
    return same, passes, single


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="fp32",
                    help="in 16 bits the model's own products round differently for another number of rows, and a near "
                         "tie may fall the other way")
    args = ap.parse_args()
    main(args.steps, args.dtype)
