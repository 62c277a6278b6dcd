"""Tree decoding, host side: argument blocks, C-level checks, depths, refusals
(CPU only; the calls are rejected before any CUDA work)."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import bfa_lib
import tree_decoding as td

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_argument_blocks_match_header_layout(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    structs = {"bfa_rope_args": bfa_lib.RopeArgs, "bfa_tree_args": bfa_lib.TreeArgs, "bfa_verify_args": bfa_lib.VerifyArgs,
               "bfa_append_args": bfa_lib.AppendArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "bfa.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = {tuple(x.split()[:2]): int(x.split()[2]) for x in out.splitlines()}
    for cname, cls in structs.items():
        assert got[(cname, "size")] == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert got[(cname, f)] == getattr(cls, f).offset, (cname, f)


def block(cls, **kw):
    a = cls()
    for key, x in kw.items():
        setattr(a, key, x)
    return a


TREE = dict(batch=1, heads_q=4, heads_kv=2, nodes=3, head_dim=64, dtype=2, num_pages=1, page_size=16, max_pages=1)
VERIFY = dict(batch=1, nodes=3, vocab=10, dtype=0)
APPEND = dict(batch=1, heads_kv=2, tokens=3, head_dim=64, dtype=2, num_pages=1, page_size=16, max_pages=1)
ROPE = dict(batch=1, heads_q=1, heads_k=1, seqlen=4, head_dim=64, rotary_dim=64, dtype=2, table_rows=4)


@pytest.mark.parametrize("name,cls,base,kw,code", [
    ("bfa_tree_fwd", "TreeArgs", TREE, dict(heads_q=3), -2), ("bfa_tree_fwd", "TreeArgs", TREE, dict(nodes=65), -3),
    ("bfa_tree_fwd", "TreeArgs", TREE, dict(nodes=0), -1), ("bfa_tree_fwd", "TreeArgs", TREE, dict(head_dim=257), -3),
    ("bfa_tree_fwd", "TreeArgs", TREE, dict(dtype=5), -3), ("bfa_tree_fwd", "TreeArgs", TREE, dict(soft_cap=-1.0), -1),
    ("bfa_tree_fwd", "TreeArgs", TREE, dict(soft_cap=float("nan")), -1), ("bfa_tree_fwd", "TreeArgs", TREE, dict(page_size=0), -1),
    ("bfa_tree_fwd", "TreeArgs", TREE, dict(max_pages=2 ** 40), -3), ("bfa_tree_fwd", "TreeArgs", TREE, dict(), -1),
    ("bfa_tree_fwd", "TreeArgs", TREE, dict(batch=0), 0),
    ("bfa_verify_tree", "VerifyArgs", VERIFY, dict(nodes=65), -3), ("bfa_verify_tree", "VerifyArgs", VERIFY, dict(vocab=0), -1),
    ("bfa_verify_tree", "VerifyArgs", VERIFY, dict(), -1), ("bfa_verify_tree", "VerifyArgs", VERIFY, dict(batch=0), 0),
    ("bfa_verify_tree", "VerifyArgs", VERIFY, dict(dtype=-1), -3),
    ("bfa_cache_append", "AppendArgs", APPEND, dict(page_size=0), -1), ("bfa_cache_append", "AppendArgs", APPEND, dict(), -1),
    ("bfa_cache_append", "AppendArgs", APPEND, dict(head_dim=300), -3), ("bfa_cache_append", "AppendArgs", APPEND, dict(batch=0), 0),
    ("bfa_rope", "RopeArgs", ROPE, dict(rotary_dim=7), -1), ("bfa_rope", "RopeArgs", ROPE, dict(rotary_dim=66), -2),
    ("bfa_rope", "RopeArgs", ROPE, dict(interleaved=2), -1), ("bfa_rope", "RopeArgs", ROPE, dict(dtype=3), -3),
    ("bfa_rope", "RopeArgs", ROPE, dict(), -1), ("bfa_rope", "RopeArgs", ROPE, dict(seqlen=0), 0)])
def test_entry_points_check_their_arguments(name, cls, base, kw, code):
    lib = bfa_lib.load()
    assert getattr(lib, name)(block(getattr(bfa_lib, cls), **dict(base, **kw)), None) == code
    assert getattr(lib, name)(None, None) == -1


def test_status_has_a_message():
    assert "index" in bfa_lib.load().bfa_strerror(bfa_lib.ERR_INDEX).decode()


def test_workspace_bytes_of_invalid_problems():
    lib = bfa_lib.load()
    assert lib.bfa_tree_workspace_bytes(None) == 0
    assert lib.bfa_tree_workspace_bytes(block(bfa_lib.TreeArgs, **dict(TREE, heads_q=3))) == 0
    assert lib.bfa_tree_workspace_bytes(block(bfa_lib.TreeArgs, **dict(TREE, batch=0))) == 0
    assert lib.bfa_tree_workspace_bytes(block(bfa_lib.TreeArgs, **TREE)) > 0


def test_depths():
    t = torch.tensor([[-1, 0, 0, 1, 3, 2], [-1, 0, 1, 2, 3, 4], [5, -1, 0, 1, -1, 2]], dtype=torch.int32)
    d = td.tree_depths(t)
    assert d.dtype == torch.int32 and d[0].tolist() == [0, 1, 1, 2, 3, 2] and d[1].tolist() == [0, 1, 2, 3, 4, 5]
    assert d[2, 0] == 0 and d[2, 2] == 1 and d[2, 5] == 2
    assert td.tree_depths(t[0]).tolist() == d[0].tolist() and td.tree_depths(torch.tensor([-1])).tolist() == [0]


def test_cpu_tensors_are_refused():
    q, k = torch.randn(1, 2, 3, 64), torch.randn(1, 1, 3, 64)
    cache = td.PagedKVCache(torch.zeros(1, 1, 16, 64), torch.zeros(1, 1, 16, 64), torch.zeros(1, 1, dtype=torch.int32),
                            torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        td.tree_attention(q, k, k, cache)
    with pytest.raises(RuntimeError, match="no CPU path"):
        td.cache_append(cache, k, k)
    with pytest.raises(RuntimeError, match="no CPU path"):
        td.verify_tree(torch.ones(1, 3, 4), torch.zeros(1, 3, dtype=torch.int64), None, torch.rand(1, 3), torch.ones(1, 4))


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspace_bytes_of_windows_without_end(dtype):
    """The largest windows (no limit at all) plan like one that covers the table."""
    lib = bfa_lib.load()
    base = dict(TREE, dtype=dtype, batch=3, max_pages=50)
    want = lib.bfa_tree_workspace_bytes(block(bfa_lib.TreeArgs, **dict(base, sliding_window=800)))
    for window in (801, 2 ** 31 - 1, 2 ** 31, 2 ** 40, 2 ** 63 - 129, 2 ** 63 - 1):
        assert lib.bfa_tree_workspace_bytes(block(bfa_lib.TreeArgs, **dict(base, sliding_window=window))) == want, window


def test_verify_refuses_vocabularies_that_its_counters_cannot_pass():
    """Entries are counted in 32 bits, in steps of up to 16 x 512."""
    lib = bfa_lib.load()
    for vocab, code in ((2 ** 31 - 1 - 8192, -1), (2 ** 31 - 8192, -3), (2 ** 31 - 1 - 4096, -3), (2 ** 31 - 1, -3), (2 ** 40, -3)):
        # In range, the null pointers are the first thing wrong.
        assert lib.bfa_verify_tree(block(bfa_lib.VerifyArgs, **dict(VERIFY, vocab=vocab)), None) == code, vocab


@pytest.mark.parametrize("name,cls,base", [("bfa_rope", "RopeArgs", ROPE), ("bfa_cache_append", "AppendArgs", APPEND)])
def test_batches_that_the_grids_counter_cannot_pass_are_refused(name, cls, base):
    """A block goes on by up to 65535 sequences at a time, in 32 bits."""
    lib = bfa_lib.load()
    for batch, code in ((2 ** 31 - 1 - 65535, -1), (2 ** 31 - 65535, -3), (2 ** 31 - 1, -3), (2 ** 40, -3)):
        # In range, the null pointers are the first thing wrong.
        assert getattr(lib, name)(block(getattr(bfa_lib, cls), **dict(base, batch=batch)), None) == code, batch


def climbed(row):
    """Depths of one tree, a node at a time."""
    depth = []
    for n, up in enumerate(row):
        depth.append(0 if n == 0 else depth[up] + 1 if 0 <= up < n and depth[up] is not None else None)
    return [d or 0 for d in depth]


@pytest.mark.parametrize("row", [[-1, -1, 1, 2], [-1, 0, -1, 2, 3, 1], [7, 0, 1, -1, 3], [0, 0, 0], [-1], [-1, -1], [-5, 0, 1, 1, 0, 4]])
def test_depths_of_absent_nodes(row):
    """A node under an absent one is absent too, at depth 0."""
    assert td.tree_depths(torch.tensor(row, dtype=torch.int32)).tolist() == climbed(row)


@pytest.mark.parametrize("row", [[-1, 0, 2, 1], [-1, 0, 9, 2, 1], [-1, 2, 1, 0], [-1, 1, 0], [-1, 0, 1, 2 ** 31 - 1, 3], [-1, -2, 1, -2 ** 31, 0],
                                 [-1, 3, 1, 2]])
def test_depths_of_parents_outside_their_range(row):
    """A parent that is no earlier node is not followed: its node is absent."""
    for t in (torch.tensor(row, dtype=torch.int32), torch.tensor([row, [-1] + list(range(len(row) - 1))], dtype=torch.int32)):
        d = td.tree_depths(t)
        assert d.dtype == torch.int32 and d.shape == t.shape
        assert (d[0] if d.dim() == 2 else d).tolist() == climbed(row)
        if d.dim() == 2:
            assert d[1].tolist() == list(range(len(row)))


@pytest.mark.parametrize("n", [1, 2, 3, 31, 32, 33, 64, 200])
def test_depths_of_larger_trees(n):
    g = torch.Generator().manual_seed(n)
    rows = [[-1] + list(range(n - 1)), [-1] + [0] * (n - 1)]
    rows += [[-1] + [int(torch.randint(-1, i, (), generator=g)) for i in range(1, n)] for _ in range(6)]
    assert td.tree_depths(torch.tensor(rows, dtype=torch.int32)).tolist() == [climbed(row) for row in rows]
    assert td.tree_depths(torch.tensor(rows)).tolist() == [climbed(row) for row in rows]


def test_depths_take_few_operations():
    """A decoding step of a changing tree forms them anew: a few operations a
    doubling, not a few a node."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Count.n += 1
            return func(*args, **(kwargs or {}))
    with Count():
        td.tree_depths(torch.tensor([[-1] + list(range(63))], dtype=torch.int32))
    assert Count.n <= 50


def test_tangents_are_refused():
    """Forward-mode differentiation would lose the tangent without a word."""
    import torch.autograd.forward_ad as fwd
    q, k = torch.randn(1, 2, 3, 64), torch.randn(1, 1, 3, 64)
    pages = torch.zeros(1, 1, 16, 64)
    cache = td.PagedKVCache(pages, pages, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    slopes = torch.ones(2)
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: td.tree_attention(dual(q), k, k, cache), lambda: td.tree_attention(q, k, dual(k), cache),
                     lambda: td.tree_attention(q, k, k, cache._replace(k_pages=dual(pages))),
                     lambda: td.tree_attention(q, k, k, cache, alibi_slope=dual(slopes)),
                     lambda: td.cache_append(cache, dual(k), k), lambda: td.cache_append(cache._replace(v_pages=dual(pages)), k, k)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
