"""The tree-decoding example: whatever the draft proposes, greedy decoding with a
tree gives the tokens of decoding one by one, in fewer passes."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("tree_decoding_example", os.path.join(ROOT, "examples", "tree_decoding.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.gpu
def test_tree_decoding_equals_single_token_decoding():
    same, passes, single = example().main(steps=60, dtype="fp32", batch=3)
    assert all(same) and passes < single


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_example_runs_in_16_bits(dtype):
    m = example()
    import torch
    prompt = torch.randint(0, 512, (2, 24), generator=torch.Generator().manual_seed(1)).to("cuda:0")
    history, passes = m.decode(m.Decoder(dtype=m.DTYPES[dtype]), prompt, 30)
    assert all(len(h) >= 54 and 0 <= min(h) and max(h) < 512 for h in history) and passes <= 30
