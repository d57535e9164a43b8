"""The example that runs sparse products, rotary positions, the paged cache and attention together, against dense blocks in 64
bits.  Needs a real MI355X: run with -m gpu."""
import importlib.util
import os

import numpy as np
import pytest

from test_spmm_gpu import torch_cuda  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [dict(hidden=256, heads=4, kv_heads=2, keep=0.2, layers=2, prompts=(70, 33, 5), beams=3, steps=3, page_tokens=16),
                                   dict(hidden=320, heads=4, kv_heads=4, keep=0.3, layers=1, prompts=(150, 1), beams=2, steps=2, page_tokens=7)])
def test_pruned_attention_blocks(torch_cuda, sizes):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "pruned_attention.py")
    spec = importlib.util.spec_from_file_location("pruned_attention", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got, want, largest = example.run(**sizes)
    # roundings to fp16 (2^-11 each): of q, k, v, turned q and k, which move a score by up to four times that of itself and so the weights,
    # of weights, sums, the last product and the sum with x, in every layer
    bound = sizes["layers"] * (6 + 4 * largest) * 2.0 ** -11
    assert np.linalg.norm(got - want) <= bound * np.linalg.norm(want)
