"""Prompts, beams that attend them together, weights that cached tokens receive and their eviction, as a serving loop runs them, against the
same in 64 bits.  Needs a real MI355X: run with -m gpu."""
import importlib.util
import os

import numpy as np
import pytest

from cache_util import to64
from test_spmm_gpu import torch_cuda  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [dict(hidden=256, heads=4, kv_heads=2, keep=0.2, layers=2, prompts=(70, 33, 90), beams=3, steps=3, page_tokens=16, budget=30),
                                   dict(hidden=320, heads=4, kv_heads=4, keep=0.3, layers=1, prompts=(150, 1), beams=2, steps=2, page_tokens=7, budget=20, first=0, last=3),
                                   dict(hidden=128, heads=2, kv_heads=1, keep=0.3, layers=2, prompts=(40,), beams=1, steps=2, page_tokens=8, budget=12, first=1, last=1, window=1),
                                   dict(hidden=512, heads=8, kv_heads=1, keep=0.2, layers=1, prompts=(300, 280), beams=2, steps=2, page_tokens=32, budget=100, window=0)])
def test_a_cache_of_bounded_length(torch_cuda, sizes):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "pruned_attention.py")
    spec = importlib.util.spec_from_file_location("pruned_attention", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    outs, decoder, mirror = example.run_bounded(**sizes)
    # roundings to fp16 (2^-11 each): of q, k, v, turned q and k, which move a score by up to four times that of itself and so the weights,
    # of weights, sums, the last product and the sum with x, in every layer
    bound = sizes["layers"] * (6 + 4 * mirror.largest) * 2.0 ** -11
    for got, want in outs:
        assert np.linalg.norm(got - want) <= bound * np.linalg.norm(want)
    # Layer 0: q and k are off by two roundings an element each, so a score and the logarithm of a row's sum by up to 4 x 2^-11 of scale |q| |k|, and what a key
    # receives by their difference's exponential; fp32's own roundings, 2^-24 of sums of up to some hundred terms and of scores, by less than 2^-12.
    off = np.exp(2 * 4 * 2.0 ** -11 * 1.01 * mirror.reach + 2.0 ** -12)
    for s, held in mirror.held.items():
        want, got = held[0][2], to64(decoder.weights[0, s])
        assert int(decoder.lengths[s]) == want.shape[1]
        assert (np.abs(got[:, : want.shape[1]] - want) <= (off - 1) * want + 2.0 ** -100).all()
        assert not got[:, want.shape[1]:].any()
    # nothing leaves that has received more than what stays, but for that (either may be off)
    assert mirror.worst <= off ** 2
    # no page is lost or named twice
    named = decoder.table.cpu().numpy()
    counts = np.bincount(named[named >= 0], minlength=decoder.references.numel())
    assert np.array_equal(decoder.references.cpu().numpy(), counts)
