"""Accumulated attention weights of cached keys on the GPU, against 64 bits.  Needs a real MI355X: run with -m gpu."""
import math

import numpy as np
import pytest

from cache_util import rounded, to64
from test_cache_gpu import ATTENTIONS, attend, attention_case, device, heads_view, ints
from test_spmm_gpu import torch_cuda  # noqa: F401

pytestmark = pytest.mark.gpu


def received64(q, k, lse, position, shared, scale, causal, window, last, there=None):
    """What the tokens of one sequence give its keys: heads x keys, and how far fp32 may be off that.
    A score: dim products and sums, (dim + 4) roundings of 2^-24 of scale * sum |q k| at most; its difference to lse: a rounding of
    either and of itself, four of the larger one with the change to units of ln 2; an exponential of two ulps; a sum of rows."""
    T, H, D = q.shape
    keys, heads = len(k), H // shared
    j = np.arange(keys)
    out, off = np.zeros((heads, keys)), np.zeros((heads, keys))
    for t in range(T):
        if last and t < T - last:
            continue
        seen = np.ones(keys, bool) if there is None else there.copy()
        if causal:
            seen &= j <= position[t]
        if window:
            seen &= j > position[t] - window
        for h in range(H):
            with np.errstate(all="ignore"):
                s = scale * (k[:, h // shared] @ q[t, h])
                p = np.where(seen, np.exp(s - lse[t, h]), 0.0)
                reach = abs(scale) * (np.abs(k[:, h // shared]) @ np.abs(q[t, h]))
                size = np.where(np.isneginf(lse[t, h]), 0.0, np.abs(lse[t, h]))
                off[h // shared] += np.where(seen, p * 1.01 * ((D + 4) * 2.0 ** -24 * reach + 4 * 2.0 ** -24 * (size + np.abs(s)) + 2.0 ** -22), 0.0)
            out[h // shared] += p
    rows = (min(T, last) if last else T) * shared
    return out, off + out * (rows + 4) * 2.0 ** -24 + 2.0 ** -126


class Case:
    def __init__(self, torch, hs, dtype, number, order=0, layers=1, seed=0, gaps=True):
        self.torch = torch
        (self.st, self.batch, self.attention, self.q, self.k, self.v, self.new, self.old, self.rows, self.scale, self.window, self.causal) = attention_case(
            torch, hs, dtype, number, order, seed, layers)
        self.layer = layers - 1
        rng = np.random.default_rng(number + seed)
        st = self.st
        # (as many tokens of a row as the longest sequence has, and some)
        self.places = max(len(x) for x in self.k) + 5
        shape = (layers, st.table.shape[0], st.heads, self.places)
        # rows of weights with something between them
        big = torch.full((layers, shape[1], st.heads + 1, self.places + 3), -5.0, device="cuda")
        self.weights = big[:, :, 1:, 2:-1] if gaps else torch.zeros(shape, device="cuda")
        self.before = np.abs(rng.standard_normal(shape)).astype(np.float32)
        self.weights.copy_(torch.from_numpy(self.before))
        self.big = big
        self.handle = hs.Weights(self.weights.data_ptr(), *self.weights.stride()[:3])
        _, self.lse = attend(torch, hs, st, self.batch, self.attention, self.q, layer=self.layer)
        self.starts, self.known = np.concatenate([[0], np.cumsum(self.new)]), {}

    def run(self, hs, decay=1.0, last=0, attention=None):
        torch, attention = self.torch, attention or self.attention
        qd = device(torch, self.q, self.st.dtype)
        need = self.st.handle.weigh_workspace(self.batch, attention, last=last)
        w = torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")
        self.st.handle.weigh(self.layer, self.batch, attention, heads_view(hs, qd), self.lse.data_ptr(), self.handle, decay=decay, last=last,
                             workspace=w.data_ptr(), workspace_bytes=w.numel(), stream=torch.cuda.current_stream().cuda_stream)
        self.kept = (qd, w)
        return to64(self.weights)

    def check(self, got, decay, last, there=None):
        """`there`: the same in every call."""
        before, lse = self.before, to64(self.lse)
        want, off = before.astype(np.float64).copy(), np.zeros(before.shape)
        for b, row in enumerate(self.rows):
            a, n, o = self.starts[b], self.new[b], self.old[b]
            if not n:
                continue
            if (b, last) not in self.known:
                self.known[b, last] = received64(self.q[a:a + n], self.k[b], lse[a:a + n], np.arange(o, o + n), self.q.shape[1] // self.st.heads, self.scale, self.causal,
                                                 self.window, last, None if there is None else there[b])
            give, d = self.known[b, last]
            w = want[self.layer, row, :, :o + n]
            w[:, :o] *= float(np.float32(decay))
            w[:, o:] = 0.0
            w += give
            off[self.layer, row, :, :o + n] = d + np.abs(w) * 3 * 2.0 ** -24
        assert np.isfinite(got).all()
        # (what is behind a sequence's last token, or another sequence's or layer's, stays to the bit)
        assert (np.abs(got - want) <= off).all(), (np.abs(got - want) - off).max()


def hints(hs, c):
    return [hs.Attention(c.attention.q_heads, float(c.scale), causal=c.causal, window=c.window, longest_chunk=chunk, longest=longest)
            for chunk, longest in ((1, 0), (5000, 100000), (0, 1), (5000, 1), (300, 2000))]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", range(len(ATTENTIONS)))
def test_weigh(torch_cuda, hs, dtype, number):
    c = Case(torch_cuda, hs, dtype, number, order=number % 2, layers=1 + number % 2)
    got = c.run(hs, decay=0.75)
    c.check(got, 0.75, 0)
    outside = c.big.clone()
    outside[:, :, 1:, 2:-1] = -5.0
    assert (outside == -5.0).all()
    # the hints choose kernels and parts; the same call gives the same bits
    for a in hints(hs, c):
        c.weights.copy_(torch_cuda.from_numpy(c.before))
        c.check(c.run(hs, decay=0.75, attention=a), 0.75, 0)
    c.weights.copy_(torch_cuda.from_numpy(c.before))
    assert np.array_equal(c.run(hs, decay=0.75), got)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [4, 5, 6, 8, 9, 13, 16, 24, 26])
@pytest.mark.parametrize("last", [1, 3, 32, 100])
def test_the_last_tokens_count(torch_cuda, hs, dtype, number, last):
    c = Case(torch_cuda, hs, dtype, number, seed=1)
    c.check(c.run(hs, decay=0.5, last=last), 0.5, last)
    for a in hints(hs, c):
        c.weights.copy_(torch_cuda.from_numpy(c.before))
        c.check(c.run(hs, decay=0.5, last=last, attention=a), 0.5, last)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_the_weights_a_token_gives_are_one(torch_cuda, hs, dtype):
    # without anything before, what a sequence's keys receive is its rows' number
    torch = torch_cuda
    for number in (3, 8, 13):
        c = Case(torch, hs, dtype, number, gaps=False)
        c.weights.zero_()
        got = c.run(hs)
        shared = c.q.shape[1] // c.st.heads
        for b, row in enumerate(c.rows):
            rows, off = c.new[b] * shared, 0.0
            _, d = received64(c.q[c.starts[b]:c.starts[b] + c.new[b]], c.k[b], to64(c.lse)[c.starts[b]:c.starts[b] + c.new[b]], np.arange(c.old[b], c.old[b] + c.new[b]), shared,
                              c.scale, c.causal, c.window, 0)
            # (each lse is off by what its own test allows: its roundings are of its score's and a sum's)
            off = d.sum(1) + rows * ((c.q.shape[2] + 8) * 2.0 ** -24 * 40 + (len(c.k[b]) / 16 + 64) * 2.0 ** -24 + 2.0 ** -20)
            assert (np.abs(got[0, row, :, :len(c.k[b])].sum(1) - rows) <= off).all()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [4, 9, 13, 17, 24])
def test_keys_without_a_page_receive_nothing(torch_cuda, hs, dtype, number):
    torch = torch_cuda
    c = Case(torch, hs, dtype, number, seed=7)
    rng, page, there = np.random.default_rng(number), c.st.page_tokens, []
    for row, k in zip(c.rows, c.k):
        gone = rng.random(-(-len(k) // page)) < 0.4
        for p in np.nonzero(gone)[0]:
            c.st.table[int(row), int(p)] = int(rng.choice([-1, c.st.pages, 0x7FFFFFFF, -7]))
        there.append(~gone[np.arange(len(k)) // page])
    _, c.lse = attend(torch, hs, c.st, c.batch, c.attention, c.q)
    c.check(c.run(hs), 1.0, 0, there=there)
    for a in hints(hs, c):
        c.weights.copy_(torch.from_numpy(c.before))
        c.check(c.run(hs, attention=a), 1.0, 0, there=there)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [6, 8, 9, 13, 24])
def test_what_is_masked_receives_nothing(torch_cuda, hs, dtype, number):
    # infinities and NaN in keys: those keys alone have what they make of the rows that see them
    torch = torch_cuda
    c = Case(torch, hs, dtype, number, seed=3)
    bad = []
    for b, row in enumerate(c.rows):
        if c.new[b] < 2:
            continue
        j = c.old[b] + c.new[b] - 1
        keys = c.k[b].copy()
        keys[j] = math.nan
        c.st.store(0, int(row), 0, keys)
        bad.append((row, j))
    assert bad
    for a in [c.attention] + hints(hs, c):
        c.weights.copy_(torch.from_numpy(c.before))
        got = c.run(hs, last=0, attention=a)
        for row, j in bad:
            assert np.isnan(got[0, row, :, j]).all()
            got[0, row, :, j] = 0.0
        calm = c.before.copy()
        keep = [x.copy() for x in c.k]
        # without those keys: no row but the last ones sees them, so the others' keys have what they had
        for b, row in enumerate(c.rows):
            if c.new[b] >= 2:
                c.k[b][c.old[b] + c.new[b] - 1] = 0.0
        lse = to64(c.lse)
        want = calm.astype(np.float64)
        for b, row in enumerate(c.rows):
            n, o, s = c.new[b], c.old[b], c.starts[b]
            if not n:
                continue
            give, off = received64(c.q[s:s + n], c.k[b], lse[s:s + n], np.arange(o, o + n), c.q.shape[1] // c.st.heads, c.scale, c.causal, c.window, 0)
            w = want[0, row, :, :o + n]
            w[:, o:] = 0.0
            w += give
            m = o + n - (1 if n >= 2 else 0)
            assert (np.abs(got[0, row, :, :m] - w[:, :m]) <= off[:, :m] + np.abs(w[:, :m]) * 3 * 2.0 ** -24).all()
        c.k = keep


def test_rows_that_see_nothing_and_odd_scales(torch_cuda, hs):
    torch = torch_cuda
    c = Case(torch, hs, 2, 9, seed=2)
    for b in range(len(c.rows)):
        c.st.table[int(c.rows[b])] = -1
    _, lse = attend(torch, hs, c.st, c.batch, c.attention, c.q)
    assert torch.isneginf(lse).all()
    c.lse = lse
    c.check(c.run(hs, decay=0.25), 0.25, 0, there=[np.zeros(len(k), bool) for k in c.k])
    for scale in (0.0, -0.3):
        c = Case(torch, hs, 2, 9, seed=2)
        c.scale = np.float64(np.float32(scale))
        c.attention = hs.Attention(c.attention.q_heads, scale, causal=c.causal, window=c.window, longest_chunk=c.attention.longest_chunk, longest=c.attention.longest)
        _, c.lse = attend(torch, hs, c.st, c.batch, c.attention, c.q)
        c.check(c.run(hs), 1.0, 0)


def test_bad_numbers_and_other_sequences(torch_cuda, hs):
    torch = torch_cuda
    c = Case(torch, hs, 0, 8)
    st = c.st
    good = to64(c.weights).copy()
    for starts in ([-4, -3, -2, -1, 0], [9999] * 5, [5, 4, 3, 2, 1], [0x7FFFFFFF] * 5):
        st.kept[0].copy_(ints(torch, starts))
        assert np.array_equal(c.run(hs), good)
    st.kept[0].copy_(ints(torch, c.starts))
    st.kept[1].copy_(ints(torch, [-1, 99, 0x7FFFFFFF, -7]))
    assert np.array_equal(c.run(hs), good)


def test_a_captured_call_on_another_stream(torch_cuda, hs):
    torch = torch_cuda
    for number in (4, 8, 13):
        c = Case(torch, hs, 2, number)
        want = c.run(hs, decay=0.5)
        torch.cuda.synchronize()
        qd, side = device(torch, c.q, 2), torch.cuda.Stream()
        w = torch.zeros(max(16, c.st.handle.weigh_workspace(c.batch, c.attention)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

        def call():
            c.st.handle.weigh(c.layer, c.batch, c.attention, heads_view(hs, qd), c.lse.data_ptr(), c.handle, decay=0.5, workspace=w.data_ptr(), workspace_bytes=w.numel(),
                              stream=torch.cuda.current_stream().cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for i in range(4):
            c.weights.copy_(torch.from_numpy(c.before))
            torch.cuda.synchronize()
            if i % 2:
                with torch.cuda.stream(side):
                    call()
            else:
                graph.replay()
            torch.cuda.synchronize()
            assert np.array_equal(to64(c.weights), want)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [4, 6, 9, 13, 24])
def test_rows_whose_lse_is_infinite_give_nothing(torch_cuda, hs, dtype, number):
    # every third one says that it sees nothing, though there are keys that it would see
    c = Case(torch_cuda, hs, dtype, number, seed=5)
    full = c.lse.clone()
    c.lse.view(-1)[::3] = -np.inf
    for a in [None] + hints(hs, c):
        c.weights.copy_(torch_cuda.from_numpy(c.before))
        got = c.run(hs, decay=0.5, attention=a)
        assert np.isfinite(got).all()
    # as with those rows' lse so large that nothing is left of what they give
    c.lse = full
    c.lse.view(-1)[::3] = 1e30
    c.weights.copy_(torch_cuda.from_numpy(c.before))
    assert np.array_equal(c.run(hs, decay=0.5, attention=a), got)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [3, 4, 6, 8, 9, 11, 13, 16, 24])
def test_rows_whose_scores_are_all_minus_infinity_give_nothing(torch_cuda, hs, dtype, number):
    # an infinite element of a query: whatever a kernel has behind a head's last element, that row gives nothing
    torch = torch_cuda
    c = Case(torch, hs, dtype, number, seed=6)
    for b, row in enumerate(c.rows):
        c.k[b][..., 0] = np.abs(c.k[b][..., 0]) + 0.5
        c.st.store(c.layer, int(row), 0, c.k[b])
    rows = c.q.reshape(-1, c.q.shape[2])
    rows[::3, 0] = -math.inf
    _, c.lse = attend(torch, hs, c.st, c.batch, c.attention, c.q, layer=c.layer)
    assert torch.isneginf(c.lse.view(-1)[::3]).all()
    got = []
    for a in [None] + hints(hs, c):
        c.weights.copy_(torch.from_numpy(c.before))
        got.append(c.run(hs, decay=0.5, attention=a))
        assert np.isfinite(got[-1]).all()
    # to the bit what the others give where those rows are zeros
    rows[::3] = 0.0
    for a, x in zip([None] + hints(hs, c), got):
        c.weights.copy_(torch.from_numpy(c.before))
        assert np.array_equal(c.run(hs, decay=0.5, attention=a), x)
