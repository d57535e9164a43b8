"""Eviction from a cache on the GPU, against lists of numbers on the CPU: everything is equal to the bit.  Needs a real MI355X: run
with -m gpu."""
import math

import numpy as np
import pytest

from cache_util import State, to64
from test_cache_gpu import ints
from test_spmm_gpu import torch_cuda  # noqa: F401

pytestmark = pytest.mark.gpu


class Model:
    """The same cache as numbers: per layer and head a sequence's stored tokens by the names they were given."""

    def __init__(self, torch, hs, dtype, pages, page, heads, dim, sequences, places, layers, order=0, gap=0):
        self.st = State(torch, hs, dtype, pages, page, heads, dim, sequences, places, layers=layers, order=order, page_gap=gap, layer_gap=3 * gap)
        self.torch, self.hs = torch, hs
        self.weights = torch.zeros((layers, sequences, heads, places * page), device="cuda")
        self.handle = hs.Weights(self.weights.data_ptr(), *self.weights.stride()[:3])
        # every element its own value: keys and values of a page's slot
        for which in (0, 1):
            x = self.st.view(which)
            n = torch.arange(x.numel(), device="cuda") * 2 + which
            x.copy_(((n * 2654435761) % 2039).reshape(x.shape).to(x.dtype))

    def snapshot(self):
        st = self.st
        return dict(table=st.table.cpu().numpy().copy(), lengths=st.lengths.cpu().numpy().copy(), references=st.references.cpu().numpy().copy(),
                    pools=[to64(st.view(w)) for w in (0, 1)], weights=self.weights.cpu().numpy().copy())

    def evict(self, parents, children, keep, first, last, kept=True, status=True, workspace=None):
        torch, st = self.torch, self.st
        n = len(parents)
        need = st.handle.evict_workspace(n, keep)
        w = torch.full((max(need, 64),), 0x5A, dtype=torch.uint8, device="cuda") if workspace is None else workspace
        if workspace is None:
            w[:64] = 0
        out = torch.full((st.layers, n, st.heads, keep), 77, dtype=torch.int32, device="cuda")
        s = ints(torch, [123])
        pd, cd = ints(torch, parents), None if children is None else ints(torch, children)
        st.handle.evict(n, pd.data_ptr(), cd.data_ptr() if cd is not None else 0, self.handle, keep, first=first, last=last, kept=out.data_ptr() if kept else 0,
                        status=s.data_ptr() if status else 0, workspace=w.data_ptr(), workspace_bytes=w.numel(), stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return out.cpu().numpy(), int(s), w

    def expect(self, before, parents, children, keep, first, last):
        """The state after the call; pools only where a child's tokens are."""
        st, page = self.st, self.st.page_tokens
        children = parents if children is None else children
        table, lengths, references, weights = (before[x].copy() for x in ("table", "lengths", "references", "weights"))
        free = [i for i in range(st.pages) if before["references"][i] <= 0]
        kept = np.full((st.layers, len(parents), st.heads, keep), -1)
        given = missing = 0
        tokens = {}                                         # child: (kept by layer and head, parent)
        gave = []
        valid = lambda s: 0 <= s < len(lengths)  # noqa: E731
        for i, (p, c) in enumerate(zip(parents, children)):
            if not valid(p):
                continue
            length = max(int(before["lengths"][p]), 0)
            have = [j for j in range(min(length, table.shape[1] * page)) if 0 <= before["table"][p][j // page] < st.pages]
            anyway = [j for j in have if j < first or j >= length - last]
            m = min(keep, len(have))
            for a in range(st.layers):
                for h in range(st.heads):
                    w = before["weights"][a, p, h]
                    if m == len(have):
                        at = have
                    else:
                        rest = [j for j in have if not (j < first or j >= length - last)]
                        score = np.where(np.isnan(w[rest]), -np.inf, w[rest])
                        isnan = np.isnan(w[rest])
                        order = sorted(range(len(rest)), key=lambda x: (isnan[x], -score[x], x))
                        at = sorted(anyway + [rest[x] for x in order[:m - len(anyway)]])
                    kept[a, i, h, :m] = at
            if not valid(c) or (p == c and length <= keep):
                continue
            in_place = p == c and sum(1 for x in parents if x == p) == 1
            need = -(-m // page)
            mine = [t for t in before["table"][p][:-(-length // page)] if 0 <= t < st.pages][:need]
            row = [int(t) if in_place and before["references"][t] == 1 else None for t in mine]
            fresh = sum(t is None for t in row)
            gave.append((i, given, fresh))
            given += fresh
            tokens[c] = (i, p, m, row, given - fresh, fresh)
        found = min(given, len(free))
        missing = given - found
        done = {}
        for c, (i, p, m, row, at, fresh) in tokens.items():
            if fresh and at + fresh > found:
                continue
            new = iter(free[at:at + fresh])
            row = [next(new) if t is None else t for t in row]
            old = before["table"][c]
            for t in old:
                if 0 <= t < st.pages:
                    references[t] -= 1
            for t in row:
                references[t] += 1
            table[c] = -1
            table[c][:len(row)] = row
            lengths[c] = m
            weights[:, c] = 0
            for a in range(st.layers):
                for h in range(st.heads):
                    weights[a, c, h, :m] = before["weights"][a, p, h][kept[a, i, h, :m]]
            done[c] = (i, p, m)
        return dict(table=table, lengths=lengths, references=references, weights=weights), kept, missing, done

    def check(self, parents, children, keep, first, last, **kw):
        before = self.snapshot()
        kept, status, w = self.evict(parents, children, keep, first, last, **kw)
        after = self.snapshot()
        want, lists, missing, done = self.expect(before, parents, children, keep, first, last)
        if kw.get("kept", True):
            assert np.array_equal(kept, lists)
        if kw.get("status", True):
            assert status == missing
        for x in ("table", "lengths", "references"):
            assert np.array_equal(after[x], want[x]), x
        assert np.array_equal(after["weights"], want["weights"], equal_nan=True)
        assert not w[:64].any()
        st, page = self.st, self.st.page_tokens
        written = np.zeros((st.pages, page), bool)
        for c, (i, p, m) in done.items():
            slot = np.arange(m)
            written[want["table"][c][slot // page], slot % page] = True
            for a in range(st.layers):
                for h in range(st.heads):
                    j = lists[a, i, h, :m]
                    for b, x in zip(before["pools"], after["pools"]):
                        assert np.array_equal(x[a, want["table"][c][slot // page], h, slot % page], b[a, before["table"][p][j // page], h, j % page])
        # nothing else is written
        for b, x in zip(before["pools"], after["pools"]):
            assert np.array_equal(x.transpose(1, 3, 0, 2, 4)[~written], b.transpose(1, 3, 0, 2, 4)[~written])
        return missing


def filled(torch, hs, seed, dtype, order, lengths, page, heads, dim, layers, places, spare, extra=0, gap=0, kind="random"):
    rng = np.random.default_rng(seed)
    n = len(lengths) + extra
    pages = int(sum(-(-x // page) for x in lengths)) + spare
    m = Model(torch, hs, dtype, pages, page, heads, dim, n, places, layers, order, gap)
    m.st.place(rng, list(lengths) + [0] * extra)
    w = {"random": lambda s: rng.standard_normal(s) ** 3, "ties": lambda s: rng.integers(0, 3, s) / 4.0, "zeros": lambda s: np.zeros(s) * rng.choice([1.0, -1.0], s),
         "near": lambda s: (np.float32(1.0).view(np.int32) + rng.integers(0, 40, s)).astype(np.int32).view(np.float32),
         "odd": lambda s: rng.choice([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38, -3e38], s)}[kind](m.weights.shape)
    m.weights.copy_(torch.from_numpy(np.asarray(w, np.float32)))
    return m, rng


SIZES = [  # lengths, page, heads, dim, layers, keep, first, last
    ([1], 16, 1, 8, 1, 1, 0, 0),
    ([40, 5, 17], 16, 2, 64, 2, 16, 2, 5),
    ([33, 100, 0, 64], 7, 3, 36, 1, 20, 0, 0),
    ([700], 16, 4, 64, 2, 256, 4, 32),
    ([1030, 2500], 24, 2, 80, 2, 333, 1, 50),
    ([300, 299, 301], 1, 1, 128, 1, 300, 100, 200),
    ([5000, 20], 64, 1, 256, 1, 1500, 0, 700),
    ([90, 91], 32, 8, 5, 3, 31, 31, 0),
    ([64, 128], 16, 2, 128, 1, 64, 0, 64)]


@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
@pytest.mark.parametrize("number", range(len(SIZES)))
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_evict_in_place(torch_cuda, hs, dtype, number, kind):
    lengths, page, heads, dim, layers, keep, first, last = SIZES[number]
    m, rng = filled(torch_cuda, hs, number, dtype, number % 2, lengths, page, heads, dim, layers, -(-max(lengths) // page) + 1, 0, kind=kind)
    parents = list(rng.permutation(len(lengths)))
    assert m.check(parents, None if number % 3 else parents, keep, first, last) == 0
    # once more: nothing is left to do
    assert m.check(parents, None, keep, first, last) == 0


@pytest.mark.parametrize("kind", ["random", "zeros", "near"])
@pytest.mark.parametrize("number", range(len(SIZES)))
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_evict_into_others(torch_cuda, hs, dtype, number, kind):
    lengths, page, heads, dim, layers, keep, first, last = SIZES[number]
    n = len(lengths)
    m, rng = filled(torch_cuda, hs, number + 50, dtype, (number + 1) % 2, lengths, page, heads, dim, layers, -(-max(lengths) // page) + 2, 4 * n * (-(-keep // page)), extra=n,
                    gap=8 if number % 2 else 0, kind=kind)
    children = list(n + rng.permutation(n))
    for _ in range(3):                                      # the children's old pages are given back
        assert m.check(list(range(n)), children, keep, first, last) == 0
        m.weights[:, :n] = m.weights[:, :n].roll(1, -1)


@pytest.mark.parametrize("dtype", [0, 2])
def test_shared_pages_are_left_alone(torch_cuda, hs, dtype):
    # forks share their pages: an eviction of one of them takes new ones for those, and keeps its own
    torch = torch_cuda
    m, rng = filled(torch, hs, 5, dtype, 0, [200, 60], 16, 2, 64, 2, 20, 40, extra=3)
    st = m.st
    stream = torch.cuda.current_stream().cuda_stream
    p, c = ints(torch, [0, 0]), ints(torch, [2, 3])
    st.handle.fork(2, p.data_ptr(), c.data_ptr(), stream=stream)
    add, rows = ints(torch, [70, 9]), ints(torch, [2, 3])
    st.handle.extend(2, rows.data_ptr(), add.data_ptr(), stream=stream)
    torch.cuda.synchronize()
    m.weights.copy_(torch.from_numpy(np.abs(rng.standard_normal(m.weights.shape)).astype(np.float32)))
    assert (st.references.cpu().numpy() == 3).any()
    assert m.check([2, 1], None, 90, 3, 20) == 0
    assert m.check([0, 3, 2], None, 150, 0, 10) == 0
    assert m.check([0, 3], [4, 0], 33, 0, 0) == 0            # a parent that is another's child
    assert m.check([2, 2], [2, 1], 40, 0, 0) == 0            # one that stays and has another child
    assert m.check([1, 0, 2], [0, 2, 1], 25, 5, 5) == 0      # around


def test_pages_that_are_missing(torch_cuda, hs):
    torch = torch_cuda
    for seed in range(4):
        m, rng = filled(torch, hs, seed, 2, seed % 2, [150, 90, 200, 33], 16, 2, 32, 2, 14, 0, extra=1)
        # holes in the rows: their tokens are dropped before any other
        for s in range(4):
            for p in range(14):
                if rng.random() < 0.3:
                    t = int(m.st.table[s, p])
                    if 0 <= t < m.st.pages:
                        m.st.references[t] -= 1
                    m.st.table[s, p] = int(rng.choice([-1, m.st.pages, -9]))
        free = int((m.st.references <= 0).sum())
        assert free > 0
        m.check([0, 1, 2, 3], None, [100, 60, 31, 140][seed], 4, 8)
        m.check([2, 0], None, 20, 0, 20)


def test_a_pool_without_free_pages(torch_cuda, hs):
    m, _ = filled(torch_cuda, hs, 1, 0, 0, [100, 50, 64], 16, 2, 32, 1, 10, 3, extra=2)
    assert m.check([0, 1, 2], [3, 1, 4], 40, 0, 0) == 3       # three of six: the first child has them
    assert m.check([0, 2], [1, 4], 40, 2, 2) == 5              # (the second one gave one of its four back)
    assert m.check([0, 1, 2], None, 40, 2, 2) == 0            # in place nothing is wanted


def test_bad_numbers(torch_cuda, hs):
    m, rng = filled(torch_cuda, hs, 1, 0, 0, [100, 50, 64], 16, 2, 32, 2, 10, 30, extra=2)
    m.check([0, -1, 7, 2], [3, 4, 1, 0x7FFFFFFF], 40, 0, 0)
    m.check([0x7FFFFFFF, -5], None, 12, 0, 0)
    m.st.lengths.copy_(ints(m.torch, [100, -7, 100000, 3, 0]))     # lengths past the row, or below zero
    m.check([0, 1, 2], None, 30, 2, 0)


def test_without_lists_and_status(torch_cuda, hs):
    m, _ = filled(torch_cuda, hs, 3, 1, 0, [100, 50], 16, 2, 20, 2, 8, 8, extra=1)
    m.check([0, 1], [2, 1], 30, 2, 2, kept=False, status=False)
    s = ints(m.torch, [9])
    m.st.handle.evict(0, 0, 0, m.handle, 5, status=s.data_ptr(), stream=m.torch.cuda.current_stream().cuda_stream)
    assert int(s) == 0


def test_captured_and_on_another_stream(torch_cuda, hs):
    torch = torch_cuda
    m, _ = filled(torch, hs, 7, 2, 0, [500, 900], 16, 2, 64, 2, 60, 80, extra=2)
    st, before = m.st, m.snapshot()
    want, lists, _, _ = m.expect(before, [0, 1], [2, 3], 200, 4, 16)
    p, c, s = ints(torch, [0, 1]), ints(torch, [2, 3]), ints(torch, [0])
    need = st.handle.evict_workspace(2, 200)
    w = torch.zeros(need, dtype=torch.uint8, device="cuda")
    kept = torch.zeros(lists.shape, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()

    def call():
        st.handle.evict(2, p.data_ptr(), c.data_ptr(), m.handle, 200, first=4, last=16, kept=kept.data_ptr(), status=s.data_ptr(), workspace=w.data_ptr(), workspace_bytes=need,
                        stream=torch.cuda.current_stream().cuda_stream)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        for x in ("table", "lengths", "references"):
            getattr(st, x).copy_(torch.from_numpy(before[x]))
        m.weights.copy_(torch.from_numpy(before["weights"]))
        kept.zero_()
        torch.cuda.synchronize()
        if i % 2:
            with torch.cuda.stream(side):
                call()
        else:
            graph.replay()
        torch.cuda.synchronize()
        after = m.snapshot()
        assert np.array_equal(kept.cpu().numpy(), lists)
        for x in ("table", "lengths", "references", "weights"):
            assert np.array_equal(after[x], want[x]), x


@pytest.mark.parametrize("lengths,keep,first,last", [([9000, 40], 2100, 4, 300), ([16384, 8193], 8000, 0, 0), ([16385], 16384, 1, 1), ([30000, 12000], 5000, 100, 1000)])
@pytest.mark.parametrize("kind", ["random", "ties"])
def test_long_sequences(torch_cuda, hs, lengths, keep, first, last, kind):
    # more tokens than a workgroup's threads have in registers, and just as many
    m, rng = filled(torch_cuda, hs, keep, 2, 0, lengths, 64, 1, 8, 1, -(-max(lengths) // 64) + 1, 2 * len(lengths) * (-(-keep // 64)), extra=len(lengths), kind=kind)
    n = len(lengths)
    assert m.check(list(range(n)), list(range(n, 2 * n)), keep, first, last) == 0
    assert m.check(list(range(n)), None, keep, first, last) == 0


def test_many_entries(torch_cuda, hs):
    # more entries than a workgroup has threads, in place and into others
    n = 1100
    m, rng = filled(torch_cuda, hs, 3, 0, 0, [5 + (7 * i) % 30 for i in range(n)], 4, 1, 8, 1, 9, 2 * n * 3, extra=n)
    assert m.check(list(range(n)), list(range(n, 2 * n)), 9, 1, 2) == 0
    assert m.check(list(rng.permutation(n)), None, 9, 1, 2) == 0
