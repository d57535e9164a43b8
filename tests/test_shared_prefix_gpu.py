"""Attention over shared prefixes on the GPU, against attention in 64 bits; tolerances are derived in cache_util.  Needs a real
MI355X: run with -m gpu."""
import math

import numpy as np
import pytest

from cache_util import State, attend64, rounded, to64
from test_cache_gpu import assert_attended, device, heads_view, ints, laid_out
from test_spmm_gpu import torch_cuda  # noqa: F401

pytestmark = pytest.mark.gpu

# groups (rows of each), prefixes, own tokens behind them (a list to repeat), new tokens (a list to repeat), rows in no group in front of them, heads, shared, dim, page, window, causal
CASES = [
    ([1], [5], [0], [1], 0, 1, 1, 8, 16, 0, True),
    ([3], [40], [0, 7, 30], [1], 0, 2, 4, 64, 16, 0, True),
    ([8], [600], [5, 90, 33], [1], 0, 2, 4, 128, 16, 0, True),
    ([2, 5, 1], [33, 300, 64], [0, 1, 50], [1, 3], 2, 2, 3, 96, 24, 0, True),
    ([4, 0, 3], [100, 50, 0], [20, 5], [2, 0, 1], 1, 1, 2, 40, 7, 0, True),
    ([20], [1100], [3, 400, 0], [1], 0, 4, 8, 128, 16, 0, True),
    ([6, 3], [700, 129], [0, 40], [30, 1, 65], 1, 2, 2, 128, 64, 0, True),
    ([5], [500], [60, 0, 200], [7], 0, 2, 4, 64, 32, 90, True),
    ([5, 2], [90, 400], [10, 300], [40, 3], 0, 1, 4, 80, 10, 250, True),
    ([3, 2], [70, 130], [9, 0], [5, 1], 1, 2, 2, 64, 16, 0, False),
    ([3], [200], [4], [70, 9], 0, 1, 2, 160, 16, 0, True),
    ([2], [77], [30, 1], [3], 0, 1, 1, 256, 5, 0, True),
    ([70], [150], [2, 0, 11], [1], 3, 2, 1, 64, 1, 0, True),
    ([1] * 9, [64, 5, 200], [8], [1, 2], 0, 2, 4, 128, 16, 0, True),
    ([9], [3000], [0, 20], [16], 0, 1, 4, 104, 48, 0, True)]


def at(x, i):
    return x[i % len(x)]


class Case:
    def __init__(self, torch, hs, dtype, number, order=0, layers=1, seed=0, whole=False):
        groups, prefixes, rests, news, loose, heads, shared, dim, page, self.window, self.causal = CASES[number]
        rng = np.random.default_rng(100 * number + seed)
        n = sum(groups) + loose
        self.groups, self.loose, self.n = groups, loose, n
        self.new = np.array([at(news, i) for i in range(n)])
        group = np.concatenate([np.full(loose, -1), np.repeat(np.arange(len(groups)), groups)]).astype(int)
        self.prefix = np.array([at(prefixes, i) for i in range(len(groups))])
        common = np.where(group >= 0, np.append(self.prefix, 0)[group], 0)
        # (a loose row has something of its own)
        self.old = common + np.array([at(rests, i) for i in range(n)]) + (group < 0) * 13
        lengths = self.old + self.new
        self.st = st = State(torch, hs, dtype, int(sum(-(-x // page) for x in lengths)) + 2, page, heads, dim, n + 2, 6000 // page + 2, layers=layers, order=order)
        self.rows = rng.permutation(n + 2)[:n]
        by_row = np.zeros(n + 2, int)
        by_row[self.rows] = lengths
        st.place(rng, by_row)
        self.k, self.v = ([rounded(torch, rng.standard_normal((x, heads, dim)) * 1.5, dtype) for x in lengths] for _ in range(2))
        firsts = np.concatenate([[0], np.cumsum(groups)]) + loose
        self.firsts = firsts
        for b in range(n):
            for which, x in ((0, self.k), (1, self.v)):
                mine = x[b].copy()
                lead = firsts[group[b]] if group[b] >= 0 else b
                if lead != b:
                    # its own pages of the prefix are not read; its first sequence may hold less than the prefix
                    common_here = min(common[b], len(x[lead]))
                    x[b][:common_here] = x[lead][:common_here]
                    mine[:common_here] = math.nan
                st.store(layers - 1, int(self.rows[b]), which, mine)
        self.q = rounded(torch, rng.standard_normal((int(self.new.sum()), heads * shared, dim)) * 1.5, dtype)
        self.starts, self.rd, self.fd, self.pd = (ints(torch, x) for x in (np.concatenate([[0], np.cumsum(self.new)]), self.rows, firsts, self.prefix))
        self.batch = hs.Batch(n, int(self.new.sum()), self.starts.data_ptr(), self.rd.data_ptr())
        self.scale = np.float64(np.float32(1.0 / math.sqrt(dim)))
        self.hint = dict(most_tokens=max(int(self.new[firsts[g]:firsts[g + 1]].sum()) for g in range(len(groups))), longest=int(self.prefix.max()))
        self.attention = self.hints(hs, int(self.new.max()), int(lengths.max()))
        self.layer, self.dtype, self.dim = layers - 1, dtype, dim

    def hints(self, hs, chunk, longest):
        return hs.Attention(self.q.shape[1], float(self.scale), causal=self.causal, window=self.window, longest_chunk=chunk, longest=longest)

    def prefixes(self, hs, **hint):
        return hs.Prefix(len(self.groups), self.fd.data_ptr(), self.pd.data_ptr(), **(hint or self.hint))

    def run(self, torch, hs, attention=None, prefix=None, layout="tokens", lse=True, workspace=None):
        attention, prefix = attention or self.attention, prefix or self.prefixes(hs)
        qd = device(torch, self.q, self.dtype)
        out = laid_out(torch, torch.full(tuple(qd.shape), math.nan, dtype=qd.dtype, device="cuda"), layout)
        l = torch.full(tuple(qd.shape[:2]), math.nan, device="cuda")
        need = self.st.handle.attend_shared_workspace(self.batch, prefix, attention)
        # (no more than it asks for; what is not counters may hold anything)
        w = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda") if workspace is None else workspace
        if workspace is None:
            w[: 4 * 16384] = 0
        self.st.handle.attend_shared(self.layer, self.batch, prefix, attention, heads_view(hs, qd), heads_view(hs, out), lse=l.data_ptr() if lse else 0,
                                     workspace=w.data_ptr(), workspace_bytes=w.numel(), stream=torch.cuda.current_stream().cuda_stream)
        self.kept = (qd, w)
        return out, l

    def want(self, there=None):
        parts, t = [], 0
        for b in range(self.n):
            parts.append(attend64(self.q[t:t + self.new[b]], self.k[b], self.v[b], np.arange(self.old[b], self.old[b] + self.new[b]), self.scale, self.causal, self.window,
                                  None if there is None else there[b][None]))
            t += self.new[b]
        return [np.concatenate(x) for x in zip(*parts)]


# hints that choose other kernels and parts: many rows and keys, few of them, none
def other_hints(hs, c):
    return [(c.hints(hs, 5000, 6000), c.prefixes(hs, most_tokens=5000, longest=6000)), (c.hints(hs, 1, 0), c.prefixes(hs, most_tokens=1, longest=1)),
            (c.hints(hs, 0, 1), c.prefixes(hs, most_tokens=0, longest=0)), (c.hints(hs, 4000, 40000), c.prefixes(hs, most_tokens=100000, longest=100))]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", range(len(CASES)))
def test_attend_shared(torch_cuda, hs, dtype, number):
    torch = torch_cuda
    for order, layout, layers in ((0, "tokens", 1), (1, "features", 2)):
        c = Case(torch, hs, dtype, number, order, layers)
        want = c.want()
        out, lse = c.run(torch, hs, layout=layout)
        assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)
        again, _ = c.run(torch, hs, layout=layout, lse=False)
        assert torch.equal(out, again)
        for attention, prefix in other_hints(hs, c):
            out, lse = c.run(torch, hs, attention, prefix, layout="gaps")
            assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [2, 3, 6, 8, 10])
def test_pages_that_are_gone_are_not_seen(torch_cuda, hs, dtype, number):
    # pages of the first sequence are the prefix's; the others' pages of the same tokens do not matter
    torch = torch_cuda
    c = Case(torch, hs, dtype, number, seed=5)
    page, rng = c.st.page_tokens, np.random.default_rng(number)
    there = [np.ones(len(x), bool) for x in c.k]
    gone = [rng.random(-(-len(x) // page)) < 0.4 for x in c.k]
    for b in range(c.n):
        for p in np.nonzero(gone[b])[0]:
            c.st.table[int(c.rows[b]), int(p)] = int(rng.choice([-1, c.st.pages, 0x7FFFFFFF, -7]))
    group = np.searchsorted(c.firsts, np.arange(c.n), side="right") - 1
    for b in range(c.n):
        lead, common = (c.firsts[group[b]], int(c.prefix[group[b]])) if group[b] >= 0 else (b, 0)
        j = np.arange(len(c.k[b]))
        row = np.where(j < min(common, len(c.k[lead])), True, False)
        mine = gone[b][j // page]
        first = gone[lead][np.minimum(j // page, len(gone[lead]) - 1)] if len(gone[lead]) else mine
        there[b] = ~np.where(row, first, mine)
    want = c.want(there)
    for attention, prefix in [(None, None)] + other_hints(hs, c):
        out, lse = c.run(torch, hs, attention, prefix)
        assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_chunks_that_begin_within_the_prefix(torch_cuda, hs, dtype):
    # a prefix that is said to be longer: causal tokens see of it what stands in front of them, and its first sequence's tokens are the others'
    torch = torch_cuda
    for number in (6, 8, 10, 14):
        c = Case(torch, hs, dtype, number, seed=2)
        more = c.prefix + np.array([25, 3, 60])[np.arange(len(c.prefix)) % 3]
        group = np.searchsorted(c.firsts, np.arange(c.n), side="right") - 1
        for b in range(c.n):
            if group[b] >= 0 and b != c.firsts[group[b]]:
                lead = c.firsts[group[b]]
                n = min(int(more[group[b]]), len(c.k[lead]), len(c.k[b]))
                c.k[b][:n], c.v[b][:n] = c.k[lead][:n], c.v[lead][:n]
        c.pd.copy_(ints(torch, more))
        want = c.want()
        for attention, prefix in [(None, None)] + other_hints(hs, c):
            out, lse = c.run(torch, hs, attention, prefix)
            assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [3, 6, 8, 9])
def test_what_is_masked_does_not_reach_the_result(torch_cuda, hs, dtype, number):
    # infinities and NaN behind the first token of the prefix's rows that sees them: only those tokens have them
    torch = torch_cuda
    c = Case(torch, hs, dtype, number, seed=3)
    rng = np.random.default_rng(number)
    group = np.searchsorted(c.firsts, np.arange(c.n), side="right") - 1
    hit = [np.zeros(m, bool) for m in c.new]
    clean_k, clean_v = [x.copy() for x in c.k], [x.copy() for x in c.v]

    def spoil(b, j, value):
        which = int(rng.integers(2))
        x, h, d = (clean_k, clean_v)[which], int(rng.integers(c.st.heads)), int(rng.integers(c.dim))
        s = int(c.rows[b])
        page, slot = int(c.st.table[s, j // c.st.page_tokens]), j % c.st.page_tokens
        c.st.view(which)[c.layer][page, h, slot, d] = value
        shares = [b]
        if group[b] >= 0 and b == c.firsts[group[b]] and j < c.prefix[group[b]]:
            shares = list(range(c.firsts[group[b]], c.firsts[group[b] + 1]))
        for o in shares:
            p = np.arange(c.old[o], c.old[o] + c.new[o])
            sees = p >= j if c.causal else np.ones(len(p), bool)
            if c.window:
                sees &= p - c.window < j
            hit[o] |= sees
    for b in range(c.n):
        if c.new[b] > 1:
            spoil(b, int(c.old[b] + c.new[b] - 1), float(rng.choice([np.inf, -np.inf, np.nan])))
    if c.window:
        # a key of the prefix that only some of the group's tokens still see
        b = c.firsts[0]
        spoil(b, int(c.prefix[0]) - 1, math.nan)
        spoil(b, max(0, int(c.prefix[0]) - 60), math.inf)
    hit = np.concatenate(hit)
    assert hit.any() and not hit.all()
    want = [x[~hit] for x in c.want()]
    for attention, prefix in [(None, None)] + other_hints(hs, c):
        out, lse = c.run(torch, hs, attention, prefix)
        calm = torch.from_numpy(~hit).cuda()
        assert_attended(dtype, out[calm], lse[calm], want, clean_k, clean_v, c.dim)
        assert not np.isfinite(to64(out)[hit]).all()


@pytest.mark.parametrize("number", [2, 6])
def test_bad_numbers_stay_within_the_arrays(torch_cuda, hs, number):
    # groups out of order, sequences and tokens that are none: nothing outside is written, and rows outside every bad group keep their results
    torch = torch_cuda
    c = Case(torch, hs, 2, number, seed=1)
    good, _ = c.run(torch, hs)
    for firsts, tokens in (([-5] * len(c.firsts), c.prefix), ([c.n + 3] * len(c.firsts), c.prefix), (c.firsts[::-1].copy(), c.prefix), ([0x7FFFFFFF] * len(c.firsts), c.prefix),
                           (c.firsts, np.full(len(c.prefix), -1)), (c.firsts, np.full(len(c.prefix), 0x7FFFFFFF)), (c.firsts, np.full(len(c.prefix), -0x80000000))):
        c.fd.copy_(ints(torch, firsts))
        c.pd.copy_(ints(torch, tokens))
        guard = torch.full((c.q.shape[0] + 2, *c.q.shape[1:]), 7.0, dtype=good.dtype, device="cuda")
        qd, prefix = device(torch, c.q, 2), c.prefixes(hs)
        need = c.st.handle.attend_shared_workspace(c.batch, prefix, c.attention)
        w = torch.zeros(need + 4096, dtype=torch.uint8, device="cuda")
        c.st.handle.attend_shared(0, c.batch, prefix, c.attention, heads_view(hs, qd), heads_view(hs, guard[1:-1]), workspace=w.data_ptr(), workspace_bytes=need,
                                  stream=torch.cuda.current_stream().cuda_stream)
        assert (guard[0] == 7).all() and (guard[-1] == 7).all() and not w[need:].any()


def test_no_groups_is_attention(torch_cuda, hs):
    torch = torch_cuda
    c = Case(torch, hs, 2, 6, seed=4)
    for b in range(c.n):
        for which, x in ((0, c.k), (1, c.v)):
            c.st.store(0, int(c.rows[b]), which, x[b])
    out, lse = c.run(torch, hs, prefix=hs.Prefix(0, 0, 0))
    assert_attended(2, out, lse, c.want(), c.k, c.v, c.dim)


def test_a_captured_call_and_two_workspaces(torch_cuda, hs):
    torch = torch_cuda
    for number in (5, 6):
        c = Case(torch, hs, 0, number)
        want, _ = c.run(torch, hs)
        need = c.st.handle.attend_shared_workspace(c.batch, c.prefixes(hs), c.attention)
        side = torch.cuda.Stream()
        spaces = [torch.zeros(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
        qd = device(torch, c.q, 0)
        outs = [torch.zeros_like(want) for _ in range(2)]
        prefix = c.prefixes(hs)

        def call(i):
            c.st.handle.attend_shared(0, c.batch, prefix, c.attention, heads_view(hs, qd), heads_view(hs, outs[i]), workspace=spaces[i].data_ptr(), workspace_bytes=need,
                                      stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(0)
        for _ in range(4):
            outs[0].zero_()
            outs[1].zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                call(1)                                     # at the same time, on another stream
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


# many rows over a long prefix: tiles of 128 rows for the prefix, of 16 or of 128 for what is behind it; heads of every kernel's size
LARGE = [([64], [4001], [3, 60], [1], 0, 4, 8, 128, 16, 0, True), ([40, 23], [3500, 2900], [0, 33], [1], 1, 4, 8, 64, 24, 0, True), ([64], [3900], [20], [1], 0, 4, 8, 96, 32, 700, True),
         ([50], [4100], [9], [1], 0, 4, 8, 160, 16, 0, True), ([40], [3000], [500, 400], [3], 0, 4, 16, 128, 16, 0, True), ([33], [2200], [700], [7], 1, 4, 8, 80, 48, 0, True)]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", range(len(LARGE)))
def test_many_rows_over_a_long_prefix(torch_cuda, hs, dtype, number):
    torch = torch_cuda
    CASES.append(LARGE[number])
    try:
        c = Case(torch, hs, dtype, len(CASES) - 1, order=number % 2)
    finally:
        CASES.pop()
    want = c.want()
    for layout in ("tokens", "features"):
        out, lse = c.run(torch, hs, layout=layout)
        assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)
    again, _ = c.run(torch, hs, layout="gaps", lse=False)
    assert torch.equal(out, again)


def test_one_workspace_serves_every_call_in_turn(torch_cuda, hs):
    # the calls leave the workspace as they want to find it, each other's among them
    torch = torch_cuda
    from test_cache_gpu import attend, attention_case
    c = Case(torch, hs, 2, 5)
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, 2, 13)
    alone, lse = attend(torch, hs, st, batch, attention, q)
    want, _ = c.run(torch, hs)
    weights = torch.zeros((1, st.table.shape[0], st.heads, st.table.shape[1] * st.page_tokens), device="cuda")
    into = hs.Weights(weights.data_ptr(), *weights.stride()[:3])
    qd, stream = device(torch, q, 2), torch.cuda.current_stream().cuda_stream
    one = ints(torch, [int(rows[0])])
    need = max(st.handle.attend_workspace(batch, attention), c.st.handle.attend_shared_workspace(c.batch, c.prefixes(hs), c.attention), st.handle.weigh_workspace(batch, attention),
               st.handle.evict_workspace(1, 1500), st.handle.weigh_workspace(batch, hs.Attention(attention.q_heads, attention.scale, longest_chunk=5000, longest=2000)))
    w = torch.zeros(need, dtype=torch.uint8, device="cuda")
    many = hs.Attention(attention.q_heads, attention.scale, longest_chunk=5000, longest=2000)
    for turn in range(3):
        out, _ = attend(torch, hs, st, batch, attention, q, workspace=w)
        assert torch.equal(out, alone)
        out, _ = c.run(torch, hs, workspace=w)
        assert torch.equal(out, want)
        for a in (attention, many):
            weights.zero_()
            st.handle.weigh(0, batch, a, heads_view(hs, qd), lse.data_ptr(), into, workspace=w.data_ptr(), workspace_bytes=need, stream=stream)
            total = weights.sum().item()
            assert abs(total - q.shape[0] * q.shape[1]) <= 1e-4 * total
        # (as many tokens as it has: nothing happens but the choice)
        st.handle.evict(1, one.data_ptr(), 0, into, 1500, workspace=w.data_ptr(), workspace_bytes=need, stream=stream)
        assert not w[: 4 * 16384].any()


def widened(torch, hs, c, keys):
    """The same cache with rows of the table that have places for so many keys: what the call is told to expect."""
    st = c.st
    table = torch.full((st.table.shape[0], max(-(-keys // st.page_tokens), st.table.shape[1])), -1, dtype=torch.int32, device="cuda")
    table[:, : st.table.shape[1]] = st.table
    st.wide = table
    st.handle = hs.Cache(st.dtype, st.layers, st.pages, st.page_tokens, st.heads, st.head_dim, table.shape[0], table.shape[1], st.pool[0].data_ptr(), st.pool[1].data_ptr(),
                         table.data_ptr(), st.lengths.data_ptr(), st.references.data_ptr(), st.scratch.data_ptr(), order=st.order)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", range(len(CASES)))
def test_small_calls_that_expect_long_sequences(torch_cuda, hs, dtype, number):
    # (by tiles of the prefixes' rows and of what is behind them, which else only large calls are)
    torch = torch_cuda
    c = Case(torch, hs, dtype, number, order=number % 2, seed=1)
    size = 4 if dtype == 1 else 2
    widened(torch, hs, c, -(-(1 << 27) // (c.n * c.st.heads * c.dim * 2 * size)))
    want = c.want()
    keys = c.st.wide.shape[1] * c.st.page_tokens
    for chunk, longest in ((int(c.new.max()), keys), (1, 0), (5000, keys)):
        for prefix in (c.hint, dict(most_tokens=0, longest=0), dict(most_tokens=1, longest=1)):
            out, lse = c.run(torch, hs, c.hints(hs, chunk, longest), c.prefixes(hs, **prefix), layout="gaps" if chunk == 1 else "tokens")
            assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)


# heads of 129 to 160 elements: chunks of fewer rows than a tile has, of sequences that are said to be long
MIDDLE = [([24], [700], [40, 300], [30, 9], 1, 2, 4, 160, 16, 0, True), ([11, 9], [500, 333], [77, 0, 200], [25], 0, 2, 4, 136, 24, 400, True), ([20], [650], [90, 8], [30], 0, 2, 4, 152, 32, 0, False)]


@pytest.mark.parametrize("dtype", [0, 2])
@pytest.mark.parametrize("number", range(len(MIDDLE)))
def test_heads_between_128_and_160(torch_cuda, hs, dtype, number):
    torch = torch_cuda
    CASES.append(MIDDLE[number])
    try:
        c = Case(torch, hs, dtype, len(CASES) - 1, order=number % 2)
    finally:
        CASES.pop()
    widened(torch, hs, c, 16000)
    keys = c.st.wide.shape[1] * c.st.page_tokens
    attention, want = c.hints(hs, int(c.new.max()), keys), c.want()
    # (by tiles of the prefixes' rows: sums of whole rows are left)
    part = c.q.shape[0] * c.q.shape[1] * (c.dim + 4) * 4
    need = c.st.handle.attend_shared_workspace(c.batch, c.prefixes(hs), attention)
    assert need > 4 * 16384 and (need - 4 * 16384) % part == 0
    for layout in ("tokens", "features"):
        out, lse = c.run(torch, hs, attention, layout=layout)
        assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)


# single tokens and long chunks in one batch, behind one prefix
MIXED = [([14], [900], [5, 130, 33], [1] * 9 + [200] + [1] * 4, 0, 2, 4, 128, 16, 0, True), ([9, 6], [500, 1300], [40, 0], [1] * 4 + [333, 1, 2] + [1] * 7 + [64], 2, 2, 4, 64, 24, 0, True),
         ([12], [700], [60, 9], [1] * 5 + [150] + [3] * 6, 0, 1, 8, 96, 32, 250, True), ([10], [640], [17], [1] * 9 + [180], 1, 2, 2, 256, 7, 0, True)]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", range(len(MIXED)))
def test_single_tokens_and_long_chunks_together(torch_cuda, hs, dtype, number):
    torch = torch_cuda
    CASES.append(MIXED[number])
    try:
        c = Case(torch, hs, dtype, len(CASES) - 1, order=number % 2)
    finally:
        CASES.pop()
    want = c.want()
    out, lse = c.run(torch, hs)
    assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)
    widened(torch, hs, c, 40000)
    keys = c.st.wide.shape[1] * c.st.page_tokens
    attention = c.hints(hs, int(c.new.max()), keys)
    part = c.q.shape[0] * c.q.shape[1] * (c.dim + 4) * 4
    need = c.st.handle.attend_shared_workspace(c.batch, c.prefixes(hs), attention)
    assert need > 4 * 16384 and (need - 4 * 16384) % part == 0
    for layout in ("tokens", "features"):
        out, lse = c.run(torch, hs, attention, layout=layout)
        assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)


class LongCase(Case):
    """The same with rows of the table that have places for so many keys that the call goes by tiles of the prefixes' rows and of what is behind them; a call without other hints is
    looked at for it."""
    def __init__(self, torch, hs, dtype, number, *args, **kw):
        super().__init__(torch, hs, dtype, number, *args, **kw)
        widened(torch, hs, self, -(-(1 << 27) // (self.n * self.st.heads * self.dim * 2 * (4 if dtype == 1 else 2))))
        self.st.table = self.st.wide
        self.attention = self.hints(hs, int(self.new.max()), self.st.wide.shape[1] * self.st.page_tokens)
        part = self.q.shape[0] * self.q.shape[1] * (self.dim + 4) * 4
        need = self.st.handle.attend_shared_workspace(self.batch, self.prefixes(hs), self.attention)
        assert need > 4 * 16384 and (need - 4 * 16384) % part == 0 and need != self.st.handle.attend_workspace(self.batch, self.attention)


@pytest.fixture
def long_cases(monkeypatch):
    import sys
    monkeypatch.setattr(sys.modules[__name__], "Case", LongCase)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", range(len(CASES)))
def test_attend_shared_by_prefix_tiles(torch_cuda, hs, long_cases, dtype, number):
    test_attend_shared(torch_cuda, hs, dtype, number)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [2, 3, 6, 8, 10, 14])
def test_pages_that_are_gone_by_prefix_tiles(torch_cuda, hs, long_cases, dtype, number):
    test_pages_that_are_gone_are_not_seen(torch_cuda, hs, dtype, number)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_chunks_that_begin_within_the_prefix_by_prefix_tiles(torch_cuda, hs, long_cases, dtype):
    test_chunks_that_begin_within_the_prefix(torch_cuda, hs, dtype)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("number", [3, 6, 8, 9])
def test_what_is_masked_by_prefix_tiles(torch_cuda, hs, long_cases, dtype, number):
    test_what_is_masked_does_not_reach_the_result(torch_cuda, hs, dtype, number)


@pytest.mark.parametrize("number", [2, 3, 6, 13])
def test_bad_numbers_by_prefix_tiles(torch_cuda, hs, long_cases, number):
    test_bad_numbers_stay_within_the_arrays(torch_cuda, hs, number)


def test_a_captured_call_and_two_workspaces_by_prefix_tiles(torch_cuda, hs, long_cases):
    test_a_captured_call_and_two_workspaces(torch_cuda, hs)


def test_one_workspace_serves_every_call_by_prefix_tiles(torch_cuda, hs, long_cases):
    test_one_workspace_serves_every_call_in_turn(torch_cuda, hs)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("kind", [Case, LongCase])
@pytest.mark.parametrize("number", [2, 3, 6, 8])
def test_rows_of_groups_that_are_none_read_their_own_pages(torch_cuda, hs, dtype, kind, number):
    # every group is out of order or has no tokens: each row is attended by its own pages
    torch = torch_cuda
    c = kind(torch, hs, dtype, number, seed=6)
    for b in range(c.n):
        for which, x in ((0, c.k), (1, c.v)):
            c.st.store(0, int(c.rows[b]), which, x[b])
    want = c.want()
    for firsts, tokens in (([-5] * len(c.firsts), c.prefix), ([c.n + 3] * len(c.firsts), c.prefix), ([c.n - 1 - i for i in range(len(c.firsts))], c.prefix), ([0x7FFFFFFF] * len(c.firsts), c.prefix),
                           (c.firsts, np.full(len(c.prefix), -1)), (c.firsts, np.zeros(len(c.prefix))), (c.firsts, np.full(len(c.prefix), -0x80000000))):
        c.fd.copy_(ints(torch, firsts))
        c.pd.copy_(ints(torch, tokens))
        out, lse = c.run(torch, hs)
        assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("kind", [Case, LongCase])
@pytest.mark.parametrize("number", [3, 6, 8, 9, 13])
def test_rows_in_front_of_the_first_group_and_behind_the_last(torch_cuda, hs, dtype, kind, number):
    # some of the groups only, and groups without rows among them: the other rows are attended by their own pages
    torch = torch_cuda
    c = kind(torch, hs, dtype, number, seed=8)
    for b in range(c.n):
        for which, x in ((0, c.k), (1, c.v)):
            c.st.store(0, int(c.rows[b]), which, x[b])
    want = c.want()
    f, p = list(c.firsts), list(c.prefix)
    for firsts, prefixes in ((f[:-1], p[:-1]), (f[1:], p[1:]), (f[:2], p[:1]), ([f[0]] + f, [5] + p), (f + [f[-1]], p + [9]), (f[:2] + f[1:], p[:1] + [7] + p[1:])):
        if not 1 <= len(prefixes) <= c.n:                   # (no more groups than rows)
            continue
        fd, pd = ints(torch, firsts), ints(torch, prefixes)
        prefix = hs.Prefix(len(prefixes), fd.data_ptr(), pd.data_ptr(), **c.hint)
        out, lse = c.run(torch, hs, prefix=prefix)
        assert_attended(dtype, out, lse, want, c.k, c.v, c.dim)
