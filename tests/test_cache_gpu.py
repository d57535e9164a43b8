"""Rotary positions, the paged cache and attention over it on the GPU, against plain implementations in 64 bits; tolerances are
derived in cache_util.  Needs a real MI355X: run with -m gpu."""
import math

import numpy as np
import pytest

from cache_util import HALF_ULP, SMALLEST, State, attend64, attend_bounds, rounded, to64, torch_type
from test_spmm_gpu import torch_cuda  # noqa: F401

pytestmark = pytest.mark.gpu


def device(torch, x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch_type(torch, dtype)).cuda()


def ints(torch, x):
    return torch.from_numpy(np.asarray(x, np.int32)).cuda()


def heads_view(hs, x):
    return hs.Heads(x.data_ptr(), *x.stride())


def laid_out(torch, x, layout):
    """tokens x heads x dim in one of the orders that callers have."""
    if layout == "features":                                   # features x tokens
        return x.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    if layout == "heads":                                      # heads x tokens x dim
        return x.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    if layout == "gaps":                                       # rows with something between them
        big = torch.full((x.shape[0], x.shape[1] + 1, x.shape[2] + 3), math.nan, dtype=x.dtype, device=x.device)
        big[:, 1:, 1:-2] = x
        return big[:, 1:, 1:-2]
    return x.contiguous()


def turned64(x, table, positions, dims, interleaved, backward):
    y = x.copy()
    i = np.arange(dims // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + dims // 2)
    c, s = table[positions][:, None, :, 0], table[positions][:, None, :, 1] * (-1 if backward else 1)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size = np.zeros_like(x)
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y, size


def assert_turned(got, want, size, dtype, scale=2.0):
    # two products and a sum in fp32, the cosine's and the sine's own rounding (they are the inputs here), then the element type
    bound = HALF_ULP[dtype] * np.abs(want) + size * scale * 3 * 2.0 ** -24 + SMALLEST[dtype]
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()


ROTATIONS = [  # tokens, heads, dim, dims
    (1, 1, 2, 2), (1, 3, 64, 64), (5, 2, 128, 64), (7, 40, 128, 128), (300, 3, 80, 40), (33, 5, 96, 92), (65, 2, 37, 6), (129, 1, 256, 256), (2, 7, 24, 0), (1000, 4, 64, 32)]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,dims", ROTATIONS)
def test_rotate(torch_cuda, hs, dtype, interleaved, tokens, heads, dim, dims):
    torch = torch_cuda
    rng = np.random.default_rng(tokens * 131 + dim)
    table = hs.rotary_table(max(dims, 2), 513, "yarn", factor=4.0, original_length=128.0)
    on_gpu = torch.from_numpy(table).cuda()
    r = hs.Rotary(dims, 513, on_gpu.data_ptr(), interleaved=interleaved)
    positions = rng.integers(0, 513, tokens)
    at = ints(torch, positions)
    x = rounded(torch, rng.standard_normal((tokens, heads, dim)), dtype)
    stream = torch.cuda.current_stream().cuda_stream
    for backward in (False, True):
        want, size = turned64(x, table.astype(np.float64), positions, dims, interleaved, backward) if dims else (x, np.zeros_like(x))
        for layout, out in (("tokens", "tokens"), ("features", "tokens"), ("tokens", "features"), ("heads", "gaps"), ("features", "features"), ("gaps", "heads")):
            xd = laid_out(torch, device(torch, x, dtype), layout)
            yd = laid_out(torch, torch.full((tokens, heads, dim), math.nan, dtype=xd.dtype, device="cuda"), out)
            hs.rotate(dtype, r, tokens, heads, dim, heads_view(hs, xd), heads_view(hs, yd), at.data_ptr(), backward=backward, stream=stream)
            assert_turned(to64(yd), want, size, dtype)
            hs.rotate(dtype, r, tokens, heads, dim, heads_view(hs, xd), heads_view(hs, xd), at.data_ptr(), backward=backward, stream=stream)
            assert torch.equal(xd, yd), (layout, out)                    # in place, and whatever the layout


def test_rotation_backward_is_the_gradient(torch_cuda, hs):
    # <g, rotate(x)> has the gradient rotate_backward(g): by the formula's derivative in every element, here by differences in 32 bits
    torch = torch_cuda
    rng = np.random.default_rng(5)
    T, H, D, dims = 9, 2, 32, 24
    table = torch.from_numpy(hs.rotary_table(dims, 64, "yarn", factor=2.0, original_length=32.0)).cuda()
    at = ints(torch, rng.integers(0, 64, T))
    stream = torch.cuda.current_stream().cuda_stream
    for interleaved in (False, True):
        r = hs.Rotary(dims, 64, table.data_ptr(), interleaved=interleaved)
        x, g = (torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).cuda() for _ in range(2))
        grad = torch.empty_like(g)
        hs.rotate(hs.TF32, r, T, H, D, heads_view(hs, g), heads_view(hs, grad), at.data_ptr(), backward=True, stream=stream)
        d = torch.zeros_like(x)
        for e in range(D):
            # the operator is linear: a step of one in element e changes its output by the column of its matrix
            one = torch.zeros_like(x)
            one[:, :, e] = 1.0
            y = torch.empty_like(x)
            hs.rotate(hs.TF32, r, T, H, D, heads_view(hs, one), heads_view(hs, y), at.data_ptr(), stream=stream)
            d[:, :, e] = (y.double() * g.double()).sum(-1).float()
        assert (d - grad).abs().max().item() <= 8 * 2.0 ** -24 * 4.0 * 1.1


def test_positions_outside_the_table_are_the_nearest(torch_cuda, hs):
    torch = torch_cuda
    table = torch.from_numpy(hs.rotary_table(16, 10)).cuda()
    r = hs.Rotary(16, 10, table.data_ptr())
    x = torch.randn(4, 2, 16, device="cuda")
    for layout in ("tokens", "features"):
        xd = laid_out(torch, x, layout)
        a, b = torch.empty_like(x), torch.empty_like(x)
        hs.rotate(hs.TF32, r, 4, 2, 16, heads_view(hs, xd), heads_view(hs, a), ints(torch, [-5, 10, 0x7FFFFFFF, 3]).data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
        hs.rotate(hs.TF32, r, 4, 2, 16, heads_view(hs, xd), heads_view(hs, b), ints(torch, [0, 9, 9, 3]).data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(a, b)


# ---- append ----------------------------------------------------------------------------------------------------------

APPENDS = [  # chunks, tokens held before, heads, shared, dim, page tokens, dims
    ([1], [0], 1, 1, 8, 16, 8), ([1, 1, 1], [15, 16, 37], 2, 4, 64, 16, 64), ([5, 0, 33, 1], [0, 9, 60, 127], 3, 2, 80, 24, 40),
    ([70, 129], [3, 0], 2, 1, 128, 1, 128), ([64, 65], [0, 1], 1, 8, 36, 7, 20), ([300], [31], 4, 1, 128, 32, 64)]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(torch_cuda, hs, dtype, order, case):
    torch = torch_cuda
    new, old, heads, shared, dim, page, dims = APPENDS[case]
    rng = np.random.default_rng(case)
    n = len(new)
    lengths = np.add(new, old)
    used = int(sum(-(-x // page) for x in lengths))
    rows = rng.permutation(n + 2)[:n]                           # batch rows are not the cache's
    st = State(torch, hs, dtype, used + 3, page, heads, dim, n + 2, int(max(-(-lengths // page))) + 1, layers=2, order=order, page_gap=16 * (case % 2), layer_gap=32 * (case % 3))
    by_row = np.zeros(n + 2, int)
    by_row[rows] = lengths
    st.place(rng, by_row)
    before = [st.pool[i].clone() for i in range(2)]
    tokens = int(sum(new))
    starts = ints(torch, np.concatenate([[0], np.cumsum(new)]))
    positions = np.concatenate([np.arange(o, o + m) for o, m in zip(old, new)])
    table = hs.rotary_table(dims, int(lengths.max()))
    on_gpu = torch.from_numpy(table).cuda()
    q, k, v = (rounded(torch, rng.standard_normal((tokens, h, dim)), dtype) for h in (heads * shared, heads, heads))
    stream = torch.cuda.current_stream().cuda_stream
    rd = ints(torch, rows)
    batch = hs.Batch(n, tokens, starts.data_ptr(), rd.data_ptr())
    seq = np.repeat(rows, new)
    ids = st.table.cpu().numpy()[seq, positions // page]
    for interleaved in (False, True):
        for layout in ("tokens", "features", "gaps"):
            for turn in (True, False):
                for i in range(2):
                    st.pool[i].copy_(before[i])
                qd, kd, vd = (laid_out(torch, device(torch, x, dtype), layout) for x in (q, k, v))
                qo = torch.full((tokens, heads * shared, dim), math.nan, dtype=qd.dtype, device="cuda")
                r = hs.Rotary(dims, int(lengths.max()), on_gpu.data_ptr(), interleaved=interleaved) if turn else None
                st.handle.append(1, batch, heads_view(hs, kd), heads_view(hs, vd), rotary=r, q_heads=heads * shared, q=heads_view(hs, qd), q_out=heads_view(hs, qo), stream=stream)
                for x, got in ((q, to64(qo)), (k, to64(st.view(0)[1])[ids, :, positions % page])):
                    want, size = turned64(x, table.astype(np.float64), positions, dims, interleaved, False) if turn else (x, np.zeros_like(x))
                    assert_turned(got, want, size, dtype, 1.0)
                assert np.array_equal(to64(st.view(1)[1])[ids, :, positions % page], v)
                # nothing else has changed
                for i in range(2):
                    ref = State.__new__(State)
                    ref.__dict__.update(st.__dict__)
                    ref.pool = [before[0].clone(), before[1].clone()]
                    idt, slot = torch.from_numpy(ids).long().cuda(), torch.from_numpy(positions % page).cuda()
                    ref.view(i)[1][idt, :, slot] = st.view(i)[1][idt, :, slot]
                    assert torch.equal(ref.pool[i].view(torch.uint8), st.pool[i].view(torch.uint8))


def test_append_without_pages_or_sequences_stores_nothing(torch_cuda, hs):
    torch = torch_cuda
    rng = np.random.default_rng(3)
    st = State(torch, hs, 2, 6, 4, 2, 16, 3, 3)
    st.place(rng, [5, 9, 2])
    st.table[0, 1] = -1                                        # the page of token 4
    st.table[1, 0] = 6                                         # not a page's number
    before = [p.clone() for p in st.pool]
    k = torch.randn(9, 2, 16, device="cuda").bfloat16()
    # rows: 0 (tokens 3, 4), 1 (0 .. 3 of a chunk of 9 > length), a sequence that is not there, a chunk longer than the sequence
    starts, rows = ints(torch, [0, 2, 6, 7, 9]), ints(torch, [0, 1, 99, -1])
    st.lengths[1] = 4
    st.handle.append(0, hs.Batch(4, 9, starts.data_ptr(), rows.data_ptr()), heads_view(hs, k), heads_view(hs, k), stream=torch.cuda.current_stream().cuda_stream)
    changed = torch.nonzero((st.pool[0].view(torch.int16) != before[0].view(torch.int16)).view(6, 2, 4, 16).any(-1).any(1))
    assert changed.tolist() == [[int(st.table[0, 0]), 3]]


# ---- attention -------------------------------------------------------------------------------------------------------

ATTENTIONS = [  # chunks, tokens held before, heads, shared, dim, page tokens, window, causal
    ([1], [0], 1, 1, 8, 16, 0, True),
    ([1, 1], [0, 70], 2, 1, 64, 16, 0, True),
    ([1, 1, 1, 1, 1], [1, 31, 32, 511, 1300], 2, 8, 128, 16, 0, True),
    ([1, 1], [1999, 4200], 1, 3, 96, 24, 0, True),
    ([1, 1, 1], [300, 64, 5], 2, 5, 64, 64, 40, True),
    ([3, 1, 8], [40, 0, 333], 2, 4, 128, 16, 0, True),
    ([17, 0, 2], [100, 5, 0], 1, 16, 64, 32, 7, True),
    ([64], [0], 2, 2, 128, 64, 0, True),
    ([130, 33, 1, 65], [0, 200, 90, 64], 2, 3, 80, 7, 0, True),
    ([97, 260], [500, 3], 1, 2, 128, 128, 100, True),
    ([40, 129], [21, 600], 2, 1, 256, 16, 0, True),
    ([5, 70], [45, 130], 2, 2, 40, 1, 1, True),
    ([4, 100, 1], [0, 31, 200], 2, 2, 64, 16, 0, False),
    ([300], [1000], 1, 4, 128, 32, 0, True),
    ([1] * 40, list(range(0, 800, 20)), 4, 2, 64, 16, 0, True),
    ([33, 33], [0, 95], 8, 1, 8, 5, 0, True),
    ([50, 90], [200, 0], 1, 2, 88, 16, 0, True),
    ([70, 1, 200], [0, 500, 33], 2, 1, 96, 32, 60, True),
    ([45, 140], [100, 0], 1, 2, 160, 16, 0, True),
    ([90], [300], 1, 1, 136, 24, 50, True),
    ([64], [40], 1, 1, 248, 48, 0, True),
    ([1, 1], [9000, 17], 1, 4, 128, 16, 0, True),
    ([1], [5000], 2, 1, 64, 10, 0, True),
    ([40], [6000], 1, 4, 128, 16, 0, True),
    # tiles of 256 rows: for many tiles only
    ([1] * 29 + [150, 2], [7] * 29 + [130, 0], 32, 1, 128, 16, 0, True),
    ([140] + [2] * 35, [300] + [0, 3, 50, 8, 1] * 7, 32, 1, 104, 24, 60, True),
    # windows, and so many tiles that the chunk's own kernel serves them
    ([200] + [1] * 20, [700] + [30] * 20, 16, 2, 64, 24, 60, True),
    ([90, 5] + [1] * 18, [0, 300] + [64] * 18, 16, 2, 160, 16, 100, True)]


def attention_case(torch, hs, dtype, case, order=0, seed=0, layers=1):
    new, old, heads, shared, dim, page, window, causal = ATTENTIONS[case]
    rng = np.random.default_rng(1000 * case + seed)
    n, lengths = len(new), np.add(new, old)
    used = int(sum(-(-x // page) for x in lengths))
    st = State(torch, hs, dtype, used + 2, page, heads, dim, n + 1, 100000 // page + 2, layers=layers, order=order)
    rows = rng.permutation(n + 1)[:n]
    by_row = np.zeros(n + 1, int)
    by_row[rows] = lengths
    st.place(rng, by_row)
    k, v = ([rounded(torch, rng.standard_normal((x, heads, dim)) * 1.5, dtype) for x in lengths] for _ in range(2))
    for s, a, b in zip(rows, k, v):
        st.store(layers - 1, s, 0, a)
        st.store(layers - 1, s, 1, b)
    q = rounded(torch, rng.standard_normal((sum(new), heads * shared, dim)) * 1.5, dtype)
    starts, rd = ints(torch, np.concatenate([[0], np.cumsum(new)])), ints(torch, rows)
    st.kept = (starts, rd)
    batch = hs.Batch(n, int(sum(new)), starts.data_ptr(), rd.data_ptr())
    scale = 1.0 / math.sqrt(dim)
    attention = hs.Attention(heads * shared, scale, causal=causal, window=window, longest_chunk=max(new), longest=int(lengths.max()))
    return st, batch, attention, q, k, v, new, old, rows, np.float64(np.float32(scale)), window, causal


def many(hs, st, batch, attention):
    """The same with hints of many rows and of so many keys that the chunk's own kernel serves, in parts of 512 keys."""
    tiles = st.heads * batch.sequences * -(-batch.tokens * (attention.q_heads // st.heads) // 128)
    return hs.Attention(attention.q_heads, attention.scale, causal=attention.causal, window=attention.window, longest_chunk=5000, longest=100000 // tiles)


def attend(torch, hs, st, batch, attention, q, layout="tokens", layer=0, lse=True, hints=True, workspace=None):
    qd = q if torch.is_tensor(q) else device(torch, q, st.dtype)
    out = laid_out(torch, torch.full(tuple(qd.shape), math.nan, dtype=qd.dtype, device="cuda"), layout)
    l = torch.full(tuple(qd.shape[:2]), math.nan, device="cuda")
    need = st.handle.attend_workspace(batch, attention)
    w = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda") if workspace is None else workspace
    st.handle.attend(layer, batch, attention, heads_view(hs, qd), heads_view(hs, out), lse=l.data_ptr() if lse else 0, workspace=w.data_ptr(), workspace_bytes=w.numel(),
                     stream=torch.cuda.current_stream().cuda_stream)
    st.kept = st.kept + (qd, w)
    return out, l


def expected(q, k, v, new, old, scale, causal, window):
    parts, at = [], 0
    for a, b, n, o in zip(k, v, new, old):
        parts.append(attend64(q[at:at + n], a, b, np.arange(o, o + n), scale, causal, window))
        at += n
    return [np.concatenate(x) for x in zip(*parts)]


def assert_attended(dtype, got, lse, want, k, v, dim):
    out, l, size, reach = want
    keys, largest = max(len(x) for x in k), max([np.abs(x).max() for x in v if x.size] + [0])
    bound, lse_bound = attend_bounds(dtype, out, l, size, reach, dim, keys, largest)
    got, lse = to64(got), to64(lse)
    assert np.isfinite(got).all()
    assert (np.abs(got - out) <= bound).all(), (np.abs(got - out) / bound).max()
    empty = np.isneginf(l)
    assert np.array_equal(np.isneginf(lse), empty) and (got[empty] == 0).all()
    assert (np.abs(lse[~empty] - l[~empty]) <= lse_bound[~empty]).all(), (np.abs(lse[~empty] - l[~empty]) / lse_bound[~empty]).max()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("case", range(len(ATTENTIONS)))
def test_attend(torch_cuda, hs, dtype, case):
    torch = torch_cuda
    for order, layout, layers in ((0, "tokens", 1), (1, "features", 2)):
        st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, dtype, case, order, layers=layers)
        want = expected(q, k, v, new, old, scale, causal, window)
        out, lse = attend(torch, hs, st, batch, attention, q, layout, layer=layers - 1)
        assert_attended(dtype, out, lse, want, k, v, q.shape[2])
        # the hints choose kernels and parts, not the result; lse may be left out; bits do not change from call to call
        again, _ = attend(torch, hs, st, batch, attention, q, layout, layer=layers - 1, lse=False)
        assert torch.equal(out, again)
        others = [hs.Attention(attention.q_heads, attention.scale, causal=causal, window=window, longest_chunk=chunk, longest=longest)
                  for chunk, longest in ((1, 0), (1, 1 << 30), (5000, 100000), (0, 1))]
        for other in others + [many(hs, st, batch, attention)]:
            out, lse = attend(torch, hs, st, batch, other, q, "gaps" if q.shape[2] > 3 else layout, layer=layers - 1)
            assert_attended(dtype, out, lse, want, k, v, q.shape[2])


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("case", [4, 5, 9, 12, 13, 24, 25, 26, 27])
def test_pages_that_are_gone_are_not_seen(torch_cuda, hs, dtype, case):
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, dtype, case, seed=7)
    page = st.page_tokens
    rng = np.random.default_rng(case)
    there, at, parts = [], 0, []
    for s, a in zip(rows, k):
        used = -(-len(a) // page)
        gone = rng.random(used) < 0.4
        if s == rows[-1]:
            gone[:] = True                                     # nothing at all
        for p in np.nonzero(gone)[0]:
            st.table[int(s), int(p)] = int(rng.choice([-1, st.pages, 0x7FFFFFFF, -7]))
        there.append(~gone[np.arange(len(a)) // page])
    for a, b, n, o, t in zip(k, v, new, old, there):
        parts.append(attend64(q[at:at + n], a, b, np.arange(o, o + n), scale, causal, window, t[None]))
        at += n
    want = [np.concatenate(x) for x in zip(*parts)]
    for a in (attention, many(hs, st, batch, attention)):
        out, lse = attend(torch, hs, st, batch, a, q)
        assert_attended(dtype, out, lse, want, k, v, q.shape[2])
        assert np.isneginf(to64(lse)).any()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("case", [2, 4, 6, 8, 9, 10, 17, 18, 19, 20, 24, 25, 26, 27])
def test_what_is_masked_does_not_reach_the_result(torch_cuda, hs, dtype, case):
    # infinities and NaN in keys and values: only the tokens that see them have them
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, dtype, case, seed=3)
    rng = np.random.default_rng(case + 50)
    hit = []
    for s, a, b, n, o in zip(rows, k, v, new, old):
        mine = np.zeros(n, bool)
        for _ in range(3):
            j = int(rng.integers(max(0, o - 2), o + n)) if n else 0
            if len(a) == 0:
                continue
            value = float(rng.choice([np.inf, -np.inf, np.nan]))
            if rng.random() < 0.5:
                st.store_one = st.view(0)[0]
                a[j, rng.integers(st.heads), rng.integers(st.head_dim)] = value
            else:
                b[j, rng.integers(st.heads), rng.integers(st.head_dim)] = value
            sees = np.arange(o, o + n) >= j
            if window:
                sees &= np.arange(o, o + n) - window < j
            mine |= sees
        st.store(0, int(s), 0, a)
        st.store(0, int(s), 1, b)
        hit.append(mine)
    hit = np.concatenate(hit)
    # (by the chunk's own kernel, and by that of a few rows)
    few = hs.Attention(attention.q_heads, attention.scale, causal=causal, window=window, longest_chunk=1, longest=attention.longest)
    for a in (attention, few, many(hs, st, batch, attention)):
        masked_holds(torch, hs, st, batch, a, q, k, v, new, old, scale, window, causal, hit)


def masked_holds(torch, hs, st, batch, attention, q, k, v, new, old, scale, window, causal, hit):
    dtype = st.dtype
    out, lse = attend(torch, hs, st, batch, attention, q)
    clean = [[np.where(np.isfinite(x), x, 0.0) for x in y] for y in (k, v)]
    want = expected(q, *clean, new, old, scale, causal, window)
    calm = [x[~hit] for x in want]
    assert_attended(dtype, out[torch.from_numpy(~hit).cuda()], lse[torch.from_numpy(~hit).cuda()], calm, *clean, q.shape[2])
    # and where a value, not a key, is infinite the other elements stay
    got = to64(out)
    assert hit.any() and not np.isfinite(got[hit]).all()


@pytest.mark.parametrize("dtype", [0, 2])
def test_infinite_values_stay_in_their_element(torch_cuda, hs, dtype):
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, dtype, 13, seed=3)
    j = 1100
    v[0][j, 0, 5] = np.inf
    st.store(0, int(rows[0]), 1, v[0])
    attention = many(hs, st, batch, attention)
    out, lse = attend(torch, hs, st, batch, attention, q)
    got = to64(out)
    sees = np.arange(old[0], old[0] + new[0]) >= j
    assert np.isposinf(got[sees][:, :, 5]).all()
    v[0][j, 0, 5] = 0.0
    want = expected(q, k, v, new, old, scale, causal, window)
    out[torch.from_numpy(sees).cuda()[:, None, None] & (torch.arange(q.shape[2], device="cuda") == 5)[None, None, :].expand(*out.shape)] = 0
    for x in (want[0], want[2]):
        x[np.ix_(sees, np.arange(x.shape[1]), [5])] = 0
    assert_attended(dtype, out, lse, want, k, v, q.shape[2])


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_scores_far_apart(torch_cuda, hs, dtype):
    # one key far above all others, in the first, a middle and the last tile, and scores of one size far from zero
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, dtype, 13, seed=9)
    for j in (0, 700, 1299):
        kk = [k[0].copy()]
        kk[0][j] *= 30
        kk = [rounded(torch, kk[0], dtype)]
        st.store(0, int(rows[0]), 0, kk[0])
        for a in (attention, many(hs, st, batch, attention)):
            out, lse = attend(torch, hs, st, batch, a, q)
            assert_attended(dtype, out, lse, expected(q, kk, v, new, old, scale, causal, window), kk, v, q.shape[2])
    kk = [np.ones_like(k[0])]
    st.store(0, int(rows[0]), 0, kk[0])
    for sign in (1.0, -1.0):
        qq = rounded(torch, sign * np.full_like(q, 40.0), dtype)
        for a in (attention, many(hs, st, batch, attention)):
            out, lse = attend(torch, hs, st, batch, a, qq)
            assert_attended(dtype, out, lse, expected(qq, kk, v, new, old, scale, causal, window), kk, v, q.shape[2])


def test_sequences_shorter_than_their_chunk(torch_cuda, hs):
    # tokens in front of the cache see nothing
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, 2, 8)
    st.lengths[int(rows[0])] = 50                              # a chunk of 130
    want = expected(q, [k[0][:50]] + k[1:], v[:1] and [v[0][:50]] + v[1:], new, [-80] + old[1:], scale, causal, window)
    for a in (attention, many(hs, st, batch, attention)):
        out, lse = attend(torch, hs, st, batch, a, q)
        assert_attended(2, out, lse, want, k, v, q.shape[2])
        assert (to64(out)[:80] == 0).all()


def test_pages_beyond_32_bits(torch_cuda, hs):
    # a pool of over 2^32 elements, the sequence's pages at its end
    torch = torch_cuda
    rng = np.random.default_rng(2)
    page, heads, dim = 64, 2, 128
    pages = (1 << 32) // (page * heads * dim) + 64
    st = State(torch, hs, 2, pages, page, heads, dim, 2, 2048, fill=0.0)
    ids = pages - 1 - np.arange(4)
    st.table[0, :4] = ints(torch, ids)
    st.lengths[0] = 200
    starts = ints(torch, [0, 200])
    batch = hs.Batch(1, 200, starts.data_ptr())
    k, v = (rounded(torch, rng.standard_normal((200, heads, dim)), 2) for _ in range(2))
    q = rounded(torch, rng.standard_normal((200, heads * 2, dim)), 2)
    st.kept = (starts,)
    kd, vd = device(torch, k, 2), device(torch, v, 2)
    st.handle.append(0, batch, heads_view(hs, kd), heads_view(hs, vd), stream=torch.cuda.current_stream().cuda_stream)
    for chunk in (200, 1):
        qq = q[-chunk:]
        s2 = ints(torch, [0, chunk])
        b2 = hs.Batch(1, chunk, s2.data_ptr())
        a = hs.Attention(heads * 2, 0.1, longest_chunk=chunk, longest=200)
        st.kept = st.kept + (s2,)
        want = attend64(qq, k, v, np.arange(200 - chunk, 200), np.float64(np.float32(0.1)), True, 0)
        for b in (a, many(hs, st, b2, a)):
            out, lse = attend(torch, hs, st, b2, b, qq)
            assert_attended(2, out, lse, want, [k], [v], dim)


# ---- pages -----------------------------------------------------------------------------------------------------------


def pages_for(tokens, page):
    return -(-tokens // page)


class Books:
    """What the calls on pages do to the table, lengths, references and contents, one entry after another."""

    def __init__(self, st):
        self.table, self.lengths, self.references = (x.cpu().numpy().copy() for x in (st.table, st.lengths, st.references))
        self.pool = [st.view(i).cpu().clone() for i in range(2)]
        self.page = st.page_tokens

    def free_pages(self):
        return [int(i) for i in np.nonzero(self.references <= 0)[0]]

    def extend(self, rows, add):
        free, missing = self.free_pages(), 0
        for s, a in zip(rows, add):
            have = int(self.lengths[s])
            now = min(have + max(int(a), 0), self.table.shape[1] * self.page)
            for p in range(pages_for(have, self.page), pages_for(now, self.page)):
                if free:
                    self.table[s, p] = free.pop(0)
                    self.references[self.table[s, p]] = 1
                else:
                    self.table[s, p] = -1
                    missing += 1
            self.lengths[s] = now
        return missing

    def fork(self, parents, children):
        free, missing = self.free_pages(), 0
        table, lengths = self.table.copy(), self.lengths.copy()
        for p, c in zip(parents, children):
            if p == c:
                continue
            n = int(lengths[p])
            row = np.full(table.shape[1], -1, np.int32)
            full = n // self.page
            row[:full] = table[p, :full]
            if n % self.page:
                if free:
                    row[full] = free.pop(0)
                    for x in self.pool:
                        if 0 <= table[p, full] < len(self.references):
                            x[:, int(row[full]), :, :n % self.page] = x[:, int(table[p, full]), :, :n % self.page]
                else:
                    missing += 1
            for old in table[c]:
                if 0 <= old < len(self.references):
                    self.references[old] -= 1
            for now in row:
                if 0 <= now < len(self.references):
                    self.references[now] += 1
            self.table[c], self.lengths[c] = row, n
        return missing

    def free(self, rows):
        for s in rows:
            for old in self.table[s]:
                if 0 <= old < len(self.references):
                    self.references[old] -= 1
            self.table[s], self.lengths[s] = -1, 0

    def compact(self):
        live = int((self.references > 0).sum())
        holes = [i for i in range(live) if self.references[i] <= 0]
        movers = [i for i in range(live, len(self.references)) if self.references[i] > 0]
        for i in range(live, len(self.references)):
            if self.references[i] <= 0:
                pass
        for to, source in zip(holes, movers):
            for x in self.pool:
                x[:, to] = x[:, source].clone()
            self.table[self.table == source] = to
            self.references[to], self.references[source] = self.references[source], 0
        return live

    def same(self, torch, st):
        assert np.array_equal(self.references, st.references.cpu().numpy())
        assert np.array_equal(self.table, st.table.cpu().numpy())
        assert np.array_equal(self.lengths, st.lengths.cpu().numpy())
        for i in range(2):
            a, b = self.pool[i].contiguous(), st.view(i).cpu().contiguous()
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype,order,pages,page,heads,dim,layers", [(2, 0, 90, 16, 2, 32, 3), (0, 1, 200, 7, 3, 5, 2), (1, 0, 1000, 4, 1, 6, 1), (0, 0, 150, 1, 8, 64, 1),
                                                                     (2, 1, 20000, 2, 1, 8, 1), (1, 0, 77, 5, 2, 3, 2)])
def test_a_life_of_pages(torch_cuda, hs, dtype, order, pages, page, heads, dim, layers):
    torch = torch_cuda
    rng = np.random.default_rng(pages)
    S, P = 24, 12
    st = State(torch, hs, dtype, pages, page, heads, dim, S, P, layers=layers, order=order, page_gap=3 if dim % 2 else 0)
    for i in range(2):
        st.view(i).copy_(torch.randn(st.view(i).shape, device="cuda"))
    books = Books(st)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    live = torch.zeros(1, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for step in range(14):
        what = ["extend", "fork", "extend", "free", "compact", "fork", "extend"][step % 7]
        n = int(rng.integers(1, S + 1))
        rows = rng.permutation(S)[:n]
        rd = ints(torch, rows)
        if what == "extend":
            add = rng.integers(-2, 5 * page, n)
            ad = ints(torch, add)
            st.handle.extend(n, rd.data_ptr(), ad.data_ptr(), status.data_ptr(), stream)
            assert int(status) == books.extend(rows, add)
        elif what == "fork":
            parents = rng.integers(0, S, n)
            parents[: n // 4] = rows[: n // 4]
            pd = ints(torch, parents)
            st.handle.fork(n, pd.data_ptr(), rd.data_ptr(), status.data_ptr(), stream)
            assert int(status) == books.fork(parents, rows)
        elif what == "free":
            n = n // 2 + 1
            st.handle.free(n, rd.data_ptr(), stream)
            books.free(rows[:n])
        else:
            # into other arrays first, then in place: both give the same
            t2, r2 = torch.full_like(st.table, 77), torch.full_like(st.references, 77)
            pool = [p.clone() for p in st.pool]
            st.handle.compact(live.data_ptr(), table_out=t2.data_ptr(), references_out=r2.data_ptr(), stream=stream)
            for i in range(2):
                st.pool[i].copy_(pool[i])
            st.handle.compact(live.data_ptr(), stream=stream)
            assert int(live) == books.compact()
            assert torch.equal(t2, st.table) and torch.equal(r2, st.references)
        books.same(torch, st)
    if pages < 100:
        assert books.references.max() > 1


@pytest.mark.parametrize("pages,lengths", [(20000, [5000, 4321, 2100, 600]), (20000, [8190, 2, 0, 0]), (8192, [8191, 1, 0, 0]), (8193, [4000, 4193, 0, 0]), (8193, [0, 0, 0, 0]),
                                           (8200, [3, 0, 8000, 190]), (30, [10, 9, 3, 0])])
def test_compaction_of_pools_of_every_fill(torch_cuda, hs, pages, lengths):
    # a page holds one token: live pages all over the pool, their number on either side of what a workgroup looks at at a time
    torch = torch_cuda
    rng = np.random.default_rng(pages + lengths[0])
    st = State(torch, hs, 2, pages, 1, 1, 8, 4, max(max(lengths), 1))
    for pool in st.pool:
        pool.copy_(torch.randn(pool.shape, device="cuda").bfloat16())
    st.place(rng, lengths)
    st.table[(st.table < 0) | (st.table >= pages)] = -1
    books, live, stream = Books(st), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.cuda.current_stream().cuda_stream
    for _ in range(2):
        st.handle.compact(live.data_ptr(), stream=stream)
        assert int(live) == sum(lengths) == books.compact()
        books.same(torch, st)


def test_numbers_that_are_none_are_passed_over(torch_cuda, hs):
    torch = torch_cuda
    rng = np.random.default_rng(8)
    st = State(torch, hs, 2, 40, 4, 2, 8, 6, 5)
    st.place(rng, [9, 4, 0, 13, 1, 0])
    st.table[st.table < 0] = -1
    st.table[st.table >= 40] = -1
    books, status = Books(st), torch.zeros(1, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    keep = [ints(torch, x) for x in ([-1, 3, 6, 2], [7, 7, 7, 7], [0, 1, 99], [-5, 2, 1], [3, 50, -2, 4], [5, 1, 2, 99])]
    st.handle.extend(4, keep[0].data_ptr(), keep[1].data_ptr(), status.data_ptr(), stream)
    assert int(status) == books.extend([3, 2], [7, 7])
    books.same(torch, st)
    st.handle.fork(3, keep[2].data_ptr(), keep[3].data_ptr(), status.data_ptr(), stream)
    assert int(status) == books.fork([1], [2])
    books.same(torch, st)
    st.handle.free(3, keep[3].data_ptr(), stream)
    books.free([2, 1])
    books.same(torch, st)
    st.handle.copy(4, keep[4].data_ptr(), keep[5].data_ptr(), stream)
    for x in books.pool:
        x[:, 5] = x[:, 3]
    books.same(torch, st)


def test_a_pool_without_pages_left(torch_cuda, hs):
    torch = torch_cuda
    st = State(torch, hs, 0, 5, 4, 1, 8, 4, 4, fill=1.0)
    books, status = Books(st), torch.zeros(1, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    add, parents, children = ints(torch, [6, 10, 9, 3]), ints(torch, [0, 0, 1]), ints(torch, [2, 3, 1])
    st.handle.extend(4, 0, add.data_ptr(), status.data_ptr(), stream)
    assert int(status) == books.extend(range(4), [6, 10, 9, 3]) == 4
    books.same(torch, st)
    st.handle.fork(3, parents.data_ptr(), children.data_ptr(), status.data_ptr(), stream)
    assert int(status) == books.fork([0, 0, 1], [2, 3, 1])
    books.same(torch, st)


# ---- how it is called --------------------------------------------------------------------------------------------------


def test_workspaces_are_asked_for_and_left_as_they_were(torch_cuda, hs):
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, 2, 23)
    chunks = many(hs, st, batch, attention)
    need = min(st.handle.attend_workspace(batch, a) for a in (attention, chunks))
    most = max(st.handle.attend_workspace(batch, a) for a in (attention, chunks))
    assert need > 0
    qd = device(torch, q, 2)
    out = torch.empty_like(qd)
    for size in (0, need - 1):
        w = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
        with pytest.raises(hs.HspmmError) as e:
            st.handle.attend(0, batch, attention, heads_view(hs, qd), heads_view(hs, out), workspace=w.data_ptr() if size else 0, workspace_bytes=size)
        assert e.value.code == 1 and str(st.handle.attend_workspace(batch, attention)) in str(e.value)
    # one workspace, calls of different shapes in turn: counters in front of the sums are zero again
    w = torch.zeros(most + 4096, dtype=torch.uint8, device="cuda")
    want = expected(q, k, v, new, old, scale, causal, window)
    small = hs.Attention(attention.q_heads, attention.scale, longest_chunk=1, longest=300)
    for _ in range(3):
        for a in (attention, small, chunks):
            o, l = attend(torch, hs, st, batch, a, q, workspace=w)
            assert_attended(2, o, l, want, k, v, q.shape[2])
        torch.cuda.synchronize()
        assert int(w[:65536].count_nonzero()) == 0


def test_streams_and_a_recorded_step(torch_cuda, hs):
    # extend, append and attend on a stream of their own, and recorded in a graph that replays with other inputs in place
    torch = torch_cuda
    rng = np.random.default_rng(4)
    S, page, heads, dim, steps = 6, 16, 2, 64, 5
    st = State(torch, hs, 0, 64, page, heads, dim, S, 10)
    table = torch.from_numpy(hs.rotary_table(dim, 200)).cuda()
    r = hs.Rotary(dim, 200, table.data_ptr())
    starts, one = ints(torch, np.arange(S + 1)), ints(torch, np.ones(S))
    batch = hs.Batch(S, S, starts.data_ptr())
    a = hs.Attention(heads * 2, 0.125, longest_chunk=1, longest=150)
    w = torch.zeros(max(1, st.handle.attend_workspace(batch, a)), dtype=torch.uint8, device="cuda")
    q, k, v = (torch.zeros(S, h, dim, dtype=torch.float16, device="cuda") for h in (heads * 2, heads, heads))
    q2, out = torch.zeros_like(q), torch.zeros_like(q)
    prompt = [int(x) for x in rng.integers(0, 120, S)]

    def step(stream):
        st.handle.extend(S, 0, one.data_ptr(), 0, stream)
        st.handle.append(0, batch, heads_view(hs, k), heads_view(hs, v), rotary=r, q_heads=heads * 2, q=heads_view(hs, q), q_out=heads_view(hs, q2), stream=stream)
        st.handle.attend(0, batch, a, heads_view(hs, q2), heads_view(hs, out), workspace=w.data_ptr(), workspace_bytes=w.numel(), stream=stream)

    def begin():
        st.table.fill_(-1)
        st.lengths.zero_()
        st.references.zero_()
        for p in st.pool:
            p.copy_(filled)
        st.handle.extend(S, 0, ints(torch, prompt).data_ptr(), 0, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()

    filled = torch.randn(st.pool[0].shape, device="cuda").half()
    inputs = [[torch.randn(x.shape, device="cuda").half() for x in (q, k, v)] for _ in range(steps)]
    begin()
    side = torch.cuda.Stream()
    results = []
    for x in inputs:
        for to, y in zip((q, k, v), x):
            to.copy_(y)
        side.wait_stream(torch.cuda.current_stream())
        step(side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        results.append(out.clone())
        out.zero_()
    begin()
    with torch.cuda.stream(side):
        step(side.cuda_stream)                                # (eagerly once: the device is known)
    torch.cuda.synchronize()
    begin()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(side.cuda_stream)
    begin()
    for x, want in zip(inputs, results):
        for to, y in zip((q, k, v), x):
            to.copy_(y)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert st.lengths.tolist() == [p + steps for p in prompt]


@pytest.mark.parametrize("chunks", [False, True])
def test_two_streams_with_workspaces_of_their_own(torch_cuda, hs, chunks):
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, 2, 23)
    if chunks:
        attention = many(hs, st, batch, attention)
    want = expected(q, k, v, new, old, scale, causal, window)
    qd = device(torch, q, 2)
    need = st.handle.attend_workspace(batch, attention)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, spaces = [torch.zeros_like(qd) for _ in range(2)], [torch.zeros(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    lses = [torch.zeros(qd.shape[:2], device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(8):
        for s, o, l, w in zip(streams, outs, lses, spaces):
            st.handle.attend(0, batch, attention, heads_view(hs, qd), heads_view(hs, o), lse=l.data_ptr(), workspace=w.data_ptr(), workspace_bytes=need, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for o, l in zip(outs, lses):
        assert_attended(2, o, l, want, k, v, q.shape[2])


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("dtype,case", [(0, 2), (2, 8), (1, 8), (0, 18)])
def test_other_scales(torch_cuda, hs, scale, dtype, case):
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, _, window, causal = attention_case(torch, hs, dtype, case, seed=1)
    other = hs.Attention(attention.q_heads, scale, causal=causal, window=window, longest_chunk=max(new), longest=attention.longest)
    for a in (other, many(hs, st, batch, other)):
        out, lse = attend(torch, hs, st, batch, a, q)
        assert_attended(dtype, out, lse, expected(q, k, v, new, old, np.float64(np.float32(scale)), causal, window), k, v, q.shape[2])


def test_tokens_of_no_chunk_are_left_alone(torch_cuda, hs):
    # chunks that begin in front of the batch, end behind it or belong to no sequence
    torch = torch_cuda
    st, batch, attention, q, k, v, new, old, rows, scale, window, causal = attention_case(torch, hs, 2, 5)
    T = q.shape[0]
    starts, rd = ints(torch, [0, 3, 4, T + 5]), ints(torch, [int(rows[0]), 1 << 20, int(rows[2])])
    out = torch.full(q.shape, 7.0, device="cuda").bfloat16()
    qd = device(torch, q, 2)
    for a in (hs.Attention(attention.q_heads, attention.scale, longest_chunk=1, longest=400), many(hs, st, batch, attention)):
        b = hs.Batch(3, T, starts.data_ptr(), rd.data_ptr())
        w = torch.zeros(max(1, st.handle.attend_workspace(b, a)), dtype=torch.uint8, device="cuda")
        st.handle.attend(0, b, a, heads_view(hs, qd), heads_view(hs, out), workspace=w.data_ptr(), workspace_bytes=w.numel(), stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert (out[3:] == 7).all() and not (out[:3] == 7).all()
