"""Batches and lists of many sequences: more than a wave looks at at a time (64), more than a workgroup keeps near (256) and than a workgroup has threads (1024).
Needs a real MI355X: run with -m gpu."""
import numpy as np
import pytest

from cache_util import State, rounded, to64
from test_cache_edges_gpu import Lives
from test_cache_gpu import assert_attended, assert_turned, attend, device, expected, heads_view, ints, laid_out, many, turned64
from test_spmm_gpu import torch_cuda  # noqa: F401

pytestmark = pytest.mark.gpu


def ragged(torch, hs, dtype, sequences, most_new, most_old, heads, dim, page, seed):
    """Chunks of 0 to most_new tokens behind 0 to most_old older ones, batch rows in another order than the cache's."""
    rng = np.random.default_rng(seed)
    new, old = rng.integers(0, most_new + 1, sequences), rng.integers(0, most_old + 1, sequences)
    new[-1] = most_new
    lengths, rows = new + old, rng.permutation(sequences + 3)[:sequences]
    used = int((-(-lengths // page)).sum())
    st = State(torch, hs, dtype, used + 5, page, heads, dim, sequences + 3, (most_new + most_old) // page + 2)
    by_row = np.zeros(sequences + 3, int)
    by_row[rows] = lengths
    st.place(rng, by_row)
    starts, rd = ints(torch, np.concatenate([[0], np.cumsum(new)])), ints(torch, rows)
    st.kept = (starts, rd)
    return st, hs.Batch(sequences, int(new.sum()), starts.data_ptr(), rd.data_ptr()), new, old, rows, rng


def stored(torch, st, rows, lengths, which, values):
    """Puts the sequences' values (a list, tokens x heads x dim) into their pages."""
    seq, at = np.repeat(rows, lengths), np.concatenate([np.arange(n) for n in lengths])
    ids = torch.from_numpy(st.table.cpu().numpy()[seq, at // st.page_tokens].astype(np.int64)).cuda()
    st.view(which)[0][ids, :, torch.from_numpy(at % st.page_tokens).cuda()] = device(torch, np.concatenate(values), st.dtype)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("sequences,most_new,most_old,page", [(65, 1, 90, 16), (100, 9, 40, 16), (255, 3, 20, 7), (256, 2, 20, 7), (300, 5, 30, 4), (4097, 2, 9, 2), (5000, 1, 12, 16)])
def test_batches_of_many_sequences(torch_cuda, hs, dtype, sequences, most_new, most_old, page):
    torch = torch_cuda
    heads, shared, dim = 1, 2, 32
    st, batch, new, old, rows, rng = ragged(torch, hs, dtype, sequences, most_new, most_old, heads, dim, page, sequences)
    k, v = ([rounded(torch, rng.standard_normal((n, heads, dim)), dtype) for n in new + old] for _ in range(2))
    q = rounded(torch, rng.standard_normal((int(new.sum()), heads * shared, dim)), dtype)
    stored(torch, st, rows, new + old, 0, k)
    stored(torch, st, rows, new + old, 1, v)
    scale = np.float64(np.float32(0.2))
    want = expected(q, k, v, new, old, scale, True, 0)
    a = hs.Attention(heads * shared, float(scale), longest_chunk=most_new, longest=most_new + most_old)
    for b in (a, many(hs, st, batch, a)):
        out, lse = attend(torch, hs, st, batch, b, q)
        assert_attended(dtype, out, lse, want, k, v, dim)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("sequences,most_new,page", [(65, 1, 16), (100, 40, 16), (255, 3, 7), (256, 2, 7), (300, 9, 4), (4097, 2, 2)])
def test_appending_to_many_sequences(torch_cuda, hs, dtype, sequences, most_new, page):
    torch = torch_cuda
    heads, shared, dim, dims = 2, 2, 16, 8
    st, batch, new, old, rows, rng = ragged(torch, hs, dtype, sequences, most_new, 30, heads, dim, page, sequences + 1)
    tokens = int(new.sum())
    positions, seq = np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)]), np.repeat(rows, new)
    ids = st.table.cpu().numpy()[seq, positions // page]
    table = hs.rotary_table(dims, most_new + 30)
    on_gpu = torch.from_numpy(table).cuda()
    r = hs.Rotary(dims, most_new + 30, on_gpu.data_ptr())
    q, k, v = (rounded(torch, rng.standard_normal((tokens, h, dim)), dtype) for h in (heads * shared, heads, heads))
    before = [p.clone() for p in st.pool]
    for layout in ("tokens", "features"):
        for pool, x in zip(st.pool, before):
            pool.copy_(x)
        qd, kd, vd = (laid_out(torch, device(torch, x, dtype), layout) for x in (q, k, v))
        out = torch.empty((tokens, heads * shared, dim), dtype=qd.dtype, device="cuda")
        st.handle.append(0, batch, heads_view(hs, kd), heads_view(hs, vd), rotary=r, q_heads=heads * shared, q=heads_view(hs, qd), q_out=heads_view(hs, out),
                         stream=torch.cuda.current_stream().cuda_stream)
        for x, got in ((q, to64(out)), (k, to64(st.view(0)[0])[ids, :, positions % page])):
            want, size = turned64(x, table.astype(np.float64), positions, dims, False, False)
            assert_turned(got, want, size, dtype, 1.0)
        assert np.array_equal(to64(st.view(1)[0])[ids, :, positions % page], v)
        # nothing else has changed
        idt, slot = torch.from_numpy(ids.astype(np.int64)).cuda(), torch.from_numpy(positions % page).cuda()
        for i in range(2):
            now = st.view(i)[0].clone()
            st.pool[i].copy_(before[i])
            st.view(i)[0][idt, :, slot] = now[idt, :, slot]
            assert torch.equal(st.view(i)[0].contiguous().view(torch.uint8), now.view(torch.uint8))


@pytest.mark.parametrize("S,pages", [(1024, 9000), (1025, 9000), (3000, 20000), (3000, 7000)])
def test_page_lists_of_many_entries(torch_cuda, hs, S, pages):
    torch = torch_cuda
    rng = np.random.default_rng(S + pages)
    page, P = 4, 6
    st = State(torch, hs, 2, pages, page, 1, 8, S, P)
    for pool in st.pool:
        pool.copy_(torch.randn(pool.shape, device="cuda").bfloat16())
    books, status, stream = Lives(st), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.cuda.current_stream().cuda_stream
    for step in range(6):
        rows = rng.permutation(S)
        n = S if step < 3 else int(rng.integers(S // 2, S))
        rows = rows[:n]
        rd = ints(torch, rows)
        if step in (0, 3, 5):
            add = rng.integers(0, 3 * page, n)
            ad = ints(torch, add)
            st.handle.extend(n, rd.data_ptr(), ad.data_ptr(), status.data_ptr(), stream)
            assert int(status) == books.extend(rows, add)
        elif step in (1, 4):
            parents = rng.integers(0, S, n)
            pd = ints(torch, parents)
            st.handle.fork(n, pd.data_ptr(), rd.data_ptr(), status.data_ptr(), stream)
            assert int(status) == books.fork(parents, rows)
        else:
            st.handle.free(n // 2, rd.data_ptr(), stream)
            books.free(rows[: n // 2])
        books.same(torch, st)
