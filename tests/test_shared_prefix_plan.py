"""How attention over shared prefixes is split, as far as its workspace shows it.  No GPU needed."""
import random

import pytest

from test_cache import ADDRESS, cache

COUNTERS = 4 * 16384


def planned(hs, dtype, groups, chunks, prefix, behind, heads, shared, dim, page=16, hint=None, sequences=None):
    """Bytes of a shared attention's workspace and of plain attention's, and those of a part of its sums: the sums over some keys of all rows.  chunks: new tokens of
    every sequence; hint: what the call says in place of the longest chunk, the longest sequence, the tokens of a group and the longest prefix."""
    n, tokens, longest = len(chunks), sum(chunks), prefix + behind + max(chunks)
    c = cache(hs, dtype=dtype, heads=heads, head_dim=dim, page_tokens=page, sequences=n, table_pages=-(-longest // page), pages=1 << 20)
    chunk, most_keys, most, common = hint or (max(chunks), longest, tokens, prefix)
    b, a = hs.Batch(n, tokens, ADDRESS), hs.Attention(heads * shared, 0.125, longest_chunk=chunk, longest=most_keys)
    p = hs.Prefix(groups, ADDRESS, ADDRESS, most_tokens=most, longest=common)
    return c.attend_shared_workspace(b, p, a), c.attend_workspace(b, a), tokens * heads * shared * (dim + 4) * 4


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("seed", range(60))
def test_sums_are_no_more_than_the_rows_and_a_launch_of_tiles(hs, dtype, seed):
    # A prefix and what is behind it are in P <= W / cells + 2 parts each, W workgroups of the chip and cells >= 1 tiles and heads, of R rows; there are no more than R (cells + heads) rows, and
    # heads are no more than cells.  So rows times parts are at most 2 W R + 2 rows of either, W R = 512 x 128 or 2048 x 16.
    rng = random.Random(seed)
    cases = [(1, [4096] * 8, 16000, 300, 8, 4, 128), (1, [1000] * 16, 8000, 300, 8, 4, 128), (1, [250] * 16, 6000, 300, 8, 4, 128), (1, [16] * 128, 16000, 300, 8, 4, 128),
             (1, [8] * 256, 8000, 300, 8, 4, 128), (1, [1] * 256, 128000, 300, 8, 4, 128)]
    if seed < len(cases):
        groups, chunks, prefix, behind, heads, shared, dim = cases[seed]
    else:
        n = int(2 ** rng.uniform(0, 11))
        groups, chunks = rng.randint(1, min(n, 8)), [int(2 ** rng.uniform(0, rng.choice([1, 6, 11]))) for _ in range(n)]
        prefix, behind, heads, shared, dim = int(2 ** rng.uniform(4, 18)), int(2 ** rng.uniform(0, 14)), rng.choice([1, 2, 4, 8, 32]), rng.choice([1, 3, 4, 8]), rng.choice([64, 96, 128, 160, 256])
    for hint in (None, (1, 0, 1, 1), (0, 0, 0, 0), (100000, 0, 100000, 0)):
        got, plain, part = planned(hs, dtype, groups, chunks, prefix, behind, heads, shared, dim, hint=hint)
        rows = part // (4 * (dim + 4))
        assert got <= max(plain, COUNTERS + (4 * 512 * 128 + 4 * rows) * (dim + 4) * 4), (got / part, got, plain)


def by_prefixes(got, plain, part):
    """Whether a call goes by tiles of the prefixes' rows: it leaves sums of all rows, and plain attention's tiles leave others."""
    return got != plain and got > COUNTERS and (got - COUNTERS) % part == 0


@pytest.mark.parametrize("dtype", [0, 2])
@pytest.mark.parametrize("chunk", [1, 31, 32, 33, 200, 1000, 2500])
def test_a_long_chunk_takes_the_prefix_from_no_single_token(hs, dtype, chunk):
    assert by_prefixes(*planned(hs, dtype, 1, [1] * 63 + [chunk], 8000, 300, 8, 4, 128))
    assert by_prefixes(*planned(hs, dtype, 2, [1] * 40 + [chunk] + [2] * 23, 6000, 700, 4, 8, 64))


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_chunks_that_fill_tiles_leave_no_sums(hs, dtype):
    for chunks in ([4096] * 8, [1500, 1200, 1100], [2000] * 3):
        got, plain, _ = planned(hs, dtype, 1, chunks, 16000, 300, 8, 4, 128)
        assert got == plain


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_hints_that_are_not_there_leave_large_calls_their_prefixes(hs, dtype):
    for groups, chunks in ((1, [1] * 64), (4, [1, 2, 3, 4] * 20), (2, [20] * 30)):
        for hint in ((0, 0, 0, 0), (0, 9000, 0, 8000), (1, 9000, 0, 0)):
            assert by_prefixes(*planned(hs, dtype, groups, chunks, 8000, 300, 8, 4, 128, hint=hint))
