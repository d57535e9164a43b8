"""Calls of the paged cache that are larger than one launch: refused, before anything reaches a device.  No GPU needed."""
import pytest

from test_cache import ADDRESS, cache, refused


@pytest.mark.parametrize("tokens", [1 << 26, 0x7FFFFFFE])
def test_rotations_of_more_tokens_than_a_launch_has(hs, tokens):
    r = hs.Rotary(64, 9, ADDRESS)
    x, apart = hs.Heads(ADDRESS, 256, 64), hs.Heads(ADDRESS, 1, 256, 4)
    refused(hs, 5, lambda: hs.rotate(hs.FP16, r, tokens, 1, 64, x, x, ADDRESS), "several calls")
    refused(hs, 5, lambda: hs.rotate(hs.FP16, r, max(tokens, 1 << 30), 1, 64, apart, apart, ADDRESS), "several calls")
    refused(hs, 5, lambda: cache(hs).append(0, hs.Batch(3, tokens, ADDRESS), x, x), "several calls")
    # (as many as a launch has: that there is no device, or that it was given no memory, is another matter)
    refused(hs, 5, lambda: hs.rotate(hs.FP16, r, (1 << 29) + 7, 1, 64, apart, apart, ADDRESS), "several calls")


def test_heads_at_any_strides_of_more_than_a_launch_has(hs):
    c, apart = cache(hs, heads=32768, page_tokens=1, head_dim=8), hs.Heads(ADDRESS, 1, 64, 8)
    refused(hs, 5, lambda: c.append(0, hs.Batch(3, 4, ADDRESS), apart, apart), "several calls")


@pytest.mark.parametrize("n", [(1 << 24) - 1, 1 << 24, 1 << 27])
def test_lists_of_more_entries_than_a_launch_has(hs, n):
    c = cache(hs, sequences=1 << 27, table_pages=1, pages=1 << 28, heads=1, page_tokens=1)
    refused(hs, 5, lambda: c.fork(n, ADDRESS, ADDRESS), "several calls")
    refused(hs, 5, lambda: c.fork(min(n, (1 << 22) - 1), ADDRESS, ADDRESS), "several calls")
    refused(hs, 5, lambda: c.free(n, ADDRESS), "several calls")
    refused(hs, 5, lambda: c.copy(n, ADDRESS, ADDRESS), "several calls")
