"""Attention over shared prefixes, accumulated attention weights and eviction: the refusals, which come before anything reaches
a device.  No GPU needed."""
import ctypes as C
import math

import pytest

from test_cache import ADDRESS, cache, refused


def shared(hs, c=None, batch=None, prefix=None, attention=None, q=None, out=None, layer=0, **kw):
    x = hs.Heads(ADDRESS, 512, 64)
    c = c or cache(hs)
    a = dict(lse=0, workspace=0, workspace_bytes=0)
    a.update(kw)
    return c.attend_shared(layer, batch or hs.Batch(3, 4, ADDRESS), prefix or hs.Prefix(1, ADDRESS, ADDRESS), attention or hs.Attention(8, 0.125), q or x, out or x, **a)


BAD_CACHES = [(dict(dtype=7), 1), (dict(pages=0), 1), (dict(keys=0), 1), (dict(scratch=0), 1), (dict(page_stride=4095), 1), (dict(heads=1 << 16), 5)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_every_call_refuses_a_cache_that_is_none(hs, kw, code):
    c, b, a, w = cache(hs, **kw), hs.Batch(1, 4, ADDRESS), hs.Attention(4, 1.0), hs.Weights(ADDRESS, 1, 1, 1)
    p, x = hs.Prefix(1, ADDRESS, ADDRESS), hs.Heads(ADDRESS, 256, 64)
    for f in (lambda: c.attend_shared(0, b, p, a, x, x), lambda: c.attend_shared_workspace(b, p, a), lambda: c.weigh(0, b, a, x, ADDRESS, w), lambda: c.weigh_workspace(b, a),
              lambda: c.evict(1, ADDRESS, 0, w, 4), lambda: c.evict_workspace(1, 4)):
        refused(hs, code, f)


def test_attend_shared_refuses(hs):
    c, b, a, x = cache(hs), hs.Batch(3, 4, ADDRESS), hs.Attention(8, 0.125), hs.Heads(ADDRESS, 512, 64)
    refused(hs, 1, lambda: shared(hs, layer=2), "layer")
    for p in (hs.Prefix(4, ADDRESS, ADDRESS), hs.Prefix(1, 0, ADDRESS), hs.Prefix(1, ADDRESS, 0)):
        refused(hs, 1, lambda: shared(hs, prefix=p), "groups")
        refused(hs, 1, lambda: c.attend_shared_workspace(b, p, a), "groups")
    for q in (hs.Attention(0, 1.0), hs.Attention(6, 1.0), hs.Attention(8, math.nan), hs.Attention(8, 1.0, causal=False, window=5)):
        refused(hs, 1, lambda: shared(hs, attention=q))
    for q in (hs.Heads(ADDRESS + 8, 512, 64), hs.Heads(ADDRESS, 516, 64), hs.Heads(ADDRESS, 1, 256, 4)):
        refused(hs, 5, lambda: shared(hs, q=q), "q")
    refused(hs, 1, lambda: shared(hs, out=hs.Heads(ADDRESS, 1, 256, 0)), "out")
    refused(hs, 1, lambda: shared(hs, lse=ADDRESS + 2), "lse")
    # (a small call joins nothing; one that expects long sequences leaves sums)
    assert c.attend_shared_workspace(b, hs.Prefix(1, ADDRESS, ADDRESS), a) == 0
    far = cache(hs, table_pages=1 << 13)
    need = far.attend_shared_workspace(b, hs.Prefix(1, ADDRESS, ADDRESS), a)
    assert need >= 4 * 8 * 68 * 4
    for w in ((0, need), (ADDRESS, need - 1), (ADDRESS + 8, need)):
        refused(hs, 1, lambda: shared(hs, c=far, workspace=w[0], workspace_bytes=w[1]), "workspace")
    refused(hs, 5, lambda: shared(hs, c=cache(hs, head_dim=60)), "elements")
    wide = hs.Batch(3, 1 << 29, ADDRESS)
    refused(hs, 5, lambda: shared(hs, batch=wide, attention=hs.Attention(4, 1.0, longest_chunk=1 << 29)), "several calls")
    shared(hs, batch=hs.Batch(3, 0, 0))                      # no tokens
    L = hs.load_library()
    assert L.hspmm_cache_attend_shared_workspace(c._c, b, None, a, C.byref(C.c_uint64())) == 1
    assert L.hspmm_cache_attend_shared_workspace(c._c, b, hs.Prefix(1, ADDRESS, ADDRESS), a, None) == 1
    # without groups it is the other call, with that one's workspace
    assert c.attend_shared_workspace(b, hs.Prefix(0, 0, 0), a) == c.attend_workspace(b, a)


def test_weigh_refuses(hs):
    c, b, a, x, w = cache(hs), hs.Batch(3, 4, ADDRESS), hs.Attention(8, 0.125), hs.Heads(ADDRESS, 512, 64), hs.Weights(ADDRESS, 3 * 4 * 64, 4 * 64, 64)
    refused(hs, 1, lambda: c.weigh(2, b, a, x, ADDRESS, w), "layer")
    for lse in (0, ADDRESS + 2):
        refused(hs, 1, lambda: c.weigh(0, b, a, x, lse, w), "lse")
    for d in (math.nan, math.inf):
        refused(hs, 1, lambda: c.weigh(0, b, a, x, ADDRESS, w, decay=d), "decay")
    for bad in (hs.Weights(0, 1, 1, 1), hs.Weights(ADDRESS + 2, 1, 1, 1), hs.Weights(ADDRESS, -1, 1, 1), hs.Weights(ADDRESS, 1, -1, 1), hs.Weights(ADDRESS, 1, 1, -1)):
        refused(hs, 1, lambda: c.weigh(0, b, a, x, ADDRESS, bad), "weights")
    refused(hs, 1, lambda: c.weigh(0, b, hs.Attention(6, 1.0), x, ADDRESS, w))
    refused(hs, 5, lambda: c.weigh(0, b, a, hs.Heads(ADDRESS, 1, 256, 4), ADDRESS, w), "q")
    refused(hs, 5, lambda: cache(hs, head_dim=60).weigh(0, b, a, x, ADDRESS, w), "elements")
    many = cache(hs, sequences=1 << 22, table_pages=1)
    refused(hs, 5, lambda: many.weigh(0, hs.Batch(1 << 22, 4, ADDRESS), a, x, ADDRESS, w), "several calls")
    c.weigh(0, hs.Batch(3, 0, 0), a, None, 0, w)             # no tokens
    L = hs.load_library()
    assert L.hspmm_cache_weigh(c._c, 0, b, a, x, ADDRESS, None, 1.0, 0, None, 0, None) == 1
    assert L.hspmm_cache_weigh_workspace(c._c, b, a, 0, None) == 1


def test_evict_refuses(hs):
    c, w = cache(hs), hs.Weights(ADDRESS, 3 * 4 * 64, 4 * 64, 64)
    need = c.evict_workspace(2, 8)
    ok = dict(workspace=ADDRESS, workspace_bytes=need)
    refused(hs, 1, lambda: c.evict(4, ADDRESS, 0, w, 8, **ok), "list")
    refused(hs, 1, lambda: c.evict(2, 0, ADDRESS, w, 8, **ok), "parents")
    for keep in (0, 65):
        refused(hs, 1, lambda: c.evict(2, ADDRESS, 0, w, keep, **ok), "keep")
        refused(hs, 1, lambda: c.evict_workspace(2, keep), "keep")
    for first, last in ((9, 0), (0, 9), (4, 5), (0xFFFFFFFF, 0xFFFFFFFF)):
        refused(hs, 1, lambda: c.evict(2, ADDRESS, 0, w, 8, first=first, last=last, **ok), "first")
    refused(hs, 1, lambda: c.evict(2, ADDRESS, 0, hs.Weights(0, 1, 1, 1), 8, **ok), "weights")
    for a, n in ((0, need), (ADDRESS, need - 1), (ADDRESS + 4, need)):
        refused(hs, 1, lambda: c.evict(2, ADDRESS, 0, w, 8, workspace=a, workspace_bytes=n), "workspace")
    big = cache(hs, sequences=1 << 20, table_pages=1, layers=64)
    refused(hs, 5, lambda: big.evict(1 << 20, ADDRESS, 0, w, 8, **ok), "several calls")
    refused(hs, 5, lambda: big.evict_workspace(1 << 20, 8), "several calls")
    c.evict(0, 0, 0, w, 8)                                  # nothing to do
    assert c.evict_workspace(0, 8) == 0
    L = hs.load_library()
    assert L.hspmm_cache_evict_workspace(c._c, 1, 8, None) == 1
    assert L.hspmm_cache_evict(c._c, 1, ADDRESS, None, None, 8, 0, 0, None, None, ADDRESS, need, None) == 1


def test_calls_fail_loudly_without_a_gfx950_device(hs):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    c, b, a, x, w = cache(hs), hs.Batch(3, 4, ADDRESS), hs.Attention(8, 0.125), hs.Heads(ADDRESS, 512, 64), hs.Weights(ADDRESS, 3 * 4 * 64, 4 * 64, 64)
    big = dict(workspace=ADDRESS, workspace_bytes=1 << 30)
    for f in (lambda: c.attend_shared(0, b, hs.Prefix(1, ADDRESS, ADDRESS), a, x, x, **big), lambda: c.weigh(0, b, a, x, ADDRESS, w, **big),
              lambda: c.evict(2, ADDRESS, 0, w, 8, **big), lambda: c.evict(0, 0, 0, w, 8, status=ADDRESS)):
        refused(hs, 2, f)


def test_rows_of_weights_that_overlap_are_refused(hs):
    c, b, a, x, w = cache(hs), hs.Batch(3, 4, ADDRESS), hs.Attention(8, 0.125), hs.Heads(ADDRESS, 512, 64), hs.Weights(ADDRESS, 3 * 4 * 64, 4 * 64, 64)
    need = c.evict_workspace(2, 8)
    for bad in (hs.Weights(ADDRESS, 768, 256, 63), hs.Weights(ADDRESS, 768, 63, 256), hs.Weights(ADDRESS, 0, 256, 64), hs.Weights(ADDRESS, 768, 256, 0)):
        refused(hs, 1, lambda: c.evict(2, ADDRESS, 0, bad, 8, workspace=ADDRESS, workspace_bytes=need), "overlap")
    for bad in (hs.Weights(ADDRESS, 768, 0, 64), hs.Weights(ADDRESS, 768, 256, 0)):
        refused(hs, 1, lambda: c.weigh(0, b, a, x, ADDRESS, bad), "overlap")
    assert w.head_stride == 64


def test_an_eviction_of_very_many_tokens_has_room_for_its_pages(hs):
    # (what is to be kept and a page of tokens pass 32 bits together)
    c = cache(hs, layers=1, heads=1, head_dim=8, page_tokens=1 << 24, table_pages=256, sequences=1, pages=256)
    keep = 0x7FFFFFFF
    assert c.evict_workspace(1, keep) >= 4 * (2 * keep + 256 + 128 + 128)
    for keep in (0x80000000, 0xFFFFFFFF):
        refused(hs, 1, lambda: c.evict_workspace(1, keep), "keep")


def test_rows_of_weights_that_meet_others_of_another_kind_are_refused(hs):
    # (2 layers of 3 sequences of 4 heads of 64 tokens; each stride passes a row, but a head's rows are where another sequence's or layer's are)
    c = cache(hs)
    ok = dict(workspace=ADDRESS, workspace_bytes=c.evict_workspace(2, 8))
    for bad in ((768, 64, 64), (64, 256, 64), (64, 64, 256), (256, 256, 64), (767, 256, 64), (768, 255, 64), (191, 384, 64), (768, 64, 191)):
        refused(hs, 1, lambda: c.evict(2, ADDRESS, 0, hs.Weights(ADDRESS, *bad), 8, **ok), "overlap")
    # in any order, and with something between: refused for what comes behind
    for good in ((768, 256, 64), (64, 512, 128), (256, 512, 64), (64, 128, 384), (5000, 300, 70), (1 << 62, 1 << 60, 64)):
        refused(hs, 1, lambda: c.evict(2, ADDRESS, 0, hs.Weights(ADDRESS, *good), 8), "workspace")
