"""Rotary positions, the paged cache and attention: what needs no GPU - the table of rotary positions against its formulas, and
the refusals, which come before anything reaches a device."""
import ctypes as C
import math

import numpy as np
import pytest


def angles64(dims, positions, kind, base, factor, original, fast, slow):
    i = np.arange(dims // 2)
    if kind == "base":
        base = base * factor ** (dims / (dims - 2))
    f = base ** (-2.0 * i / dims)
    scale = 1.0
    if kind == "linear":
        f = f / factor
    if kind == "yarn":
        # turns within the original context: 2 pi / f is a wavelength
        def pair(turns):
            return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dims - 1)
        ramp = np.clip((i - low) / (max(high, low + 0.001) - low), 0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        scale = 0.1 * math.log(factor) + 1
    a = np.arange(positions)[:, None] * f[None]
    return np.stack([np.cos(a), np.sin(a)], -1) * scale


@pytest.mark.parametrize("kind,factor", [("plain", 1.0), ("linear", 4.0), ("base", 8.0), ("yarn", 16.0), ("yarn", 1.0)])
@pytest.mark.parametrize("dims,positions,base", [(2, 5, 10000.0), (6, 1, 500.0), (64, 700, 10000.0), (128, 9001, 500000.0)])
def test_rotary_table_is_its_formula(hs, kind, factor, dims, positions, base):
    if kind == "base" and dims == 2:
        with pytest.raises(hs.HspmmError):
            hs.rotary_table(dims, positions, kind, base, factor)
        return
    got = hs.rotary_table(dims, positions, kind, base, factor, original_length=2048.0)
    want = angles64(dims, positions, kind, base, factor, 2048.0, 32.0, 1.0)
    # one rounding to fp32 of values up to the scale; the angles in 64 bits carry 2^-52 of themselves
    assert got.shape == want.shape
    assert np.abs(got - want).max() <= 2.0 ** -24 * (0.1 * math.log(factor) + 1) + positions * 2.0 ** -48


def test_scaled_frequencies_keep_the_fast_pairs_and_slow_the_last(hs):
    plain, yarn = hs.rotary_table(64, 2), hs.rotary_table(64, 2, "yarn", factor=8.0, original_length=4096.0)
    angle = lambda t: np.arctan2(t[1, :, 1].astype(np.float64), t[1, :, 0].astype(np.float64))  # noqa: E731
    assert angle(yarn)[0] == pytest.approx(angle(plain)[0], rel=1e-6)
    assert angle(yarn)[-1] == pytest.approx(angle(plain)[-1] / 8, rel=1e-4)
    based = hs.rotary_table(64, 2, "base", factor=8.0)
    assert angle(based)[0] == pytest.approx(angle(plain)[0], rel=1e-6) and angle(based)[-1] == pytest.approx(angle(plain)[-1] / 8, rel=1e-4)


@pytest.mark.parametrize("bad", [dict(dims=0), dict(dims=7), dict(base=1.0), dict(base=math.inf), dict(kind="linear", factor=0.5), dict(kind="base", factor=math.nan),
                                 dict(kind="yarn", factor=2.0, original_length=0.0), dict(kind="yarn", factor=2.0, original_length=64.0, fast_turns=1.0, slow_turns=1.0)])
def test_rotary_table_refuses(hs, bad):
    a = dict(dims=8, positions=4)
    a.update(bad)
    with pytest.raises(hs.HspmmError) as e:
        hs.rotary_table(**a)
    assert e.value.code == 1
    with pytest.raises(ValueError):
        hs.rotary_table(8, 4, "other")


ADDRESS = 1 << 20      # never read: every call here is refused


def cache(hs, **kw):
    a = dict(dtype=hs.BF16, layers=2, pages=8, page_tokens=16, heads=4, head_dim=64, sequences=3, table_pages=4, keys=ADDRESS, values=ADDRESS,
             table=ADDRESS, lengths=ADDRESS, references=ADDRESS, scratch=ADDRESS)
    a.update(kw)
    return hs.Cache(**a)


def refused(hs, code, f, *words):
    with pytest.raises(hs.HspmmError) as e:
        f()
    assert e.value.code == code, str(e.value)
    for w in words:
        assert w in str(e.value), str(e.value)


@pytest.mark.parametrize("kw,code", [(dict(dtype=7), 1), (dict(order=2), 1), (dict(layers=0), 1), (dict(pages=0), 1), (dict(page_tokens=0), 1), (dict(heads=0), 1),
                                     (dict(head_dim=0), 1), (dict(sequences=0), 1), (dict(table_pages=0), 1), (dict(keys=0), 1), (dict(values=ADDRESS + 8), 1), (dict(table=0), 1),
                                     (dict(lengths=0), 1), (dict(references=0), 1), (dict(scratch=0), 1), (dict(page_stride=4095), 1), (dict(page_stride=-1), 1),
                                     (dict(layer_stride=-5), 1), (dict(sequences=1 << 16, table_pages=1 << 16), 5), (dict(heads=1 << 16), 5), (dict(page_tokens=1 << 30), 5)])
def test_every_call_refuses_a_cache_that_is_none(hs, kw, code):
    c, b, a = cache(hs, **kw), hs.Batch(1, 4, ADDRESS), hs.Attention(4, 1.0)
    x = hs.Heads(ADDRESS, 256, 64)
    for f in (lambda: c.append(0, b, x, x), lambda: c.attend(0, b, a, x, x), lambda: c.attend_workspace(b, a), lambda: c.extend(1, 0, ADDRESS), lambda: c.fork(1, ADDRESS, ADDRESS),
              lambda: c.free(1, ADDRESS), lambda: c.compact(), lambda: c.copy(1, ADDRESS, ADDRESS)):
        refused(hs, code, f)


def test_append_refuses(hs):
    c, b, x = cache(hs), hs.Batch(3, 4, ADDRESS), hs.Heads(ADDRESS, 256, 64)
    refused(hs, 1, lambda: c.append(2, b, x, x), "layer")
    refused(hs, 1, lambda: c.append(0, hs.Batch(3, 4, 0), x, x), "starts")
    refused(hs, 1, lambda: c.append(0, hs.Batch(0, 4, ADDRESS), x, x))
    refused(hs, 1, lambda: c.append(0, hs.Batch(4, 4, ADDRESS), x, x), "sequences")
    refused(hs, 1, lambda: c.append(0, b, hs.Heads(0, 256, 64), x), "k")
    refused(hs, 1, lambda: c.append(0, b, x, hs.Heads(ADDRESS + 1, 256, 64)), "v", "align")
    refused(hs, 1, lambda: c.append(0, b, x, hs.Heads(ADDRESS, -1, 64)), "strides")
    refused(hs, 1, lambda: c.append(0, b, x, x, q_heads=8, q=x), "q_out")
    for r in (hs.Rotary(3, 9, ADDRESS), hs.Rotary(66, 9, ADDRESS), hs.Rotary(64, 0, ADDRESS), hs.Rotary(64, 9, 0), hs.Rotary(64, 9, ADDRESS + 4)):
        refused(hs, 1, lambda: c.append(0, b, x, x, rotary=r))
    L = hs.load_library()
    assert L.hspmm_cache_append(c._c, 0, None, x, x, None, 0, None, None, None) == 1 and b"batch" in L.hspmm_last_error()


def test_rotate_refuses(hs):
    x, r = hs.Heads(ADDRESS, 256, 64), hs.Rotary(64, 9, ADDRESS)
    refused(hs, 1, lambda: hs.rotate(5, r, 4, 4, 64, x, x, ADDRESS), "dtype")
    refused(hs, 1, lambda: hs.rotate(hs.FP16, None, 4, 4, 64, x, x, ADDRESS), "rotary")
    refused(hs, 1, lambda: hs.rotate(hs.FP16, r, 4, 4, 0, x, x, ADDRESS))
    refused(hs, 1, lambda: hs.rotate(hs.FP16, r, 4, 4, 32, x, x, ADDRESS), "64 of 32")
    refused(hs, 1, lambda: hs.rotate(hs.FP16, r, 4, 4, 64, x, x, 0), "positions")
    refused(hs, 1, lambda: hs.rotate(hs.FP16, r, 4, 4, 64, None, x, ADDRESS), "x")
    refused(hs, 1, lambda: hs.rotate(hs.TF32, r, 4, 4, 64, x, hs.Heads(ADDRESS + 2, 256, 64), ADDRESS), "y")
    hs.rotate(hs.FP16, r, 0, 4, 64, None, None, 0)         # nothing to do


def test_attend_refuses(hs):
    c, b, a, x = cache(hs), hs.Batch(3, 4, ADDRESS), hs.Attention(8, 0.125), hs.Heads(ADDRESS, 512, 64)
    refused(hs, 1, lambda: c.attend(2, b, a, x, x), "layer")
    for q in (hs.Attention(0, 1.0), hs.Attention(6, 1.0), hs.Attention(8, math.nan), hs.Attention(8, math.inf), hs.Attention(8, 1.0, causal=False, window=5)):
        refused(hs, 1, lambda: c.attend(0, b, q, x, x))
        refused(hs, 1, lambda: c.attend_workspace(b, q))
    for q in (hs.Heads(ADDRESS + 8, 512, 64), hs.Heads(ADDRESS, 516, 64), hs.Heads(ADDRESS, 512, 68), hs.Heads(ADDRESS, 1, 256, 4)):
        refused(hs, 5, lambda: c.attend(0, b, a, q, x), "q")
    refused(hs, 1, lambda: c.attend(0, b, a, x, hs.Heads(ADDRESS, 1, 256, 0)), "out")
    refused(hs, 1, lambda: c.attend(0, b, a, x, x, lse=ADDRESS + 2), "lse")
    for d in (4, 60, 264):
        refused(hs, 5, lambda: cache(hs, head_dim=d).attend(0, b, a, x, x), "elements")
    refused(hs, 5, lambda: cache(hs, page_stride=16 * 4 * 64 + 4).attend(0, b, a, x, x), "16 bytes")
    # more tiles than a launch has workgroups
    wide = hs.Batch(3, 1 << 29, ADDRESS)
    for f in (lambda: c.attend(0, wide, hs.Attention(4, 1.0, longest_chunk=1 << 29), x, x), lambda: c.attend_workspace(wide, hs.Attention(4, 1.0, longest_chunk=1 << 29))):
        refused(hs, 5, f, "several calls")
    c.attend(0, hs.Batch(3, 0, 0), a, None, None)           # no tokens
    L = hs.load_library()
    assert L.hspmm_cache_attend_workspace(c._c, b, a, None) == 1


def test_page_calls_refuse(hs):
    c = cache(hs)
    refused(hs, 1, lambda: c.extend(4, 0, ADDRESS), "list")
    refused(hs, 1, lambda: c.extend(1, 0, 0), "add")
    refused(hs, 1, lambda: c.fork(1, 0, ADDRESS), "parents")
    refused(hs, 1, lambda: c.fork(1, ADDRESS, 0), "children")
    refused(hs, 1, lambda: c.free(4, ADDRESS), "list")
    refused(hs, 1, lambda: c.free(1, 0), "rows")
    refused(hs, 1, lambda: c.copy(9, ADDRESS, ADDRESS), "copy")
    refused(hs, 1, lambda: c.copy(1, ADDRESS, 0))
    c.free(0, 0)
    c.fork(0, 0, 0)
    c.copy(0, 0, 0)


def test_calls_fail_loudly_without_a_gfx950_device(hs):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    c, b, x = cache(hs), hs.Batch(3, 4, ADDRESS), hs.Heads(ADDRESS, 512, 64)
    for f in (lambda: c.append(0, b, x, x), lambda: c.attend(0, b, hs.Attention(8, 1.0), x, x), lambda: c.extend(1, 0, ADDRESS), lambda: c.fork(1, ADDRESS, ADDRESS),
              lambda: c.free(1, ADDRESS), lambda: c.compact(), lambda: c.copy(1, ADDRESS, ADDRESS), lambda: hs.rotate(hs.FP16, hs.Rotary(64, 9, ADDRESS), 4, 4, 64, x, x, ADDRESS)):
        refused(hs, 2, f)


def test_null_structures_are_refused(hs):
    L = hs.load_library()
    c = cache(hs)
    n = C.c_uint64()
    assert L.hspmm_cache_extend(None, 1, None, None, None, None) == 1
    assert L.hspmm_cache_attend_workspace(c._c, None, hs.Attention(8, 1.0), C.byref(n)) == 1
    assert L.hspmm_cache_attend_workspace(c._c, hs.Batch(1, 1, ADDRESS), None, C.byref(n)) == 1


@pytest.mark.parametrize("d", [1, 2, 3, 7, 16, 24, 96, 1000, 65535, (1 << 30) - 1, 1 << 30])
def test_division_by_multiplication(d):
    # the rule of Divisor (cache_device.h), restated: every quotient of 31 bits is exact
    l = 0
    while l < 31 and (1 << l) < d:
        l += 1
    m = (1 << (31 + l)) // d + 1
    assert m < 1 << 32
    rng = np.random.default_rng(d)
    ns = np.concatenate([rng.integers(0, 1 << 31, 2000), np.arange(50), (1 << 31) - 1 - np.arange(50), d * rng.integers(0, ((1 << 31) - 1) // d, 500, endpoint=True)])
    for n in ns.tolist() + [x - 1 for x in ns.tolist() if x]:
        assert (n * m) >> (31 + l) == n // d and n * m < 1 << 64
