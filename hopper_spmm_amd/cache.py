"""Rotary positions, a paged cache of keys and values and the attention over it (include/hspmm.h): what lies between two
products of a pruned decoder layer.

As in `Plan.run`, tensors are given by their device addresses (e.g. torch's `.data_ptr()`), and every call only launches
kernels on the stream it is given; what the addresses name stays the caller's.  The classes hold a call's
fixed part, so that a decoding loop makes them once.
"""
import ctypes as C

import numpy as np

from .capi import _check, load_library

HEADS_FIRST, TOKENS_FIRST = 0, 1
ROTARY_KINDS = {"plain": 0, "linear": 1, "base": 2, "yarn": 3}


class Heads(C.Structure):
    """A tensor tokens x heads x elements, strides in elements: `Heads(x.data_ptr(), *x.stride())`; of C of `Plan.run`
    (features x tokens) token_stride is 1."""
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64), ("dim_stride", C.c_int64)]

    def __init__(self, data, token_stride, head_stride, dim_stride=1):
        super().__init__(data, token_stride, head_stride, dim_stride)


class Rotary(C.Structure):
    """The first `dims` elements of a head turn, in pairs (i, i + dims / 2) or, interleaved, (2 i, 2 i + 1); table: address of
    positions x dims / 2 x (cosine, sine) in device memory (`rotary_table` makes it)."""
    _fields_ = [("dims", C.c_uint32), ("interleaved", C.c_int32), ("positions", C.c_uint32), ("table", C.c_void_p)]

    def __init__(self, dims, positions, table, interleaved=False):
        super().__init__(dims, int(bool(interleaved)), positions, table)


class Batch(C.Structure):
    """Tokens starts[b] .. starts[b + 1] - 1 are the last ones of the cache's sequence rows[b] (rows 0: b)."""
    _fields_ = [("sequences", C.c_uint32), ("tokens", C.c_uint32), ("starts", C.c_void_p), ("rows", C.c_void_p)]

    def __init__(self, sequences, tokens, starts, rows=0):
        super().__init__(sequences, tokens, starts, rows or None)


class Attention(C.Structure):
    """What of an attention stays the same from call to call; longest_chunk and longest choose kernels only."""
    _fields_ = [("q_heads", C.c_uint32), ("scale", C.c_float), ("causal", C.c_int32), ("window", C.c_uint32),
                ("longest_chunk", C.c_uint32), ("longest", C.c_uint32)]

    def __init__(self, q_heads, scale, causal=True, window=0, longest_chunk=1, longest=0):
        super().__init__(q_heads, scale, int(bool(causal)), window, longest_chunk, longest)


class Prefix(C.Structure):
    """Groups of a batch's rows that begin with the same tokens: rows firsts[g] .. firsts[g + 1] - 1 share the first tokens[g], which the first
    one's pages hold; most_tokens (of the batch, of a group) and longest (of a prefix) choose kernels only."""
    _fields_ = [("groups", C.c_uint32), ("most_tokens", C.c_uint32), ("longest", C.c_uint32), ("firsts", C.c_void_p), ("tokens", C.c_void_p)]

    def __init__(self, groups, firsts, tokens, most_tokens=0, longest=0):
        super().__init__(groups, most_tokens, longest, firsts or None, tokens or None)


class Weights(C.Structure):
    """Attention weight that cached keys have received, layers x sequences x heads x tokens floats (a head's tokens side by side):
    `Weights(w.data_ptr(), *w.stride()[:3])`."""
    _fields_ = [("data", C.c_void_p), ("layer_stride", C.c_int64), ("sequence_stride", C.c_int64), ("head_stride", C.c_int64)]


class _Cache(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("order", C.c_int32), ("layers", C.c_uint32), ("pages", C.c_uint32), ("page_tokens", C.c_uint32),
                ("heads", C.c_uint32), ("head_dim", C.c_uint32), ("sequences", C.c_uint32), ("table_pages", C.c_uint32),
                ("page_stride", C.c_int64), ("layer_stride", C.c_int64), ("keys", C.c_void_p), ("values", C.c_void_p),
                ("table", C.c_void_p), ("lengths", C.c_void_p), ("references", C.c_void_p), ("scratch", C.c_void_p)]


_declared = None


def _library():
    global _declared
    if _declared is None:
        L = load_library()
        u32, i32, vp, f64, P = C.c_uint32, C.c_int, C.c_void_p, C.c_double, C.POINTER
        L.hspmm_rotary_table.argtypes = [i32, u32, f64, f64, f64, f64, f64, u32, vp]
        L.hspmm_rotate.argtypes = [P(Rotary), i32, u32, u32, u32, P(Heads), vp, P(Heads), i32, vp]
        L.hspmm_cache_scratch_words.argtypes = [u32, u32, u32]
        L.hspmm_cache_scratch_words.restype = C.c_uint64
        L.hspmm_cache_append.argtypes = [P(_Cache), u32, P(Batch), P(Heads), P(Heads), P(Rotary), u32, P(Heads), P(Heads), vp]
        L.hspmm_cache_attend_workspace.argtypes = [P(_Cache), P(Batch), P(Attention), P(C.c_uint64)]
        L.hspmm_cache_attend.argtypes = [P(_Cache), u32, P(Batch), P(Attention), P(Heads), P(Heads), vp, vp, C.c_uint64, vp]
        L.hspmm_cache_attend_shared_workspace.argtypes = [P(_Cache), P(Batch), P(Prefix), P(Attention), P(C.c_uint64)]
        L.hspmm_cache_attend_shared.argtypes = [P(_Cache), u32, P(Batch), P(Prefix), P(Attention), P(Heads), P(Heads), vp, vp, C.c_uint64, vp]
        L.hspmm_cache_weigh_workspace.argtypes = [P(_Cache), P(Batch), P(Attention), u32, P(C.c_uint64)]
        L.hspmm_cache_weigh.argtypes = [P(_Cache), u32, P(Batch), P(Attention), P(Heads), vp, P(Weights), C.c_float, u32, vp, C.c_uint64, vp]
        L.hspmm_cache_evict_workspace.argtypes = [P(_Cache), u32, u32, P(C.c_uint64)]
        L.hspmm_cache_evict.argtypes = [P(_Cache), u32, vp, vp, P(Weights), u32, u32, u32, vp, vp, vp, C.c_uint64, vp]
        L.hspmm_cache_extend.argtypes = [P(_Cache), u32, vp, vp, vp, vp]
        L.hspmm_cache_fork.argtypes = [P(_Cache), u32, vp, vp, vp, vp]
        L.hspmm_cache_free.argtypes = [P(_Cache), u32, vp, vp]
        L.hspmm_cache_compact.argtypes = [P(_Cache), vp, vp, vp, vp]
        L.hspmm_cache_copy.argtypes = [P(_Cache), u32, vp, vp, vp]
        _declared = L
    return _declared


def rotary_table(dims, positions, kind="plain", base=10000.0, factor=1.0, original_length=0.0, fast_turns=32.0, slow_turns=1.0):
    """hspmm_rotary_table: numpy array positions x dims / 2 x 2 (cosine, sine) for the caller to put on the device."""
    if kind not in ROTARY_KINDS:
        raise ValueError("kind must be one of %s" % ", ".join(ROTARY_KINDS))
    table = np.empty((positions, dims // 2, 2), np.float32)
    _check(_library().hspmm_rotary_table(ROTARY_KINDS[kind], dims, base, factor, original_length, fast_turns, slow_turns, positions,
                                         table.ctypes.data_as(C.c_void_p)))
    return table


def rotate(dtype, rotary, tokens, heads, head_dim, x, y, positions, backward=False, stream=0):
    """hspmm_rotate: y = x turned by positions[tokens]; backward: the gradient of x from that of y."""
    rc = _library().hspmm_rotate(rotary, dtype, tokens, heads, head_dim, x, positions, y, backward, stream)
    if rc:
        _check(rc)


def cache_scratch_words(pages, sequences, table_pages):
    """32-bit words of a cache's scratch array."""
    return _library().hspmm_cache_scratch_words(pages, sequences, table_pages)


class Cache:
    """hspmm_cache: keys and values of `layers` layers in pages, by the addresses of the caller's arrays."""

    def __init__(self, dtype, layers, pages, page_tokens, heads, head_dim, sequences, table_pages, keys, values, table, lengths, references,
                 scratch, order=HEADS_FIRST, page_stride=0, layer_stride=0):
        L = _library()
        self._c = _Cache(dtype, order, layers, pages, page_tokens, heads, head_dim, sequences, table_pages, page_stride, layer_stride,
                         keys, values, table, lengths, references, scratch)
        # (bound once: small calls are made of their host time)
        self._append, self._attend, self._fork, self._compact = L.hspmm_cache_append, L.hspmm_cache_attend, L.hspmm_cache_fork, L.hspmm_cache_compact
        self._attend_shared, self._weigh, self._evict = L.hspmm_cache_attend_shared, L.hspmm_cache_weigh, L.hspmm_cache_evict

    def append(self, layer, batch, k, v, rotary=None, q_heads=0, q=None, q_out=None, stream=0):
        """hspmm_cache_append: keys and values of the batch's tokens into their pages, turned before if rotary is given; q_out = q turned."""
        rc = self._append(self._c, layer, batch, k, v, rotary, q_heads, q, q_out, stream)
        if rc:
            _check(rc)

    def attend_workspace(self, batch, attention):
        """Bytes of workspace (zeros at first) that `attend` wants for these."""
        n = C.c_uint64()
        _check(_library().hspmm_cache_attend_workspace(self._c, batch, attention, n))
        return n.value

    def attend(self, layer, batch, attention, q, out, lse=0, workspace=0, workspace_bytes=0, stream=0):
        """hspmm_cache_attend: out = softmax(scale q k) v of the batch's tokens; lse: address of tokens x q_heads floats, or 0."""
        rc = self._attend(self._c, layer, batch, attention, q, out, lse, workspace, workspace_bytes, stream)
        if rc:
            _check(rc)

    def attend_shared_workspace(self, batch, prefix, attention):
        """Bytes of workspace (zeros at first) that `attend_shared` wants for these."""
        n = C.c_uint64()
        _check(_library().hspmm_cache_attend_shared_workspace(self._c, batch, prefix, attention, n))
        return n.value

    def attend_shared(self, layer, batch, prefix, attention, q, out, lse=0, workspace=0, workspace_bytes=0, stream=0):
        """hspmm_cache_attend_shared: `attend` of groups of sequences that begin with the same tokens, whose keys and values are read by the first
        one's pages, and once for all of a group where each sequence has few new tokens."""
        rc = self._attend_shared(self._c, layer, batch, prefix, attention, q, out, lse, workspace, workspace_bytes, stream)
        if rc:
            _check(rc)

    def weigh_workspace(self, batch, attention, last=0):
        """Bytes of workspace (zeros at first) that `weigh` wants for these."""
        n = C.c_uint64()
        _check(_library().hspmm_cache_weigh_workspace(self._c, batch, attention, last, n))
        return n.value

    def weigh(self, layer, batch, attention, q, lse, weights, decay=1.0, last=0, workspace=0, workspace_bytes=0, stream=0):
        """hspmm_cache_weigh: weights of cached keys = decay * weights + what the batch's tokens give them; q and lse are those of `attend`."""
        rc = self._weigh(self._c, layer, batch, attention, q, lse, weights, decay, last, workspace, workspace_bytes, stream)
        if rc:
            _check(rc)

    def evict_workspace(self, n, keep):
        """Bytes of workspace (zeros at first) that `evict` wants for a list of n sequences that keep so many tokens."""
        b = C.c_uint64()
        _check(_library().hspmm_cache_evict_workspace(self._c, n, keep, b))
        return b.value

    def evict(self, n, parents, children, weights, keep, first=0, last=0, kept=0, status=0, workspace=0, workspace_bytes=0, stream=0):
        """hspmm_cache_evict: sequence children[i] (children 0: the parent itself) becomes what parents[i] was, with `keep` of its tokens at most."""
        rc = self._evict(self._c, n, parents, children, weights, keep, first, last, kept, status, workspace, workspace_bytes, stream)
        if rc:
            _check(rc)

    def extend(self, n, rows, add, status=0, stream=0):
        """hspmm_cache_extend: add[i] more tokens for sequence rows[i] (rows 0: i), and their pages."""
        _check(_library().hspmm_cache_extend(self._c, n, rows, add, status, stream))

    def fork(self, n, parents, children, status=0, stream=0):
        """hspmm_cache_fork: sequence children[i] becomes what parents[i] was."""
        rc = self._fork(self._c, n, parents, children, status, stream)
        if rc:
            _check(rc)

    def free(self, n, rows, stream=0):
        """hspmm_cache_free: sequences rows[i] have no tokens any more."""
        _check(_library().hspmm_cache_free(self._c, n, rows, stream))

    def compact(self, live=0, table_out=0, references_out=0, stream=0):
        """hspmm_cache_compact: live pages to the low end of the pool."""
        rc = self._compact(self._c, table_out, references_out, live, stream)
        if rc:
            _check(rc)

    def copy(self, n, source, to, stream=0):
        """hspmm_cache_copy: pages source[i] to to[i]."""
        _check(_library().hspmm_cache_copy(self._c, n, source, to, stream))
