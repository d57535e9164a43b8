"""A paged cache on the GPU for the tests, and plain implementations in 64 bits on the CPU."""
import math

import numpy as np

HALF_ULP = {0: 2.0 ** -11, 1: 2.0 ** -24, 2: 2.0 ** -8}        # of the result, by element type (fp16, fp32, bf16: 11, 24 and 8 bits)
SMALLEST = {0: 2.0 ** -25, 1: 2.0 ** -140, 2: 2.0 ** -134}     # half the spacing of the type's subnormals


def torch_type(torch, dtype):
    return {0: torch.float16, 1: torch.float32, 2: torch.bfloat16}[dtype]


def to64(x):
    return x.detach().cpu().double().numpy()


class State:
    """Arrays of a cache and its handle.  Free slots hold NaN: nothing may read them into a result."""

    def __init__(self, torch, hs, dtype, pages, page_tokens, heads, head_dim, sequences, table_pages, layers=1, order=0, page_gap=0, layer_gap=0, fill=math.nan):
        self.torch, self.dtype, self.order = torch, dtype, order
        self.pages, self.page_tokens, self.heads, self.head_dim, self.layers = pages, page_tokens, heads, head_dim, layers
        self.page_stride = page_tokens * heads * head_dim + page_gap
        self.layer_stride = self.page_stride * pages + layer_gap
        self.pool = [torch.full((layers * self.layer_stride,), fill, dtype=torch_type(torch, dtype), device="cuda") for _ in range(2)]
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((sequences, table_pages), -1, **i32)
        self.lengths, self.references = torch.zeros(sequences, **i32), torch.zeros(pages, **i32)
        self.scratch = torch.full((hs.cache_scratch_words(pages, sequences, table_pages),), 0x5A5A5A5A, **i32)
        self.handle = hs.Cache(dtype, layers, pages, page_tokens, heads, head_dim, sequences, table_pages, self.pool[0].data_ptr(), self.pool[1].data_ptr(),
                               self.table.data_ptr(), self.lengths.data_ptr(), self.references.data_ptr(), self.scratch.data_ptr(), order=order,
                               page_stride=self.page_stride if page_gap else 0, layer_stride=self.layer_stride if layer_gap or page_gap else 0)

    def view(self, which):
        """layers x pages x heads x page_tokens x head_dim of keys (0) or values (1), in place."""
        x = self.pool[which].as_strided((self.layers, self.pages, self.page_tokens * self.heads * self.head_dim), (self.layer_stride, self.page_stride, 1))
        if self.order == 0:
            return x.view(self.layers, self.pages, self.heads, self.page_tokens, self.head_dim)
        return x.view(self.layers, self.pages, self.page_tokens, self.heads, self.head_dim).transpose(2, 3)

    def place(self, rng, lengths, keep=()):
        """Gives sequences pages in a random order; table places behind a row's last page hold numbers that are no page's."""
        table = rng.choice(np.array([-1, self.pages, 0x7FFFFFFF, -0x80000000]), self.table.shape)
        ids = rng.permutation(self.pages)
        references = np.zeros(self.pages, np.int64)
        at = 0
        for s, n in enumerate(lengths):
            used = -(-int(n) // self.page_tokens)
            table[s, :used] = ids[at:at + used]
            references[ids[at:at + used]] = 1
            at += used
        t = self.torch
        self.table.copy_(t.from_numpy(table.astype(np.int32)))
        self.lengths.copy_(t.from_numpy(np.asarray(lengths, np.int32)))
        self.references.copy_(t.from_numpy(references.astype(np.int32)))

    def store(self, layer, s, which, values):
        """values: tokens x heads x head_dim (64 bits) of sequence s from its first token on."""
        t = self.torch
        v = t.from_numpy(np.ascontiguousarray(values)).to(torch_type(t, self.dtype)).cuda()
        n = np.arange(len(values))
        ids = self.table[s].long()[t.from_numpy(n // self.page_tokens).cuda()] if len(n) else None
        if ids is not None:
            self.view(which)[layer][ids, :, t.from_numpy(n % self.page_tokens).cuda()] = v

    def load(self, layer, s, which, tokens):
        n = np.arange(tokens)
        table = self.table[s].cpu().numpy()
        return to64(self.view(which)[layer])[table[n // self.page_tokens], :, n % self.page_tokens]


def rounded(torch, x, dtype):
    """64-bit values of x rounded to an element type."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float64)).to(torch_type(torch, dtype)).double().numpy()


def attend64(q, k, v, positions, scale, causal, window, there=None):
    """q: tokens x heads x dim, k and v: keys x kv heads x dim, positions of the tokens.  Returns out, lse, and per output
    sum p |v| and per (token, head) the largest scale * sum |q k| of a key seen."""
    T, H, D = q.shape
    shared = H // k.shape[1]
    j = np.arange(len(k))
    seen = np.ones((T, len(k)), bool) if there is None else np.broadcast_to(there, (T, len(k))).copy()
    if causal:
        seen &= j[None] <= positions[:, None]
    if window:
        seen &= j[None] > positions[:, None] - window
    out, size = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse, reach = np.full((T, H), -np.inf), np.zeros((T, H))
    for t in range(T):
        at = np.nonzero(seen[t])[0]
        if not len(at):
            continue
        for h in range(H):
            kk, vv = k[at, h // shared], v[at, h // shared]
            with np.errstate(all="ignore"):
                s = scale * (kk @ q[t, h])
                m = s.max()
                p = np.exp(s - m)
                total = p.sum()
                p /= total
                out[t, h], size[t, h] = p @ vv, p @ np.abs(vv)
                lse[t, h] = m + np.log(total)
                reach[t, h] = abs(scale) * (np.abs(kk) @ np.abs(q[t, h])).max()
    return out, lse, size, reach


def attend_bounds(dtype, out, lse, size, reach, dim, keys, largest):
    """How far a result in fp32 with weights of the element type may be off.
    A score: dim products and sums, (dim + 4) roundings of 2^-24 of scale * sum |q k| at most, its exponential four more;
    a weight: exp of that, and for 16-bit types half an ulp of its own; sums over the keys: two roundings a
    tile of 32, which are at most keys / 16 + 64; the result's own rounding.  16-bit floats of five exponent bits: weights below
    2^-14 of the largest are off by 2^-25 of that."""
    score = (dim + 4) * 2.0 ** -24 * reach + 4 * 2.0 ** -24
    weight = 2 * score + (HALF_ULP[dtype] if dtype != 1 else 0.0) + (keys / 16 + 64) * 2.0 ** -24
    bound = HALF_ULP[dtype] * np.abs(out) + size * weight[..., None] * 1.01 + SMALLEST[dtype] + 2.0 ** -126
    if dtype == 0:
        bound = bound + keys * 2.0 ** -25 * largest
    return bound, score + (keys / 16 + 64) * 2.0 ** -24 + np.where(np.isfinite(lse), np.abs(lse), 0) * 2.0 ** -22
