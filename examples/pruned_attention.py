"""The attention block of a decoder whose four projections are pruned: sparse products, rotary positions, a paged cache and
the attention over it, as a serving loop runs them.

    python examples/pruned_attention.py [--hidden 1024] [--heads 8] [--kv-heads 2] [--keep 0.1] [--layers 2]

Prompts of different lengths go through as one ragged batch, every prompt is forked into beams, the beams decode and are
reordered, one prompt's beams end and its pages are compacted away.  Activations lie features x tokens, which is what
`Plan.run` reads and writes; `append` and `attend` take them by their strides, so nothing is transposed in between.
"""
import argparse
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import hopper_spmm_amd as hs  # noqa: E402
from hopper_spmm_amd import generators as G  # noqa: E402

DTYPE, TORCH = hs.FP16, torch.float16


def stream():
    return torch.cuda.current_stream().cuda_stream


def heads_of(x, dim):
    """features x tokens as tokens x heads x dim."""
    return x.view(-1, dim, x.shape[1]).permute(2, 0, 1)


def view(x):
    return hs.Heads(x.data_ptr(), *x.stride())


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).cuda()


class PrunedLayer:
    """Wq, Wk, Wv and Wo of one layer, with the fraction `keep` of largest magnitude kept."""

    def __init__(self, hidden, heads, kv_heads, dim, keep, seed):
        self.csr, self.plans = [], []
        for i, (rows, cols) in enumerate(((heads * dim, hidden), (kv_heads * dim, hidden), (kv_heads * dim, hidden), (hidden, heads * dim))):
            w = G.pruned_weight(rows, cols, keep, seed + i, std=1.0 / math.sqrt(keep * cols), dtype=DTYPE)
            self.csr.append(w)
            self.plans.append(hs.Plan(hs.csr_to_btcf(rows, cols, w["row_ptr"], w["col_idx"], w["values"], DTYPE)))

    def product(self, i, x):
        y = torch.empty((self.plans[i].rows, x.shape[1]), dtype=TORCH, device="cuda")
        self.plans[i].run(x.data_ptr(), y.data_ptr(), x.shape[1], stream())
        return y

    def dense(self, i):
        """The weight in 64 bits, for checks."""
        w = self.csr[i]
        d = np.zeros((w["rows"], w["cols"]))
        d[np.repeat(np.arange(w["rows"]), np.diff(w["row_ptr"].astype(np.int64))), w["col_idx"]] = np.asarray(w["values"]).view(np.float16).astype(np.float64)
        return d


class Decoder:
    """Attention blocks over one paged cache."""

    def __init__(self, hidden, heads, kv_heads, layers, keep, pages, page_tokens, sequences, longest):
        self.heads, self.kv_heads, self.dim, self.longest = heads, kv_heads, hidden // heads, longest
        self.layers = [PrunedLayer(hidden, heads, kv_heads, self.dim, keep, 100 * i) for i in range(layers)]
        places = -(-longest // page_tokens)
        shape = (layers, pages, kv_heads, page_tokens, self.dim)
        self.keys, self.values = (torch.zeros(shape, dtype=TORCH, device="cuda") for _ in range(2))
        self.table, self.lengths, self.references = i32(np.full((sequences, places), -1)), i32(np.zeros(sequences)), i32(np.zeros(pages))
        self.scratch, self.status = i32(np.zeros(hs.cache_scratch_words(pages, sequences, places))), i32([0])
        self.cache = hs.Cache(DTYPE, layers, pages, page_tokens, kv_heads, self.dim, sequences, places, self.keys.data_ptr(), self.values.data_ptr(),
                              self.table.data_ptr(), self.lengths.data_ptr(), self.references.data_ptr(), self.scratch.data_ptr())
        self.angles = torch.from_numpy(hs.rotary_table(self.dim, longest, "yarn", factor=2.0, original_length=longest / 2)).cuda()
        self.rotary = hs.Rotary(self.dim, longest, self.angles.data_ptr())
        self.workspace = torch.zeros(1, dtype=torch.uint8, device="cuda")

    def forward(self, x, rows, new):
        """x: hidden x tokens, the new tokens of sequences `rows`, `new` of each, one after another."""
        rows_d, new_d, starts = i32(rows), i32(new), i32(np.concatenate([[0], np.cumsum(new)]))
        self.cache.extend(len(rows), rows_d.data_ptr(), new_d.data_ptr(), self.status.data_ptr(), stream())
        batch = hs.Batch(len(rows), x.shape[1], starts.data_ptr(), rows_d.data_ptr())
        attention = hs.Attention(self.heads, 1.0 / math.sqrt(self.dim), longest_chunk=max(new), longest=self.longest)
        need = self.cache.attend_workspace(batch, attention)
        if need > self.workspace.numel():
            self.workspace = torch.zeros(need, dtype=torch.uint8, device="cuda")
        for i, layer in enumerate(self.layers):
            q, k, v = (heads_of(layer.product(j, x), self.dim) for j in range(3))
            turned = torch.empty((x.shape[1], self.heads, self.dim), dtype=TORCH, device="cuda")
            self.cache.append(i, batch, view(k), view(v), rotary=self.rotary, q_heads=self.heads, q=view(q), q_out=view(turned), stream=stream())
            mixed = torch.empty((self.heads * self.dim, x.shape[1]), dtype=TORCH, device="cuda")
            self.cache.attend(i, batch, attention, view(turned), view(heads_of(mixed, self.dim)), workspace=self.workspace.data_ptr(),
                              workspace_bytes=self.workspace.numel(), stream=stream())
            x = x + layer.product(3, mixed)
        if int(self.status):
            raise RuntimeError("%d pages are missing" % int(self.status))
        return x

    def fork(self, parents, children):
        p, c = i32(parents), i32(children)
        self.cache.fork(len(parents), p.data_ptr(), c.data_ptr(), self.status.data_ptr(), stream())
        if int(self.status):
            raise RuntimeError("%d pages are missing" % int(self.status))

    def end(self, rows):
        """Sequences that are done; returns the pages still in use, which lie at the low end of the pool from here on."""
        r, live = i32(rows), i32([0])
        self.cache.free(len(rows), r.data_ptr(), stream())
        self.cache.compact(live.data_ptr(), stream=stream())
        return int(live)


def reference(decoder, histories):
    """The blocks in 64 bits over whole histories (hidden x tokens each), layer by layer; also the largest score."""
    outs, largest = [], 0.0
    for x in histories:
        x = x.astype(np.float64)
        T, D, angles = x.shape[1], decoder.dim, decoder.angles.cpu().double().numpy()[: x.shape[1]]
        for layer in decoder.layers:
            q, k, v = ((layer.dense(j) @ x).reshape(-1, D, T) for j in range(3))

            def turn(y):
                a, b, c, s = y[:, : D // 2], y[:, D // 2:], angles[:, :, 0].T, angles[:, :, 1].T
                return np.concatenate([a * c - b * s, a * s + b * c], 1)
            q, k = turn(q), turn(k)
            mixed = np.zeros_like(q)
            for h in range(decoder.heads):
                g = h // (decoder.heads // decoder.kv_heads)
                scores = q[h].T @ k[g] / math.sqrt(D)
                scores[np.triu_indices(T, 1)] = -np.inf
                largest = max(largest, np.abs(scores[np.isfinite(scores)]).max())
                p = np.exp(scores - scores.max(1, keepdims=True))
                mixed[h] = v[g] @ (p / p.sum(1, keepdims=True)).T
            x = x + layer.dense(3) @ mixed.reshape(-1, T)
        outs.append(x)
    return outs, largest


def run(hidden=1024, heads=8, kv_heads=2, keep=0.1, layers=2, prompts=(70, 33, 5), beams=3, steps=4, page_tokens=16, seed=0):
    """Serves `prompts` with `beams` beams each; returns the outputs of the last step, what the reference says of them and its largest score."""
    rng = np.random.default_rng(seed)
    n = len(prompts)
    longest = max(prompts) + 2 * steps
    decoder = Decoder(hidden, heads, kv_heads, layers, keep, n * beams * (-(-longest // page_tokens) + 1), page_tokens, n * beams, longest)
    history = [rng.standard_normal((hidden, p)).astype(np.float16) for p in prompts]
    # prompts, as sequences 0, beams, 2 beams, ..
    first = [i * beams for i in range(n)]
    decoder.forward(torch.from_numpy(np.concatenate(history, 1)).cuda(), first, list(prompts))
    history = [h for h in history for _ in range(beams)]
    decoder.fork([f for f in first for _ in range(beams - 1)], [f + b for f in first for b in range(1, beams)])
    alive = list(range(n * beams))
    for step in range(2 * steps):
        if step == steps:
            # the last prompt's beams are done
            alive = alive[:-beams]
            live = decoder.end(list(range((n - 1) * beams, n * beams)))
            print("pages in use: %d of %d" % (live, decoder.references.numel()), flush=True)
        new = rng.standard_normal((hidden, len(alive))).astype(np.float16)
        out = decoder.forward(torch.from_numpy(new).cuda(), alive, [1] * len(alive))
        history = [np.concatenate([history[s], new[:, i:i + 1]], 1) for i, s in enumerate(alive)] + history[len(alive):]
        if step % 2 == 0:
            # a beam search's choice: beams go on from others of their prompt
            parents = [s - s % beams + int(rng.integers(beams)) for s in alive]
            decoder.fork(parents, alive)
            history = [history[p] for p in parents] + history[len(alive):]
            out = None
    want, largest = reference(decoder, [history[s] for s in alive])
    return out.cpu().double().numpy(), np.stack([w[:, -1] for w in want], 1), largest


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("hidden", 1024), ("heads", 8), ("kv-heads", 2), ("layers", 2), ("beams", 3), ("steps", 4)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--keep", type=float, default=0.1)
    a = ap.parse_args()
    got, want, _ = run(a.hidden, a.heads, a.kv_heads, a.keep, a.layers, beams=a.beams, steps=a.steps)
    print("last tokens of %d beams: relative difference to 64 bits %.2g" % (got.shape[1], np.linalg.norm(got - want) / np.linalg.norm(want)))


if __name__ == "__main__":
    main()
