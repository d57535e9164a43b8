"""The attention block of a decoder whose four projections are pruned: sparse products, rotary positions, a paged cache and
the attention over it, as a serving loop runs them.

    python examples/pruned_attention.py [--hidden 1024] [--heads 8] [--kv-heads 2] [--keep 0.1] [--layers 2] [--budget 40]

Prompts of different lengths go through as one ragged batch, every prompt is forked into beams, the beams decode and are
reordered, one prompt's beams end and its pages are compacted away.  Activations lie features x tokens, which is what
`Plan.run` reads and writes; `append` and `attend` take them by their strides, so nothing is transposed in between.

With a budget a sequence holds no more tokens than that: beams attend their prompt together (`attend_shared`), what every cached
token receives is added up (`weigh`), and the tokens that received least leave (`evict`).
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


class BoundedDecoder(Decoder):
    """The same with prompts that beams read together and a cache of bounded length.  Where tokens have left, a sequence's next position is no
    longer its length: the caller says the positions, by which queries and keys are turned before they are appended."""

    def __init__(self, *args):
        super().__init__(*args)
        self.weights = torch.zeros(len(self.layers), self.lengths.numel(), self.kv_heads, self.table.shape[1] * self.keys.shape[3], device="cuda")
        self.received = hs.Weights(self.weights.data_ptr(), *self.weights.stride()[:3])

    def reserve(self, need):
        if need > self.workspace.numel():
            self.workspace = torch.zeros(need, dtype=torch.uint8, device="cuda")
        return dict(workspace=self.workspace.data_ptr(), workspace_bytes=self.workspace.numel())

    def turn(self, x, positions):
        """features x tokens, as tokens x heads x dim at their positions."""
        y = torch.empty((x.shape[1], x.shape[0] // self.dim, self.dim), dtype=TORCH, device="cuda")
        hs.rotate(DTYPE, self.rotary, y.shape[0], y.shape[1], self.dim, view(heads_of(x, self.dim)), view(y), positions.data_ptr(), stream=stream())
        return y

    def forward(self, x, rows, new, positions, groups=(), decay=1.0, last=0):
        """groups: (rows of the batch, tokens) that begin alike, of all rows in order, or none; decay, last: of the weights."""
        rows_d, new_d, starts, positions = i32(rows), i32(new), i32(np.concatenate([[0], np.cumsum(new)])), i32(positions)
        self.cache.extend(len(rows), rows_d.data_ptr(), new_d.data_ptr(), self.status.data_ptr(), stream())
        batch = hs.Batch(len(rows), x.shape[1], starts.data_ptr(), rows_d.data_ptr())
        attention = hs.Attention(self.heads, 1.0 / math.sqrt(self.dim), longest_chunk=max(new), longest=self.longest)
        firsts, tokens = i32(np.cumsum([0] + [n for n, _ in groups])), i32([t for _, t in groups])
        prefix = hs.Prefix(len(groups), firsts.data_ptr(), tokens.data_ptr() if groups else 0, longest=max([t for _, t in groups], default=0))
        space = self.reserve(max(self.cache.attend_shared_workspace(batch, prefix, attention), self.cache.weigh_workspace(batch, attention, last)))
        lse = torch.empty((x.shape[1], self.heads), device="cuda")
        for i, layer in enumerate(self.layers):
            q, k, v = (layer.product(j, x) for j in range(3))
            q, k = self.turn(q, positions), self.turn(k, positions)
            self.cache.append(i, batch, view(k), view(heads_of(v, self.dim)), stream=stream())
            mixed = torch.empty((self.heads * self.dim, x.shape[1]), dtype=TORCH, device="cuda")
            self.cache.attend_shared(i, batch, prefix, attention, view(q), view(heads_of(mixed, self.dim)), lse=lse.data_ptr(), stream=stream(), **space)
            self.cache.weigh(i, batch, attention, view(q), lse.data_ptr(), self.received, decay=decay, last=last, stream=stream(), **space)
            x = x + layer.product(3, mixed)
        if int(self.status):
            raise RuntimeError("%d pages are missing" % int(self.status))
        return x

    def fork(self, parents, children):
        super().fork(parents, children)
        self.weights[:, children] = self.weights[:, parents]

    def evict(self, parents, children, keep, first, last):
        """The tokens kept, layers x entries x heads x keep."""
        p, c, kept = i32(parents), i32(children), i32(np.empty((len(self.layers), len(parents), self.kv_heads, keep)))
        self.cache.evict(len(parents), p.data_ptr(), c.data_ptr(), self.received, keep, first=first, last=last, kept=kept.data_ptr(), status=self.status.data_ptr(),
                         stream=stream(), **self.reserve(self.cache.evict_workspace(len(parents), keep)))
        if int(self.status):
            raise RuntimeError("%d pages are missing" % int(self.status))
        return kept.cpu().numpy()


class Mirror:
    """What a BoundedDecoder does, in 64 bits.  Which tokens are kept is taken from it, and looked at: `worst` is the largest
    weight in layer 0 that left, relative to the smallest one that stayed in its place; `reach` its largest scale |q| |k|."""

    def __init__(self, decoder):
        self.decoder, self.dense = decoder, [[layer.dense(j) for j in range(4)] for layer in decoder.layers]
        self.angles = decoder.angles.cpu().double().numpy()
        empty = np.zeros((decoder.kv_heads, 0, decoder.dim))
        self.held = {s: [(empty, empty, empty[:, :, 0]) for _ in decoder.layers] for s in range(decoder.lengths.numel())}
        self.largest = self.reach = self.worst = 0.0

    def turn(self, y, positions):
        half, a = self.decoder.dim // 2, self.angles[positions]
        return np.concatenate([y[..., :half] * a[:, :, 0] - y[..., half:] * a[:, :, 1], y[..., :half] * a[:, :, 1] + y[..., half:] * a[:, :, 0]], -1)

    def forward(self, s, x, positions, decay, last):
        d, x = self.decoder, x.astype(np.float64)
        n, shared = x.shape[1], d.heads // d.kv_heads
        for i, w in enumerate(self.dense):
            q, k, v = ((w[j] @ x).reshape(-1, d.dim, n).transpose(0, 2, 1) for j in range(3))
            keys, values, weights = self.held[s][i]
            old = keys.shape[1]
            q, keys, values = self.turn(q, positions), np.concatenate([keys, self.turn(k, positions)], 1), np.concatenate([values, v], 1)
            weights = np.concatenate([weights * decay, np.zeros((d.kv_heads, n))], 1)
            mixed = np.zeros_like(q)
            for h in range(d.heads):
                g = h // shared
                scores = q[h] @ keys[g].T / math.sqrt(d.dim)
                scores[np.arange(old + n)[None] > old + np.arange(n)[:, None]] = -np.inf
                self.largest = max(self.largest, np.abs(scores[np.isfinite(scores)]).max())
                if i == 0:
                    self.reach = max(self.reach, np.linalg.norm(q[h], axis=1).max() * np.linalg.norm(keys[g], axis=1).max() / math.sqrt(d.dim))
                p = np.exp(scores - scores.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                mixed[h] = p @ values[g]
                weights[g] += p[-last:].sum(0)
            self.held[s][i] = keys, values, weights
            x = x + w[3] @ mixed.transpose(0, 2, 1).reshape(-1, n)
        return x

    def fork(self, parents, children):
        self.held.update({c: list(h) for c, h in [(c, self.held[p]) for p, c in zip(parents, children)]})

    def evict(self, parents, children, keep, first, last, kept):
        now = {}
        for e, (p, c) in enumerate(zip(parents, children)):
            now[c] = []
            for i, (keys, values, weights) in enumerate(self.held[p]):
                n = keys.shape[1]
                at = [list(x[x >= 0]) for x in kept[i, e]]
                for g in range(self.decoder.kv_heads):
                    assert len(at[g]) == min(n, keep) and at[g] == sorted(set(at[g])) and (kept[i, e, g, len(at[g]):] == -1).all()
                    gone, sure = set(range(n)) - set(at[g]), set(range(first)) | set(range(n - last, n))
                    assert not gone & sure
                    chosen = [weights[g, j] for j in at[g] if j not in sure]
                    if i == 0 and gone and chosen:
                        self.worst = max(self.worst, max(weights[g, j] for j in gone) / min(chosen))
                now[c].append(tuple(np.stack([x[g][at[g]] for g in range(self.decoder.kv_heads)]) for x in (keys, values, weights)))
        self.held.update(now)


def run_bounded(hidden=1024, heads=8, kv_heads=2, keep=0.1, layers=2, prompts=(70, 33, 90), beams=3, steps=4, page_tokens=16, budget=40, first=2, last=8, decay=0.875, window=16, seed=0):
    """Serves `prompts` with `beams` beams each that hold `budget` tokens at most; returns the outputs of every step, what the mirror says of them, and both."""
    rng = np.random.default_rng(seed)
    n = len(prompts)
    longest = max(prompts) + 3 * steps
    decoder = BoundedDecoder(hidden, heads, kv_heads, layers, keep, 2 * n * beams * (-(-longest // page_tokens) + 1), page_tokens, n * beams, longest)
    mirror, outs = Mirror(decoder), []
    position = np.zeros(n * beams, int)

    def forward(rows, new, groups=(), last=0):
        x = [rng.standard_normal((hidden, m)).astype(np.float16) for m in new]
        at = [np.arange(position[s], position[s] + m) for s, m in zip(rows, new)]
        got = decoder.forward(torch.from_numpy(np.concatenate(x, 1)).cuda(), rows, new, np.concatenate(at), groups, decay, last)
        want = np.concatenate([mirror.forward(s, y, p, decay, last) for s, y, p in zip(rows, x, at)], 1)
        position[rows] += new
        outs.append((got.cpu().double().numpy(), want))

    def fork(parents, children):
        decoder.fork(parents, children)
        mirror.fork(parents, children)
        position[children] = position[parents]

    def evict(parents, children, keep):
        mirror.evict(parents, children, keep, first, last, decoder.evict(parents, children, keep, first, last))
        position[children] = position[parents]

    # (of a prompt its last tokens say what is wanted)
    begin = [i * beams for i in range(n)]
    forward(begin, list(prompts), last=window)
    fork([f for f in begin for _ in range(beams - 1)], [f + b for f in begin for b in range(1, beams)])
    rows = list(range(n * beams))
    for step in range(steps):
        forward(rows, [1] * len(rows), [(beams, p) for p in prompts])
        if step % 2 == 0:
            fork([s - s % beams + int(rng.integers(beams)) for s in rows], rows)
    # every beam keeps tokens of its own choice: nothing is shared from here on
    evict(rows, rows, budget)
    for step in range(steps):
        forward(rows, [1] * len(rows))
        if step % 2 == 0:
            evict(rows, rows, budget)
    # a prompt's first beam goes on in all of them, with half as many tokens
    evict([s - s % beams for s in rows], rows, max(budget // 2, first + last))
    for step in range(steps):
        forward(rows, [1] * len(rows))
    print("tokens held: %s of %s" % (decoder.lengths.tolist(), position.tolist()), flush=True)
    return outs, decoder, mirror


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("hidden", 1024), ("heads", 8), ("kv-heads", 2), ("layers", 2), ("beams", 3), ("steps", 4)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--keep", type=float, default=0.1)
    ap.add_argument("--budget", type=int, default=0, help="tokens that a sequence holds at most (0: all)")
    a = ap.parse_args()
    if a.budget:
        outs, _, _ = run_bounded(a.hidden, a.heads, a.kv_heads, a.keep, a.layers, beams=a.beams, steps=a.steps, budget=a.budget)
        print("outputs of %d steps: relative difference to 64 bits %.2g" % (len(outs), max(np.linalg.norm(g - w) / np.linalg.norm(w) for g, w in outs)))
        return
    got, want, _ = run(a.hidden, a.heads, a.kv_heads, a.keep, a.layers, beams=a.beams, steps=a.steps)
    print("last tokens of %d beams: relative difference to 64 bits %.2g" % (got.shape[1], np.linalg.norm(got - want) / np.linalg.norm(want)))


if __name__ == "__main__":
    main()
