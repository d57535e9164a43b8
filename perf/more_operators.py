"""Performance cases of the operators that serve many sequences from one long prompt with a bounded cache: attention that
reads a shared prefix once, the attention weight that every cached token has received, and the eviction of the tokens that
received least.

A case names an operator, sizes and an element type; one pass is one call of that operator with everything resident on
the GPU:

  shared   softmax(scale q k) v of new tokens whose sequences begin with the same tokens, group by group: those keys and
           values are one sequence's, the others' behind them their own
  weigh    weights of cached keys += what the softmax of the batch's tokens gives them, summed over the heads of queries that
           share a head of keys
  evict    sequences that take over what others hold, as many tokens as they may keep: the first and the last ones, and those of
           the greatest weight between, for every layer and head of keys by itself

Heads of 128 of a hidden size of 4096 (32 heads, 8 of them of keys and values) are those of the layers that the
products are benchmarked at; the rest is generic.  Inputs are made on the GPU from the seed alone.
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
NAMES = {"fp16": "FP16", "bf16": "BF16", "fp32": "TF32"}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _shared(groups, rows_least, rows_most, prefix_least, prefix_most, rest_least, rest_most, new_least, new_most, heads, shared, dim, page, dtype, transposed):
    """rows_*: sequences of a group; prefix_*: tokens that they begin with; rest_*: tokens of their own behind those; new_*: tokens
    of the batch, the last ones; shared: heads of queries to one of keys and values; transposed: the output lies features x
    tokens, as the next product wants it."""
    return {"op": "shared", "groups": groups, "rows_least": rows_least, "rows_most": rows_most, "prefix_least": prefix_least, "prefix_most": prefix_most,
            "rest_least": rest_least, "rest_most": rest_most, "new_least": new_least, "new_most": new_most, "heads": heads, "shared": shared, "dim": dim,
            "page": page, "dtype": dtype, "transposed": transposed}


def _weigh(sequences, new_least, new_most, old_least, old_most, last, heads, shared, dim, page, dtype):
    """new_*, old_*: tokens of a sequence's chunk, and of what its cache holds already; last: how many of a chunk's tokens count
    (0: all)."""
    return {"op": "weigh", "sequences": sequences, "new_least": new_least, "new_most": new_most, "old_least": old_least, "old_most": old_most, "last": last,
            "heads": heads, "shared": shared, "dim": dim, "page": page, "dtype": dtype}


def _evict(sequences, length_least, length_most, keep, first, last, layers, heads, dim, page, dtype):
    """length_*: tokens that a sequence holds; keep: tokens that it may keep, the first and the last ones among them."""
    return {"op": "evict", "sequences": sequences, "length_least": length_least, "length_most": length_most, "keep": keep, "first": first, "last": last,
            "layers": layers, "heads": heads, "dim": dim, "page": page, "dtype": dtype}


def listed():
    return [
        # the beams of one prompt, a token each: latency
        dict(_shared(1, 8, 8, 1000, 1000, 5, 200, 1, 1, 8, 4, 128, 16, "fp16", False), name="shared_beams"),
        # a server's batch behind one long system prompt, a token each
        dict(_shared(1, 64, 64, 8000, 8000, 20, 1500, 1, 1, 8, 4, 128, 16, "bf16", True), name="shared_step"),
        # several prompts, few tokens for each of their continuations (drafts that are checked), full precision, odd page size
        dict(_shared(5, 3, 12, 300, 6000, 0, 800, 1, 12, 4, 3, 64, 24, "fp32", False), name="shared_drafts"),
        # questions of many tokens about two long documents
        dict(_shared(2, 7, 9, 3000, 6000, 0, 500, 50, 250, 8, 4, 128, 64, "bf16", True), name="shared_questions"),
        # three short sequences, a token each, full precision: latency
        dict(_weigh(3, 1, 1, 20, 300, 0, 8, 1, 64, 16, "fp32"), name="weigh_step_small"),
        # a server's batch that decodes: the keys are read once
        dict(_weigh(48, 1, 1, 500, 16000, 0, 8, 4, 128, 16, "bf16"), name="weigh_step"),
        # prompts of different lengths, of which the last tokens choose what is kept: odd head, page and chunk sizes
        dict(_weigh(17, 1, 700, 0, 5000, 32, 4, 3, 96, 24, "fp16"), name="weigh_last"),
        # all tokens of the second half of a long prompt
        dict(_weigh(1, 4096, 4096, 4096, 4096, 0, 8, 4, 128, 64, "bf16"), name="weigh_prompt"),
        # one sequence of a small model: latency
        dict(_evict(1, 700, 700, 256, 4, 32, 2, 4, 64, 16, "fp16"), name="evict_small"),
        # odd sizes in full precision
        dict(_evict(5, 100, 3001, 333, 1, 50, 3, 5, 80, 24, "fp32"), name="evict_odd"),
        # a server's batch of long prompts, of which a thousand tokens stay
        dict(_evict(12, 500, 8000, 1024, 4, 256, 8, 8, 128, 16, "bf16"), name="evict_batch"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["shared", "shared", "weigh", "weigh", "evict"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    dim = rng.choice([64, 128, 128, 8 * rng.randint(4, 20)])
    page = rng.choice([16, 64, _log(rng, 7, 128)])
    heads, shared = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    # (no more scores than the largest listed case of the operator has)
    if op == "shared":
        most = 16 * 250 * 6750 * 32
        prefix, rest = _log(rng, 64, 16000), _log(rng, 1, 2000)
        new = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 16, 300)])
        while 2 * new * (prefix + rest + new) * heads * shared > most:
            new, prefix = (new + 1) // 2, (prefix + 1) // 2
        rows = _log(rng, 2, max(2, min(128, most // (new * (prefix + rest + new) * heads * shared))))
        groups = _log(rng, 1, max(1, min(16, rows // 2)))
        each = max(1, rows // groups)
        return _shared(groups, (each + 1) // 2, each, (prefix + 1) // 2, prefix, rest // 3, rest, (new + 1) // 2, new, heads, shared, dim, page, dtype, rng.random() < 0.5)
    if op == "weigh":
        kind = rng.choice(["step", "last", "prompt"])
        new = {"step": 1, "last": _log(rng, 16, 2000), "prompt": _log(rng, 16, 4096)}[kind]
        last = rng.randint(1, 64) if kind == "last" else 0
        old = _log(rng, 1, 16000)
        most = 4096 * 8192 * 32
        count = min(new, last) if last else new
        while count * (new + old) * heads * shared > most:
            new, old = (new + 1) // 2, old // 2
            count = min(new, last) if last else new
        most = min(64, most // (count * (new + old) * heads * shared), 48 * 16000 * 8 * 128 // ((new + old) * heads * dim))
        return _weigh(_log(rng, 1, max(1, most)), (new + 1) // 2, new, old // 2, old, last, heads, shared, dim, page, dtype)
    layers, length = _log(rng, 1, 16), _log(rng, 64, 16000)
    keep = _log(rng, 16, length)
    first = rng.randint(0, min(8, keep // 4))
    token = 2 * layers * heads * dim * BYTES[dtype]
    most = max(1, min(64, 12 * 8000 * (1 << 15) // (token * (length + 2 * keep))))
    return _evict(_log(rng, 1, most), (length + 3) // 4, length, keep, first, rng.randint(0, keep // 2), layers, heads, dim, page, dtype)


# ---- inputs -------------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, dtype, scale=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=g)


def _spread(low, high, count):
    return [low + i * (high - low) // (count - 1) for i in range(count)] if count > 1 else [high]


def _between(seed, low, high, count, salt):
    """`count` whole numbers spread evenly from low to high: every seed has the same ones, in an order of its own."""
    g = torch.Generator()
    g.manual_seed(int(seed) * 31 + salt)
    return torch.tensor(_spread(low, high, count))[torch.randperm(count, generator=g)]


def _out_of(tokens, heads, dim, dtype, transposed):
    """A tensor tokens x heads x dim, in memory like that or, transposed, features x tokens."""
    x = torch.empty((heads, dim, tokens) if transposed else (tokens, heads, dim), dtype=dtype, device="cuda")
    return x.permute(2, 0, 1) if transposed else x


def _i32(x):
    return x.to(torch.int32).cuda()


def _sums(x):
    """0, x[0], x[0] + x[1], ..."""
    s = torch.zeros(x.numel() + 1, dtype=torch.int64)
    s[1:] = torch.cumsum(x, 0)
    return s


def _pool(s, g, layers, pages, heads, page, dim, dtype):
    s["keys"], s["values"] = (_normal(g, (layers, pages, heads, page, dim), dtype) for _ in range(2))
    s["references"] = _i32(torch.bincount(s["table"][s["table"] >= 0].flatten().cpu().long(), minlength=pages))


def _handle(s, dtype):
    """The framework's description of the cache in the state (its arrays stay the state's own)."""
    import hopper_spmm_amd as hs
    sequences, table_pages = s["table"].shape
    layers, pages, heads, page, dim = s["keys"].shape
    s["scratch"] = torch.zeros(hs.cache_scratch_words(pages, sequences, table_pages), dtype=torch.int32, device="cuda")
    s["cache"] = hs.Cache(getattr(hs, NAMES[dtype]), layers, pages, page, heads, dim, sequences, table_pages, s["keys"].data_ptr(), s["values"].data_ptr(),
                          s["table"].data_ptr(), s["lengths"].data_ptr(), s["references"].data_ptr(), s["scratch"].data_ptr())


def _weights_handle(s):
    import hopper_spmm_amd as hs
    return hs.Weights(s["weights"].data_ptr(), *s["weights"].stride()[:3])


def _view(x):
    import hopper_spmm_amd as hs
    return hs.Heads(x.data_ptr(), *x.stride())


def _workspace(s, need):
    s["workspace"] = torch.zeros(max(1, need), dtype=torch.uint8, device="cuda")


def prepare(case, seed):
    return {"shared": _prepare_shared, "weigh": _prepare_weigh, "evict": _prepare_evict}[case["op"]](case, seed)


def _chunks(s, new, length):
    """Every new token's sequence and position, which the plain forms index with."""
    starts = _sums(new)
    s["starts"], s["lengths"] = _i32(starts), _i32(length)
    s["sequence"] = torch.repeat_interleave(torch.arange(new.numel()), new).cuda()
    s["position"] = torch.arange(int(starts[-1]), device="cuda") - s["starts"].long()[s["sequence"]] + _i32(length - new).long()[s["sequence"]]


def _prepare_shared(case, seed):
    g = _generator(seed)
    dtype, page, groups = TYPES[case["dtype"]], case["page"], case["groups"]
    rows = _between(seed, case["rows_least"], case["rows_most"], groups, 1)
    n = int(rows.sum())
    prefix = _between(seed, case["prefix_least"], case["prefix_most"], groups, 2)
    rest, new = _between(seed, case["rest_least"], case["rest_most"], n, 3), _between(seed, case["new_least"], case["new_most"], n, 4)
    firsts = _sums(rows)
    group = torch.repeat_interleave(torch.arange(groups), rows)
    length = prefix[group] + rest + new
    # pages that lie within the prefix are the group's, the others a sequence's own
    common, held = prefix // page, (length + page - 1) // page
    table_pages = -(-(case["prefix_most"] + case["rest_most"] + case["new_most"]) // page)
    pages = (sum(_spread(case["prefix_least"], case["prefix_most"], groups)) + int(rest.sum()) + int(new.sum())) // page + 2 * n + groups
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 5))
    place = torch.arange(table_pages)
    first_common, first_own = _sums(common), _sums(held - common[group]) + int(common.sum())
    at = torch.where(place[None, :] < common[group][:, None], first_common[:-1][group][:, None] + place[None, :],
                     first_own[:-1][:, None] + place[None, :] - common[group][:, None])
    table = torch.where(place[None, :] < held[:, None], order[at.clamp(0, pages - 1)], torch.full_like(at, -1))
    s = {"case": case, "table": _i32(table), "prefix": _i32(prefix), "firsts": _i32(firsts), "longest": int(length.max())}
    _chunks(s, new, length)
    _pool(s, g, 1, pages, case["heads"], page, case["dim"], dtype)
    # a page that the prefix ends in is every sequence's own, and begins alike
    for i in range(groups):
        if int(prefix[i]) % page:
            ids = s["table"][firsts[i]:firsts[i + 1], common[i]].long()
            for x in (s["keys"], s["values"]):
                x[0][ids, :, : int(prefix[i]) % page] = x[0][ids[0], :, : int(prefix[i]) % page].clone()
    tokens, queries = int(new.sum()), case["heads"] * case["shared"]
    s["q"] = _normal(g, (tokens, queries, case["dim"]), dtype, 1.5)
    s["out"] = _out_of(tokens, queries, case["dim"], dtype, case["transposed"])
    s["lse"] = torch.empty((tokens, queries), dtype=torch.float32, device="cuda")
    if own:
        import hopper_spmm_amd as hs
        _handle(s, case["dtype"])
        s["batch"] = hs.Batch(n, tokens, s["starts"].data_ptr())
        most = max(int(new[firsts[i]:firsts[i + 1]].sum()) for i in range(groups))
        s["shared"] = hs.Prefix(groups, s["firsts"].data_ptr(), s["prefix"].data_ptr(), most_tokens=most, longest=case["prefix_most"])
        s["attention"] = hs.Attention(queries, 1.0 / math.sqrt(case["dim"]), longest_chunk=case["new_most"], longest=s["longest"])
        s["views"] = [_view(s[x]) for x in ("q", "out")]
        _workspace(s, s["cache"].attend_shared_workspace(s["batch"], s["shared"], s["attention"]))
    return s


def _pages_of(s, case, seed, length, table_pages, spare, sequences):
    """A table of `sequences` rows, of which the first ones hold so many tokens, in pages in a random order; spare: free pages."""
    held = (length + case["page"] - 1) // case["page"]
    pages = int(length.sum()) // case["page"] + length.numel() + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 5))
    table = torch.full((sequences, table_pages), -1, dtype=torch.int64)
    inside = torch.arange(table_pages)[None, :] < held[:, None]
    table[: length.numel()][inside] = order[: int(held.sum())]
    s["table"] = _i32(table)
    return pages


def _prepare_weigh(case, seed):
    g = _generator(seed)
    dtype, n, page = TYPES[case["dtype"]], case["sequences"], case["page"]
    new = _between(seed, case["new_least"], case["new_most"], n, 1)
    length = new + _between(seed, case["old_least"], case["old_most"], n, 2)
    table_pages = -(-(case["new_most"] + case["old_most"]) // page)
    s = {"case": case, "longest": case["new_most"] + case["old_most"]}
    pages = _pages_of(s, case, seed, length, table_pages, 0, n)
    _chunks(s, new, length)
    _pool(s, g, 1, pages, case["heads"], page, case["dim"], dtype)
    tokens, queries = int(new.sum()), case["heads"] * case["shared"]
    s["q"] = _normal(g, (tokens, queries, case["dim"]), dtype, 1.5)
    # what the keys have received so far
    s["weights"] = torch.exp(_normal(g, (1, n, case["heads"], table_pages * page), torch.float32, 1.5)) * 0.01
    # the attention of these tokens left the logarithms of its softmax's denominators
    s["lse"] = torch.zeros((tokens, queries), dtype=torch.float32, device="cuda")
    starts = _sums(new).tolist()
    for b in range(n):
        scores, rows = _scores(s, b, starts, torch.float32)
        s["lse"][rows] = torch.logsumexp(scores, -1).permute(1, 0, 2).reshape(len(rows), queries)
    if own:
        import hopper_spmm_amd as hs
        _handle(s, case["dtype"])
        s["batch"] = hs.Batch(n, tokens, s["starts"].data_ptr())
        s["attention"] = hs.Attention(queries, 1.0 / math.sqrt(case["dim"]), longest_chunk=case["new_most"], longest=s["longest"])
        s["view"], s["into"] = _view(s["q"]), _weights_handle(s)
        _workspace(s, s["cache"].weigh_workspace(s["batch"], s["attention"], last=case["last"]))
    return s


def _scores(s, b, starts, dtype):
    """Scores of the tokens of sequence b that count: heads x tokens x shared x keys, and the tokens' numbers."""
    c = s["case"]
    t0, t1 = starts[b], starts[b + 1]
    if c["last"]:
        t0 = max(t0, t1 - c["last"])
    length = int(s["position"][t1 - 1]) + 1
    key = torch.arange(length, device="cuda")
    k = s["keys"][0][s["table"][b][key // c["page"]].long(), :, key % c["page"]].to(dtype)
    q = s["q"][t0:t1].to(dtype).reshape(t1 - t0, c["heads"], c["shared"], c["dim"])
    scores = torch.matmul(q.permute(1, 0, 2, 3).reshape(c["heads"], -1, c["dim"]), k.permute(1, 2, 0).contiguous()).mul_(1.0 / math.sqrt(c["dim"]))
    scores = scores.reshape(c["heads"], t1 - t0, c["shared"], length)
    scores.masked_fill_((key[None, :] > s["position"][t0:t1, None])[None, :, None, :], -math.inf)
    return scores, torch.arange(t0, t1, device="cuda")


def _prepare_evict(case, seed):
    g = _generator(seed)
    n, page, keep = case["sequences"], case["page"], case["keep"]
    length = _between(seed, case["length_least"], case["length_most"], n, 1)
    table_pages = -(-case["length_most"] // page)
    # sequences 0 .. n - 1 hold the prompts, n .. 2 n - 1 take over what stays of them (twice its pages: the old ones are given back last)
    s = {"case": case, "parents": _i32(torch.arange(n)), "children": _i32(torch.arange(n, 2 * n)), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    pages = _pages_of(s, case, seed, length, table_pages, 2 * n * -(-keep // page), 2 * n)
    s["lengths"] = _i32(torch.cat([length, torch.zeros_like(length)]))
    _pool(s, g, case["layers"], pages, case["heads"], page, case["dim"], TYPES[case["dtype"]])
    # accumulated weights are spread over orders of magnitude; some tokens have received nothing
    w = torch.exp(_normal(g, (case["layers"], 2 * n, case["heads"], table_pages * page), torch.float32, 2.0)) * 0.01
    w.masked_fill_(torch.rand(w.shape, generator=g, device="cuda") < 0.05, 0.0)
    s["weights"] = w.masked_fill_(torch.arange(w.shape[-1], device="cuda")[None, None, None, :] >= s["lengths"][None, :, None, None], 0.0)
    s["kept"] = torch.empty((case["layers"], n, case["heads"], keep), dtype=torch.int32, device="cuda")
    if own:
        _handle(s, case["dtype"])
        s["into"] = _weights_handle(s)
        _workspace(s, s["cache"].evict_workspace(n, keep))
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------


def run(state):
    return (RUN_OWN if own else RUN_PLAIN)[state["case"]["op"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_shared(s):
    q, out = s["views"]
    s["cache"].attend_shared(0, s["batch"], s["shared"], s["attention"], q, out, lse=s["lse"].data_ptr(), workspace=s["workspace"].data_ptr(),
                             workspace_bytes=s["workspace"].numel(), stream=_stream())
    return s["out"], s["lse"]


def _own_weigh(s):
    s["cache"].weigh(0, s["batch"], s["attention"], s["view"], s["lse"].data_ptr(), s["into"], decay=DECAY, last=s["case"]["last"],
                     workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(), stream=_stream())
    return s["weights"]


def _own_evict(s):
    c = s["case"]
    s["cache"].evict(c["sequences"], s["parents"].data_ptr(), s["children"].data_ptr(), s["into"], c["keep"], first=c["first"], last=c["last"],
                     kept=s["kept"].data_ptr(), status=s["status"].data_ptr(), workspace=s["workspace"].data_ptr(),
                     workspace_bytes=s["workspace"].numel(), stream=_stream())
    return s["table"], s["lengths"], s["references"], s["status"], s["kept"], s["weights"], s["keys"], s["values"]


# of what keys have received before
DECAY = 0.96875


def _padded(s, chunk):
    """Scores of the last `chunk` tokens of every sequence, those of short ones at the front: sequence, head, token, head that
    shares, key; which keys a token sees; the tokens' numbers, and their places there."""
    c = s["case"]
    n, heads, shared, dim = s["starts"].numel() - 1, c["heads"], c["shared"], c["dim"]
    keys = s["table"].shape[1] * c["page"]
    ids = s["table"].clamp_min(0).long()
    k = s["keys"][0][ids].permute(0, 2, 1, 3, 4).reshape(n, heads, keys, dim).float()
    count = (s["starts"][1:] - s["starts"][:-1]).clamp_max(chunk)
    place = torch.arange(s["sequence"].numel(), device="cuda") - (s["starts"][1:] - count)[s["sequence"]]
    tokens = torch.nonzero(place >= 0)[:, 0]
    sequence, place = s["sequence"][tokens], place[tokens]
    q = torch.zeros((n, chunk, heads * shared, dim), dtype=torch.float32, device="cuda")
    q[sequence, place] = s["q"][tokens].float()
    q = q.reshape(n, chunk, heads, shared, dim).permute(0, 2, 1, 3, 4).reshape(n, heads, chunk * shared, dim)
    at = (s["lengths"] - count)[:, None] + torch.arange(chunk, device="cuda")[None, :]
    key = torch.arange(keys, device="cuda")
    seen = (key[None, None, :] <= at[:, :, None]) & (key[None, None, :] < s["lengths"][:, None, None])
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(dim)).reshape(n, heads, chunk, shared, keys)
    return scores, seen, tokens, (sequence, place)


def _plain_shared(s):
    c = s["case"]
    heads, shared, dim, chunk = c["heads"], c["shared"], c["dim"], c["new_most"]
    scores, seen, _, place = _padded(s, chunk)
    n, keys = scores.shape[0], scores.shape[-1]
    v = s["values"][0][s["table"].clamp_min(0).long()].permute(0, 2, 1, 3, 4).reshape(n, heads, keys, dim).float()
    scores = scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    most = scores.amax(-1, keepdim=True)
    weights = scores.sub_(most).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.reshape(n, heads, chunk * shared, keys), v).reshape(n, heads, chunk, shared, dim) / total
    s["out"].copy_(out.permute(0, 2, 1, 3, 4).reshape(n, chunk, heads * shared, dim)[place])
    s["lse"].copy_((most + total.log())[..., 0].permute(0, 2, 1, 3).reshape(n, chunk, heads * shared)[place])
    return s["out"], s["lse"]


def _plain_weigh(s):
    c = s["case"]
    heads, shared, chunk = c["heads"], c["shared"], min(c["new_most"], c["last"] or c["new_most"])
    scores, seen, tokens, place = _padded(s, chunk)
    n, keys = scores.shape[0], scores.shape[-1]
    counts = torch.zeros((n, chunk), dtype=torch.bool, device="cuda")
    counts[place] = True
    lse = torch.zeros((n, chunk, heads * shared), dtype=torch.float32, device="cuda")
    lse[place] = s["lse"][tokens]
    scores = scores.sub_(lse.reshape(n, chunk, heads, shared).permute(0, 2, 1, 3)[..., None]).masked_fill_(~(seen & counts[:, :, None])[:, None, :, None, :], -math.inf)
    received = scores.exp_().sum((2, 3))
    key, old = torch.arange(keys, device="cuda")[None, :], (s["lengths"] - (s["starts"][1:] - s["starts"][:-1]))[:, None]
    before = torch.where((key < old)[:, None, :], s["weights"][0] * DECAY, torch.zeros((), device="cuda"))
    s["weights"][0] = torch.where((key < s["lengths"][:, None])[:, None, :], before + received, s["weights"][0])
    return s["weights"]


def _plain_evict(s):
    c = s["case"]
    n, page, keep = c["sequences"], c["page"], c["keep"]
    parents, children = s["parents"].long(), s["children"].long()
    length = s["lengths"][parents]
    stays = length.clamp_max(keep)
    w = s["weights"][:, parents]
    position = torch.arange(w.shape[-1], device="cuda")
    anyway = (position[None, :] < c["first"]) | (position[None, :] >= length[:, None] - c["last"])
    rank = w.masked_fill(anyway[None, :, None, :], math.inf).masked_fill((position[None, :] >= length[:, None])[None, :, None, :], -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :keep]
    valid = torch.arange(keep, device="cuda")[None, :] < stays[:, None]
    kept = torch.where(valid[None, :, None, :], order, torch.full_like(order, 1 << 40)).sort(-1)[0]
    kept = torch.where(valid[None, :, None, :], kept, torch.zeros_like(kept))
    s["kept"].copy_(torch.where(valid[None, :, None, :], kept, torch.full_like(kept, -1)))
    s["weights"][:, children] = torch.nn.functional.pad(w.gather(-1, kept).masked_fill(~valid[None, :, None, :], 0.0), (0, w.shape[-1] - keep))
    # the free pages of lowest number, in the children's order
    need = (stays + page - 1) // page
    places = -(-keep // page)
    free = torch.argsort((s["references"] > 0).int(), stable=True).to(torch.int32)
    at = (torch.cumsum(need, 0) - need)[:, None] + torch.arange(places, device="cuda")[None, :]
    rows = torch.where(torch.arange(places, device="cuda")[None, :] < need[:, None], free[at.clamp_max(free.numel() - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
    # keys and values, layer by layer; what is behind a child's last token is left as it was
    slot = torch.arange(keep, device="cuda")
    to_page = torch.where(valid, rows[:, slot // page], rows[:, :1]).long()[:, None, :].expand(n, c["heads"], keep)
    to_slot = torch.where(valid, (slot % page)[None, :], torch.zeros_like(slot)[None, :])[:, None, :].expand(n, c["heads"], keep)
    head = torch.arange(c["heads"], device="cuda")[None, :, None].expand(n, c["heads"], keep)
    for i in range(c["layers"]):
        # (where there is no token the first one is copied once more)
        source = torch.where(valid[:, None, :], kept[i], kept[i][..., :1])
        from_page = s["table"][parents[:, None, None], source // page].long()
        for x in (s["keys"], s["values"]):
            x[i][to_page, head, to_slot] = x[i][from_page, head, source % page]
    old = s["table"][children]
    s["references"].index_add_(0, old.clamp_min(0).flatten().long(), -(old >= 0).flatten().int())
    s["references"].index_add_(0, rows.clamp_min(0).flatten().long(), (rows >= 0).flatten().int())
    s["table"][children] = torch.nn.functional.pad(rows, (0, s["table"].shape[1] - places), value=-1)
    s["lengths"][children] = stays
    s["status"].zero_()
    return s["table"], s["lengths"], s["references"], s["status"], s["kept"], s["weights"], s["keys"], s["values"]


RUN_OWN = {"shared": _own_shared, "weigh": _own_weigh, "evict": _own_evict}
RUN_PLAIN = {"shared": _plain_shared, "weigh": _plain_weigh, "evict": _plain_evict}


# ---- what a pass cannot do without --------------------------------------------------------------------------------


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "evict":
        lengths = _spread(case["length_least"], case["length_most"], case["sequences"])
        kept = sum(min(x, case["keep"]) for x in lengths)
        rows = case["layers"] * case["heads"]
        table_pages = -(-case["length_most"] // case["page"])
        # weights of all tokens read; a child's row of them and its list written; keys and values moved; rows of the table
        numbers = 4 * rows * (sum(lengths) + case["sequences"] * (table_pages * case["page"] + case["keep"])) + 8 * case["sequences"] * table_pages
        return {"bytes": numbers + 4 * kept * rows * case["dim"] * size, "flops": 0}
    queries = case["heads"] * case["shared"]
    if case["op"] == "weigh":
        new, old = (_spread(case[x + "_least"], case[x + "_most"], case["sequences"]) for x in ("new", "old"))
        count = [min(m, case["last"]) if case["last"] else m for m in new]
        # (the order of the chunks and that of what lies in front of them are drawn apart: means of both)
        pairs = sum(c * (m - c) + c * (c + 1) / 2 for c, m in zip(count, new)) + sum(count) * sum(old) / len(old)
        keys = sum(new) + sum(old)
        kept = keys * case["heads"] * (case["dim"] * size + 4) + 4 * sum(old) * case["heads"]
        return {"bytes": kept + sum(count) * queries * (case["dim"] * size + 4), "flops": 2 * pairs * queries * case["dim"]}
    rows = _spread(case["rows_least"], case["rows_most"], case["groups"])
    prefix = _spread(case["prefix_least"], case["prefix_most"], case["groups"])
    rest, new = (_spread(case[x + "_least"], case[x + "_most"], sum(rows)) for x in ("rest", "new"))
    tokens = sum(new)
    pairs = tokens * (sum(prefix) / len(prefix) + sum(rest) / len(rest)) + sum(m * (m + 1) / 2 for m in new)
    kv = 2 * (sum(prefix) + sum(rest) + tokens) * case["heads"] * case["dim"] * size
    return {"bytes": kv + 2 * tokens * queries * case["dim"] * size + 4 * tokens * queries, "flops": 4 * pairs * queries * case["dim"]}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------


def exact(case, seed):
    return {"shared": _exact_shared, "weigh": _exact_weigh, "evict": _exact_evict}[case["op"]](case, prepare(case, seed))


def _exact_shared(case, s):
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    starts, lengths, firsts, prefix = (s[x].tolist() for x in ("starts", "lengths", "firsts", "prefix"))
    for g in range(case["groups"]):
        for b in range(firsts[g], firsts[g + 1]):
            t0, t1 = starts[b], starts[b + 1]
            key = torch.arange(lengths[b], device="cuda")
            hidden = key[None, :] > torch.arange(lengths[b] - (t1 - t0), lengths[b], device="cuda")[:, None]
            # the prefix by the group's first sequence
            row = torch.where(key < prefix[g], s["table"][firsts[g]][key // case["page"]], s["table"][b][key // case["page"]]).long()
            for h in range(case["heads"]):
                k, v = s["keys"][0][row, h, key % case["page"]].double(), s["values"][0][row, h, key % case["page"]].double()
                for r in range(h * case["shared"], (h + 1) * case["shared"]):
                    logits = (s["q"][t0:t1, r].double() @ k.T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
                    lse[t0:t1, r] = torch.logsumexp(logits, -1)
                    out[t0:t1, r] = torch.softmax(logits, -1) @ v
    return out, lse


def _exact_weigh(case, s):
    weights, starts = s["weights"].double(), s["starts"].tolist()
    for b in range(case["sequences"]):
        t0, t1, length = starts[b], starts[b + 1], int(s["lengths"][b])
        weights[0, b, :, : length - (t1 - t0)] *= DECAY
        weights[0, b, :, length - (t1 - t0): length] = 0.0
        if case["last"]:
            t0 = max(t0, t1 - case["last"])
        key = torch.arange(length, device="cuda")
        hidden = key[None, :] > s["position"][t0:t1, None]
        for h in range(case["heads"]):
            k = s["keys"][0][s["table"][b][key // case["page"]].long(), h, key % case["page"]].double()
            for r in range(h * case["shared"], (h + 1) * case["shared"]):
                logits = (s["q"][t0:t1, r].double() @ k.T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
                weights[0, b, h, :length] += torch.exp(logits - s["lse"][t0:t1, r, None].double()).sum(0)
    return weights


def _exact_evict(case, s):
    page, first, last, keep = case["page"], case["first"], case["last"], case["keep"]
    keys, values, weights = s["keys"].double(), s["values"].double(), s["weights"].double()
    table, lengths = s["table"].cpu(), s["lengths"].tolist()
    free = torch.nonzero(s["references"].cpu() <= 0)[:, 0].tolist()
    for b in range(case["sequences"]):
        length, child = lengths[b], case["sequences"] + b
        m = min(length, keep)
        pages = [free.pop(0) for _ in range(-(-m // page))]
        to = torch.tensor(pages)[torch.arange(m) // page].cuda()
        w = s["weights"][:, b].cpu().double()
        weights[:, child] = 0.0
        for i in range(case["layers"]):
            for h in range(case["heads"]):
                middle = w[i, h, first: max(first, length - last)]
                chosen = torch.sort(middle, descending=True, stable=True)[1][: keep - first - last] + first
                at = (torch.arange(length) if length <= keep else torch.cat([torch.arange(first), chosen.sort()[0], torch.arange(length - last, length)])).cuda()
                weights[i, child, h, :m] = s["weights"][i, b, h, at].double()
                source = s["table"][b][at // page].long()
                for x, y in ((keys, s["keys"]), (values, s["values"])):
                    x[i, to, h, torch.arange(m, device="cuda") % page] = y[i, source, h, at % page].double()
    return None, None, None, None, None, weights, keys, values
