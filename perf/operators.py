"""Performance cases of the operators between two products of a pruned decoder layer: rotary positions, a paged cache of
keys and values, the attention of new tokens over it, and the work on its pages.

A case names an operator, sizes and an element type; one pass is one call of that operator with everything resident on
the GPU:

  rotate    turn the pairs of elements of every head by their token's position; `backward`: the gradient of that
  append    keys and values of new tokens into their pages, queries and keys turned on the way
  attend    softmax(scale q k) v of a ragged batch of new tokens (a chunk, or a single one) over pages
  fork      sequences that take over others' states: shared pages, a copy of the last one where it is partly filled
  compact   live pages to the low end of the pool, tables renamed

Heads of 128 of a hidden size of 4096 (32 heads, 8 of them of keys and values) are those of the layers that the
products are benchmarked at; the rest is generic.  Inputs are made on the GPU from the seed alone.
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
NAMES = {"fp16": "FP16", "bf16": "BF16", "fp32": "TF32"}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _rotate(tokens, heads, dim, dims, dtype, interleaved, backward, positions):
    return {"op": "rotate", "tokens": tokens, "heads": heads, "dim": dim, "dims": dims, "dtype": dtype, "interleaved": interleaved,
            "backward": backward, "positions": positions}


def _batch(op, sequences, new_least, new_most, old_least, old_most, heads, shared, dim, page, dtype):
    """new_*, old_*: tokens of a sequence's chunk, and of what its cache holds already; shared: heads of queries that share
    one of keys and values."""
    return {"op": op, "sequences": sequences, "new_least": new_least, "new_most": new_most, "old_least": old_least, "old_most": old_most,
            "heads": heads, "shared": shared, "dim": dim, "page": page, "dtype": dtype}


def _append(sequences, new_least, new_most, old_least, old_most, heads, shared, dim, page, dtype, dims, interleaved, transposed):
    """transposed: queries, keys and values lie features x tokens, as a product of weights leaves them."""
    return dict(_batch("append", sequences, new_least, new_most, old_least, old_most, heads, shared, dim, page, dtype),
                dims=dims, interleaved=interleaved, transposed=transposed)


def _attend(sequences, new_least, new_most, old_least, old_most, heads, shared, dim, page, dtype, window, transposed):
    """window: 0, or how many keys a token sees; transposed: the output lies features x tokens, as the next product wants it."""
    return dict(_batch("attend", sequences, new_least, new_most, old_least, old_most, heads, shared, dim, page, dtype),
                window=window, transposed=transposed)


def _fork(groups, beams, length_least, length_most, layers, heads, dim, page, dtype):
    return {"op": "fork", "groups": groups, "beams": beams, "length_least": length_least, "length_most": length_most, "layers": layers,
            "heads": heads, "dim": dim, "page": page, "dtype": dtype}


def _compact(sequences, length_least, length_most, pages, layers, heads, dim, page, dtype):
    return {"op": "compact", "sequences": sequences, "length_least": length_least, "length_most": length_most, "pages": pages, "layers": layers,
            "heads": heads, "dim": dim, "page": page, "dtype": dtype}


def listed():
    return [
        # the queries and keys of a small batch that decodes: launch latency
        dict(_rotate(8, 40, 128, 128, "bf16", False, False, 32768), name="rotate_step"),
        # the gradient of a training batch's queries: half of each head turned, neighbours in pairs
        dict(_rotate(16384, 32, 128, 64, "fp16", True, True, 4096), name="rotate_train"),
        # one new token for each of 64 sequences, as the products leave them
        dict(_append(64, 1, 1, 100, 8000, 8, 4, 128, 16, "bf16", 128, False, True), name="append_step"),
        # prompts of odd lengths in full precision
        dict(_append(5, 700, 4099, 0, 333, 10, 3, 80, 24, "fp32", 40, True, False), name="append_prompts"),
        # three short sequences, a token each, full precision: launch latency
        dict(_attend(3, 1, 1, 20, 300, 8, 1, 64, 16, "fp32", 0, False), name="attend_step_small"),
        # a server's batch that decodes: the cache is read once
        dict(_attend(48, 1, 1, 500, 16000, 8, 4, 128, 16, "bf16", 0, True), name="attend_step"),
        # prompts and single tokens mixed, each token sees a thousand keys: odd head, page and chunk sizes
        dict(_attend(17, 1, 700, 0, 5000, 4, 3, 96, 24, "fp16", 1000, False), name="attend_mixed"),
        # the last quarter of a long prompt
        dict(_attend(1, 4096, 4096, 12288, 12288, 8, 4, 128, 64, "bf16", 0, True), name="attend_chunk"),
        # beam search of one prompt, one layer's cache
        dict(_fork(1, 8, 100, 1000, 1, 8, 128, 16, "fp16"), name="fork_beams"),
        # a server's batch of beams, all layers
        dict(_fork(48, 4, 100, 1500, 32, 8, 128, 16, "bf16"), name="fork_batch"),
        # a small pool with holes
        dict(_compact(7, 20, 500, 300, 2, 4, 64, 16, "fp32"), name="compact_small"),
        # a pool two thirds full, all layers: a third of what it holds moves
        dict(_compact(40, 20, 1000, 2048, 32, 8, 128, 16, "bf16"), name="compact_pool"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend", "attend", "attend", "attend", "fork", "compact"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    dim = rng.choice([64, 128, 128, 8 * rng.randint(4, 20)])
    page = rng.choice([16, 64, _log(rng, 8, 128)])
    if op == "rotate":
        heads = rng.randint(1, 48)
        tokens = _log(rng, 1, max(1, 16384 * 32 * 128 // (heads * dim)))
        return _rotate(tokens, heads, dim, 2 * rng.randint(dim // 8, dim // 2), dtype, rng.random() < 0.5, rng.random() < 0.5, _log(rng, 512, 131072))
    if op in ("append", "attend"):
        heads, shared = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        if op == "append":
            new = _log(rng, 1, 4096)
            sequences = _log(rng, 1, max(1, min(128, 16384 // new)))
            return _append(sequences, (new + 1) // 2, new, 0, _log(rng, 1, 4000), heads, shared, dim, page, dtype, 2 * rng.randint(dim // 8, dim // 2),
                           rng.random() < 0.5, rng.random() < 0.5)
        window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        kind = rng.choice(["step", "few", "chunk", "mixed"])
        new = {"step": 1, "few": rng.randint(2, 16), "chunk": _log(rng, 64, 4096), "mixed": _log(rng, 16, 1024)}[kind]
        old = _log(rng, 1, 16000)
        while new * (new + old) * heads * shared > 4096 * 16384 * 32:
            new, old = (new + 1) // 2, old // 2
        # (no more scores than the largest listed case has, nor keys than the largest batch)
        most = min(64, 4096 * 16384 * 32 // (new * (new + old) * heads * shared), 48 * 16000 * 8 * 128 // ((new + old) * heads * dim))
        sequences = _log(rng, 1, max(1, most))
        return _attend(sequences, 1 if kind == "mixed" else new, new, old // 2, old, heads, shared, dim, page, dtype, window, rng.random() < 0.5)
    layers, heads = _log(rng, 1, 32), rng.choice([1, 2, 4, 8])
    page_bytes = 2 * layers * heads * page * dim * BYTES[dtype]
    if op == "fork":
        most = 48 * 4 * (1 << 21) // page_bytes
        length = min(_log(rng, 16, 1500), 90 * page)
        beams = rng.randint(2, 8)
        return _fork(_log(rng, 1, max(1, min(64, most // (beams + length // page + 1)))), beams, (length + 1) // 2, length, layers, heads, dim, page, dtype)
    pages = _log(rng, 64, max(65, min(65536, 2048 * (1 << 21) // page_bytes)))
    length = _log(rng, page, page * max(1, min(64, pages // 6)))
    return _compact(max(1, min(512, pages * page // (2 * length))), (length + 1) // 2, length, pages, layers, heads, dim, page, dtype)


# ---- inputs -------------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, dtype, scale=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=g)


def _between(case, seed, low, high, count, salt):
    """`count` whole numbers spread evenly from low to high: every seed has the same ones, in an order of its own."""
    g = torch.Generator()
    g.manual_seed(int(seed) * 31 + salt)
    return torch.tensor(_spread(low, high, count))[torch.randperm(count, generator=g)]


def _table(positions, dims):
    """(cos, sin) by position and pair, frequencies 10000^(-2 i / dims)."""
    f = torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), -torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f[None, :]
    return torch.stack([torch.cos(a), torch.sin(a)], dim=-1).to(torch.float32).contiguous()


def _heads_of(g, tokens, heads, dim, dtype, transposed, scale=1.0, empty=False):
    """A tensor tokens x heads x dim, in memory like that or, transposed, features x tokens."""
    shape = (heads, dim, tokens) if transposed else (tokens, heads, dim)
    x = torch.empty(shape, dtype=dtype, device="cuda") if empty else _normal(g, shape, dtype, scale)
    return x.permute(2, 0, 1) if transposed else x


def _pool(g, layers, pages, heads, page, dim, dtype):
    return _normal(g, (layers, pages, heads, page, dim), dtype), _normal(g, (layers, pages, heads, page, dim), dtype)


def _i32(x):
    return x.to(torch.int32).cuda()


def _handle(s, layers, pages, heads, page, dim, dtype):
    """The framework's description of the cache in the state (its arrays stay the state's own)."""
    import hopper_spmm_amd as hs
    sequences, table_pages = s["table"].shape
    s["scratch"] = torch.zeros(hs.cache_scratch_words(pages, sequences, table_pages), dtype=torch.int32, device="cuda")
    s["cache"] = hs.Cache(getattr(hs, NAMES[dtype]), layers, pages, page, heads, dim, sequences, table_pages, s["keys"].data_ptr(), s["values"].data_ptr(),
                          s["table"].data_ptr(), s["lengths"].data_ptr(), s["references"].data_ptr(), s["scratch"].data_ptr())


def _view(x):
    import hopper_spmm_amd as hs
    return hs.Heads(x.data_ptr(), *x.stride())


def prepare(case, seed):
    return {"rotate": _prepare_rotate, "append": _prepare_batch, "attend": _prepare_batch, "fork": _prepare_fork, "compact": _prepare_compact}[case["op"]](case, seed)


def _prepare_rotate(case, seed):
    g = _generator(seed)
    dtype = TYPES[case["dtype"]]
    s = {"case": case, "x": _normal(g, (case["tokens"], case["heads"], case["dim"]), dtype), "table": _table(case["positions"], case["dims"]),
         "positions": torch.randint(0, case["positions"], (case["tokens"],), generator=g, device="cuda", dtype=torch.int32)}
    s["y"] = torch.empty_like(s["x"])
    if own:
        import hopper_spmm_amd as hs
        s["rotary"] = hs.Rotary(case["dims"], case["positions"], s["table"].data_ptr(), interleaved=case["interleaved"])
        s["type"], s["x_heads"], s["y_heads"] = getattr(hs, NAMES[case["dtype"]]), _view(s["x"]), _view(s["y"])
    return s


def _prepare_batch(case, seed):
    g = _generator(seed)
    dtype, n, page, dim, heads, shared = TYPES[case["dtype"]], case["sequences"], case["page"], case["dim"], case["heads"], case["shared"]
    new = _between(case, seed, case["new_least"], case["new_most"], n, 1)
    length = new + _between(case, seed, case["old_least"], case["old_most"], n, 2)
    starts = torch.zeros(n + 1, dtype=torch.int64)
    starts[1:] = torch.cumsum(new, 0)
    tokens, longest = int(starts[-1]), case["new_most"] + case["old_most"]
    held = (length + page - 1) // page
    # (the pool is the same for every seed, whichever chunk meets whichever sequence)
    table_pages, pages = -(-longest // page), int(length.sum()) // page + n
    places = torch.arange(table_pages)[None, :] < held[:, None]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 5))
    table = torch.full((n, table_pages), -1, dtype=torch.int64)
    table[places] = order[: int(held.sum())]
    s = {"case": case, "longest": longest, "longest_chunk": case["new_most"], "table": _i32(table), "lengths": _i32(length), "starts": _i32(starts),
         "references": _i32(torch.bincount(table[table >= 0], minlength=pages))}
    # what the plain form indexes with: every token's sequence and position
    s["sequence"] = _i32(torch.repeat_interleave(torch.arange(n), new)).long()
    s["position"] = (torch.arange(tokens, device="cuda") - s["starts"][s["sequence"]] + (s["lengths"] - _i32(new))[s["sequence"]]).long()
    s["keys"], s["values"] = _pool(g, 1, pages, heads, page, dim, dtype)
    if case["op"] == "append":
        t = case["transposed"]
        s["q"], s["k"], s["v"] = (_heads_of(g, tokens, h, dim, dtype, t) for h in (heads * shared, heads, heads))
        s["q_out"] = torch.empty((tokens, heads * shared, dim), dtype=dtype, device="cuda")
        s["angles"] = _table(longest, case["dims"])
    else:
        s["q"] = _normal(g, (tokens, heads * shared, dim), dtype, 1.5)
        s["out"] = _heads_of(g, tokens, heads * shared, dim, dtype, case["transposed"], empty=True)
        s["lse"] = torch.empty((tokens, heads * shared), dtype=torch.float32, device="cuda")
    if own:
        import hopper_spmm_amd as hs
        _handle(s, 1, pages, heads, page, dim, case["dtype"])
        s["batch"] = hs.Batch(n, tokens, s["starts"].data_ptr())
        if case["op"] == "append":
            s["rotary"] = hs.Rotary(case["dims"], longest, s["angles"].data_ptr(), interleaved=case["interleaved"])
            s["views"] = [_view(s[x]) for x in ("k", "v", "q", "q_out")]
        else:
            s["attention"] = hs.Attention(heads * shared, 1.0 / math.sqrt(dim), causal=True, window=case["window"], longest_chunk=s["longest_chunk"], longest=longest)
            s["views"] = [_view(s[x]) for x in ("q", "out")]
            s["workspace"] = torch.zeros(max(1, s["cache"].attend_workspace(s["batch"], s["attention"])), dtype=torch.uint8, device="cuda")
    return s


def _prepare_fork(case, seed):
    g = _generator(seed)
    dtype, beams, groups, page = TYPES[case["dtype"]], case["beams"], case["groups"], case["page"]
    n = beams * groups
    # a group's beams share what they have in common, and have a last page each
    length = _between(case, seed, case["length_least"], case["length_most"], groups, 1)
    common, part = length // page, length % page > 0
    table_pages = int(((length + page - 1) // page).max()) + 1
    used = int(common.sum()) + beams * int(part.sum())
    pages = used + n + n // 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 5))
    table = torch.full((groups, beams, table_pages), -1, dtype=torch.int64)
    first = torch.cumsum(common, 0) - common
    inside = torch.arange(table_pages)[None, :] < common[:, None]
    table[inside[:, None, :].expand(groups, beams, table_pages)] = order[(first[:, None] + torch.arange(table_pages)[None, :])[:, None, :].expand(groups, beams, table_pages)[
        inside[:, None, :].expand(groups, beams, table_pages)]]
    own_pages = order[int(common.sum()):][: beams * int(part.sum())].reshape(-1, beams)
    table[torch.nonzero(part)[:, 0][:, None], torch.arange(beams)[None, :], common[part][:, None]] = own_pages
    table = table.reshape(n, table_pages)
    references = torch.bincount(table[table >= 0], minlength=pages)
    pick = torch.Generator().manual_seed(int(seed) + 6)
    parents = torch.randint(0, beams, (groups, beams), generator=pick) + torch.arange(groups)[:, None] * beams
    s = {"case": case, "table": _i32(table), "lengths": _i32(torch.repeat_interleave(length, beams)), "references": _i32(references),
         "parents": _i32(parents.reshape(-1)), "children": _i32(torch.arange(n)), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    s["keys"], s["values"] = _pool(g, case["layers"], pages, case["heads"], page, case["dim"], dtype)
    if own:
        _handle(s, case["layers"], pages, case["heads"], page, case["dim"], case["dtype"])
    return s


def _prepare_compact(case, seed):
    g = _generator(seed)
    n, page, pages = case["sequences"], case["page"], case["pages"]
    length = _between(case, seed, case["length_least"], case["length_most"], n, 1)
    held = (length + page - 1) // page
    fits = torch.cumsum(held, 0) <= pages
    length, held = length * fits, held * fits
    table_pages, used = max(1, int(held.max())), int(held.sum())
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 5))
    table = torch.full((n, table_pages), -1, dtype=torch.int64)
    table[torch.arange(table_pages)[None, :] < held[:, None]] = order[:used]
    references = torch.bincount(table[table >= 0], minlength=pages)
    s = {"case": case, "table": _i32(table), "lengths": _i32(length), "references": _i32(references)}
    s["table_out"], s["references_out"], s["live"] = torch.empty_like(s["table"]), torch.empty_like(s["references"]), torch.zeros(1, dtype=torch.int32, device="cuda")
    s["keys"], s["values"] = _pool(g, case["layers"], pages, case["heads"], page, case["dim"], TYPES[case["dtype"]])
    if own:
        _handle(s, case["layers"], pages, case["heads"], page, case["dim"], case["dtype"])
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------


def run(state):
    return (RUN_OWN if own else RUN_PLAIN)[state["case"]["op"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_rotate(s):
    import hopper_spmm_amd as hs
    c = s["case"]
    hs.rotate(s["type"], s["rotary"], c["tokens"], c["heads"], c["dim"], s["x_heads"], s["y_heads"], s["positions"].data_ptr(), backward=c["backward"], stream=_stream())
    return s["y"]


def _own_append(s):
    k, v, q, q_out = s["views"]
    s["cache"].append(0, s["batch"], k, v, rotary=s["rotary"], q_heads=s["case"]["heads"] * s["case"]["shared"], q=q, q_out=q_out, stream=_stream())
    return s["q_out"], s["keys"], s["values"]


def _own_attend(s):
    q, out = s["views"]
    s["cache"].attend(0, s["batch"], s["attention"], q, out, lse=s["lse"].data_ptr(), workspace=s["workspace"].data_ptr(),
                      workspace_bytes=s["workspace"].numel(), stream=_stream())
    return s["out"], s["lse"]


def _own_fork(s):
    s["cache"].fork(s["parents"].numel(), s["parents"].data_ptr(), s["children"].data_ptr(), s["status"].data_ptr(), stream=_stream())
    return s["table"], s["lengths"], s["references"], s["status"], s["keys"], s["values"]


def _own_compact(s):
    s["cache"].compact(s["live"].data_ptr(), table_out=s["table_out"].data_ptr(), references_out=s["references_out"].data_ptr(), stream=_stream())
    return s["table_out"], s["references_out"], s["live"], s["keys"], s["values"]


def _turned(x, cos, sin, dims, interleaved):
    """x in 32 bits: tokens x heads x dim; cos, sin: tokens x 1 x dims / 2."""
    part = x[..., :dims]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., : dims // 2], part[..., dims // 2:])
    first, second = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([first, second], dim=-1).flatten(-2) if interleaved else torch.cat([first, second], dim=-1)
    return torch.cat([turned, x[..., dims:]], dim=-1)


def _plain_rotate(s):
    c = s["case"]
    angles = s["table"][s["positions"].long()][:, None]
    sin = -angles[..., 1] if c["backward"] else angles[..., 1]
    s["y"].copy_(_turned(s["x"].float(), angles[..., 0], sin, c["dims"], c["interleaved"]))
    return s["y"]


def _plain_append(s):
    c = s["case"]
    angles = s["angles"][s["position"]][:, None]
    turn = lambda x: _turned(x.float(), angles[..., 0], angles[..., 1], c["dims"], c["interleaved"])  # noqa: E731
    s["q_out"].copy_(turn(s["q"]))
    pages, slots = s["table"][s["sequence"], s["position"] // c["page"]].long(), s["position"] % c["page"]
    s["keys"][0][pages, :, slots] = turn(s["k"]).to(s["keys"].dtype)
    s["values"][0][pages, :, slots] = s["v"]
    return s["q_out"], s["keys"], s["values"]


def _plain_attend(s):
    c = s["case"]
    n, page, dim, heads, shared = c["sequences"], c["page"], c["dim"], c["heads"], c["shared"]
    chunk, keys = s["longest_chunk"], s["table"].shape[1] * page
    # keys and values: sequence, head, position, element; queries: sequence, head, (token, head that shares), element
    ids = s["table"].clamp_min(0).long()
    k, v = (s[x][0][ids].permute(0, 2, 1, 3, 4).reshape(n, heads, keys, dim).float() for x in ("keys", "values"))
    place = torch.arange(s["sequence"].numel(), device="cuda") - s["starts"][s["sequence"]]
    q = torch.zeros((n, chunk, heads * shared, dim), dtype=torch.float32, device="cuda")
    q[s["sequence"], place] = s["q"].float()
    q = q.reshape(n, chunk, heads, shared, dim).permute(0, 2, 1, 3, 4).reshape(n, heads, chunk * shared, dim)
    new = s["starts"][1:] - s["starts"][:-1]
    at = (s["lengths"] - new)[:, None] + torch.arange(chunk, device="cuda")[None, :]
    key = torch.arange(keys, device="cuda")
    seen = (key[None, None, :] <= at[:, :, None]) & (key[None, None, :] < s["lengths"][:, None, None])
    if c["window"]:
        seen &= key[None, None, :] > at[:, :, None] - c["window"]
    v = torch.where((key[None, :] < s["lengths"][:, None])[:, None, :, None], v, torch.zeros((), device="cuda"))
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(dim))
    scores = scores.reshape(n, heads, chunk, shared, keys).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    most = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(most > -math.inf, most, torch.zeros_like(most))).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.reshape(n, heads, chunk * shared, keys), v).reshape(n, heads, chunk, shared, dim) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 2, 1, 3, 4).reshape(n, chunk, heads * shared, dim)[s["sequence"], place]
    lse = (most + total.log())[..., 0].permute(0, 2, 1, 3).reshape(n, chunk, heads * shared)[s["sequence"], place]
    s["out"].copy_(out)
    s["lse"].copy_(lse)
    return s["out"], s["lse"]


def _plain_fork(s):
    c = s["case"]
    page, table, references = c["page"], s["table"], s["references"]
    parents, children = s["parents"].long(), s["children"].long()
    rows, old, lengths = table[parents], table[children], s["lengths"][parents]
    full = (lengths // page).long()[:, None]
    last = rows.gather(1, full)[:, 0]
    part = (lengths % page > 0) & (parents != children)
    free = torch.argsort((references > 0).int(), stable=True)[torch.cumsum(part, 0).clamp_min(1) - 1].to(torch.int32)
    source = torch.where(last >= 0, last, rows[:, 0])
    taken = torch.where(part, free, source)
    rows = rows.scatter(1, full, torch.where(part, free, last)[:, None])
    references.index_add_(0, old.clamp_min(0).flatten().long(), -(old >= 0).flatten().int())
    references.index_add_(0, rows.clamp_min(0).flatten().long(), (rows >= 0).flatten().int())
    table[children], s["lengths"][children] = rows, lengths
    s["status"].zero_()
    held = (torch.arange(page, device="cuda")[None, :] < (lengths % page)[:, None])[None, :, None, :, None]
    for x in (s["keys"], s["values"]):
        x[:, taken.long()] = torch.where(held, x[:, source.long()], x[:, taken.long()])
    return s["table"], s["lengths"], s["references"], s["status"], s["keys"], s["values"]


def _plain_compact(s):
    live = s["references"] > 0
    count = live.sum()
    ids = torch.arange(live.numel(), device="cuda")
    movers, holes = torch.nonzero(live & (ids >= count))[:, 0], torch.nonzero(~live & (ids < count))[:, 0]
    new = ids.to(torch.int32)
    new[movers] = holes.to(torch.int32)
    s["table_out"].copy_(torch.where(s["table"] >= 0, new[s["table"].clamp_min(0).long()], s["table"]))
    s["references_out"].copy_(s["references"])
    s["references_out"][holes] = s["references"][movers]
    s["references_out"][movers] = 0
    s["live"].copy_(count)
    for x in (s["keys"], s["values"]):
        x[:, holes] = x[:, movers]
    return s["table_out"], s["references_out"], s["live"], s["keys"], s["values"]


RUN_OWN = {"rotate": _own_rotate, "append": _own_append, "attend": _own_attend, "fork": _own_fork, "compact": _own_compact}
RUN_PLAIN = {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend, "fork": _plain_fork, "compact": _plain_compact}


# ---- what a pass cannot do without --------------------------------------------------------------------------------


def _spread(low, high, count):
    return [low + i * (high - low) // (count - 1) for i in range(count)] if count > 1 else [high]


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "rotate":
        values = case["tokens"] * case["heads"] * case["dim"]
        pairs = case["tokens"] * case["dims"] // 2
        return {"bytes": 2 * values * size + 8 * min(pairs, case["positions"] * case["dims"] // 2) + 4 * case["tokens"], "flops": 6 * pairs * case["heads"]}
    if case["op"] in ("append", "attend"):
        new, old = (_spread(case[x + "_least"], case[x + "_most"], case["sequences"]) for x in ("new", "old"))
        tokens, queries = sum(new), case["heads"] * case["shared"]
        if case["op"] == "append":
            moved = 2 * tokens * (queries + 2 * case["heads"]) * case["dim"] * size
            return {"bytes": moved + tokens * (4 * case["dims"] + 4), "flops": 3 * tokens * case["dims"] * (queries + case["heads"])}
        window = case["window"] or (1 << 40)
        # (the order of the chunks and that of what lies in front of them are drawn apart: means of both)
        pairs = held = 0.0
        for o in old:
            for m in new:
                # sum over i of min(o + i + 1, window)
                grows = max(0, min(m, window - o))
                pairs += (grows * o + grows * (grows + 1) / 2 + (m - grows) * window) / len(old)
                held += min(o + m, window + m - 1) / len(old)
        kv = 2 * held * case["heads"] * case["dim"] * size
        return {"bytes": kv + 2 * tokens * queries * case["dim"] * size + 4 * tokens * queries, "flops": 4 * pairs * queries * case["dim"]}
    token = 2 * case["layers"] * case["heads"] * case["dim"] * size
    if case["op"] == "fork":
        lengths, n = _spread(case["length_least"], case["length_most"], case["groups"]), case["groups"] * case["beams"]
        # a beam stays where it is with probability 1 / beams
        copied = sum(x % case["page"] for x in lengths) * (case["beams"] - 1)
        table = 2 * 4 * case["beams"] * sum(-(-x // case["page"]) for x in lengths)
        return {"bytes": 2 * copied * token + table + 16 * n, "flops": 0}
    held, total = [], 0
    for x in _spread(case["length_least"], case["length_most"], case["sequences"]):
        total += -(-x // case["page"])
        if total <= case["pages"]:
            held.append(-(-x // case["page"]))
    live, pages = sum(held), case["pages"]
    moved = live * (pages - live) / pages
    table = 2 * 4 * case["sequences"] * max(held + [1])
    return {"bytes": 2 * moved * case["page"] * token + table + 2 * 4 * pages, "flops": 0}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------


def _exact_turn(x, table, positions, dims, interleaved, sign):
    y = x.double().clone()
    for i in range(dims // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + dims // 2)
        c, t = table[positions, i, 0].double()[:, None], sign * table[positions, i, 1].double()[:, None]
        y[:, :, a] = x[:, :, a].double() * c - x[:, :, b].double() * t
        y[:, :, b] = x[:, :, a].double() * t + x[:, :, b].double() * c
    return y


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "rotate":
        return _exact_turn(s["x"], s["table"], s["positions"].long(), case["dims"], case["interleaved"], -1.0 if case["backward"] else 1.0)
    if op == "append":
        at = s["position"]
        q, k = (_exact_turn(s[x], s["angles"], at, case["dims"], case["interleaved"], 1.0) for x in ("q", "k"))
        keys, values = s["keys"].double(), s["values"].double()
        page = s["table"][s["sequence"], at // case["page"]].long()
        keys[0][page, :, at % case["page"]] = k
        values[0][page, :, at % case["page"]] = s["v"].double()
        return q, keys, values
    if op == "attend":
        out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
        starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
        for b in range(case["sequences"]):
            t0, t1, length = starts[b], starts[b + 1], lengths[b]
            where = torch.arange(length - (t1 - t0), length, device="cuda")
            first = max(0, length - (t1 - t0) - case["window"] + 1) if case["window"] else 0
            key = torch.arange(first, length, device="cuda")
            hidden = key[None, :] > where[:, None]
            if case["window"]:
                hidden |= where[:, None] - key[None, :] >= case["window"]
            ids, slots = s["table"][b][key // case["page"]].long(), key % case["page"]
            for h in range(case["heads"]):
                k, v = s["keys"][0][ids, h, slots].double(), s["values"][0][ids, h, slots].double()
                for r in range(h * case["shared"], (h + 1) * case["shared"]):
                    logits = (s["q"][t0:t1, r].double() @ k.T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
                    lse[t0:t1, r] = torch.logsumexp(logits, -1)
                    out[t0:t1, r] = torch.softmax(logits, -1) @ v
        return out, lse
    keys, values = s["keys"].double(), s["values"].double()
    if op == "fork":
        # by the beams' own rows, one at a time
        table, references, page = s["table"].cpu(), s["references"].cpu(), case["page"]
        free = [i for i in range(references.numel()) if references[i] == 0]
        for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
            length = int(s["lengths"][parent])
            if parent == child or length % page == 0:
                continue
            source, to = int(table[parent][length // page]), free.pop(0)
            for x in (keys, values):
                x[:, to, :, : length % page] = x[:, source, :, : length % page].clone()
        return None, None, None, None, keys, values
    references = s["references"].cpu()
    live = int((references > 0).sum())
    holes = [i for i in range(live) if references[i] == 0]
    for to, source in zip(holes, [i for i in range(live, references.numel()) if references[i] > 0]):
        keys[:, to], values[:, to] = keys[:, source].clone(), values[:, source].clone()
    return None, None, None, keys, values
