"""Calls of a block-sparse serving step over the paged KV pool: append, index, select, attend.

A model that reads only the blocks of its context that a cheap score selects does four things a layer: it rotates the
new tokens' queries and keys by their positions and puts K and V into the pool's pages; it puts a small 8-bit index key
of each new token beside them; it scores every block of a request's context with index queries against those keys and
takes the Top-K blocks; and it attends to the tokens of those blocks. Each case below is one of those calls, on buffers
that a serving loop keeps.

listed() names the cases, draw() gives others of the same ranges; prepare() builds what the caller holds before the
call, run() makes one pass, work() states what a pass cannot do without, exact() gives its outputs in 64 bits. With
`own` false, run() computes the operators in plain form, in 32 bits from elementary torch operations; angles and the
quotients that are rounded to 8 bits are taken in 64.

The index scores are numbers of 32 bits by their definition, so that a selection is the same wherever it is made: whole
products, summed without a rounding, times a key's scale (rounded), the largest of a block's tokens, times the query
head's scale (rounded), the largest of a group's heads.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
_PACKAGE = Path(__file__).resolve().parents[1] / "elastic-kv-vmm_amd"
_NO_SCORE = float("-inf")


def listed():
    return [
        # One layer of a decode step of 128 requests: one token each, at positions up to 65536. Latency is all.
        {"name": "append_decode", "kind": "append", "dtype": "bfloat16", "batch": 128, "added": 1, "context": 65536,
         "page": 16, "layout": "planes", "heads": 16, "kv_heads": 2, "dim": 128, "rotary": 128, "pairs": "half",
         "scaling": "none", "factor": 1.0, "fused": True, "padded": 0},
        # Prompt pieces of up to 4096 tokens far into long contexts, their frequencies scaled for those; 0.2 GB of
        # queries in, as much out.
        {"name": "append_prompts", "kind": "append", "dtype": "bfloat16", "batch": 8, "added": 4096,
         "context": 1000000, "page": 64, "layout": "blocks", "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "pairs": "half", "scaling": "ramp", "factor": 32.0, "fused": True, "padded": 0},
        # Neighbouring elements as pairs, a part of an odd head rotated, float16, places behind the last token.
        {"name": "append_part", "kind": "append", "dtype": "float16", "batch": 11, "added": 301, "context": 8192,
         "page": 1, "layout": "planes", "heads": 12, "kv_heads": 4, "dim": 80, "rotary": 24, "pairs": "neighbours",
         "scaling": "linear", "factor": 4.0, "fused": False, "padded": 37},
        # The index keys of a decode step's tokens: 16 KB in.
        {"name": "index_decode", "kind": "index", "dtype": "bfloat16", "tokens": 128, "page": 16, "dim": 64},
        # The index keys of a batch of prompts.
        {"name": "index_prompts", "kind": "index", "dtype": "bfloat16", "tokens": 50000, "page": 64, "dim": 128},
        # The smallest selection: four requests of up to 8192 tokens, 16 blocks of 128 (the lookup microbenchmark's).
        {"name": "select_small", "kind": "select", "dtype": "bfloat16", "batch": 4, "query": 1, "context": 8192,
         "page": 16, "layout": "planes", "block": 128, "chosen": 16, "heads": 4, "groups": 1, "dim": 128, "first": 1,
         "last": 1},
        # One layer of the largest decode batch, a list for each of 2 KV heads: 5.2 million index keys.
        {"name": "select_step", "kind": "select", "dtype": "bfloat16", "batch": 128, "query": 1, "context": 65536,
         "page": 16, "layout": "planes", "block": 64, "chosen": 32, "heads": 8, "groups": 2, "dim": 128, "first": 1,
         "last": 2},
        # Top-K tokens instead of blocks: 2048 of up to 40000, what the resident lookup takes with blocks of one.
        {"name": "select_tokens", "kind": "select", "dtype": "float16", "batch": 24, "query": 1, "context": 40000,
         "page": 64, "layout": "blocks", "block": 1, "chosen": 2048, "heads": 4, "groups": 1, "dim": 64, "first": 0,
         "last": 1},
        # Prompt pieces of up to 1024 tokens, each token with its own selection: large whole-number products.
        {"name": "select_prompts", "kind": "select", "dtype": "bfloat16", "batch": 6, "query": 1024, "context": 16384,
         "page": 16, "layout": "planes", "block": 128, "chosen": 16, "heads": 4, "groups": 2, "dim": 128, "first": 1,
         "last": 1},
        # The smallest attention over blocks: four requests.
        {"name": "blocks_small", "kind": "blocks", "dtype": "bfloat16", "batch": 4, "query": 1, "context": 8192,
         "page": 16, "layout": "planes", "block": 128, "chosen": 4, "lists": 1, "heads": 16, "kv_heads": 2,
         "dim": 128, "lse": True},
        # One layer of the largest decode batch: 2048 tokens in 32 blocks of 64 for each KV head.
        {"name": "blocks_step", "kind": "blocks", "dtype": "bfloat16", "batch": 128, "query": 1, "context": 65536,
         "page": 16, "layout": "planes", "block": 64, "chosen": 32, "lists": 2, "heads": 16, "kv_heads": 2,
         "dim": 128, "lse": False},
        # Prompt pieces of up to 512 tokens, each token with its own blocks, most of them its neighbours' too.
        {"name": "blocks_prompts", "kind": "blocks", "dtype": "bfloat16", "batch": 4, "query": 512, "context": 16384,
         "page": 16, "layout": "planes", "block": 128, "chosen": 16, "lists": 2, "heads": 16, "kv_heads": 2,
         "dim": 128, "lse": True},
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def _reduced(case, size, measure, largest):
    """The case with one of its sizes made smaller until its work is no more than that of the listed case."""
    limit = work(next(c for c in listed() if c["name"] == largest))[measure]
    while work(case)[measure] > limit and case[size] > 1:
        case[size] = max(1, case[size] * 3 // 4)
    return case


def draw(rng):
    kind = rng.choice(["append", "append", "index", "select", "select", "select", "blocks", "blocks", "blocks"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    page = rng.choice([1, 16, 16, 64, 100])
    layout = rng.choice(["planes", "planes", "blocks"])
    if kind == "append":
        kv_heads = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        scaling = rng.choice(["none", "none", "linear", "base", "ramp"])
        case = {"kind": kind, "dtype": dtype, "batch": _log(rng, 1, 256), "added": _log(rng, 1, 4096),
                "context": _log(rng, 64, 1000000), "page": page, "layout": layout,
                "heads": kv_heads * rng.choice([1, 2, 4, 8]), "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2, 24]), "pairs": rng.choice(["half", "half", "neighbours"]),
                "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]),
                "fused": rng.random() < 0.5, "padded": rng.choice([0, 0, rng.randint(1, 100)])}
        return _reduced(_reduced(case, "added", "bytes", "append_prompts"), "batch", "bytes", "append_prompts")
    if kind == "index":
        case = {"kind": kind, "dtype": dtype, "tokens": _log(rng, 1, 100000), "page": page,
                "dim": rng.choice([32, 64, 128, 128, 256])}
        return _reduced(case, "tokens", "bytes", "index_prompts")
    query = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 16, 1024)])
    context = query + _log(rng, 2048 if kind == "select" else 16, 65536)
    if kind == "select":
        groups = rng.choice([1, 1, 2, 4])
        block = rng.choice([1, 4, 16, 64, 64, 100, 128, 128]) if query <= 8 else rng.choice([16, 32, 64, 128])
        chosen = rng.choice([512, 2048]) if block <= 4 else rng.choice([4, 8, 16, 17, 32, 64])
        case = {"kind": kind, "dtype": dtype, "batch": _log(rng, 1, 128), "query": query, "context": context,
                "page": page, "layout": layout, "block": block, "chosen": chosen,
                "heads": groups * rng.choice([1, 2, 4]), "groups": groups, "dim": rng.choice([32, 64, 128, 128]),
                "first": rng.choice([0, 1, 2]), "last": rng.choice([0, 1, 2])}
        case = _reduced(_reduced(case, "batch", "flops", "select_prompts"), "query", "flops", "select_prompts")
        # A selection leaves half of the longest context's blocks out, or there would be nothing to choose.
        case["chosen"] = max(4, min(chosen, case["context"] // block // 2))
        case["first"] = min(case["first"], case["chosen"] // 8)
        return _reduced(case, "batch", "bytes", "select_step")
    kv_heads = rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "dtype": dtype, "batch": _log(rng, 1, 128), "query": min(query, 512), "context": context,
            "page": page, "layout": layout, "block": rng.choice([16, 32, 64, 64, 100, 128]),
            "chosen": rng.choice([1, 4, 8, 16, 17, 32]), "lists": rng.choice([1, kv_heads]),
            "heads": kv_heads * rng.choice([1, 2, 4, 8, 8, 16]), "kv_heads": kv_heads,
            "dim": rng.choice([64, 80, 96, 128, 128, 256]), "lse": rng.random() < 0.5}
    case = _reduced(_reduced(case, "batch", "flops", "blocks_prompts"), "query", "flops", "blocks_prompts")
    # A selected token is read for every query token by the plain form, so its rows are bounded too.
    while case["query"] * case["batch"] * case["chosen"] * case["block"] * case["kv_heads"] * case["dim"] > 2 ** 30:
        case["batch" if case["batch"] > 1 else "query"] //= 2
    return _reduced(case, "batch", "bytes", "blocks_step")


# ---------------------------------------------------------------- sizes that follow from a case


def _spread(batch, low, high):
    """Ragged whole numbers between low and high, the highest among them: what work() and prepare() both go by."""
    if batch == 1:
        return [high]
    step = 0.6180339887498949
    return [high] + [low + int((high - low) * ((i * step) % 1.0)) for i in range(1, batch)]


def _sizes(case):
    """(query tokens, tokens in all) of every batch row: the new tokens are the last ones."""
    batch, query = case["batch"], case["added" if case["kind"] == "append" else "query"]
    tokens = [1] * batch if query == 1 else _spread(batch, max(1, query // 2), query)
    context = max(case["context"], query)
    lengths = _spread(batch, max(1, context // 4), context)
    return tokens, [max(n, t) for n, t in zip(lengths, tokens)]


def _seen_in_blocks(case, position):
    """Tokens that a query token at this position sees through a full list that holds its newest block."""
    block = case["block"]
    count = min(case["chosen"], position // block + 1)
    return (count - 1) * block + position % block + 1


def work(case):
    """Bytes of each input read once and each output written once; multiplications and additions of the products."""
    kind = case["kind"]
    if kind == "index":
        return {"bytes": case["tokens"] * (3 * case["dim"] + 8), "flops": 0}
    tokens, lengths = _sizes(case)
    total = sum(tokens)
    if kind == "append":
        rows = total * case["dim"] * 2 * 2
        return {"bytes": rows * (case["heads"] + 2 * case["kv_heads"]) + 8 * total, "flops": 0}
    tables = 4 * sum(-(-n // case["page"]) for n in lengths)
    if kind == "select":
        pairs = sum(t * n - t * (t - 1) // 2 for t, n in zip(tokens, lengths))
        return {"bytes": sum(lengths) * (case["dim"] + 4) + tables + total * case["heads"] * case["dim"] * 2
                + 4 * total * case["groups"] * case["chosen"], "flops": 2 * pairs * case["heads"] * case["dim"]}
    seen = [[_seen_in_blocks(case, n - t + i) for i in range(t)] for t, n in zip(tokens, lengths)]
    row = case["kv_heads"] * case["dim"] * 2 * 2
    read = sum(min(n, sum(s)) for n, s in zip(lengths, seen))
    stats = 4 * case["heads"] if case["lse"] else 0
    return {"bytes": read * row + 4 * total * case["lists"] * case["chosen"]
            + total * (case["heads"] * case["dim"] * 4 + stats),
            "flops": 4 * sum(map(sum, seen)) * case["heads"] * case["dim"]}


def _frequencies(case):
    """Radians a position of every pair, and the factor of the rotated parts."""
    size, base, factor = case["rotary"], 10000.0, case["factor"]
    if case["scaling"] == "base":
        base *= factor ** (size / (size - 2))
    plain = [base ** (-2 * i / size) for i in range(size // 2)]
    if case["scaling"] == "linear":
        return [f / factor for f in plain], 1.0
    if case["scaling"] != "ramp":
        return plain, 1.0
    # Pairs that turn more than 32 times in the original 32768 positions keep their frequency, those that turn less
    # than once are slowed by the factor, the others lie between.
    place = [size * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
    low, high = max(math.floor(place[0]), 0), min(math.ceil(place[1]), size - 1)
    slow = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(size // 2)]
    return [f * (1 - s) + f / factor * s for f, s in zip(plain, slow)], 0.1 * math.log(factor) + 1.0


# ---------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _shuffled(values, gen):
    """The ragged sizes in another order for every seed (the first place keeps the largest)."""
    order = torch.randperm(len(values) - 1, generator=gen, device=DEVICE).tolist() if len(values) > 1 else []
    return [values[0]] + [values[1 + i] for i in order]


def _cache(gen, dtype, layout, pages, page, kv_heads, dim):
    """The pool's memory and its keys and values as [pages, page, kv_heads, dim] views.

    planes: one plane of token rows for K and one for V; blocks: a page's planes of two layers lie together, and the
    second layer is read."""
    if layout == "planes":
        pool = torch.empty((1, 2, pages, page, kv_heads, dim), dtype=dtype, device=DEVICE).normal_(generator=gen)
        return pool, pool[0, 0], pool[0, 1]
    pool = torch.empty((pages, 2, 2, page, kv_heads, dim), dtype=dtype, device=DEVICE).normal_(generator=gen)
    return pool, pool[:, 1, 0], pool[:, 1, 1]


def _batch(case, gen):
    """Lengths, query tokens and their rows: what a step knows of its batch, as lists and as tensors."""
    tokens, lengths = _sizes(case)
    order = list(zip(tokens, lengths))
    order = _shuffled(order, gen)
    tokens, lengths = [t for t, _ in order], [n for _, n in order]
    counts = _int(tokens, torch.int64)
    row = torch.repeat_interleave(torch.arange(len(tokens), device=DEVICE), counts, output_size=sum(tokens))
    starts = torch.cumsum(counts, 0) - counts
    at = torch.arange(sum(tokens), device=DEVICE) - starts[row]
    position = (_int(lengths, torch.int64) - counts)[row] + at
    return {"tokens": tokens, "sizes": lengths, "lengths": _int(lengths), "row": row, "at": at, "position": position,
            "most": max(tokens), "widest": max(lengths), "page": case["page"], "layout": case["layout"],
            "query_starts": None if max(tokens) == 1 else torch.cat([starts, starts[-1:] + counts[-1:]]).int()}


def _tables(s, gen):
    """Pages of all rows in random order (page 0 is the sink and belongs to nobody), requests in another order."""
    page, lengths = s["page"], s["sizes"]
    batch = len(lengths)
    held = [-(-n // page) for n in lengths]
    s["pages"] = 1 + sum(held)
    order = torch.randperm(s["pages"] - 1, generator=gen, device=DEVICE).to(torch.int32) + 1
    s["rows"] = torch.randperm(batch, generator=gen, device=DEVICE)
    held = _int(held, torch.int64)
    first = torch.cumsum(held, 0) - held
    column = torch.arange(int(held.max()) + 1, device=DEVICE).view(1, -1)
    s["tables"] = torch.zeros((batch, column.shape[1]), dtype=torch.int32, device=DEVICE)
    mine = column < held.view(-1, 1)
    s["tables"][s["rows"]] = torch.where(mine, order[(first.view(-1, 1) + column).clamp_max(len(order) - 1)], 0)


def _append_inputs(case, seed):
    gen = _generator(seed)
    dtype = getattr(torch, case["dtype"])
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    s = _batch(case, gen)
    total, padded = len(s["row"]), case["padded"]
    # The pages that the new tokens touch, each a place of its own in the pool.
    counts = _int(s["tokens"], torch.int64)
    begin = (s["lengths"].long() - counts) // page
    touched = (s["lengths"].long() - 1) // page - begin + 1
    first = torch.cumsum(touched, 0) - touched
    pages = 1 + int(touched.sum()) + 16
    order = torch.randperm(pages - 1, generator=gen, device=DEVICE) + 1
    slots = order[first[s["row"]] + s["position"] // page - begin[s["row"]]] * page + s["position"] % page
    blank = torch.full((padded,), -1, dtype=torch.int64, device=DEVICE)
    pool, keys, values = _cache(gen, dtype, case["layout"], pages, page, kv_heads, dim)
    if case["fused"]:
        # One projection's output: queries, keys and values of a token side by side.
        both = torch.randn((total + padded, heads + 2 * kv_heads, dim), generator=gen, device=DEVICE).to(dtype)
        query, key, value = both.split([heads, kv_heads, kv_heads], 1)
    else:
        query, key, value = (torch.randn((total + padded, n, dim), generator=gen, device=DEVICE).to(dtype)
                             for n in (heads, kv_heads, kv_heads))
    output = torch.zeros((total + padded, heads, dim), dtype=dtype, device=DEVICE)
    frequencies, magnitude = _frequencies(case)
    return {"kind": "append", "query": query, "key": key, "value": value, "pool": pool, "keys": keys,
            "values": values, "page": page, "layout": case["layout"], "output": output, "magnitude": magnitude,
            "positions": torch.cat([s["position"], blank]).int(), "slots": torch.cat([slots, blank]).int(),
            "neighbours": case["pairs"] == "neighbours", "rotary_dim": case["rotary"],
            "frequencies": _int(frequencies, torch.float64),
            "making": {"rotary_dim": case["rotary"], "scaling": None if case["scaling"] == "none" else case["scaling"],
                       "factor": case["factor"], "original": 32768, "interleaved": case["pairs"] == "neighbours"}}


def _index_inputs(case, seed):
    gen = _generator(seed)
    dtype, tokens, page, dim = getattr(torch, case["dtype"]), case["tokens"], case["page"], case["dim"]
    pages = 17 + -(-tokens // page)
    order = torch.randperm(pages - 1, generator=gen, device=DEVICE) + 1
    token = torch.arange(tokens, device=DEVICE)
    # Keys of unlike sizes, as tokens have them.
    size = torch.exp(0.5 * torch.randn((tokens, 1), generator=gen, device=DEVICE))
    return {"kind": "index", "page": page, "layout": "planes",
            "index_key": (torch.randn((tokens, dim), generator=gen, device=DEVICE) * size).to(dtype),
            "slots": (order[token // page] * page + token % page).int(),
            "pool": torch.zeros((pages, page, dim), dtype=torch.int8, device=DEVICE),
            "scales": torch.zeros(pages * page, dtype=torch.float32, device=DEVICE)}


def _select_inputs(case, seed):
    gen = _generator(seed)
    dtype, page, dim = getattr(torch, case["dtype"]), case["page"], case["dim"]
    s = _batch(case, gen)
    _tables(s, gen)
    pool = torch.empty((s["pages"], page, dim), dtype=torch.float16, device=DEVICE).normal_(0, 40, generator=gen)
    scales = torch.exp(0.3 * torch.randn(s["pages"] * page, generator=gen, device=DEVICE)) * 0.02
    total = len(s["row"])
    s.update(kind="select", pool=pool.round().clamp(-127, 127).to(torch.int8), scales=scales, block=case["block"],
             first=case["first"], last=case["last"],
             index_query=torch.randn((total, case["heads"], dim), generator=gen, device=DEVICE).to(dtype),
             blocks=torch.empty((total, case["groups"], case["chosen"]), dtype=torch.int32, device=DEVICE))
    return s


def _blocks_inputs(case, seed):
    gen = _generator(seed)
    dtype, page = getattr(torch, case["dtype"]), case["page"]
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    s = _batch(case, gen)
    _tables(s, gen)
    pool, keys, values = _cache(gen, dtype, case["layout"], s["pages"], page, kv_heads, dim)
    total, lists, chosen = len(s["row"]), case["lists"], case["chosen"]
    # Selections as scores give them: some blocks matter to all of a request's tokens, others come and go over some tens
    # of tokens. The newest block is always there.
    newest = s["position"] // block
    count = int(newest.max()) + 1
    common = torch.randn((len(s["tokens"]), lists, count), generator=gen, device=DEVICE)
    steps = torch.randn((s["most"] // 32 + 2, lists, count), generator=gen, device=DEVICE)
    part = ((s["at"] % 32).float() / 32).view(-1, 1, 1)
    score = common[s["row"]] + steps[s["at"] // 32] * (1 - part) + steps[s["at"] // 32 + 1] * part
    block_id = torch.arange(count, device=DEVICE).view(1, 1, -1)
    score = torch.where(block_id == newest.view(-1, 1, 1), 100.0, score)
    score = torch.where(block_id > newest.view(-1, 1, 1), _NO_SCORE, score)
    best, found = torch.topk(score, min(chosen, count), dim=-1)
    found = torch.where(best == _NO_SCORE, count, found).sort(-1).values
    blocks = torch.full((total, lists, chosen), -1, dtype=torch.int32, device=DEVICE)
    blocks[..., :found.shape[-1]] = torch.where(found == count, -1, found)
    # Scores of a standard deviation of two: a few keys carry most of a row's weight.
    query = (torch.randn((total, heads, dim), generator=gen, device=DEVICE) * 2).to(dtype)
    s.update(kind="blocks", pool=pool, keys=keys, values=values, kv_heads=kv_heads, block=block, blocks=blocks,
             query=query, scale=dim ** -0.5, output=torch.empty((total, heads, dim), dtype=dtype, device=DEVICE),
             lse=torch.empty((total, heads), dtype=torch.float32, device=DEVICE) if case["lse"] else None)
    return s


def _inputs(case, seed):
    return {"append": _append_inputs, "index": _index_inputs, "select": _select_inputs,
            "blocks": _blocks_inputs}[case["kind"]](case, seed)


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        _prepare_own(state)
    return state


def _prepare_own(s):
    """The pool's description, the rotation and the workspace that a serving loop keeps."""
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    from adaptive_sparse import append, attention, block_selection
    from adaptive_sparse.kv_pool import KVPlanes

    pool, page, layer = s["pool"], s["page"], 0
    if s["kind"] in ("index", "select"):
        pages, _, row = pool.shape
        if s["layout"] == "planes":
            sizes = dict(layers=1, kv=1, row_stride=row, row_bytes=row, rows=pages * page)
        else:
            sizes = dict(layers=1, kv=1, row_stride=row * page, row_bytes=row * page, rows=pages)
        sizes.update(layer_stride=pages * page * row, kv_stride=pages * page * row)
    else:
        pages, _, kv_heads, dim = s["keys"].shape
        row = kv_heads * dim * 2
        plane = pages * page * row
        if s["layout"] == "planes":
            sizes = dict(layers=1, kv=2, layer_stride=2 * plane, kv_stride=plane, row_stride=row, row_bytes=row,
                         rows=pages * page)
        else:
            row *= page
            layer = 1
            sizes = dict(layers=2, kv=2, layer_stride=2 * row, kv_stride=row, row_stride=4 * row, row_bytes=row,
                         rows=pages)
    s["layer"] = layer
    s["planes"] = KVPlanes(base=pool.data_ptr(), device=pool.device.index, owner=pool, **sizes)
    if s["kind"] == "append":
        s["call"] = append.append_rotary
        s["rotary"] = append.make_rotary(device=pool.device, **s["making"])
    elif s["kind"] == "index":
        s["call"] = append.append_index
    elif s["kind"] == "select":
        s["call"] = block_selection.select_blocks
        tokens, groups, _ = s["blocks"].shape
        size = block_selection.selection_workspace(tokens, groups, s["tables"].shape[1], page, s["block"])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEVICE)
    else:
        s["call"] = attention.block_attention
        tokens, heads, dim = s["query"].shape
        size = attention.block_workspace(tokens, s["blocks"].shape[2], s["block"], heads, s["kv_heads"], dim,
                                         s["most"])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEVICE)


# ---------------------------------------------------------------- one pass


def run(state):
    if own:
        return _OWN[state["kind"]](state)
    return _PLAIN[state["kind"]](state)


def _attention_outputs(s):
    return [s["output"]] if s["lse"] is None else [s["output"], s["lse"]]


def _own_append(s):
    s["call"](s["query"], s["key"], s["value"], s["planes"], s["slots"], s["positions"], s["rotary"], s["output"],
              page_size=s["page"], layer=s["layer"])
    return [s["output"], s["pool"]]


def _own_index(s):
    s["call"](s["index_key"], s["planes"], s["scales"], s["slots"], page_size=s["page"], layer=s["layer"])
    return [s["pool"], s["scales"]]


def _own_select(s):
    s["call"](s["index_query"], s["planes"], s["scales"], s["tables"], s["rows"], s["lengths"], s["blocks"],
              page_size=s["page"], block_size=s["block"], layer=s["layer"], query_starts=s["query_starts"],
              max_query=s["most"], first=s["first"], last=s["last"], workspace=s["workspace"])
    return [s["blocks"]]


def _own_blocks(s):
    s["call"](s["query"], s["planes"], s["tables"], s["rows"], s["lengths"], s["blocks"], s["output"],
              page_size=s["page"], block_size=s["block"], kv_heads=s["kv_heads"], layer=s["layer"],
              query_starts=s["query_starts"], max_query=s["most"], scale=s["scale"], lse=s["lse"],
              workspace=s["workspace"])
    return _attention_outputs(s)


_OWN = {"append": _own_append, "index": _own_index, "select": _own_select, "blocks": _own_blocks}


def _plain_append(s):
    size, page = s["rotary_dim"], s["page"]
    live = s["positions"] >= 0
    angle = s["positions"].double().view(-1, 1) * s["frequencies"]
    cos = (torch.cos(angle) * s["magnitude"]).float().unsqueeze(1)
    sin = (torch.sin(angle) * s["magnitude"]).float().unsqueeze(1)

    def rotated(x):
        y = x.float()
        if s["neighbours"]:
            a, b = y[..., 0:size:2], y[..., 1:size:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :size // 2], y[..., size // 2:size]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, y[..., size:]], -1).to(x.dtype)

    s["output"].copy_(torch.where(live.view(-1, 1, 1), rotated(s["query"]), s["output"]))
    slot = s["slots"][live].long()
    s["keys"][slot // page, slot % page] = rotated(s["key"])[live]
    s["values"][slot // page, slot % page] = s["value"][live]
    return [s["output"], s["pool"]]


def _codes(x):
    """Rows of 8-bit whole numbers and the scale of each: quotients rounded to 32 bits, halves to even."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True) / 127.0).float()
    quotient = (x / torch.where(scale > 0, scale, 1.0).double()).float()
    return torch.round(quotient), scale.squeeze(-1)


def _plain_index(s):
    codes, scale = _codes(s["index_key"])
    slot, page = s["slots"].long(), s["page"]
    s["pool"][slot // page, slot % page] = codes.to(torch.int8)
    s["scales"][slot] = scale
    return [s["pool"], s["scales"]]


def _plain_select(s):
    page, block, row, at, most = s["page"], s["block"], s["row"], s["at"], s["most"]
    total, groups, chosen = s["blocks"].shape
    heads, dim = s["index_query"].shape[1:]
    batch, width = len(s["sizes"]), -(-s["widest"] // block) * block
    codes, scale = _codes(s["index_query"])
    q = codes.new_zeros((batch, most, heads, dim))
    q[row, at] = codes
    token = torch.arange(width, device=DEVICE)
    pages = s["tables"][s["rows"]][:, (token // page).clamp_max(s["tables"].shape[1] - 1)].long()
    inside = (token % page).view(1, -1).expand_as(pages)
    keys = s["pool"][pages, inside].float().transpose(1, 2).contiguous()
    scores = torch.matmul(q.view(batch, most * heads, dim), keys).view(batch, most, heads, width)
    scores = scores * s["scales"].view(-1, page)[pages, inside].view(batch, 1, 1, width)
    last = s["lengths"].long().view(-1, 1) - torch.bincount(row, minlength=batch).view(-1, 1)
    last = last + torch.arange(most, device=DEVICE).view(1, -1)
    seen = (token.view(1, 1, -1) <= last.unsqueeze(-1)) & (pages >= 1).unsqueeze(1)
    scores = scores.masked_fill(~seen.unsqueeze(2), _NO_SCORE)
    scores = scores.view(batch, most, heads, -1, block).amax(-1)[row, at] * scale.unsqueeze(-1)
    scores = torch.where(scores.isnan(), _NO_SCORE, scores)        # nothing seen, times a scale of 0
    scores = scores.view(total, groups, heads // groups, -1).amax(2)
    block_id = torch.arange(scores.shape[-1], device=DEVICE)
    newest = (s["position"] // block).view(-1, 1)
    forced = (block_id < s["first"]) | ((block_id > newest - s["last"]) & (block_id <= newest))
    scores = torch.where(forced.unsqueeze(1) & (scores > _NO_SCORE), math.inf, scores)
    best, order = torch.sort(scores, dim=-1, descending=True, stable=True)
    best, order = best[..., :chosen], order[..., :chosen]
    none = len(block_id)
    found = torch.where(best > _NO_SCORE, order, none).sort(-1).values
    s["blocks"].fill_(-1)
    s["blocks"][..., :found.shape[-1]] = torch.where(found == none, -1, found)
    return [s["blocks"]]


def _plain_blocks(s):
    page, block, kv_heads = s["page"], s["block"], s["kv_heads"]
    total, heads, dim = s["query"].shape
    lists = s["blocks"].shape[1]
    each = kv_heads // lists
    blocks = s["blocks"].long().unsqueeze(-1)
    token = blocks * block + torch.arange(block, device=DEVICE)
    seen = (blocks >= 0) & (token <= s["position"].view(-1, 1, 1, 1))
    token = torch.where(seen, token, 0).view(total, lists, -1)
    pages = torch.gather(s["tables"][s["rows"][s["row"]]].long().unsqueeze(1).expand(-1, lists, -1), 2, token // page)
    seen = seen.view(total, lists, -1) & (pages >= 1)
    which = torch.arange(lists, device=DEVICE).view(1, -1, 1)

    def read(cache):
        return cache.unflatten(2, (lists, each))[pages, token % page, which].float()       # [N, lists, T, each, D]

    query = (s["query"].float() * s["scale"]).view(total, lists, each, heads // kv_heads, dim)
    scores = torch.matmul(query, read(s["keys"]).permute(0, 1, 3, 4, 2).contiguous())
    scores = scores.masked_fill(~seen.view(total, lists, 1, 1, -1), _NO_SCORE)
    top = scores.amax(-1, keepdim=True)
    safe = torch.where(top == _NO_SCORE, 0.0, top)
    weights = torch.exp(scores - safe)
    mass = weights.sum(-1, keepdim=True)
    value = torch.matmul(weights, read(s["values"]).permute(0, 1, 3, 2, 4).contiguous())
    s["output"].copy_(torch.where(mass > 0, value / mass, 0.0).view(total, heads, dim))
    if s["lse"] is not None:
        s["lse"].copy_((torch.log(mass) + safe).view(total, heads))
    return _attention_outputs(s)


_PLAIN = {"append": _plain_append, "index": _plain_index, "select": _plain_select, "blocks": _plain_blocks}


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    """The outputs of run() for these inputs in 64 bits, one request after the other."""
    s = _inputs(case, seed)
    return {"append": _exact_append, "index": _exact_index, "select": _exact_select,
            "blocks": _exact_blocks}[case["kind"]](case, s)


def _exact_append(case, s):
    size = case["rotary"]
    half = size // 2
    first = torch.arange(half, device=DEVICE)
    first, second = (2 * first, 2 * first + 1) if case["pairs"] == "neighbours" else (first, first + half)
    angle = s["positions"].double().unsqueeze(1) * s["frequencies"].unsqueeze(0)
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle).unsqueeze(1)
    live = torch.nonzero(s["positions"] >= 0).squeeze(1)

    def rotated(x):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    output, pool = s["output"].double(), s["pool"].double()
    output[live] = rotated(s["query"])[live]
    keys, values = (pool[0, 0], pool[0, 1]) if case["layout"] == "planes" else (pool[:, 1, 0], pool[:, 1, 1])
    slot = s["slots"][live].long()
    at = (torch.div(slot, s["page"], rounding_mode="floor"), slot % s["page"])
    keys[at] = rotated(s["key"])[live]
    values[at] = s["value"][live].double()
    return [output, pool]


def _exact_codes(x):
    """As _codes, by way of the host's numbers of 32 bits."""
    x = x.cpu().numpy() if x.dtype == torch.float16 else x.float().cpu().numpy()
    x = x.astype("float32")
    scale = abs(x).max(-1, keepdims=True) / x.dtype.type(127)
    codes = (x / (scale + (scale == 0))).round()
    return torch.from_numpy(codes).to(DEVICE).double(), torch.from_numpy(scale[..., 0]).to(DEVICE).double()


def _exact_index(case, s):
    codes, scale = _exact_codes(s["index_key"])
    pool, scales = s["pool"].view(-1, case["dim"]), s["scales"].double()
    slot = s["slots"].long()
    pool[slot] = codes.to(torch.int8)
    scales[slot] = scale
    return [s["pool"], scales]


def _exact_select(case, s):
    page, block, groups, chosen = case["page"], case["block"], case["groups"], case["chosen"]
    if sum(t * n for t, n in zip(s["tokens"], s["sizes"])) * case["heads"] > 1 << 31:
        return None
    codes, scale = _exact_codes(s["index_query"])
    place, start = s["rows"].tolist(), 0
    keys, scales = s["pool"].view(-1, case["dim"]), s["scales"]
    for b, (count, length) in enumerate(zip(s["tokens"], s["sizes"])):
        position = torch.arange(length, device=DEVICE)
        slot = s["tables"][place[b]].long()[position // page] * page + position % page
        q = codes[start:start + count].reshape(-1, case["dim"])
        product = (q @ keys[slot].double().t().contiguous()).view(count, case["heads"], length)
        score = (product * scales[slot].double()).float()          # rounded to 32 bits by definition
        last = length - count + torch.arange(count, device=DEVICE).view(-1, 1)
        blocks = -(-length // block)
        score = score.masked_fill((position.view(1, -1) > last).unsqueeze(1), _NO_SCORE)
        score = torch.nn.functional.pad(score, (0, blocks * block - length), value=_NO_SCORE)
        score = score.view(count, case["heads"], blocks, block).amax(-1).double()
        score = (score * scale[start:start + count].unsqueeze(-1)).float()
        score = score.nan_to_num(nan=_NO_SCORE, neginf=_NO_SCORE, posinf=math.inf)
        score = score.view(count, groups, -1, blocks).amax(2)
        there = torch.arange(blocks, device=DEVICE).view(1, -1)
        newest = last // block
        forced = ((there < case["first"]) | (there > newest - case["last"])) & (there <= newest)
        score[forced.unsqueeze(1).expand_as(score) & (score > _NO_SCORE)] = math.inf
        # A block is chosen when fewer than `chosen` others stand before it.
        order = torch.argsort(-score, dim=-1, stable=True)
        rank = torch.argsort(order, dim=-1)
        take = (rank < chosen) & (score > _NO_SCORE)
        column = torch.cumsum(take, -1) - 1
        found = torch.full((count, groups, chosen + 1), -1, dtype=torch.int32, device=DEVICE)
        found.scatter_(2, torch.where(take, column, chosen), there.int().unsqueeze(1).expand_as(score).contiguous())
        s["blocks"][start:start + count] = found[..., :chosen]
        start += count
    return [s["blocks"]]


def _exact_blocks(case, s):
    page, block, heads, kv_heads = case["page"], case["block"], case["heads"], case["kv_heads"]
    share, lists = heads // kv_heads, case["lists"]
    if sum(t * n for t, n in zip(s["tokens"], s["sizes"])) * share > 1 << 30:
        return None
    outs, sums, start = [], [], 0
    place = s["rows"].tolist()
    for b, (count, length) in enumerate(zip(s["tokens"], s["sizes"])):
        pages = s["tables"][place[b]][:-(-length // page)].long()
        keys, values = (cache[pages].reshape(-1, kv_heads, case["dim"])[:length] for cache in (s["keys"], s["values"]))
        position = torch.arange(length, device=DEVICE)
        last = length - count + torch.arange(count, device=DEVICE).view(-1, 1)
        listed_here = s["blocks"][start:start + count].long()
        per_head = []
        for h in range(kv_heads):
            found = listed_here[:, h * lists // kv_heads]
            holds = torch.zeros((count, -(-length // block) + 1), dtype=torch.bool, device=DEVICE)
            holds.scatter_(1, torch.where(found < 0, holds.shape[1] - 1, found), True)
            holds[:, -1] = False
            seen = holds[:, position // block] & (position.view(1, -1) <= last)
            q = s["query"][start:start + count, h * share:(h + 1) * share].double().reshape(count * share, -1)
            scores = (q @ keys[:, h].double().t().contiguous() * s["scale"]).view(count, share, length)
            scores = scores.masked_fill(~seen.unsqueeze(1), _NO_SCORE)
            lse = torch.logsumexp(scores, -1)
            weights = torch.exp(scores - torch.where(lse == _NO_SCORE, 0.0, lse).unsqueeze(-1))
            per_head.append((torch.matmul(weights.view(count * share, -1), values[:, h].double())
                             .view(count, share, -1), lse))
        outs.append(torch.cat([o for o, _ in per_head], 1))
        sums.append(torch.cat([l for _, l in per_head], 1))
        start += count
    return [torch.cat(outs)] if s["lse"] is None else [torch.cat(outs), torch.cat(sums)]
