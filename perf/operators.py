"""Calls of the attention operators over the paged KV pool and of the block tables that feed them, over the range that
a server meets.

A serving step extends every request's block table by its new tokens, writes their K/V rows through the slot map, and
attends: to a prefix that a whole batch shares and each request's own pages, or to the Top-K slots that the resident
lookup returned. Each case below is one of those calls, on buffers that a serving loop keeps.

listed() names the cases, draw() gives others of the same ranges; prepare() builds what the caller holds before the
call, run() makes one pass, work() states what a pass cannot do without, exact() gives its outputs in 64 bits. With
`own` false, run() computes the operators in plain form, in 32 bits from elementary torch operations.
"""

import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
_PACKAGE = Path(__file__).resolve().parents[1] / "elastic-kv-vmm_amd"
_NO_SCORE = float("-inf")


def listed():
    return [
        # One decode step's block tables: 128 requests get one token each, one in sixteen a new page. Latency is all.
        {"name": "tables_decode", "kind": "tables", "batch": 128, "page": 16, "context": 65536, "added": 1,
         "decoding": 1.0},
        # A mixed batch: three quarters decode, the others bring ragged prompt pieces of up to 4096 tokens.
        {"name": "tables_mixed", "kind": "tables", "batch": 48, "page": 16, "context": 32768, "added": 4096,
         "decoding": 0.75},
        # Prompts only, up to 32768 tokens each: millions of slots and positions written.
        {"name": "tables_prompts", "kind": "tables", "batch": 251, "page": 64, "context": 4096, "added": 32768,
         "decoding": 0.0},
        # The smallest decode call: four requests behind a short common instruction. Latency counts.
        {"name": "prefix_small", "kind": "prefix", "dtype": "bfloat16", "batch": 4, "groups": 1, "heads": 16,
         "kv_heads": 2, "dim": 128, "page": 16, "prefix": 1024, "own": 64, "query": 1, "layout": "planes"},
        # An ordinary decode batch behind one system prompt with examples: the prefix is longer than what is own.
        {"name": "prefix_decode", "kind": "prefix", "dtype": "bfloat16", "batch": 32, "groups": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "prefix": 8192, "own": 1024, "query": 1, "layout": "planes"},
        # The largest decode batch, a shared document of 32768 tokens, own contexts of up to 4096.
        {"name": "prefix_step", "kind": "prefix", "dtype": "bfloat16", "batch": 128, "groups": 1, "heads": 16,
         "kv_heads": 2, "dim": 128, "page": 64, "prefix": 32768, "own": 4096, "query": 1, "layout": "planes"},
        # Seven prompts' groups of unlike sizes in one batch (sampling several answers to each), token pages, padded
        # batch rows that see nothing, float16.
        {"name": "prefix_groups", "kind": "prefix", "dtype": "float16", "batch": 91, "groups": 7, "heads": 32,
         "kv_heads": 8, "dim": 64, "page": 1, "prefix": 4096, "own": 1500, "query": 1, "layout": "planes",
         "lse": True},
        # Verification of drafted tokens: up to five query tokens a request, an odd head size, block-major pages.
        {"name": "prefix_verify", "kind": "prefix", "dtype": "bfloat16", "batch": 24, "groups": 2, "heads": 12,
         "kv_heads": 4, "dim": 96, "page": 128, "prefix": 5000, "own": 700, "query": 5, "layout": "blocks",
         "lse": True},
        # Prompt pieces of up to 1024 tokens behind a shared prompt: two large products a KV head, causal at the end.
        {"name": "prefix_prompts", "kind": "prefix", "dtype": "bfloat16", "batch": 8, "groups": 1, "heads": 16,
         "kv_heads": 2, "dim": 128, "page": 16, "prefix": 16384, "own": 4096, "query": 1024, "layout": "planes"},
        # The smallest Top-K read: a few requests, few lanes.
        {"name": "topk_small", "kind": "topk", "dtype": "bfloat16", "batch": 4, "lanes": 256, "heads": 16,
         "kv_heads": 2, "dim": 128},
        # One layer of the Top-K decode read of 128 requests: 2048 lanes each, 2 KV heads of 128.
        {"name": "topk_step", "kind": "topk", "dtype": "bfloat16", "batch": 128, "lanes": 2048, "heads": 16,
         "kv_heads": 2, "dim": 128},
        # A small batch of a model with many heads, an odd number of lanes, float16, the log sums returned for a merge.
        {"name": "topk_heads", "kind": "topk", "dtype": "float16", "batch": 11, "lanes": 1501, "heads": 64,
         "kv_heads": 8, "dim": 64, "lse": True},
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def _reduced(case, size, measure, largest):
    """The case with one of its sizes made smaller until its work is no more than that of the listed case."""
    limit = work(next(c for c in listed() if c["name"] == largest))[measure]
    while work(case)[measure] > limit and case[size] > 1:
        case[size] = max(1, case[size] * 3 // 4)
        if "groups" in case:
            case["groups"] = min(case["groups"], case["batch"])
    return case


def draw(rng):
    kind = rng.choice(["tables", "prefix", "prefix", "prefix", "topk", "topk"])
    if kind == "tables":
        batch = _log(rng, 1, 256)
        case = {"kind": kind, "batch": batch, "page": rng.choice([1, 16, 16, 64, 100]),
                "context": _log(rng, 64, 65536), "added": _log(rng, 1, 16384),
                "decoding": rng.choice([0.0, 0.5, 0.9, 1.0])}
        return _reduced(case, "batch", "bytes", "tables_prompts")
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 80, 96, 128, 128, 128])
    heads = kv_heads * rng.choice([1, 2, 4, 6, 8, 8])
    if kind == "topk":
        case = {"kind": kind, "dtype": dtype, "batch": _log(rng, 1, 160), "lanes": _log(rng, 33, 4096),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "lse": rng.random() < 0.5}
        return _reduced(case, "batch", "bytes", "topk_step")
    query = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 16, 1024)])
    batch = _log(rng, 1, 128)
    case = {"kind": kind, "dtype": dtype, "batch": batch, "groups": min(batch, rng.choice([1, 1, 2, 5])),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([1, 16, 16, 64, 128]),
            "prefix": _log(rng, 100, 32768), "own": query + _log(rng, 16, 4096), "query": query,
            "layout": rng.choice(["planes", "planes", "blocks"]), "lse": rng.random() < 0.5}
    case = _reduced(case, "batch", "flops", "prefix_prompts")
    return _reduced(_reduced(case, "prefix", "bytes", "prefix_step"), "batch", "bytes", "prefix_step")


# ---------------------------------------------------------------- sizes that follow from a case


def _spread(batch, low, high):
    """Ragged whole numbers between low and high, the highest among them: what work() and prepare() both go by."""
    if batch == 1:
        return [high]
    step = 0.6180339887498949
    return [high] + [low + int((high - low) * ((i * step) % 1.0)) for i in range(1, batch)]


def _table_sizes(case):
    """Own lengths and new tokens of every batch row."""
    lengths = _spread(case["batch"], case["context"] // 4, case["context"])
    added = _spread(case["batch"], max(1, case["added"] // 8), case["added"])
    decoding = round(case["batch"] * case["decoding"])
    return lengths, [1 if i >= case["batch"] - decoding else n for i, n in enumerate(added)]


def _prefix_sizes(case):
    """(first rows of the groups, prefix lengths, query tokens per row, own lengths per row)."""
    batch, groups = case["batch"], case["groups"]
    padded = batch // 30 if groups > 1 else 0           # padded batch rows at the end belong to no group
    weight = [1 + i % 3 for i in range(groups)]
    edges = [0]
    for i in range(groups):
        edges.append(round((batch - padded) * sum(weight[:i + 1]) / sum(weight)))
    prefixes = _spread(groups, case["prefix"] // 3, case["prefix"])
    if case["query"] == 1:
        tokens = [1] * batch
    else:
        tokens = _spread(batch, max(1, case["query"] // 2), case["query"])
    owns = _spread(batch, case["own"] // 8, case["own"])
    owns = [max(n, t) for n, t in zip(owns, tokens)]
    for row in range(batch - padded, batch):
        owns[row] = 0
    return edges, prefixes, tokens, owns


def work(case):
    """Bytes of each input read once and each output written once; flops of both products."""
    if case["kind"] == "tables":
        lengths, added = _table_sizes(case)
        page = case["page"]
        new = sum(-(-(n + a) // page) - -(-n // page) for n, a in zip(lengths, added))
        held = sum(1 for n in lengths if n % page)
        total = sum(added)
        # lengths, added, rows, starts, new lengths; the free list's pages read, written; open pages' entries; slots,
        # positions
        return {"bytes": 24 * case["batch"] + 8 * new + 4 * held + 8 * total, "flops": 0}
    heads, dim = case["heads"], case["dim"]
    row = case["kv_heads"] * dim * 2 * 2
    stats = 4 * heads if case.get("lse") else 0
    if case["kind"] == "topk":
        lanes = case["batch"] * case["lanes"]
        return {"bytes": lanes * (4 + row) + case["batch"] * (heads * dim * 4 + stats),
                "flops": 4 * lanes * heads * dim}
    edges, prefixes, tokens, owns = _prefix_sizes(case)
    total = sum(tokens)
    keys = sum(prefixes) + sum(owns)
    pairs = 0
    for g, prefix in enumerate(prefixes):
        pairs += prefix * sum(tokens[edges[g]:edges[g + 1]])
    pairs += sum(max(0, t * n - t * (t - 1) // 2) for t, n in zip(tokens, owns))
    return {"bytes": keys * row + 4 * (keys // case["page"]) + total * (heads * dim * 4 + stats) + 24 * case["batch"],
            "flops": 4 * pairs * heads * dim}


# ---------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _shuffled(values, gen):
    """The ragged sizes in another order for every seed (the first place keeps the largest)."""
    order = torch.randperm(len(values) - 1, generator=gen, device=DEVICE).tolist() if len(values) > 1 else []
    return [values[0]] + [values[1 + i] for i in order]


def _table_inputs(case, seed):
    gen = _generator(seed)
    page, batch = case["page"], case["batch"]
    lengths, added = _table_sizes(case)
    lengths, added = _shuffled(lengths, gen), _shuffled(added, gen)
    columns = -(-(case["context"] + case["added"]) // page) + 1
    held = [-(-n // page) for n in lengths]
    new = sum(-(-(n + a) // page) - h for n, a, h in zip(lengths, added, held))
    pool = torch.randperm(sum(held) + new + 64, generator=gen, device=DEVICE).to(torch.int32) + 1
    tables = torch.zeros((batch, columns), dtype=torch.int32, device=DEVICE)
    rows = torch.randperm(batch, generator=gen, device=DEVICE)
    column = torch.arange(columns, device=DEVICE).view(1, -1)
    held = _int(held, torch.int64)
    first = torch.cumsum(held, 0) - held
    mine = column < held.view(-1, 1)
    tables[rows] = torch.where(mine, pool[(first.view(-1, 1) + column).clamp_max(len(pool) - 1)], 0)
    start = int(held.sum())
    return {"kind": "tables", "page": page, "tables": tables, "rows": rows, "lengths": _int(lengths),
            "added": _int(added), "free": pool[start:].contiguous(), "head": _int([17]), "total": sum(added)}


def _cache(gen, dtype, layout, pages, page, kv_heads, dim):
    """The pool's memory and its keys and values as [pages, page, kv_heads, dim] views.

    planes: one plane of token rows for K and one for V; blocks: a page's planes of two layers lie together, and the
    second layer is read."""
    if layout == "planes":
        pool = torch.empty((1, 2, pages, page, kv_heads, dim), dtype=dtype, device=DEVICE).normal_(generator=gen)
        return pool, pool[0, 0], pool[0, 1]
    pool = torch.empty((pages, 2, 2, page, kv_heads, dim), dtype=dtype, device=DEVICE).normal_(generator=gen)
    return pool, pool[:, 1, 0], pool[:, 1, 1]


def _prefix_inputs(case, seed):
    gen = _generator(seed)
    dtype = getattr(torch, case["dtype"])
    page, batch, heads, kv_heads, dim = case["page"], case["batch"], case["heads"], case["kv_heads"], case["dim"]
    edges, prefixes, tokens, owns = _prefix_sizes(case)
    prefix_pages = [-(-n // page) for n in prefixes]
    own_pages = [-(-n // page) for n in owns]
    pages = 1 + sum(prefix_pages) + sum(own_pages)
    pool, keys, values = _cache(gen, dtype, case["layout"], pages, page, kv_heads, dim)
    # Pages in random order: page 0 is the sink and belongs to nobody.
    order = torch.randperm(pages - 1, generator=gen, device=DEVICE).to(torch.int32) + 1
    prefix_tables = torch.zeros((len(prefixes), max(prefix_pages)), dtype=torch.int32, device=DEVICE)
    at = 0
    for g, n in enumerate(prefix_pages):
        prefix_tables[g, :n] = order[at:at + n]
        at += n
    tables = torch.zeros((batch, max(own_pages) + 1), dtype=torch.int32, device=DEVICE)
    rows = torch.randperm(batch, generator=gen, device=DEVICE)
    place = rows.tolist()
    for b, n in enumerate(own_pages):
        tables[place[b], :n] = order[at:at + n]
        at += n
    total = sum(tokens)
    # Scores of a standard deviation of two: a few keys carry most of a row's weight.
    query = (torch.randn((total, heads, dim), generator=gen, device=DEVICE) * 2).to(dtype)
    starts = [0]
    for n in tokens:
        starts.append(starts[-1] + n)
    return {"kind": "prefix", "pool": pool, "keys": keys, "values": values, "page": page, "kv_heads": kv_heads,
            "query": query, "tables": tables, "rows": rows, "lengths": _int(owns), "prefix_tables": prefix_tables,
            "prefix_lengths": _int(prefixes), "group_starts": _int(edges),
            "query_starts": None if case["query"] == 1 else _int(starts), "most": max(tokens), "widest": max(owns),
            "edges": edges, "prefixes": prefixes, "tokens": tokens, "owns": owns, "starts": starts,
            "layout": case["layout"], "scale": dim ** -0.5,
            "out": torch.empty((total, heads, dim), dtype=dtype, device=DEVICE),
            "lse": torch.empty((total, heads), dtype=torch.float32, device=DEVICE) if case.get("lse") else None}


def _topk_inputs(case, seed):
    gen = _generator(seed)
    dtype = getattr(torch, case["dtype"])
    batch, lanes, heads, kv_heads, dim = (case["batch"], case["lanes"], case["heads"], case["kv_heads"], case["dim"])
    hot = 2 * lanes                                     # slots of a request's hot buffer
    pool, keys, values = _cache(gen, dtype, "planes", 1 + batch * hot, 1, kv_heads, dim)
    slots = torch.rand((batch, hot), generator=gen, device=DEVICE).argsort(-1)[:, :lanes]
    slots = slots + torch.arange(batch, device=DEVICE).view(-1, 1) * hot + 1
    # One lane in fifty is not resident (slot 0); short requests end in padding lanes.
    slots = slots.masked_fill(torch.rand((batch, lanes), generator=gen, device=DEVICE) < 0.02, 0)
    filled = _int(_shuffled(_spread(batch, lanes * 3 // 4, lanes), gen), torch.int64)
    slots = torch.where(torch.arange(lanes, device=DEVICE).view(1, -1) < filled.view(-1, 1), slots, -1)
    query = (torch.randn((batch, heads, dim), generator=gen, device=DEVICE) * 2).to(dtype)
    return {"kind": "topk", "pool": pool, "keys": keys, "values": values, "page": 1, "kv_heads": kv_heads,
            "query": query, "slots": slots.to(torch.int32), "layout": "planes", "scale": dim ** -0.5,
            "out": torch.empty((batch, heads, dim), dtype=dtype, device=DEVICE),
            "lse": torch.empty((batch, heads), dtype=torch.float32, device=DEVICE) if case.get("lse") else None}


def _inputs(case, seed):
    return {"tables": _table_inputs, "prefix": _prefix_inputs, "topk": _topk_inputs}[case["kind"]](case, seed)


def prepare(case, seed):
    state = _inputs(case, seed)
    if state["kind"] == "tables":
        batch, total = len(state["rows"]), state["total"]
        state["slots"] = torch.empty(total, dtype=torch.int32, device=DEVICE)
        state["positions"] = torch.empty(total, dtype=torch.int32, device=DEVICE)
        state["starts"] = torch.empty(batch + 1, dtype=torch.int32, device=DEVICE)
        state["new_lengths"] = torch.empty(batch, dtype=torch.int32, device=DEVICE)
        state["new_head"] = torch.empty(1, dtype=torch.int32, device=DEVICE)
    if own:
        _prepare_own(state)
    return state


def _prepare_own(state):
    """The pool's description and the workspace that a serving loop keeps."""
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    if state["kind"] == "tables":
        from adaptive_sparse.block_tables import extend_block_tables
        state["call"] = extend_block_tables
        state["status"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        return
    from adaptive_sparse import attention
    from adaptive_sparse.kv_pool import KVPlanes

    pool, keys = state["pool"], state["keys"]
    pages, page, kv_heads, dim = keys.shape
    row = kv_heads * dim * 2
    if state["layout"] == "planes":
        plane = pages * page * row
        state["layer"] = 0
        state["planes"] = KVPlanes(base=pool.data_ptr(), device=pool.device.index, layers=1, kv=2,
                                   layer_stride=2 * plane, kv_stride=plane, row_stride=row, row_bytes=row,
                                   rows=pages * page, owner=pool)
    else:
        row *= page
        state["layer"] = 1
        state["planes"] = KVPlanes(base=pool.data_ptr(), device=pool.device.index, layers=2, kv=2,
                                   layer_stride=2 * row, kv_stride=row, row_stride=4 * row, row_bytes=row, rows=pages,
                                   owner=pool)
    tokens, heads, dim = state["query"].shape
    if state["kind"] == "topk":
        state["call"] = attention.topk_attention
        size = attention.topk_workspace(tokens, state["slots"].shape[1], heads, kv_heads, dim)
    else:
        state["call"] = attention.shared_prefix_attention
        size = attention.shared_prefix_workspace(tokens, len(state["rows"]), len(state["prefixes"]), heads, kv_heads,
                                                 dim, state["most"])
    state["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEVICE)


# ---------------------------------------------------------------- one pass


def run(state):
    if own:
        return _OWN[state["kind"]](state)
    return _PLAIN[state["kind"]](state)


def _table_outputs(s):
    return [s["tables"], s["slots"], s["positions"], s["starts"], s["new_lengths"], s["new_head"]]


def _attention_outputs(s):
    return [s["out"]] if s["lse"] is None else [s["out"], s["lse"]]


def _own_tables(s):
    s["call"](s["tables"], s["rows"], s["lengths"], s["added"], s["free"], s["head"], s["page"], slots=s["slots"],
              positions=s["positions"], starts=s["starts"], new_lengths=s["new_lengths"], new_head=s["new_head"],
              status=s["status"])
    return _table_outputs(s)


def _own_prefix(s):
    s["call"](s["query"], s["planes"], s["tables"], s["rows"], s["lengths"], s["prefix_tables"], s["prefix_lengths"],
              s["out"], page_size=s["page"], kv_heads=s["kv_heads"], layer=s["layer"], group_starts=s["group_starts"],
              query_starts=s["query_starts"], max_query=s["most"], scale=s["scale"], lse=s["lse"],
              workspace=s["workspace"])
    return _attention_outputs(s)


def _own_topk(s):
    s["call"](s["query"], s["planes"], s["slots"], s["out"], kv_heads=s["kv_heads"], layer=s["layer"],
              scale=s["scale"], lse=s["lse"], workspace=s["workspace"])
    return _attention_outputs(s)


_OWN = {"tables": _own_tables, "prefix": _own_prefix, "topk": _own_topk}


def _plain_tables(s):
    page, tables, lengths, added = s["page"], s["tables"], s["lengths"].long(), s["added"].long()
    held, need = (lengths + page - 1) // page, (lengths + added + page - 1) // page
    last = torch.cumsum(need - held, 0)
    base = last - (need - held) + s["head"]
    column = torch.arange(tables.shape[1], device=DEVICE).view(1, -1)
    new = (column >= held.view(-1, 1)) & (column < need.view(-1, 1))
    source = (base.view(-1, 1) + column - held.view(-1, 1)).clamp(0, len(s["free"]) - 1)
    tables[s["rows"]] = torch.where(new, s["free"][source], tables[s["rows"]])
    ends = torch.cumsum(added, 0)
    token = torch.arange(s["total"], device=DEVICE)
    row = torch.searchsorted(ends, token, right=True)
    position = lengths[row] + token - (ends - added)[row]
    s["slots"].copy_(tables[s["rows"][row], position // page] * page + position % page)
    s["positions"].copy_(position)
    s["starts"][:1].zero_()
    s["starts"][1:].copy_(ends)
    s["new_lengths"].copy_(lengths + added)
    s["new_head"].copy_(s["head"] + last[-1:])
    return _table_outputs(s)


def _weights(scores):
    """Unnormalised softmax weights of masked scores, their sum and their largest score."""
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == _NO_SCORE, 0.0, top))
    return weights, weights.sum(-1, keepdim=True), top


def _finish(weighted, total, top):
    """A part's outputs, sums and largest scores joined: each a list over the parts."""
    most = top[0]
    for t in top[1:]:
        most = torch.maximum(most, t)
    safe = torch.where(most == _NO_SCORE, 0.0, most)
    factor = [torch.exp(t - safe) for t in top]
    mass = sum(f * t for f, t in zip(factor, total))
    value = sum(f * w for f, w in zip(factor, weighted))
    return torch.where(mass > 0, value / mass, 0.0), (torch.log(mass) + safe).squeeze(-1)


def _plain_prefix(s):
    page, kv_heads, scale = s["page"], s["kv_heads"], s["scale"]
    tokens, heads, dim = s["query"].shape
    share = heads // kv_heads
    batch, widest, most = len(s["rows"]), s["widest"], s["most"]
    query = s["query"].float() * scale
    # The prefix: all rows of a group against one set of keys.
    weighted = query.new_zeros((tokens, heads, dim))
    total = query.new_zeros((tokens, heads, 1))
    top = query.new_full((tokens, heads, 1), _NO_SCORE)
    for g, prefix in enumerate(s["prefixes"]):
        low, high = s["starts"][s["edges"][g]], s["starts"][s["edges"][g + 1]]
        if low == high or not prefix:
            continue
        pages = s["prefix_tables"][g, :-(-prefix // page)].long()
        keys = s["keys"][pages].reshape(-1, kv_heads, dim)[:prefix].float().permute(1, 2, 0).contiguous()
        values = s["values"][pages].reshape(-1, kv_heads, dim)[:prefix].float().permute(1, 0, 2).contiguous()
        q = query[low:high].view(-1, kv_heads, share, dim).transpose(0, 1).reshape(kv_heads, -1, dim)
        weights, mass, peak = _weights(torch.matmul(q, keys))
        for part, found in ((weighted, torch.matmul(weights, values)), (total, mass), (top, peak)):
            part[low:high] = found.view(kv_heads, high - low, share, -1).transpose(0, 1).reshape(high - low, heads, -1)
    # What is each request's own: padded to the longest, masked by position.
    pages = s["tables"][s["rows"]][:, :-(-widest // page)].long()
    keys = s["keys"][pages].reshape(batch, -1, kv_heads, dim).float().permute(0, 2, 3, 1).contiguous()
    values = s["values"][pages].reshape(batch, -1, kv_heads, dim).float().permute(0, 2, 1, 3).contiguous()
    token = torch.arange(tokens, device=DEVICE)
    if s["query_starts"] is None:
        row, at = token, torch.zeros_like(token)
        count = torch.ones(batch, dtype=torch.int64, device=DEVICE)
    else:
        starts = s["query_starts"].long()
        row = torch.searchsorted(starts[1:].contiguous(), token, right=True)
        at = token - starts[row]
        count = starts[1:] - starts[:-1]
    q = query.new_zeros((batch, most, heads, dim))
    q[row, at] = query
    q = q.view(batch, most, kv_heads, share, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, most * share, dim)
    scores = torch.matmul(q, keys).view(batch, kv_heads, most, share, -1)
    last = s["lengths"].long().view(-1, 1) - count.view(-1, 1) + torch.arange(most, device=DEVICE).view(1, -1)
    seen = torch.arange(keys.shape[-1], device=DEVICE).view(1, 1, -1) <= last.unsqueeze(-1)
    scores = scores.masked_fill(~seen.view(batch, 1, most, 1, -1), _NO_SCORE)
    weights, mass, peak = _weights(scores)
    value = torch.matmul(weights.view(batch, kv_heads, most * share, -1), values)
    value, mass, peak = (t.view(batch, kv_heads, most, share, -1).permute(0, 2, 1, 3, 4)
                         .reshape(batch, most, heads, -1)[row, at] for t in (value, mass, peak))
    result, stats = _finish([weighted, value], [total, mass], [top, peak])
    s["out"].copy_(result)
    if s["lse"] is not None:
        s["lse"].copy_(stats)
    return _attention_outputs(s)


def _plain_topk(s):
    kv_heads, slots = s["kv_heads"], s["slots"].long()
    batch, heads, dim = s["query"].shape
    seen = (slots >= 1) & (slots < s["keys"].shape[0])
    at = torch.where(seen, slots, 0)
    keys = s["keys"][at, 0].float().permute(0, 2, 3, 1).contiguous()
    values = s["values"][at, 0].float().permute(0, 2, 1, 3).contiguous()
    q = (s["query"].float() * s["scale"]).view(batch, kv_heads, heads // kv_heads, dim)
    scores = torch.matmul(q, keys).masked_fill(~seen.view(batch, 1, 1, -1), _NO_SCORE)
    weights, mass, peak = _weights(scores)
    result, stats = _finish([torch.matmul(weights, values)], [mass], [peak])
    s["out"].copy_(result.reshape(batch, heads, dim))
    if s["lse"] is not None:
        s["lse"].copy_(stats.reshape(batch, heads))
    return _attention_outputs(s)


_PLAIN = {"tables": _plain_tables, "prefix": _plain_prefix, "topk": _plain_topk}


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    """The outputs of run() for these inputs, one request after the other, in 64 bits."""
    s = _inputs(case, seed)
    return {"tables": _exact_tables, "prefix": _exact_prefix, "topk": _exact_topk}[case["kind"]](s)


def _exact_tables(s):
    page = s["page"]
    tables, free = s["tables"].cpu(), s["free"].cpu()
    head, start = int(s["head"]), 0
    slots, positions, starts, grown = [], [], [0], []
    for row, length, added in zip(s["rows"].tolist(), s["lengths"].tolist(), s["added"].tolist()):
        for column in range(-(-length // page), -(-(length + added) // page)):
            tables[row, column] = free[head]
            head += 1
        position = torch.arange(length, length + added)
        slots.append(tables[row, position // page].long() * page + position % page)
        positions.append(position)
        start += added
        starts.append(start)
        grown.append(length + added)
    outputs = [tables, torch.cat(slots), torch.cat(positions), torch.tensor(starts), torch.tensor(grown),
               torch.tensor([head])]
    return [t.to(torch.int32) for t in outputs]


def _attend(query, keys, values, scale, seen=None):
    """Softmax attention of [n, heads, dim] queries to [t, kv_heads, dim] keys in 64 bits: outputs and log sums."""
    n, heads, dim = query.shape
    kv_heads = keys.shape[1]
    share = heads // kv_heads
    if not keys.shape[0]:
        return query.new_zeros((n, heads, dim)).double(), query.new_full((n, heads), _NO_SCORE).double()
    outs, sums = [], []
    for h in range(kv_heads):
        q = query[:, h * share:(h + 1) * share].double().reshape(n * share, dim)
        scores = (q @ keys[:, h].double().t().contiguous() * scale).view(n, share, -1)
        if seen is not None:
            scores = scores.masked_fill(~seen.view(n, 1, -1), _NO_SCORE)
        lse = torch.logsumexp(scores, -1)
        weights = torch.exp(scores - torch.where(lse == _NO_SCORE, 0.0, lse).unsqueeze(-1))
        outs.append((weights.view(n * share, -1) @ values[:, h].double()).view(n, share, dim))
        sums.append(lse)
    return torch.cat(outs, 1), torch.cat(sums, 1)


def _exact_prefix(s):
    page = s["page"]
    _, heads, dim = s["query"].shape
    kv_heads = s["kv_heads"]

    def read(cache, table, count):
        pages = table[:-(-count // page)].long()
        return cache[pages].reshape(-1, kv_heads, dim)[:count]

    outs, sums = [], []
    place = s["rows"].tolist()
    for b, (count, length) in enumerate(zip(s["tokens"], s["owns"])):
        group = next((g for g in range(len(s["prefixes"])) if s["edges"][g] <= b < s["edges"][g + 1]), None)
        prefix = 0 if group is None else s["prefixes"][group]
        table = s["tables"][place[b]]
        parts = [[read(cache, table, length)] for cache in (s["keys"], s["values"])]
        if prefix:
            for part, cache in zip(parts, (s["keys"], s["values"])):
                part.insert(0, read(cache, s["prefix_tables"][group], prefix))
        keys, values = (torch.cat(part) for part in parts)
        last = prefix + length - count + torch.arange(count, device=DEVICE)
        seen = torch.arange(prefix + length, device=DEVICE).view(1, -1) <= last.view(-1, 1)
        out, lse = _attend(s["query"][s["starts"][b]:s["starts"][b] + count], keys, values, s["scale"], seen)
        outs.append(out)
        sums.append(lse)
    return [torch.cat(outs)] if s["lse"] is None else [torch.cat(outs), torch.cat(sums)]


def _exact_topk(s):
    outs, sums = [], []
    for b in range(s["query"].shape[0]):
        slots = s["slots"][b].long()
        slots = slots[(slots >= 1) & (slots < s["keys"].shape[0])]
        out, lse = _attend(s["query"][b:b + 1], s["keys"][slots, 0], s["values"][slots, 0], s["scale"])
        outs.append(out)
        sums.append(lse)
    return [torch.cat(outs)] if s["lse"] is None else [torch.cat(outs), torch.cat(sums)]
