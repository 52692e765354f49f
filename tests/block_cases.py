"""Random problems of the block-sparse operators and their answers, for the GPU tests.

Selections are compared exactly: scores are numbers of 32 bits by their definition (whole-number products, two roundings),
which numpy's float32 on the host gives likewise. Attention over blocks is compared with a 64-bit answer by the bounds of
attention_cases.py.
"""

from dataclasses import dataclass

import numpy as np
import torch

from adaptive_sparse.kv_pool import KVPlanes

from attention_cases import answer_of, attend, make_pool


def codes_of(x):
    """(codes int64, scales float32) of rows of 16-bit floats: the definition of append_index, on the host."""
    x = x.float().cpu().numpy()
    scale = (np.abs(x).max(-1, keepdims=True) / np.float32(127)).astype(np.float32)
    quotient = (x / np.where(scale > 0, scale, np.float32(1))).astype(np.float32)
    return np.rint(quotient).astype(np.int64), scale[..., 0]


@dataclass
class IndexPool:
    """Index keys of `layers` layers; keys [pages, page, dim] int8 of one layer, scales [pages * page] of it."""

    memory: torch.Tensor
    planes: KVPlanes
    keys: torch.Tensor
    scales: torch.Tensor
    page: int
    layer: int


def make_index_pool(device, pages, page, dim, layout="planes", layers=2, layer=1, seed=0, small=False):
    gen = torch.Generator(device=device).manual_seed(seed)
    high = 3 if small else 128            # small codes make equal scores
    shape = (layers, pages, page, dim) if layout == "planes" else (pages, layers, page, dim)
    memory = torch.randint(1 - high, high, shape, generator=gen, device=device, dtype=torch.int8)
    scales = torch.rand((layers, pages * page), generator=gen, device=device) * 0.02 + 0.005
    if small:
        scales.fill_(0.5)
    if layout == "planes":
        planes = KVPlanes(base=memory.data_ptr(), device=device.index or 0, layers=layers, kv=1,
                          layer_stride=pages * page * dim, kv_stride=pages * page * dim, row_stride=dim, row_bytes=dim,
                          rows=pages * page, owner=memory)
        keys = memory[layer]
    else:
        row = page * dim
        planes = KVPlanes(base=memory.data_ptr(), device=device.index or 0, layers=layers, kv=1, layer_stride=row,
                          kv_stride=row, row_stride=layers * row, row_bytes=row, rows=pages, owner=memory)
        keys = memory[:, layer]
    return IndexPool(memory, planes, keys, scales[layer], page, layer)


@dataclass
class Batch:
    """Batch rows with pages of their own: lengths and query tokens of each, page tables, requests in another order."""

    lengths: list
    counts: list
    tables: torch.Tensor
    rows: torch.Tensor
    pages: int
    page: int
    index: torch.dtype

    def starts(self):
        at = [0]
        for n in self.counts:
            at.append(at[-1] + n)
        return at

    def ints(self, values):
        return torch.tensor(values, dtype=self.index, device=self.tables.device)

    def given(self, tokens):
        """The arguments of a call that say where its `tokens` query tokens are."""
        ragged = any(n != 1 for n in self.counts) or tokens != len(self.counts)
        return dict(query_starts=self.ints(self.starts()) if ragged else None, max_query=max([1, *self.counts]))

    def places(self, tokens):
        """(batch row or None, position) of every query token."""
        found = [(b, length - count + i) for b, (length, count) in enumerate(zip(self.lengths, self.counts))
                 for i in range(count)]
        return found + [(None, -1)] * (tokens - len(found))

    def table(self, b):
        place = int(self.rows[b]) if self.rows is not None else b
        return self.tables[place].tolist() if 0 <= place < self.tables.shape[0] else []

    def seen(self, b, position):
        """(token, page) of everything that a query token at `position` of row b may see."""
        table = self.table(b)
        last = min(position + 1, self.lengths[b], len(table) * self.page)
        return [(t, table[t // self.page]) for t in range(last) if 1 <= table[t // self.page] < self.pages]


def make_batch(device, lengths, counts=None, page=16, index=torch.int32, seed=0, spare=3, permute=True):
    gen = torch.Generator(device=device).manual_seed(seed + 7)
    lengths = list(lengths)
    counts = list(counts) if counts is not None else [1] * len(lengths)
    held = [max(0, -(-n // page)) for n in lengths]
    pages = 1 + sum(held) + spare
    order = (torch.randperm(pages - 1, generator=gen, device=device) + 1).to(index)
    tables = torch.zeros((len(lengths), max([1, *held])), dtype=index, device=device)
    rows = torch.randperm(len(lengths), generator=gen, device=device) if permute else None
    place = rows.tolist() if rows is not None else list(range(len(lengths)))
    at = 0
    for b, n in enumerate(held):
        tables[place[b], :n] = order[at:at + n]
        at += n
    return Batch(lengths, counts, tables, rows, pages, page, index)


def selection(batch, pool, query, groups, chosen, block, first, last):
    """The lists of select_blocks [N, G, K], by sorting the scores of the definition."""
    tokens, heads, _ = query.shape
    codes, q_scale = codes_of(query)
    keys = pool.keys.cpu().numpy().astype(np.int64)
    scales = pool.scales.cpu().numpy()
    share = heads // groups
    out = np.full((tokens, groups, chosen), -1, np.int32)
    for n, (b, position) in enumerate(batch.places(tokens)):
        if b is None:
            continue
        seen = batch.seen(b, position)
        if not seen:
            continue
        token = np.array([t for t, _ in seen])
        page = np.array([p for _, p in seen])
        inside = token % batch.page
        product = codes[n] @ keys[page, inside].T                                # [Hi, T], whole numbers
        scores = product.astype(np.float32) * scales[page * batch.page + inside]
        ids = token // block
        newest = position // block
        for g in range(groups):
            best = {}
            for h in range(g * share, (g + 1) * share):
                for j in np.unique(ids):
                    score = np.float32(scores[h][ids == j].max()) * q_scale[n, h]
                    best[j] = max(best.get(j, -np.inf), score)
            rank = sorted(best, key=lambda j: (0 if j < first or j > newest - last else 1,
                                               0 if j < first or j > newest - last else -best[j], j))
            taken = sorted(rank[:chosen])
            out[n, g, :len(taken)] = taken
    return torch.from_numpy(out)


@dataclass
class BlockProblem:
    """A block_attention call."""

    batch: Batch
    pool: object
    query: torch.Tensor
    blocks: torch.Tensor
    block: int
    scale: float

    def answer(self):
        tokens, heads, dim = self.query.shape
        kv_heads = self.pool.keys.shape[2]
        lists = self.blocks.shape[1]
        listed = self.blocks.cpu().tolist()
        parts = []
        for n, (b, position) in enumerate(self.batch.places(tokens)):
            seen = {} if b is None else dict(self.batch.seen(b, position))
            per_head = []
            for h in range(kv_heads):
                mine = []
                for j in listed[n][h * lists // kv_heads]:
                    if 0 <= j and j * self.block <= position:
                        mine += [(t, seen[t]) for t in range(j * self.block, min((j + 1) * self.block, position + 1))
                                 if t in seen]
                at = torch.tensor([p for _, p in mine], dtype=torch.int64, device=self.query.device)
                inside = torch.tensor([t % self.batch.page for t, _ in mine], dtype=torch.int64,
                                      device=self.query.device)
                keys, values = (cache[at, inside, h:h + 1].reshape(-1, 1, dim)
                                for cache in (self.pool.keys, self.pool.values))
                share = heads // kv_heads
                good = torch.ones(len(mine), dtype=torch.bool, device=self.query.device)
                per_head.append(attend(self.query[n, h * share:(h + 1) * share], keys, values, self.scale, good))
            parts.append(tuple(torch.cat([x[i] for x in per_head]) for i in range(4))
                         + (max(x[4] for x in per_head),))
        return answer_of(parts)

    def call(self, run, output, lse=None, **extra):
        given = dict(page_size=self.batch.page, block_size=self.block, kv_heads=self.pool.keys.shape[2],
                     layer=self.pool.layer, scale=self.scale, lse=lse)
        given.update(self.batch.given(self.query.shape[0]))
        given.update(extra)
        run(self.query, self.pool.planes, self.batch.tables, self.batch.rows, self.batch.ints(self.batch.lengths),
            self.blocks, output, **given)


def make_block_problem(device, *, dtype=torch.bfloat16, heads=8, kv_heads=2, dim=128, page=16, lengths=(500, 40),
                       counts=None, block=64, chosen=4, lists=1, layout="planes", index=torch.int32, seed=0, tail=0,
                       permute=True, together=False):
    """Lists of random blocks up to the newest, some entries -1, in random order; together: neighbours' lists are alike."""
    batch = make_batch(device, lengths, counts, page, index, seed, permute=permute)
    pool = make_pool(device, dtype, batch.pages, page, kv_heads, dim, layout, seed=seed)
    gen = torch.Generator(device=device).manual_seed(seed + 2)
    tokens = sum(batch.counts) + tail
    query = (torch.randn((tokens, heads, dim), generator=gen, device=device) * 2).to(dtype)
    rng = np.random.default_rng(seed)
    blocks = np.full((tokens, lists, chosen), -1, np.int64)
    common = rng.random((len(batch.lengths) + 1, lists, 1 + max([1, *batch.lengths]) // block))
    for n, (b, position) in enumerate(batch.places(tokens)):
        count = max(position, 0) // block + 1
        for g in range(lists):
            weight = rng.random(count) * (0.2 if together else 1.0)
            if together and b is not None:
                weight = weight + common[b, g, :count]
            found = np.argsort(-weight)[:chosen]
            if count > 1 and rng.random() < 0.7:
                found[0] = count - 1                        # mostly the newest one, perhaps twice
            found = rng.permutation(np.concatenate([found, np.full(chosen - len(found), -1)]))
            blocks[n, g] = found
    return BlockProblem(batch, pool, query, torch.from_numpy(blocks).to(device=device, dtype=index), block, dim ** -0.5)
