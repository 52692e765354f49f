"""Random paged-attention problems and their answers in 64 bits, for the GPU tests of the attention operators.

A problem is built from plain Python sizes; its answer is computed token by token from the definition, reading
every seen K and V row through the tables on the host side of the copy. The bounds are derived from the number
formats: with u the unit roundoff of the 16-bit type (2^-8 bfloat16, 2^-11 float16), the weights are rounded once
before they multiply V (at most u * sum p|v| / sum p) and the result once (u |o|); sums and statistics are held in 32
bits (a relative 2^-12 of sum p|v| / sum p covers them by far). An error that is random from key to key adds up to u times
the root of sum (p v)^2, which bounds the root mean square over many outputs.
"""

import math
from dataclasses import dataclass, field

import torch

from adaptive_sparse.kv_pool import KVPlanes

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@dataclass
class Pool:
    """K and V planes of `layers` layers; keys/values [pages, page, kv_heads, dim] views of one layer."""

    memory: torch.Tensor
    planes: KVPlanes
    keys: torch.Tensor
    values: torch.Tensor
    page: int
    layer: int


def make_pool(device, dtype, pages, page, kv_heads, dim, layout="planes", layers=2, layer=1, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    row = kv_heads * dim * 2
    if layout == "planes":
        memory = torch.empty((layers, 2, pages, page, kv_heads, dim), dtype=dtype, device=device)
        memory.normal_(generator=gen)
        plane = pages * page * row
        planes = KVPlanes(base=memory.data_ptr(), device=device.index or 0, layers=layers, kv=2,
                          layer_stride=2 * plane, kv_stride=plane, row_stride=row, row_bytes=row, rows=pages * page,
                          owner=memory)
        return Pool(memory, planes, memory[layer, 0], memory[layer, 1], page, layer)
    memory = torch.empty((pages, layers, 2, page, kv_heads, dim), dtype=dtype, device=device).normal_(generator=gen)
    row *= page
    planes = KVPlanes(base=memory.data_ptr(), device=device.index or 0, layers=layers, kv=2, layer_stride=2 * row,
                      kv_stride=row, row_stride=2 * layers * row, row_bytes=row, rows=pages, owner=memory)
    return Pool(memory, planes, memory[:, layer, 0], memory[:, layer, 1], page, layer)


@dataclass
class Answer:
    out: torch.Tensor          # [N, Hq, D] float64
    lse: torch.Tensor          # [N, Hq] float64
    mass: torch.Tensor         # [N, Hq, D]: sum p|v| / sum p
    spread: torch.Tensor       # [N, Hq, D]: sum (p v)^2 / (sum p)^2
    size: float                # the largest sum of |scale q_d k_d| over the scores


def attend(query, keys, values, scale, seen):
    """One query token [Hq, D] against keys/values [T, Hkv, D] in 64 bits; seen [T] bool."""
    heads, dim = query.shape
    kv_heads = keys.shape[1]
    keys, values = keys[seen].double(), values[seen].double()
    q = query.double().view(kv_heads, heads // kv_heads, dim)
    if not keys.shape[0]:
        zero = torch.zeros((heads, dim), dtype=torch.float64, device=query.device)
        return zero, torch.full((heads,), -math.inf, dtype=torch.float64, device=query.device), zero, zero, 0.0
    k, v = keys.permute(1, 0, 2), values.permute(1, 0, 2)
    scores = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
    lse = torch.logsumexp(scores, -1)
    p = torch.exp(scores - lse.unsqueeze(-1))
    size = float((torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous()) * abs(scale)).nan_to_num().max())
    return (torch.matmul(p, v).reshape(heads, dim), lse.reshape(heads), torch.matmul(p, v.abs()).reshape(heads, dim),
            torch.matmul(p * p, v * v).reshape(heads, dim), size)


def answer_of(parts):
    outs, sums, masses, spreads, sizes = zip(*parts)
    return Answer(torch.stack(outs), torch.stack(sums), torch.stack(masses), torch.stack(spreads), max(sizes))


def read(pool, table, count):
    """(keys, values, seen) of the first `count` tokens of a table row; unseen ones are zeros."""
    page = pool.page
    count = max(0, min(count, table.shape[0] * page))
    pages = table[:-(-count // page)].long()
    good = (pages >= 1) & (pages < pool.keys.shape[0])
    at = torch.where(good, pages, 0)
    shape = (-1, *pool.keys.shape[2:])
    keys = pool.keys[at].reshape(shape)[:count]
    values = pool.values[at].reshape(shape)[:count]
    return keys, values, good.repeat_interleave(page)[:count]


@dataclass
class Problem:
    """A shared_prefix_attention call: tensors on the device and the sizes as Python lists."""

    pool: Pool
    query: torch.Tensor
    tables: torch.Tensor
    rows: torch.Tensor
    lengths: list
    prefix_tables: torch.Tensor
    prefix_lengths: list
    group_starts: list
    counts: list
    scale: float
    index: torch.dtype = torch.int32
    extra: dict = field(default_factory=dict)

    def starts(self):
        at = [0]
        for n in self.counts:
            at.append(at[-1] + n)
        return at

    def group(self, b):
        if self.prefix_tables is None:
            return None
        for g in range(len(self.prefix_lengths)):
            if self.group_starts[g] <= b < self.group_starts[g + 1]:
                return g
        return None

    def answer(self):
        parts = []
        starts = self.starts()
        place = self.rows.tolist() if self.rows is not None else list(range(len(self.lengths)))
        empty = self.tables.new_zeros(0)
        for b, (count, length) in enumerate(zip(self.counts, self.lengths)):
            g = self.group(b)
            first = read(self.pool, empty if g is None else self.prefix_tables[g],
                         0 if g is None else self.prefix_lengths[g])
            own = empty if not 0 <= place[b] < self.tables.shape[0] else self.tables[place[b]]
            for i in range(count):
                second = read(self.pool, own, length - count + i + 1)
                keys, values, seen = (torch.cat(pair) for pair in zip(first, second))
                parts.append(attend(self.query[starts[b] + i], keys, values, self.scale, seen))
        for t in range(starts[-1], self.query.shape[0]):
            keys, values, seen = read(self.pool, empty, 0)
            parts.append(attend(self.query[t], keys, values, self.scale, seen))
        return answer_of(parts)

    def call(self, run, output, lse=None, **extra):
        device = self.query.device
        ints = lambda v: torch.tensor(v, dtype=self.index, device=device)  # noqa: E731
        ragged = any(n != 1 for n in self.counts) or self.query.shape[0] != len(self.counts)
        given = dict(page_size=self.pool.page, kv_heads=self.pool.keys.shape[2], layer=self.pool.layer,
                     group_starts=ints(self.group_starts) if self.group_starts is not None else None,
                     query_starts=ints(self.starts()) if ragged else None, max_query=max([1, *self.counts]),
                     scale=self.scale, lse=lse)
        given.update(self.extra)
        given.update(extra)
        prefix = self.prefix_tables is not None
        run(self.query, self.pool.planes, self.tables, self.rows, ints(self.lengths), self.prefix_tables,
            ints(self.prefix_lengths) if prefix else None, output, **given)


def make_problem(device, *, dtype=torch.bfloat16, heads=8, kv_heads=2, dim=128, page=16, lengths=(5, 40), counts=None,
                 prefixes=(100,), groups=None, layout="planes", index=torch.int32, seed=0, spare=2, magnitude=2.0,
                 permute=True, tail=0):
    """Shuffled pages, permuted requests; groups: first batch rows (None: one group of all rows)."""
    gen = torch.Generator(device=device).manual_seed(seed + 1)
    lengths = list(lengths)
    batch = len(lengths)
    counts = list(counts) if counts is not None else [1] * batch
    prefixes = list(prefixes) if prefixes is not None else []
    own_pages = [max(0, -(-n // page)) for n in lengths]
    prefix_pages = [-(-n // page) for n in prefixes]
    total = 1 + sum(own_pages) + sum(prefix_pages) + spare
    pool = make_pool(device, dtype, total, page, kv_heads, dim, layout, seed=seed)
    order = (torch.randperm(total - 1, generator=gen, device=device) + 1).to(index)
    tables = torch.zeros((batch, max([1, *own_pages])), dtype=index, device=device)
    rows = torch.randperm(batch, generator=gen, device=device) if permute else None
    place = rows.tolist() if rows is not None else list(range(batch))
    at = 0
    for b, n in enumerate(own_pages):
        tables[place[b], :n] = order[at:at + n]
        at += n
    prefix_tables = None
    if prefixes:
        prefix_tables = torch.zeros((len(prefixes), max([1, *prefix_pages])), dtype=index, device=device)
        for g, n in enumerate(prefix_pages):
            prefix_tables[g, :n] = order[at:at + n]
            at += n
    query = (torch.randn((sum(counts) + tail, heads, dim), generator=gen, device=device) * magnitude).to(dtype)
    if groups is None and prefixes:
        groups = [0, batch]
    return Problem(pool, query, tables, rows, lengths, prefix_tables, prefixes, groups, counts, dim ** -0.5, index)


def check(out, lse, want, dim):
    """The output and statistics against the 64-bit answer, by the bounds in this file's head."""
    unit = UNIT[out.dtype]
    got = out.double()
    error = (got - want.out).abs()
    bound = unit * want.out.abs() + (unit + 2.0 ** -12) * want.mass + 2.0 ** -24
    worst = float((error / bound).max()) if error.numel() else 0.0
    assert torch.isfinite(got).all(), "an output is not finite"
    assert worst <= 1.0, f"an output is {worst:.3f} times its bound away"
    if error.numel() >= 256:
        rms = math.sqrt(float(error.square().mean()))
        limit = unit * math.sqrt(float((want.out.square() + want.spread).mean())) + 2.0 ** -24
        assert rms <= limit, f"root mean square error {rms:.3e}, bound {limit:.3e}"
    if lse is not None:
        empty = want.lse == -math.inf
        assert torch.equal(lse == -math.inf, empty), "empty rows and lse = -inf differ"
        off = (lse.double() - want.lse).abs()[~empty]
        # A score's rounding errors grow with the root of the head size; 4 of those, and the sum's own.
        limit = 4 * math.sqrt(dim) * 2.0 ** -24 * want.size + 2.0 ** -20 * (1 + want.lse.abs()[~empty])
        if off.numel():
            assert float((off / limit).max()) <= 1.0, f"lse off by {float((off / limit).max()):.3f} times its bound"
