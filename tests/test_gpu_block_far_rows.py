"""The block-sparse step's operators where offsets pass 32 bits, and in two streams at once.

The same step runs over a small pool and over one whose pages lie far behind its beginning: what is written and what
comes out are the same to the bit.
"""

import pytest
import torch

from adaptive_sparse.append import append_index, append_rotary, make_rotary
from adaptive_sparse.attention import block_attention, block_workspace
from adaptive_sparse.block_selection import select_blocks, selection_workspace
from adaptive_sparse.kv_pool import KVPlanes

pytestmark = pytest.mark.gpu

PAGE, HEADS, KV_HEADS, DIM, INDEX_DIM, INDEX_HEADS = 16, 8, 2, 128, 128, 4
ROW = KV_HEADS * DIM * 2


class Pool:
    """K, V and index keys of `pages` pages; the step uses pages from `first` on."""

    def __init__(self, gpu, pages, first):
        rows = pages * PAGE
        self.first, self.rows = first, rows
        self.kv = torch.empty(2 * rows * ROW, dtype=torch.uint8, device=gpu)
        self.keys = torch.empty(rows * INDEX_DIM, dtype=torch.uint8, device=gpu)
        self.scales = torch.empty(rows, device=gpu)
        self.planes = KVPlanes(base=self.kv.data_ptr(), device=0, layers=1, kv=2, layer_stride=2 * rows * ROW,
                               kv_stride=rows * ROW, row_stride=ROW, row_bytes=ROW, rows=rows, owner=self.kv)
        self.index = KVPlanes(base=self.keys.data_ptr(), device=0, layers=1, kv=1, layer_stride=rows * INDEX_DIM,
                              kv_stride=rows * INDEX_DIM, row_stride=INDEX_DIM, row_bytes=INDEX_DIM, rows=rows,
                              owner=self.keys)

    def used(self, pages):
        """The bytes of the pages that the step uses."""
        at, n = self.first * PAGE, pages * PAGE
        kv, keys = self.kv.view(2, self.rows, ROW), self.keys.view(self.rows, INDEX_DIM)
        return kv[:, at:at + n], keys[at:at + n], self.scales[at:at + n]


def run(gpu, pool, counts, lengths, index, chosen, block, seed=0, workspaces=None):
    """Contexts written, then `counts` query tokens of each of two requests; returns lists, outputs, statistics."""
    gen = torch.Generator(device=gpu).manual_seed(seed)
    held = [-(-n // PAGE) for n in lengths]
    order = torch.randperm(sum(held), generator=gen, device=gpu) + pool.first
    tables = torch.zeros((2, max(held)), dtype=index, device=gpu)
    tables[0, :held[0]], tables[1, :held[1]] = order[:held[0]].to(index), order[held[0]:].to(index)
    positions = torch.cat([torch.arange(n, device=gpu) for n in lengths]).to(index)
    slots = torch.cat([tables[b].long()[torch.arange(n, device=gpu) // PAGE] * PAGE + torch.arange(n, device=gpu) % PAGE
                       for b, n in enumerate(lengths)]).to(index)
    total = sum(lengths)
    draw = lambda *shape: torch.randn(shape, generator=gen, device=gpu).to(torch.bfloat16)  # noqa: E731
    rotary = make_rotary(DIM, device=gpu)
    append_rotary(None, draw(total, KV_HEADS, DIM), draw(total, KV_HEADS, DIM), pool.planes, slots, positions, rotary,
                  None, page_size=PAGE)
    append_index(draw(total, INDEX_DIM), pool.index, pool.scales, slots, page_size=PAGE)
    tokens = sum(counts)
    blocks = torch.full((tokens, 2, chosen), 9, dtype=torch.int32, device=gpu)
    starts = torch.tensor([0, counts[0], tokens], dtype=index, device=gpu)
    given = dict(page_size=PAGE, block_size=block, query_starts=starts, max_query=max(counts))
    row_lengths = torch.tensor(lengths, dtype=index, device=gpu)
    select_blocks(draw(tokens, INDEX_HEADS, INDEX_DIM), pool.index, pool.scales, tables, None, row_lengths, blocks,
                  workspace=None if workspaces is None else workspaces[0], **given)
    query = draw(tokens, HEADS, DIM)
    out, lse = torch.empty_like(query), torch.empty((tokens, HEADS), device=gpu)
    block_attention(query, pool.planes, tables, None, row_lengths, blocks, out, kv_heads=KV_HEADS, lse=lse,
                    workspace=None if workspaces is None else workspaces[1], **given)
    return blocks, out, lse


SHAPES = [
    ([1, 1], [700, 400]),              # single tokens
    ([700, 400], [700, 900]),          # prompts: 2200 pairs of a token and a KV head
]


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("counts,lengths", SHAPES)
def test_pages_behind_4_gib(gpu, counts, lengths, index):
    print(f"[far] {counts} {lengths} {index}", flush=True)
    held = sum(-(-n // PAGE) for n in lengths)
    near = Pool(gpu, held + 1, 1)
    for part in near.used(held):
        part.zero_()
    want = run(gpu, near, counts, lengths, index, 5, 64)
    # 2^32 bytes of index keys before the first page, four times as many of K.
    first = (1 << 32) // (PAGE * INDEX_DIM) + 7
    far = Pool(gpu, first + held, first)
    for part in far.used(held):
        part.zero_()
    got = run(gpu, far, counts, lengths, index, 5, 64)
    assert all(torch.isfinite(x.float()).all() for x in want)
    for mine, other in zip(got, want):
        assert torch.equal(mine, other)
    for mine, other in zip(far.used(held), near.used(held)):
        assert torch.equal(mine, other) and bool(mine.any())


def test_slots_past_31_bits(gpu):
    """Rows of 16 bytes: the last of more than 2^31 slots."""
    rows = (1 << 31) + 64
    memory = torch.empty(2 * rows * 16, dtype=torch.uint8, device=gpu)
    planes = KVPlanes(base=memory.data_ptr(), device=0, layers=1, kv=2, layer_stride=2 * rows * 16, kv_stride=rows * 16,
                      row_stride=16, row_bytes=16, rows=rows, owner=memory)
    last = memory.view(2, rows, 8, 2)[:, -64:].view(torch.bfloat16).view(2, 64, 8)
    last.fill_(3.0)
    slots = torch.tensor([rows - 1, rows - 64, rows, rows + (1 << 32)], device=gpu)
    key = torch.arange(32, device=gpu).view(4, 1, 8).to(torch.bfloat16)
    value = key + 100
    zero = torch.zeros(4, dtype=torch.int64, device=gpu)        # position 0: nothing turns
    append_rotary(None, key, value, planes, slots, zero, make_rotary(8, device=gpu), None, page_size=16)
    assert torch.equal(last[0, 63], key[0, 0]) and torch.equal(last[1, 63], value[0, 0])
    assert torch.equal(last[0, 0], key[1, 0]) and torch.equal(last[1, 0], value[1, 0])
    assert bool((last[:, 1:63] == 3.0).all())


def test_two_streams_at_once(gpu):
    """Steps of two streams over pools, workspaces and outputs of their own: as one after the other."""
    pools = [Pool(gpu, 120, 1) for _ in range(2)]
    shapes = [([1, 1], [700, 400]), ([700, 400], [700, 900])]
    want = [run(gpu, pools[i], *shapes[i], torch.int32, 5, 64, seed=i) for i in range(2)]
    spaces = []
    for counts, lengths in shapes:
        columns = -(-max(lengths) // PAGE)
        sizes = (selection_workspace(sum(counts), 2, columns, PAGE, 64),
                 block_workspace(sum(counts), 5, 64, HEADS, KV_HEADS, DIM, max(counts)))
        spaces.append([torch.empty(n, dtype=torch.uint8, device=gpu) for n in sizes])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(run(gpu, pools[i], *shapes[i], torch.int32, 5, 64, seed=i, workspaces=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            for mine, other in zip(one, want[i]):
                assert torch.equal(mine, other)
