"""extend_block_tables against a row-by-row restatement: whole numbers, equal in every entry."""

import random

import pytest
import torch

from adaptive_sparse.block_tables import (TABLES_BAD_ROW, TABLES_MAP_FULL, TABLES_NO_PAGES, TABLES_ROW_FULL,
                                          TABLES_SLOT_RANGE, check_table_status, extend_block_tables)

pytestmark = pytest.mark.gpu

OLD = -77     # what entries and places hold that must not be written


def restate(table, rows, lengths, added, free, head, page, capacity, narrow=True):
    """The documented rules over Python lists; table is changed in place."""
    flags = 0
    columns = len(table[0]) if table else 0
    slots, positions, starts, grown = [], [], [], []
    taken, total = 0, 0
    for b, (length, count) in enumerate(zip(lengths, added)):
        r = rows[b] if rows is not None else b
        room = columns * page
        if not 0 <= r < len(table) or not 0 <= length <= room or count < 0:
            flags |= TABLES_BAD_ROW
            r, length, count = 0, min(max(length, 0), room), 0
        if count > room - length:
            flags |= TABLES_ROW_FULL
            count = room - length
        starts.append(min(total, capacity))
        grown.append(length + count)
        for j in range(-(-length // page), -(-(length + count) // page)):
            at = head + taken
            taken += 1
            if not 0 <= at < len(free):
                flags |= TABLES_NO_PAGES
            table[r][j] = free[at] if 0 <= at < len(free) else 0
        for i in range(count):
            p = length + i
            entry = table[r][p // page]
            slot = entry * page + p % page if entry >= 1 else -1
            if narrow and slot > 0x7fffffff and total < capacity:
                flags |= TABLES_SLOT_RANGE
                slot = -1
            if total < capacity:
                slots.append(slot)
                positions.append(p)
            total += 1
    if total > capacity:
        flags |= TABLES_MAP_FULL
    if head < 0:
        flags |= TABLES_NO_PAGES
    pad = [-1] * (capacity - len(slots))
    return slots + pad, positions + pad, starts + [min(total, capacity)], grown, head + taken, flags


def run(gpu, table, rows, lengths, added, free, head, page, capacity, *, dtype=torch.int32, slot_dtype=torch.int32,
        spread=False, offset=0):
    """The call on tensors of these lists; spread: every tensor with gaps between its elements."""
    def tensor(values, kind=dtype):
        t = torch.tensor(values, dtype=kind, device=gpu)
        if not spread:
            return t
        wide = torch.full(tuple(2 * n for n in t.shape), OLD, dtype=kind, device=gpu)
        view = wide[tuple(slice(None, None, 2) for _ in t.shape)]
        view.copy_(t)
        return view

    def fresh(count, kind=slot_dtype):
        # `offset` elements into a buffer: not 16-byte aligned
        return tensor([OLD] * (count + offset), kind)[offset:]

    given = tensor(table)
    slots, positions = fresh(capacity), fresh(capacity)
    starts, grown, next_head = fresh(len(lengths) + 1, dtype), fresh(len(lengths), dtype), fresh(1, dtype)
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    print(f"[tables] batch {len(lengths)} page {page} capacity {capacity} added {added[:6]}", flush=True)
    extend_block_tables(given, None if rows is None else tensor(rows, torch.int64), tensor(lengths), tensor(added),
                        tensor(free), tensor([head]), page, slots=slots, positions=positions, starts=starts,
                        new_lengths=grown, new_head=next_head, status=status)
    torch.cuda.synchronize()
    return [given.tolist(), slots.tolist(), positions.tolist(), starts.tolist(), grown.tolist(), int(next_head),
            int(status)]


def compare(gpu, table, rows, lengths, added, free, head, page, capacity, **how):
    got = run(gpu, table, rows, lengths, added, free, head, page, capacity, **how)
    want_table = [list(row) for row in table]
    want = restate(want_table, rows, lengths, added, free, head, page, capacity,
                   how.get("slot_dtype", torch.int32) == torch.int32)
    for name, a, b in zip(("table", "slots", "positions", "starts", "new_lengths", "new_head", "status"),
                          got, [want_table, *want]):
        assert a == b, name


def problem(seed, batch, page, most, columns=None, requests=None):
    rng = random.Random(seed)
    lengths = [rng.choice([0, 1, page - 1, page, page + 1, rng.randrange(0, 5 * page + 1)]) for _ in range(batch)]
    added = [rng.choice([0, 1, 1, page, rng.randrange(0, most + 1)]) for _ in range(batch)]
    columns = columns or max(-(-(n + a) // page) for n, a in zip(lengths, added)) + 2
    requests = requests or batch + 3
    rows = rng.sample(range(requests), batch)
    table = [[OLD] * columns for _ in range(requests)]
    ids = list(range(1, 200000))
    rng.shuffle(ids)
    at = 0
    for b, n in enumerate(lengths):
        for j in range(-(-n // page)):
            table[rows[b]][j] = ids[at]
            at += 1
    needed = sum(-(-(n + a) // page) - -(-n // page) for n, a in zip(lengths, added))
    return table, rows, lengths, added, ids[at:at + needed + 5], sum(added)


@pytest.mark.parametrize("page", [1, 2, 7, 16, 64, 100])
@pytest.mark.parametrize("batch", [1, 3, 130])
def test_ragged_batches(gpu, page, batch):
    table, rows, lengths, added, free, total = problem(page * 31 + batch, batch, page, 6 * page)
    compare(gpu, table, rows, lengths, added, [9] * 4 + free, 4, page, total + 3)


@pytest.mark.parametrize("how", [dict(dtype=torch.int64), dict(slot_dtype=torch.int64), dict(spread=True),
                                 dict(offset=1), dict(dtype=torch.int64, slot_dtype=torch.int64, spread=True)])
def test_types_strides_and_alignment(gpu, how):
    table, rows, lengths, added, free, total = problem(5, 40, 16, 100)
    compare(gpu, table, rows, lengths, added, free, 0, 16, total + 9, **how)


@pytest.mark.parametrize("batch", [1023, 1024, 1025, 2600])
def test_more_rows_than_a_workgroup_sums_at_once(gpu, batch):
    table, rows, lengths, added, free, total = problem(batch, batch, 4, 9)
    compare(gpu, table, rows, lengths, added, free, 0, 4, total)


def test_long_prompts(gpu):
    table, rows, lengths, added, free, total = problem(77, 9, 16, 30000)
    added[4] = 50001
    table = [row + [OLD] * 4000 for row in table]
    free = list(range(300000, 320000))
    compare(gpu, table, rows, lengths, added, free, 3, 16, sum(added) + 5000)


def test_rows_none_zero_tokens_and_no_rows(gpu):
    table = [[OLD, OLD], [5, OLD], [6, 7]]
    compare(gpu, table, None, [0, 3, 8], [4, 0, 0], [11, 12], 0, 4, 6)
    compare(gpu, table, None, [0, 3, 8], [0, 0, 0], [11, 12], 1, 4, 3)
    compare(gpu, table, [], [], [], [11, 12], 1, 4, 3)
    compare(gpu, table, None, [0, 3, 8], [1, 1, 0], [11, 12], 0, 4, 0)


def test_what_does_not_fit_is_left_out(gpu):
    table = [[OLD] * 4 for _ in range(5)]
    full = [[21, 22, 23, 24]] + table[1:]
    # past the columns; a full row
    compare(gpu, full, [1, 0], [0, 13], [100, 9], list(range(30, 60)), 0, 4, 200)
    # bad rows among good ones
    compare(gpu, full, [7, 1, -1, 0, 2], [0, -3, 2, 17, 0], [3, 3, 3, 1, 5], list(range(30, 60)), 2, 4, 30)
    compare(gpu, full, [1, 2], [0, 0], [-1, 6], list(range(30, 60)), 2, 4, 30)
    # no pages left, a head outside the list
    compare(gpu, table, [0, 1, 2], [0, 0, 0], [9, 9, 9], [31, 32, 33, 34], 0, 4, 27)
    compare(gpu, table, [0, 1], [0, 0], [9, 9], [31, 32, 33, 34], 9, 4, 27)
    compare(gpu, table, [0, 1], [0, 0], [9, 9], [31, 32, 33, 34], -2, 4, 27)
    # a map that is too short; ids below 1 in the list
    compare(gpu, table, [0, 1, 2], [0, 0, 0], [9, 9, 9], list(range(30, 60)), 0, 4, 13)
    compare(gpu, table, [0, 1], [0, 0], [9, 9], [31, 0, -4, 34, 35, 36], 0, 4, 18)


def test_a_slot_past_31_bits(gpu):
    table = [[OLD] * 3 for _ in range(2)]
    ids = [5, 1 << 30, 6, (1 << 30) + 1]
    compare(gpu, table, [1, 0], [0, 0], [7, 5], ids, 0, 4, 12)
    compare(gpu, table, [1, 0], [0, 0], [7, 5], ids, 0, 4, 12, slot_dtype=torch.int64)


def test_status_is_raised_once(gpu):
    status = torch.tensor([TABLES_NO_PAGES | TABLES_MAP_FULL], dtype=torch.int32, device=gpu)
    with pytest.raises(RuntimeError, match="ran out of pages; more new tokens"):
        check_table_status(status)
    check_table_status(status)


def test_outputs_must_not_share_memory_with_inputs(gpu):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    table, lengths, added, free, head = ints(0, 0).view(1, 2), ints(0), ints(1), ints(3, 4), ints(0)
    slots, starts = ints(0), ints(0, 0)
    with pytest.raises(RuntimeError, match="new_lengths must not share memory"):
        extend_block_tables(table, None, lengths, added, free, head, 4, slots=slots, starts=starts,
                            new_lengths=lengths, new_head=ints(0))
    with pytest.raises(RuntimeError, match="new_head must not share memory"):
        extend_block_tables(table, None, lengths, added, free, head, 4, slots=slots, starts=starts,
                            new_lengths=ints(0), new_head=head)


def test_graph_replays(gpu):
    """A captured call replayed with new lengths: every replay equals the restatement."""
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    page, batch = 4, 3
    start = [[OLD] * 6 for _ in range(batch)]
    table, lengths, added, head = ints(start), ints([0] * batch), ints([5, 1, 3]), ints([0])
    free = ints(list(range(50, 90)))
    slots, starts, grown, next_head = ints([0] * 12), ints([0] * 4), ints([0] * 3), ints([0])

    def call():
        extend_block_tables(table, None, lengths, added, free, head, page, slots=slots, starts=starts,
                            new_lengths=grown, new_head=next_head)

    call()
    torch.cuda.synchronize()
    table.copy_(ints(start))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    held, want_head, want_table = [0] * batch, 0, [list(r) for r in start]
    for step in range(4):
        more = [5 - step, 1, 3 + step]
        added.copy_(ints(more))
        graph.replay()
        torch.cuda.synchronize()
        want = restate(want_table, None, held, more, list(range(50, 90)), want_head, page, 12)
        assert table.tolist() == want_table and slots.tolist() == want[0] and starts.tolist() == want[2]
        held, want_head = want[3], want[4]
        assert grown.tolist() == held and int(next_head) == want_head
        lengths.copy_(grown)
        head.copy_(next_head)
