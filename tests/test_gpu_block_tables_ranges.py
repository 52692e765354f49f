"""extend_block_tables where a number does not fit the type that it is written in, and where tensors lie in one another."""

import pytest
import torch

from adaptive_sparse import block_tables
from adaptive_sparse.block_tables import TABLES_NO_PAGES, TABLES_SLOT_RANGE, check_table_status, extend_block_tables

pytestmark = pytest.mark.gpu

I32, I64 = torch.int32, torch.int64


def call(gpu, table, lengths, added, free, page, *, table_type=I32, slot_type=I64, head=0):
    """One call whose free list and head are int64: table, slots, next head, status."""
    total = sum(added)
    tensor = lambda v, kind: torch.tensor(v, dtype=kind, device=gpu)  # noqa: E731
    table = tensor(table, table_type)
    slots = torch.full((total,), -77, dtype=slot_type, device=gpu)
    starts, grown = tensor([0] * (len(lengths) + 1), I32), tensor([0] * len(lengths), I32)
    next_head, status = tensor([0], I64), tensor([0], I32)
    print(f"[tables] page {page} head {head} ids {free[:6]}", flush=True)
    extend_block_tables(table, None, tensor(lengths, I32), tensor(added, I32), tensor(free, I64), tensor([head], I64),
                        page, slots=slots, starts=starts, new_lengths=grown, new_head=next_head, status=status)
    assert grown.tolist() == [n + a for n, a in zip(lengths, added)]
    return table.tolist(), slots.tolist(), int(next_head), status


# 2^32 + 6 and 5 - 2^32 keep a page's number in their low words.
@pytest.mark.parametrize("wrong", [1 << 31, (1 << 32) + 6, 5 - (1 << 32), -(1 << 31) - 1, (1 << 62) + 3])
@pytest.mark.parametrize("slot_type", [I32, I64])
def test_a_page_id_that_an_int32_table_cannot_hold(gpu, wrong, slot_type):
    table, slots, head, status = call(gpu, [[9, 0, 0, 0]], [3], [10], [4, wrong, 7], 4, slot_type=slot_type)
    assert table == [[9, 4, 0, 7]]                      # the sink in its place
    assert slots == [39, 16, 17, 18, 19, -1, -1, -1, -1, 28]
    assert head == 3
    assert int(status) == block_tables.TABLES_ID_RANGE
    with pytest.raises(RuntimeError, match="a page id does not fit the int32 block table"):
        check_table_status(status)
    check_table_status(status)


def test_the_same_ids_in_an_int64_table(gpu):
    wide = (1 << 32) + 6
    table, slots, head, status = call(gpu, [[9, 0, 0, 0]], [3], [10], [4, wide, 7], 4, table_type=I64)
    assert table == [[9, 4, wide, 7]]
    assert slots == [39, 16, 17, 18, 19, *(wide * 4 + i for i in range(4)), 28]
    assert int(status) == 0


@pytest.mark.parametrize("wrong", [(1 << 61), (1 << 62) + 1, (1 << 63) - 1])
def test_a_slot_that_64_bits_cannot_hold(gpu, wrong):
    # 2^61 * 4 = 2^63; (2^62 + 1) * 4 would be 4 again.
    table, slots, head, status = call(gpu, [[wrong, 0, 0]], [3], [6], [4, wrong], 4, table_type=I64)
    assert table == [[wrong, 4, wrong]]
    assert slots == [-1, 16, 17, 18, 19, -1]
    assert int(status) == TABLES_SLOT_RANGE


def test_the_largest_slot_of_64_bits(gpu):
    most = ((1 << 63) - 4) // 4
    table, slots, head, status = call(gpu, [[0]], [0], [4], [most], 4, table_type=I64)
    assert table == [[most]] and slots == [most * 4 + i for i in range(4)] and slots[-1] == (1 << 63) - 1
    assert int(status) == 0


@pytest.mark.parametrize("head", [(1 << 63) - 1, (1 << 63) - 2, 1 << 40, -1, -(1 << 63)])
def test_heads_far_outside_the_list(gpu, head):
    table, slots, _, status = call(gpu, [[0, 0, 0]], [0], [9], [4, 5, 6], 4, head=head)
    assert int(status) == TABLES_NO_PAGES
    inside = [4, 5] if head == -1 else [0, 0]
    assert table == [[0, *inside]]
    assert slots == [-1] * 4 + ([16, 17, 18, 19, 20] if head == -1 else [-1] * 5)


def test_columns_of_one_tensor_do_not_share_memory(gpu):
    """Lengths, new lengths, heads and starts side by side in the rows of one tensor: no element is another's."""
    state = torch.tensor([[3, -77, 1, 0], [0, -77, 5, 1], [6, -77, 2, 2]], dtype=I32, device=gpu)
    heads = torch.tensor([1, -77], dtype=I32, device=gpu)
    table = torch.tensor([[9, 0, 0], [0, 0, 0], [7, 8, 0]], dtype=I32, device=gpu)
    slots, starts = torch.zeros(8, dtype=I32, device=gpu), torch.zeros(4, dtype=I32, device=gpu)
    status = torch.zeros(1, dtype=I32, device=gpu)
    extend_block_tables(table, state[:, 3], state[:, 0], state[:, 2], torch.tensor([1, 2, 3, 4], dtype=I32, device=gpu),
                        heads[:1], 4, slots=slots, starts=starts, new_lengths=state[:, 1], new_head=heads[1:],
                        status=status)
    assert state.tolist() == [[3, 4, 1, 0], [0, 5, 5, 1], [6, 8, 2, 2]]
    assert table.tolist() == [[9, 0, 0], [2, 3, 0], [7, 8, 0]]
    assert heads.tolist() == [1, 3] and starts.tolist() == [0, 1, 6, 8] and int(status) == 0
    assert slots.tolist() == [39, 8, 9, 10, 11, 12, 34, 35]
