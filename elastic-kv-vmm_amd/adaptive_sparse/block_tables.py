"""Block tables and slot maps of a serving step, built on the GPU from request lengths (HIP).

The reference extends its tables on the host, with a device read per step
(adaptive_sparse/request_residency.py:739-790, .tolist() and torch.tensor);
here one launch of csrc/block_tables.hip does it, so a step needs no host
round trip and can be captured in a HIP graph. The pages come from a device
list that the pool's owner fills with pages it has taken (PlanePagedPool.take);
the slot map is what scatter_kv takes to write the new tokens' rows, and the
new lengths and starts are what shared_prefix_attention takes.
"""

from elastic_kv import _native

from .profile_ranges import profile_range

TABLES_BAD_ROW = 1     # EKV_TABLES_BAD_ROW
TABLES_ROW_FULL = 2    # EKV_TABLES_ROW_FULL
TABLES_NO_PAGES = 4    # EKV_TABLES_NO_PAGES
TABLES_MAP_FULL = 8    # EKV_TABLES_MAP_FULL
TABLES_SLOT_RANGE = 16  # EKV_TABLES_SLOT_RANGE
TABLES_ID_RANGE = 32   # EKV_TABLES_ID_RANGE

_REASONS = (
    (TABLES_BAD_ROW, "a row names no request, or its length or new tokens are negative or past its table"),
    (TABLES_ROW_FULL, "a row's new tokens pass its table's columns"),
    (TABLES_NO_PAGES, "the free list ran out of pages"),
    (TABLES_MAP_FULL, "more new tokens than the slot map holds"),
    (TABLES_SLOT_RANGE, "a slot does not fit the slot map's type"),
    (TABLES_ID_RANGE, "a page id does not fit the int32 block table"),
)


@profile_range("native/block_tables")
def extend_block_tables(block_tables, rows, lengths, added, free_pages, free_head, page_size, *, slots, starts,
                        new_lengths, new_head, positions=None, status=None):
    """Extend every batch row's block table by `added` tokens and map the new tokens to slots.

    block_tables [R, M]; rows [B] (None: batch row b is request b): distinct
    requests; lengths, added [B]: tokens held and tokens new; free_pages [F]
    and free_head [1]: the page ids to take, in order, from entry free_head
    on. Each page that a row's new tokens open is written to block_tables;
    slots [N] gets page * page_size + offset of every new token, batch row
    after batch row, positions [N] its position; starts [B + 1] the rows'
    first tokens there, new_lengths [B] = lengths + added, new_head [1] the
    next unused entry of the free list. No output may share memory with an input
    or another output, so a call can be repeated or replayed. Places past the
    last token are -1. Index tensors are int32 or int64. What does not fit is
    left out and sets bits in status ([1] int32, OR-ed; check_table_status
    raises for them).
    """
    helper, entries = _native.launch_helper()
    result = helper.extend_tables(entries["ekv_extend_block_tables"], block_tables, rows, lengths, added, free_pages,
                                  free_head, int(page_size), slots, positions, starts, new_lengths, new_head, status)
    _native.launch_check(result, "extend_block_tables")


def check_table_status(status):
    """Raise if an extend_block_tables left something out since the last check (a synchronizing read); clears it."""
    flags = int(status.item())
    if flags:
        status.zero_()
        raise RuntimeError("extend_block_tables: " + "; ".join(text for bit, text in _REASONS if flags & bit))
