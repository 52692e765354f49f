"""The Top-K blocks of a context for every query token, by scores from 8-bit index keys (HIP).

The reference takes the selected blocks from its engine
(adaptive_sparse/request_residency.py:792-839). These kernels
(csrc/select_blocks.hip) make them: what resolve_resident, decode_step and
load_blocks_to_device_buffer_mha take as `topk`, and block_attention as its
lists.
"""

import torch

from elastic_kv import _native

from .kv_pool import KVPlanes
from .profile_ranges import profile_range


def selection_workspace(tokens, groups, columns, page_size, block_size):
    """Bytes of workspace that select_blocks needs for [tokens, groups] lists and tables of `columns` pages."""
    lib = _native.kernel_library()
    size = lib.ekv_select_workspace_bytes(int(tokens), int(groups), int(columns), int(page_size), int(block_size))
    if size == (1 << 64) - 1:
        raise ValueError(lib.ev_error().decode())
    return size


@profile_range("native/select_blocks")
def select_blocks(index_query, planes, scales, block_tables, rows, lengths, blocks, *, page_size, block_size, layer=0,
                  query_starts=None, max_query=1, first=0, last=1, workspace=None):
    """Choose the blocks of largest score for every query token and group of index heads, into `blocks`.

    index_query [N, Hi, Di] bfloat16 or float16, finite (rotated already);
    planes, scales: the index keys that append_index wrote. blocks [N, G, K]
    int32, any strides: G lists a token, each of Hi / G heads; a list is in
    ascending order, -1 behind its last block. block_tables [R, M], rows [B]
    (None: batch row b is request b), lengths [B], query_starts [B + 1] (None:
    one token a row) as in shared_prefix_attention: token i of a row's n is at
    position lengths[b] - n + i and sees the tokens up to it. max_query: the
    most query tokens of a row, as far as known: it picks kernels, never what
    is chosen.
    A block's score is the largest, over a group's heads and the block's seen
    tokens, of the product of query and key as they are held in 8 bits, and one
    past the largest or the lowest number of 32 bits counts as that. The
    `first` blocks of the context and the `last` up to the position's own are
    chosen whatever their scores; ties go to the lower block. block_size = 1
    chooses tokens. workspace: a uint8 device tensor of selection_workspace(...)
    bytes (None: one from torch's allocator); calls on several streams need one
    each.
    """
    if not isinstance(planes, KVPlanes):
        raise TypeError("planes must be a KVPlanes")
    if blocks.dim() != 3 or block_tables.dim() != 2:
        raise ValueError("blocks must be shaped [tokens, groups, K] and block_tables [requests, pages]")
    if workspace is None:
        size = selection_workspace(blocks.shape[0], blocks.shape[1], block_tables.shape[1], page_size, block_size)
        workspace = torch.empty(size, dtype=torch.uint8, device=blocks.device)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    helper, entries = _native.launch_helper()
    status = helper.select_blocks(entries["ekv_select_blocks"], index_query, planes, layer, page_size, block_size,
                                  scales, block_tables, rows, lengths, query_starts, max_query, first, last, blocks,
                                  workspace)
    _native.launch_check(status, "select_blocks")
