"""Attention over the paged K/V pool (HIP): behind a shared prefix, and over Top-K slots.

The reference resolves which pool rows a decode step reads - a shared
prefix's blocks (adaptive_sparse/shared_prefix.py:122-204) or the selected
Top-K slots (adaptive_sparse/request_residency.py:792-839) - and leaves the
attention to its engine. These calls read the same rows where they lie, with
no gather in between; the kernels are in csrc/attention.hip. One call serves
one layer.
"""

import torch

from elastic_kv import _native

from .kv_pool import KVPlanes
from .profile_ranges import profile_range


def _size(entry, *sizes):
    lib = _native.kernel_library()
    size = getattr(lib, entry)(*map(int, sizes))
    if size == (1 << 64) - 1:
        raise ValueError(lib.ev_error().decode())
    return size


def shared_prefix_workspace(tokens, batch, groups, query_heads, kv_heads, head_dim, max_query=1):
    """Bytes of workspace that shared_prefix_attention needs for these sizes."""
    return _size("ekv_shared_prefix_workspace_bytes", tokens, batch, groups, query_heads, kv_heads, head_dim,
                 max_query)


def topk_workspace(tokens, lanes, query_heads, kv_heads, head_dim):
    """Bytes of workspace that topk_attention needs for these sizes."""
    return _size("ekv_topk_workspace_bytes", tokens, lanes, query_heads, kv_heads, head_dim)


def _check(query, planes, workspace):
    if not isinstance(planes, KVPlanes):
        raise TypeError("planes must be a KVPlanes")
    if query.dim() != 3:
        raise ValueError("query must be shaped [tokens, heads, head_dim]")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")


def _scale(scale, dim):
    return max(dim, 1) ** -0.5 if scale is None else scale    # a head size of 0 is the entry point's to refuse


@profile_range("native/prefix_attention")
def shared_prefix_attention(query, planes, block_tables, rows, lengths, prefix_tables, prefix_lengths, output, *,
                            page_size, kv_heads, layer=0, group_starts=None, query_starts=None, max_query=1,
                            scale=None, lse=None, workspace=None):
    """Attention of every batch row to its group's shared prefix and to its own tokens, into `output`.

    query, output [N, Hq, D] bfloat16 or float16; query head h reads KV head
    h // (Hq // kv_heads). planes: the pool's KVPlanes, a plane row holding a
    token ([kv_heads, D]) or a whole page ([page_size, kv_heads, D]).
    block_tables [R, M], rows [B] (None: batch row b is request b), lengths
    [B]: the own pages and tokens of each batch row, the new tokens (whose K/V
    are in the pool already) among them. query_starts [B + 1]: first query
    token of each row (None: one token a row); token i of n sees the prefix and
    own tokens 0 .. lengths[b] - n + i. max_query: the most query tokens of a
    row, as far as known: it picks kernels, never which keys are seen.
    prefix_tables [G, P], prefix_lengths [G], group_starts [G + 1]: the groups
    of consecutive batch rows and their prefixes (group_starts None: one group
    of all rows; prefix_tables None: no prefix). With query rows = query tokens
    * Hq // kv_heads: if max_query makes 64 of them at most and a group has more
    on average, K and V of a prefix are read once per 128 query rows of its
    group, else once per batch row and tile of its rows. One choice serves the
    whole call: many decode rows and a few prompt pieces behind a long prefix
    are faster as two calls.
    A page id below 1 or past the pool is not seen (page 0 is the sink); a
    query token that sees nothing gets zeros and lse -inf. lse [N, Hq] float32:
    log of the sum of exp(scale q.k), which merges outputs of other parts.
    scale: D ** -0.5 by default. workspace: a uint8 device tensor of
    shared_prefix_workspace(...) bytes (None: one from torch's allocator); calls
    on several streams need one each.
    """
    _check(query, planes, workspace)
    tokens, heads, dim = query.shape
    if workspace is None:
        groups = prefix_tables.shape[0] if prefix_tables is not None else 0
        size = shared_prefix_workspace(tokens, lengths.shape[0], groups, heads, kv_heads, dim, max_query)
        workspace = torch.empty(size, dtype=torch.uint8, device=query.device)
    helper, entries = _native.launch_helper()
    status = helper.prefix_attention(entries["ekv_shared_prefix_attention"], query, planes, int(layer), int(kv_heads),
                                     int(page_size), block_tables, rows, lengths, prefix_tables, prefix_lengths,
                                     group_starts, query_starts, int(max_query),
                                     _scale(scale, dim), output, lse, workspace)
    _native.launch_check(status, "shared_prefix_attention")


@profile_range("native/topk_attention")
def topk_attention(query, planes, slots, output, *, kv_heads, layer=0, scale=None, lse=None, zero_below=1,
                   workspace=None):
    """Decode attention of each query token to its Top-K slots, into `output`: one layer, no gather.

    query, output [N, Hq, D] bfloat16 or float16; planes: the hot pool, a plane
    row holding a token ([kv_heads, D]); slots [N, K] int32 or int64, the slots
    that resolve_resident or decode_step returned for this layer (any strides).
    Lanes with slot < zero_below (0: not resident, -1: padding) or past the
    pool are not seen and not read; a slot listed twice counts twice. A token
    that sees nothing gets zeros and lse -inf. lse, scale and workspace
    (topk_workspace(...) bytes) as in shared_prefix_attention.
    """
    _check(query, planes, workspace)
    tokens, heads, dim = query.shape
    if slots.dim() != 2:
        raise ValueError("slots must be shaped [tokens, K]")
    if workspace is None:
        size = topk_workspace(tokens, slots.shape[1], heads, kv_heads, dim)
        workspace = torch.empty(size, dtype=torch.uint8, device=query.device)
    helper, entries = _native.launch_helper()
    status = helper.topk_attention(entries["ekv_topk_attention"], query, planes, int(layer), int(kv_heads), slots,
                                   int(zero_below), _scale(scale, dim), output, lse, workspace)
    _native.launch_check(status, "topk_attention")
