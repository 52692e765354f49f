"""Workspace sizes of the attentions (CPU only): parts of cut items, not a copy of the output.

Where an item that one workgroup has whole is written to the output, a workgroup leaves two parts at most, each of a row
tile of 32-bit values and two statistics a row. There are at most 512 workgroups of tiles of 128 rows or fewer and 256 of
tiles of 256 rows.
"""

import pytest

from adaptive_sparse.attention import shared_prefix_workspace, topk_workspace

SPARE = 4096     # three arrays' alignment


@pytest.mark.parametrize("tokens", [16384, 32768, 1 << 20])
@pytest.mark.parametrize("groups", [0, 1])
def test_prompts(tokens, groups):
    """Eight rows' prompt pieces, 64 query heads of 128 over 8 KV heads."""
    assert shared_prefix_workspace(tokens, 8, groups, 64, 8, 128, tokens // 8) <= 2 * 256 * 256 * (128 + 2) * 4 + SPARE


@pytest.mark.parametrize("batch", [1000, 10000])
def test_decode_without_a_prefix(batch):
    size = shared_prefix_workspace(batch, batch, 0, 64, 8, 128)
    assert size <= 2 * 512 * 16 * (128 + 2) * 4 + 8 * batch + SPARE


@pytest.mark.parametrize("tokens", [1000, 100000])
@pytest.mark.parametrize("heads,kv_heads,dim,rows", [(64, 8, 128, 16), (64, 2, 64, 32), (64, 1, 128, 64),
                                                     (128, 1, 256, 128), (256, 1, 96, 256)])
def test_topk(tokens, heads, kv_heads, dim, rows):
    assert topk_workspace(tokens, 2048, heads, kv_heads, dim) <= 2 * 512 * rows * (dim + 2) * 4 + SPARE


def test_small_calls_take_a_part_per_workgroup_and_item():
    assert topk_workspace(4, 256, 16, 2, 128) <= (512 + 8 + 8) * 16 * (128 + 2) * 4 + SPARE
