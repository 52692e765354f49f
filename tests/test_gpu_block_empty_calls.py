"""The block-sparse operators where there is nothing to choose from or to attend to: no batch rows, tokens or blocks."""

import math

import pytest
import torch

from adaptive_sparse.attention import block_attention
from adaptive_sparse.block_selection import select_blocks

from attention_cases import make_pool
from block_cases import make_index_pool

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("tokens,heads,groups,most", [(1, 8, 2, 1), (3, 4, 4, 1), (70, 2, 1, 64), (300, 4, 2, 300)])
@pytest.mark.parametrize("columns", [4, 200, 1200, 5000])
def test_tokens_without_a_batch_row_select_nothing(gpu, tokens, heads, groups, most, columns):
    print(f"[select] {tokens} tokens of no row, {heads} heads, {groups} groups, {columns} pages", flush=True)
    pool = make_index_pool(gpu, 8, 16, 64)
    query = torch.randn((tokens, heads, 64), device=gpu).to(BF16)
    tables = torch.zeros((2, columns), dtype=torch.int32, device=gpu)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    starts = torch.zeros(1, dtype=torch.int32, device=gpu)
    blocks = torch.full((tokens, groups, 5), 77, dtype=torch.int32, device=gpu)
    for rows in (None, none):
        blocks.fill_(77)
        select_blocks(query, pool.planes, pool.scales, tables, rows, none, blocks, page_size=16, block_size=16, layer=1,
                      query_starts=starts, max_query=most)
        assert bool((blocks == -1).all())


@pytest.mark.parametrize("batch", [0, 2])
def test_no_tokens_select_nothing(gpu, batch):
    pool = make_index_pool(gpu, 8, 16, 64)
    ints = lambda n: torch.zeros(n, dtype=torch.int32, device=gpu)  # noqa: E731
    select_blocks(torch.empty((0, 4, 64), dtype=BF16, device=gpu), pool.planes, pool.scales, ints((2, 4)), None, ints(batch),
                  ints((0, 2, 5)), page_size=16, block_size=16, layer=1, query_starts=ints(batch + 1), max_query=4)


@pytest.mark.parametrize("tokens,heads,kv_heads,most", [(16, 128, 128, 64), (1, 8, 2, 1), (63, 64, 64, 64), (70, 64, 32, 64),
                                                        (2100, 8, 2, 1000)])
@pytest.mark.parametrize("dim", [64, 256])
def test_tokens_without_a_batch_row_attend_to_nothing(gpu, tokens, heads, kv_heads, most, dim):
    print(f"[blocks] {tokens} tokens of no row, {heads} heads, {kv_heads} KV heads of {dim}", flush=True)
    pool = make_pool(gpu, BF16, 4, 16, kv_heads, dim)
    query = torch.randn((tokens, heads, dim), device=gpu).to(BF16)
    tables = torch.ones((2, 40), dtype=torch.int32, device=gpu)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    starts = torch.zeros(1, dtype=torch.int32, device=gpu)
    blocks = torch.zeros((tokens, 1, 3), dtype=torch.int32, device=gpu)
    out = torch.full_like(query, 7.0)
    lse = torch.full((tokens, heads), 7.0, device=gpu)
    block_attention(query, pool.planes, tables, None, none, blocks, out, page_size=16, block_size=32, kv_heads=kv_heads,
                    layer=pool.layer, query_starts=starts, max_query=most, lse=lse)
    assert not bool(out.any()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("share", [1, 4])
def test_prompts_with_lists_of_no_entries(gpu, share):
    """As many tokens as go through their lists together where there are entries."""
    tokens, kv_heads = 2100, 2
    pool = make_pool(gpu, BF16, 200, 16, kv_heads, 64)
    query = torch.randn((tokens, share * kv_heads, 64), device=gpu).to(BF16)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=gpu)  # noqa: E731
    tables = torch.arange(1, 133, dtype=torch.int32, device=gpu).view(1, -1)
    out = torch.full_like(query, 7.0)
    lse = torch.full(out.shape[:2], 7.0, device=gpu)
    block_attention(query, pool.planes, tables, None, ints([tokens]), torch.empty((tokens, 1, 0), dtype=torch.int32,
                                                                                  device=gpu),
                    out, page_size=16, block_size=32, kv_heads=kv_heads, layer=pool.layer, query_starts=ints([0, tokens]),
                    max_query=tokens, lse=lse)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
