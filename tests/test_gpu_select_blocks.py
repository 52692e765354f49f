"""select_blocks against the definition: the lists are the same, whatever the layout, the sizes or the split."""

import pytest
import torch

from adaptive_sparse.block_selection import select_blocks, selection_workspace
from adaptive_sparse.resident_lookup import resolve_resident

from block_cases import make_batch, make_index_pool, selection

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def choose(batch, pool, query, groups, chosen, block, first, last, **extra):
    tokens = query.shape[0]
    blocks = torch.full((tokens, groups, chosen), 77, dtype=torch.int32, device=query.device)
    given = dict(page_size=batch.page, block_size=block, layer=pool.layer, first=first, last=last)
    given.update(batch.given(tokens))
    given.update(extra)
    select_blocks(query, pool.planes, pool.scales, batch.tables, batch.rows, batch.ints(batch.lengths), blocks, **given)
    return blocks


def queries(gpu, tokens, heads, dim, dtype=BF16, seed=0):
    gen = torch.Generator(device=gpu).manual_seed(seed + 11)
    return torch.randn((tokens, heads, dim), generator=gen, device=gpu).to(dtype)


CASES = [
    # lengths, query tokens, heads, groups, index size, page, layout, block, chosen, first, last
    ([1], None, 1, 1, 16, 16, "planes", 16, 1, 0, 1),
    ([0, 1, 63, 64, 65, 700], None, 4, 1, 128, 16, "planes", 64, 4, 1, 1),
    ([300, 1000, 5], None, 8, 2, 64, 1, "planes", 32, 6, 0, 0),
    ([300, 999, 5], None, 6, 3, 32, 100, "blocks", 100, 3, 1, 2),       # blocks that no step divides
    ([129, 640], None, 4, 4, 48, 64, "blocks", 20, 7, 2, 1),            # blocks shorter than a step
    ([200, 2000], None, 5, 1, 80, 16, "planes", 1, 40, 3, 5),           # tokens
    ([200, 1500], None, 2, 2, 256, 16, "planes", 2, 33, 0, 1),
    ([77, 900], None, 3, 1, 128, 3, "planes", 4, 64, 0, 1),
    ([77, 900], None, 16, 1, 128, 16, "blocks", 8, 17, 1, 1),
    ([500, 901], None, 17, 1, 64, 16, "planes", 16, 5, 0, 1),           # 32 rows
    ([500, 901], None, 64, 1, 64, 16, "planes", 37, 5, 0, 1),
    ([500, 901], None, 128, 1, 64, 16, "planes", 64, 5, 0, 1),          # a group of 128 heads
    ([500, 901], None, 256, 2, 128, 16, "planes", 64, 5, 0, 1),
    ([40, 500, 333], [3, 1, 7], 4, 2, 128, 16, "planes", 32, 4, 1, 1),  # drafted tokens
    ([300, 90, 450], [100, 90, 3], 4, 2, 128, 16, "planes", 64, 3, 0, 1),
    ([300, 90, 450], [100, 90, 3], 2, 1, 256, 16, "blocks", 64, 3, 0, 1),
    ([150, 60], [70, 1], 3, 1, 64, 16, "planes", 1, 20, 0, 1),
    ([150, 60], [150, 60], 1, 1, 16, 16, "planes", 16, 2, 0, 0),        # 128 tokens a tile
    ([5000, 4100], None, 4, 1, 64, 64, "planes", 4, 100, 0, 1),         # more than 1024 blocks
    ([3000, 2500], None, 4, 2, 64, 64, "planes", 1, 2048, 1, 1),
    ([20000, 333], None, 2, 1, 64, 16, "planes", 16384, 1, 0, 0),       # a block of several segments' length
]


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{'-'.join(map(str, c[2:]))}".replace(" ", ""))
def test_selection(gpu, case, index):
    lengths, counts, heads, groups, dim, page, layout, block, chosen, first, last = case
    print(f"[select] {case} {index}", flush=True)
    batch = make_batch(gpu, lengths, counts, page, index, seed=dim)
    pool = make_index_pool(gpu, batch.pages, page, dim, layout, seed=dim)
    query = queries(gpu, sum(batch.counts), heads, dim, F16 if index == torch.int64 else BF16)
    want = selection(batch, pool, query, groups, chosen, block, first, last)
    got = choose(batch, pool, query, groups, chosen, block, first, last).cpu()
    assert torch.equal(got, want)


@pytest.mark.parametrize("block", [1, 16, 64])
@pytest.mark.parametrize("counts", [None, [9, 40]])
def test_equal_scores_go_to_lower_blocks(gpu, block, counts):
    batch = make_batch(gpu, [1900, 800], counts, 16, seed=5)
    pool = make_index_pool(gpu, batch.pages, 16, 16, seed=5, small=True)
    query = torch.ones((sum(batch.counts), 2, 16), dtype=BF16, device=gpu)
    want = selection(batch, pool, query, 1, 12, block, 0, 0)
    assert torch.equal(choose(batch, pool, query, 1, 12, block, 0, 0).cpu(), want)
    # All scores alike: the first blocks.
    query.zero_()
    got = choose(batch, pool, query, 2, 12, block, 0, 0).cpu()
    for n, (b, position) in enumerate(batch.places(query.shape[0])):
        count = min(12, position // block + 1)
        assert got[n, 0].tolist() == list(range(count)) + [-1] * (12 - count)


def test_rows_that_name_no_request_bad_pages_and_lengths(gpu):
    batch = make_batch(gpu, [300, 640, 100, 200], None, 16, seed=2)
    pool = make_index_pool(gpu, batch.pages, 16, 64, seed=2)
    query = queries(gpu, 4, 4, 64)
    batch.rows = batch.rows.clone()
    place = int(batch.rows[1])
    batch.tables[place, 0:4] = 0                    # the sink: block 0 has no token
    batch.tables[place, 5] = batch.pages            # past the pool
    batch.tables[place, 9] = -3
    batch.rows[2] = 4                               # no such request
    batch.rows[3] = -1
    for first, last in ((0, 0), (2, 1)):
        want = selection(batch, pool, query, 2, 5, 64, first, last)
        assert torch.equal(choose(batch, pool, query, 2, 5, 64, first, last).cpu(), want)
        assert bool((want[2:] == -1).all()) and 0 not in want[1].tolist()[0]
    # A length past the table, and one below zero.
    batch.lengths = [300, 5000, 100, -7]
    batch.rows[2:] = torch.tensor([0, 1], device=gpu)
    want = selection(batch, pool, query, 2, 5, 64, 1, 1)
    assert torch.equal(choose(batch, pool, query, 2, 5, 64, 1, 1).cpu(), want)


def test_scales_of_tokens_that_are_not_seen_do_not_matter(gpu):
    batch = make_batch(gpu, [100, 333], [3, 2], 16, seed=4)
    pool = make_index_pool(gpu, batch.pages, 16, 128, seed=4)
    query = queries(gpu, 5, 4, 128)
    want = selection(batch, pool, query, 1, 3, 32, 0, 1)
    for b, length in enumerate(batch.lengths):
        table = batch.table(b)
        at = table[length // 16] * 16 if length // 16 < len(table) else 0
        pool.scales[at + length % 16:at + 16] = float("nan") if b else float("inf")
    pool.scales[:16] = float("nan")
    assert torch.equal(choose(batch, pool, query, 1, 3, 32, 0, 1).cpu(), want)


@pytest.mark.parametrize("scale", [0.0, -0.25])
def test_scales_of_zero_and_below(gpu, scale):
    batch = make_batch(gpu, [700], None, 16, seed=6)
    pool = make_index_pool(gpu, batch.pages, 16, 64, seed=6)
    pool.scales[::3] = scale
    query = queries(gpu, 1, 2, 64)
    want = selection(batch, pool, query, 1, 6, 16, 0, 0)
    assert torch.equal(choose(batch, pool, query, 1, 6, 16, 0, 0).cpu(), want)


@pytest.mark.parametrize("most", [1, 9, 1000])
def test_the_hint_does_not_change_what_is_chosen(gpu, most):
    batch = make_batch(gpu, [400, 90, 77], [30, 1, 9], 16, seed=8)
    pool = make_index_pool(gpu, batch.pages, 16, 64, seed=8)
    query = queries(gpu, 43, 4, 64)           # three tokens of no batch row behind the others
    want = selection(batch, pool, query, 2, 3, 16, 1, 1)
    got = choose(batch, pool, query, 2, 3, 16, 1, 1, max_query=most)
    assert torch.equal(got.cpu(), want) and bool((got[40:] == -1).all())


def test_strided_outputs_wide_tables_and_a_workspace(gpu):
    batch = make_batch(gpu, [900, 350], None, 16, seed=9, permute=False)
    pool = make_index_pool(gpu, batch.pages, 16, 64, seed=9)
    batch.tables = torch.cat([batch.tables, torch.full((2, 4000), -1, dtype=torch.int32, device=gpu)], 1)
    query = queries(gpu, 2, 4, 64)
    both = torch.full((9, 2, 2, 3), 55, dtype=torch.int32, device=gpu)
    blocks = both.permute(2, 1, 0, 3)[..., 1]                              # [2, 2, 9], no dimension dense
    workspace = torch.empty(selection_workspace(2, 2, batch.tables.shape[1], 16, 32), dtype=torch.uint8, device=gpu)
    workspace.fill_(255)
    select_blocks(query, pool.planes, pool.scales, batch.tables, None, batch.ints(batch.lengths), blocks, page_size=16,
                  block_size=32, layer=1, first=1, last=1, workspace=workspace)
    assert torch.equal(blocks.cpu(), selection(batch, pool, query, 2, 9, 32, 1, 1))
    assert bool((both[..., 0] == 55).all()) and bool((both[..., 2] == 55).all())


def test_replays_in_a_graph_with_other_lengths(gpu):
    batch = make_batch(gpu, [900, 350, 640], None, 16, seed=10)
    pool = make_index_pool(gpu, batch.pages, 16, 128, seed=10)
    query = queries(gpu, 3, 4, 128)
    lengths = batch.ints(batch.lengths)
    blocks = torch.zeros((3, 2, 6), dtype=torch.int32, device=gpu)
    size = selection_workspace(3, 2, batch.tables.shape[1], 16, 64)
    workspace = torch.empty(size, dtype=torch.uint8, device=gpu)
    run = lambda: select_blocks(query, pool.planes, pool.scales, batch.tables, batch.rows, lengths, blocks,  # noqa: E731
                                page_size=16, block_size=64, layer=1, workspace=workspace)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run()
    torch.cuda.synchronize()
    for step in range(3):
        batch.lengths = [900 - 250 * step, 350 - step, 640 - 64 * step]
        lengths.copy_(batch.ints(batch.lengths))
        query.copy_(queries(gpu, 3, 4, 128, seed=step + 20))
        blocks.fill_(99)
        graph.replay()
        torch.cuda.synchronize()
        want = selection(batch, pool, query, 2, 6, 64, 0, 1)
        assert torch.equal(blocks.cpu(), want)


def test_the_resident_lookup_takes_the_lists(gpu):
    batch = make_batch(gpu, [900, 350], None, 16, seed=12, permute=False)
    pool = make_index_pool(gpu, batch.pages, 16, 64, seed=12)
    query = queries(gpu, 2, 4, 64)
    topk = torch.zeros((1, 2, 5), dtype=torch.int32, device=gpu)           # the lookup's [L, B, K]
    select_blocks(query, pool.planes, pool.scales, batch.tables, None, batch.ints(batch.lengths),
                  topk[0].unsqueeze(1), page_size=16, block_size=32, layer=1)
    width = batch.tables.shape[1] * 16
    position = torch.arange(width, device=gpu)
    table = (batch.tables[:, position // 16] * 16 + position % 16).to(torch.int32)
    slots = torch.full((1, 2, 5 * 32), -7, dtype=torch.int32, device=gpu)
    rows = torch.arange(2, device=gpu)
    resolve_resident(topk, table, None, rows, batch.ints(batch.lengths), rows, slots, 32)
    want = selection(batch, pool, query, 1, 5, 32, 0, 1)[:, 0]
    for b, length in enumerate(batch.lengths):
        tokens = [j * 32 + i for j in want[b].tolist() for i in range(32)]
        expected = [int(table[b, t]) if 0 <= t < length else -1 for t in tokens]
        assert slots[0, b].tolist() == expected


@pytest.mark.parametrize("chosen,first,last", [(1, 0, 1), (7, 3, 4), (300, 1, 1), (2500, 1000, 1500), (2100, 0, 0)])
def test_many_blocks_of_equal_and_forced_scores(gpu, chosen, first, last):
    """Lists of tokens: scores with few values, lists as long as what is always chosen, longer than the context."""
    batch = make_batch(gpu, [2400, 130, 2050], None, 64, seed=13)
    pool = make_index_pool(gpu, batch.pages, 64, 16, seed=13, small=True)
    query = torch.ones((3, 1, 16), dtype=BF16, device=gpu)
    want = selection(batch, pool, query, 1, chosen, 1, first, last)
    assert torch.equal(choose(batch, pool, query, 1, chosen, 1, first, last).cpu(), want)
    batch.tables = torch.cat([batch.tables, torch.zeros((3, 1100), dtype=torch.int32, device=gpu)], 1)   # > 65536 places
    assert torch.equal(choose(batch, pool, query, 1, chosen, 1, first, last).cpu(), want)
