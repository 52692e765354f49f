"""select_blocks at scores next to the limits of 32-bit numbers: the lists are those of the definition, and nothing else is
written."""

import pytest
import torch

from adaptive_sparse.block_selection import select_blocks

from block_cases import make_batch, make_index_pool, selection

pytestmark = pytest.mark.gpu


def scored(gpu, scores, chosen, block=1, places=0, **given):
    """(lists, the definition's lists) of rows of one query token whose tokens have `scores`, in tables of `places` tokens.

    A key is 1 or -1 in its first element and a query 127 with a scale of 1, so a token's score is its sign times 127 times
    its scale, but for the roundings. Nothing may be written outside the lists.
    """
    batch = make_batch(gpu, [len(s) for s in scores], None, 16, seed=3, permute=False)
    wide = max(places // 16 - batch.tables.shape[1], 0)
    batch.tables = torch.cat([batch.tables, torch.zeros((len(scores), wide), dtype=torch.int32, device=gpu)], 1)
    pool = make_index_pool(gpu, batch.pages, 16, 16, seed=3)
    pool.keys.zero_()
    for b, row in enumerate(scores):
        position = torch.arange(len(row), device=gpu)
        page = batch.tables[b, position // 16].long()
        pool.keys[page, position % 16, 0] = torch.where(row < 0, -1, 1).to(torch.int8)
        pool.scales[page * 16 + position % 16] = (row.double().abs() / 127).float()
    query = torch.zeros((len(scores), 1, 16), dtype=torch.bfloat16, device=gpu)
    query[:, :, 0] = 127
    memory = torch.full((len(scores) + 2, 1, chosen), 77, dtype=torch.int32, device=gpu)
    blocks = memory[1:-1]
    print(f"[select] {[len(s) for s in scores]} of {chosen}, {batch.tables.shape[1] * 16} places", flush=True)
    select_blocks(query, pool.planes, pool.scales, batch.tables, None, batch.ints(batch.lengths), blocks, page_size=16,
                  block_size=block, layer=pool.layer, **given)
    torch.cuda.synchronize()
    assert bool((memory[0] == 77).all()) and bool((memory[-1] == 77).all()), "written outside the lists"
    return blocks.cpu(), selection(batch, pool, query, 1, chosen, block, given.get("first", 0), given.get("last", 1))


PLACES = [4096, 20000, 70000]            # keys in few registers, in many, read again


@pytest.mark.parametrize("places", PLACES)
@pytest.mark.parametrize("factor", [1.0, 1e-2, -1.0])
def test_many_scores_alike_far_below_zero(gpu, places, factor):
    """One part of the range holds more scores than are compared with each other, and begins near the lowest number."""
    row = torch.full((4096,), -1e37, device=gpu)
    row[100], row[200] = -2e38, -1e36
    got, want = scored(gpu, [row * factor, row[:3500] * factor], 512, places=places, last=0)
    assert torch.equal(got, want)


@pytest.mark.parametrize("places", PLACES)
def test_the_lowest_scores_are_reached(gpu, places):
    row = torch.full((2500,), -1e38, device=gpu)
    row[::1000] = 0.0
    row[5] = -3e38
    for chosen in (3, 300, 2499):
        got, want = scored(gpu, [row, row.flip(0)], chosen, places=places, last=0)
        assert torch.equal(got, want)


@pytest.mark.parametrize("places", PLACES)
@pytest.mark.parametrize("low,high", [(36.0, 38.4), (-44.0, 38.4), (-45.0, -38.0)])
def test_scores_of_all_magnitudes(gpu, places, low, high):
    gen = torch.Generator(device=gpu).manual_seed(9)
    rows = []
    for n in (3000, 2200):
        size = 10.0 ** (low + (high - low) * torch.rand(n, generator=gen, device=gpu, dtype=torch.float64))
        sign = torch.where(torch.rand(n, generator=gen, device=gpu) < 0.9, -1.0, 1.0)
        rows.append((size * sign).float())
    for chosen in (64, 1500):
        got, want = scored(gpu, rows, chosen, places=places, first=2)
        assert torch.equal(got, want)


@pytest.mark.parametrize("places", [256, 1024, *PLACES])
@pytest.mark.parametrize("block", [1, 2, 4, 16, 100])
def test_scores_past_the_lowest_number_are_scores(gpu, places, block):
    """Blocks whose products pass the lowest number are the last to be chosen, but are chosen: no block is without a score."""
    print(f"[select] blocks of {block}, {places} places", flush=True)
    batch = make_batch(gpu, [240, 33], None, 16, seed=4, permute=False)
    pool = make_index_pool(gpu, batch.pages, 16, 16, seed=4)
    wide = max(places // 16 - batch.tables.shape[1], 0)
    batch.tables = torch.cat([batch.tables, torch.zeros((2, wide), dtype=torch.int32, device=gpu)], 1)
    pool.keys.zero_()
    pool.keys[..., 0] = -1
    pool.scales.fill_(3e38)                                         # 127 times it passes the lowest number
    # The scores of the first two blocks of the long row do not.
    for t in range(2 * block):
        pool.scales[int(batch.tables[0, t // 16]) * 16 + t % 16] = 1.0 + t // block
    query = torch.zeros((2, 1, 16), dtype=torch.bfloat16, device=gpu)
    query[:, :, 0] = 127
    for chosen, first, last in ((1, 0, 1), (3, 0, 1), (3, 0, 0), (4, 2, 1), (300, 0, 0)):
        blocks = torch.full((2, 1, chosen), 77, dtype=torch.int32, device=gpu)
        select_blocks(query, pool.planes, pool.scales, batch.tables, None, batch.ints(batch.lengths), blocks,
                      page_size=16, block_size=block, layer=pool.layer, first=first, last=last)
        for b, length in enumerate(batch.lengths):
            count = (length - 1) // block + 1
            cost = [1.0 + j if b == 0 and j < 2 else float("inf") for j in range(count)]
            rank = sorted(range(count), key=lambda j: (not (j < first or j >= count - last), cost[j], j))
            want = sorted(rank[:chosen])
            assert blocks[b, 0].tolist() == want + [-1] * (chosen - len(want))


@pytest.mark.parametrize("counts", [None, [70, 90]])
def test_scores_past_the_largest_number_go_to_lower_blocks(gpu, counts):
    batch = make_batch(gpu, [300, 200], counts, 16, seed=5)
    pool = make_index_pool(gpu, batch.pages, 16, 16, seed=5)
    pool.keys.zero_()
    pool.keys[..., 0] = 1
    pool.scales.fill_(3e38)
    tokens = sum(batch.counts)
    query = torch.zeros((tokens, 2, 16), dtype=torch.bfloat16, device=gpu)
    query[:, 0, 0] = 127                                            # the other head's scores are 0
    blocks = torch.full((tokens, 1, 3), 77, dtype=torch.int32, device=gpu)
    for block in (1, 8, 64):
        select_blocks(query, pool.planes, pool.scales, batch.tables, batch.rows, batch.ints(batch.lengths), blocks,
                      page_size=16, block_size=block, layer=pool.layer, last=0, **batch.given(tokens))
        for n, (_, position) in enumerate(batch.places(tokens)):
            count = min(position // block + 1, 3)
            assert blocks[n, 0].tolist() == list(range(count)) + [-1] * (3 - count)
