"""select_blocks out of many candidates, at the numbers of places where the kernel that chooses changes, and for tokens of
prompts: the lists are those of the definition."""

import numpy as np
import pytest
import torch

from adaptive_sparse.block_selection import select_blocks

from block_cases import codes_of, make_batch, make_index_pool, selection

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def chosen_of(batch, pool, query, groups, chosen, block, first, last):
    """The lists of select_blocks [N, G, K] of long rows, all of whose pages are good."""
    tokens, heads, _ = query.shape
    codes, q_scale = codes_of(query)
    keys, scales = pool.keys.cpu().numpy(), pool.scales.cpu().numpy()
    out = np.full((tokens, groups, chosen), -1, np.int32)
    for n, (b, position) in enumerate(batch.places(tokens)):
        if b is None or position < 0:
            continue
        token = np.arange(position + 1)
        page = np.array(batch.table(b))[token // batch.page]
        inside = token % batch.page
        product = (keys[page, inside].astype(np.int32) @ codes[n].astype(np.int32).T).T
        scores = product.astype(np.float32) * scales[page * batch.page + inside]
        most = np.maximum.reduceat(scores, np.arange(0, position + 1, block), axis=1) * q_scale[n][:, None]
        most = most.reshape(groups, heads // groups, -1).max(1)
        j = np.arange(most.shape[1])
        forced = (j < first) | (j > position // block - last)
        for g in range(groups):
            rank = np.lexsort((j, np.where(forced, 0, -most[g]), ~forced))
            taken = np.sort(rank[:chosen])
            out[n, g, :len(taken)] = taken
    return torch.from_numpy(out)


def check(gpu, lengths, counts, heads, groups, dim, page, block, chosen, first, last, columns=0, small=False):
    batch = make_batch(gpu, lengths, counts, page, seed=dim + chosen)
    wide = max(columns - batch.tables.shape[1], 0)
    batch.tables = torch.cat([batch.tables, torch.zeros((len(lengths), wide), dtype=torch.int32, device=gpu)], 1)
    pool = make_index_pool(gpu, batch.pages, page, dim, seed=dim, small=small)
    tokens = sum(batch.counts)
    gen = torch.Generator(device=gpu).manual_seed(chosen)
    query = torch.randn((tokens, heads, dim), generator=gen, device=gpu).to(BF16)
    if small:
        query.fill_(1.0)
    blocks = torch.full((tokens, groups, chosen), 77, dtype=torch.int32, device=gpu)
    print(f"[select] {lengths} {counts} heads {heads} groups {groups} dim {dim}, {batch.tables.shape[1] * page} places, "
          f"blocks of {block}, {chosen} chosen", flush=True)
    select_blocks(query, pool.planes, pool.scales, batch.tables, batch.rows, batch.ints(batch.lengths), blocks,
                  page_size=page, block_size=block, layer=pool.layer, first=first, last=last, **batch.given(tokens))
    want = chosen_of(batch, pool, query, groups, chosen, block, first, last)
    assert torch.equal(blocks.cpu(), want)
    return batch, pool, query, want


LONG = [
    # lengths, page, block, chosen, first, last, columns
    ([256, 3, 200], 1, 1, 20, 1, 2, 256),                  # by one wave
    ([257, 3, 200], 1, 1, 20, 1, 2, 257),                  # by four
    ([2048, 700], 1, 1, 100, 1, 2, 2048),
    ([2049, 700], 1, 1, 100, 1, 2, 2049),                  # by sixteen, keys in registers
    ([16384, 700, 9000], 1, 1, 2048, 0, 1, 16384),
    ([16385, 700, 9000], 1, 1, 2048, 0, 1, 16385),         # in more of them
    ([40000, 1, 0, 12345], 16, 1, 2048, 0, 1, 0),
    ([40000, 33000], 16, 1, 31000, 3, 5, 0),
    ([65536, 17000], 16, 1, 512, 2, 2, 0),
    ([65000, 65536], 1, 1, 1, 0, 0, 65536),
    ([65537, 50000], 1, 1, 700, 1, 1, 65537),              # read again
    ([90001, 20000, 5], 1, 1, 4096, 1, 1, 0),
    ([100000, 65600], 16, 4, 300, 1, 1, 0),                # 25000 blocks of 4
    ([300000], 16, 16, 300, 1, 1, 0),                      # 18750 of 16
    ([30000, 20], 16, 1, 100, 0, 1, 8192),                 # a table far wider than its contexts
]


@pytest.mark.parametrize("small", [False, True], ids=["", "ties"])
@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_many_candidates(gpu, case, small):
    lengths, page, block, chosen, first, last, columns = case
    check(gpu, lengths, None, 2, 1, 32, page, block, chosen, first, last, columns, small)


def test_the_two_definitions_agree(gpu):
    given = ([700, 333], [3, 5], 4, 2, 32, 16, 20, 6, 1, 2)
    batch, pool, query, want = check(gpu, *given)
    assert torch.equal(selection(batch, pool, query, 2, 6, 20, 1, 2), want)


@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("block,heads,groups", [(1, 2, 2), (2, 2, 2), (1, 1, 1), (4, 4, 4), (1, 4, 2), (64, 3, 3)])
def test_prompts_that_choose_tokens_and_short_blocks(gpu, dim, block, heads, groups):
    """A head a group: 128 query tokens of it are a tile, and the scores of their tokens' steps take the most LDS."""
    check(gpu, [400, 230, 64], [130, 100, 64], heads, groups, dim, 16, block, 17, 1, 1)
