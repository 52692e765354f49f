"""Attention with tables so wide that a launch's places would pass 31 bits, and starts out of order whose places do.

Work is cut in units of keys that are counted over all rows, row tiles and KV heads from the tables' widths; where
those counts could pass 31 bits the unit is made larger. The tables here are 2^30 - 16 tokens wide, their rows
overlapping windows of one list of page ids, so that they cost one row's memory. The bounds are those of
attention_cases.py.
"""

import pytest
import torch

from adaptive_sparse.attention import shared_prefix_attention

from attention_cases import check, make_problem

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
PAGE = 16
COLUMNS = ((1 << 30) - 1) // PAGE       # of the widest table


def widen(table):
    """The table with its columns in front of others up to COLUMNS, which hold the next rows' ids and then 0."""
    rows, step = table.shape
    ids = torch.zeros((rows - 1) * step + COLUMNS, dtype=table.dtype, device=table.device)
    ids[:table.numel()] = table.reshape(-1)
    return ids.as_strided((rows, COLUMNS), (step, 1))


def run(problem, **extra):
    out = torch.full_like(problem.query, float("nan"))
    lse = torch.full(out.shape[:2], float("nan"), device=out.device)
    problem.call(shared_prefix_attention, out, lse, **extra)
    return out, lse


def verify_wide(problem):
    print(f"[attention] {tuple(problem.query.shape)} rows {len(problem.lengths)}", flush=True)
    want = problem.answer()
    problem.tables = widen(problem.tables)
    if problem.prefix_tables is not None:
        problem.prefix_tables = widen(problem.prefix_tables)
    out, lse = run(problem)
    check(out, lse, want, problem.query.shape[2])


def ragged(count, most):
    return [int(most * ((i * 0.6180339887498949) % 1.0) ** 3) for i in range(count)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prefixes,groups", [(None, None), ([5000, 0, 700], [3, 100, 200, 290])])
def test_decode_with_tables_of_2_30_tokens(gpu, dtype, prefixes, groups):
    # 8 KV heads of 300 rows: units of 2048 keys instead of 128.
    lengths = ragged(300, 2500)
    lengths[7] = 40000
    verify_wide(make_problem(gpu, dtype=dtype, heads=16, kv_heads=8, dim=64, lengths=lengths, prefixes=prefixes,
                             groups=groups, seed=1))


@pytest.mark.parametrize("prefixes,groups", [(None, None), ([3000, 40], [0, 2, 24])])
def test_prompts_with_tables_of_2_30_tokens(gpu, prefixes, groups):
    # 32 KV heads of 25 rows of up to 300 tokens, 2 query heads each.
    counts = [(37 * i) % 60 for i in range(25)]
    counts[3] = 300
    lengths = [n + (211 * i) % 900 for i, n in enumerate(counts)]
    verify_wide(make_problem(gpu, heads=64, kv_heads=32, dim=64, lengths=lengths, counts=counts, prefixes=prefixes,
                             groups=groups, seed=2))


@pytest.mark.parametrize("tokens,rows", [(16, 1025), (4096, 9)])
def test_starts_out_of_order_whose_places_pass_32_bits(gpu, tokens, rows):
    """Every other row claims all query tokens and 2^30 - 16 keys: 2^32 places in all, and the last row's few.

    16 tokens are one tile of 2^23 units a row, 512 rows and the last; 4096 are 256 tiles of 2^22 units, 4 rows and the
    last. What such starts give is not defined; nothing around the output changes, and a later call is right.
    """
    problem = make_problem(gpu, heads=1, kv_heads=1, dim=64, page=PAGE, lengths=[PAGE] * rows,
                           counts=[tokens] + [0] * (rows - 1), prefixes=None, seed=4)
    want = problem.answer()
    memory = torch.full((tokens + 2, 1, 64), 7.0, dtype=BF16, device=gpu)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    lengths = [COLUMNS * PAGE] * (rows - 1) + [100]
    print(f"[attention] {tokens} tokens claimed by {(rows + 1) // 2} rows", flush=True)
    shared_prefix_attention(problem.query, problem.pool.planes, widen(problem.tables), problem.rows, ints(lengths), None,
                            None, memory[1:-1], page_size=PAGE, kv_heads=1, layer=1, max_query=1,
                            query_starts=ints([tokens * (i % 2) for i in range(rows + 1)]))
    torch.cuda.synchronize()
    assert (memory[0] == 7).all() and (memory[-1] == 7).all()
    out, lse = run(problem)
    check(out, lse, want, 64)
