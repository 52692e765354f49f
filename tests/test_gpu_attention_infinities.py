"""Infinities and NaN in V: the query tokens that see such a key get them, the others do not.

A key in a tile that only some rows see has weight 0 for the others, and 0 times infinity is not 0, so the kernels add
what is not finite apart from the product. Expected per output element, over the keys that its token sees: NaN if V
holds NaN or infinities of both signs there, the infinity if it holds one, else the answer without them, within the
bounds of attention_cases.py. Scores are of standard deviation one, so that no weight is rounded to zero.
"""

import math

import pytest
import torch

from adaptive_sparse.attention import shared_prefix_attention

from attention_cases import check, make_problem, read

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def spoil(problem):
    """Puts values that are not finite into V, among keys that all, some and one of a row's tokens see."""
    values, page, dim = problem.pool.values, problem.pool.page, problem.query.shape[2]
    place = problem.rows.tolist()
    last = values.shape[2] - 1

    def put(table, position, head, column, value):
        values[int(table[position // page]), position % page, head, column] = value

    for b, (length, count) in enumerate(zip(problem.lengths, problem.counts)):
        table = problem.tables[place[b]]
        put(table, length - 1, 0, 0, INF)
        put(table, length - 1, 0, 3, NAN)
        put(table, length - 2, 0, 0, -INF)
        put(table, length - 2, last, 1, -INF)
        put(table, length - 1 - count // 2, last, dim - 1, INF)
        put(table, 5, last, 2, -INF)
    for g, length in enumerate(problem.prefix_lengths):
        put(problem.prefix_tables[g], length // 2, 0, 4, INF)
        put(problem.prefix_tables[g], length - 1, 0, 5, NAN)


def seen_specials(problem):
    """[N, Hq, D] truth values: the token sees +infinity, -infinity, NaN there."""
    kv_heads, dim = problem.pool.values.shape[2:]
    share = problem.query.shape[1] // kv_heads
    place = problem.rows.tolist()
    found = []
    for b, (length, count) in enumerate(zip(problem.lengths, problem.counts)):
        g = problem.group(b)
        parts = [] if g is None else [read(problem.pool, problem.prefix_tables[g], problem.prefix_lengths[g])[1]]
        for i in range(count):
            own = read(problem.pool, problem.tables[place[b]], length - count + i + 1)[1]
            v = torch.cat([*parts, own])
            found.append([kind.any(0).repeat_interleave(share, 0) for kind in (v == INF, v == -INF, v.isnan())])
    return [torch.stack(kind) for kind in zip(*found)]


CASES = [
    # heads, KV heads, head size, query tokens and lengths of each row, prefixes, groups
    ("16 rows", 8, 2, 128, [1, 3, 4], [3000, 200, 85], None, None),
    ("32 rows", 8, 2, 64, [8, 2, 5], [128, 3001, 21], None, None),
    ("64 rows", 8, 2, 128, [16, 2, 15], [64, 2300, 95], None, None),
    ("128 rows", 8, 2, 96, [32, 2, 9], [100, 2500, 33], None, None),
    ("256 rows", 8, 2, 128, [60, 2, 33], [2900, 77, 130], None, None),
    ("16 rows of 256", 8, 2, 256, [4, 2, 3], [700, 40, 33], None, None),
    ("32 rows of 256", 8, 2, 256, [7, 2, 8], [700, 40, 33], None, None),
    ("128 rows of 256", 8, 2, 256, [30, 2, 17], [700, 40, 95], None, None),
    ("16 rows and their own prefixes", 8, 2, 64, [4, 2], [300, 40], [100, 65], [0, 1, 2]),
    ("256 rows and their own prefixes", 8, 2, 128, [40, 64], [300, 70], [100, 65], [0, 1, 2]),
    ("a prefix of its own, 16 rows", 8, 2, 128, [1, 3, 4, 2, 4, 1], [900, 200, 85, 31, 64, 40], [1000], [0, 6]),
    ("a prefix of its own, 128 rows", 8, 2, 64, [16, 3, 9, 12, 4, 1], [900, 200, 85, 32, 64, 40], [99, 500], [0, 2, 6]),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", CASES, ids=[case[0].replace(" ", "_") for case in CASES])
def test_what_is_not_finite_reaches_the_tokens_that_see_it(gpu, dtype, case):
    name, heads, kv_heads, dim, counts, lengths, prefixes, groups = case
    print(f"[attention] {name} {dtype}", flush=True)
    problem = make_problem(gpu, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, lengths=lengths, counts=counts,
                           prefixes=prefixes, groups=groups, magnitude=1.0, seed=dim)
    # Unlike rows share no page, so each spoiled key belongs to one row or one prefix.
    spoil(problem)
    plus, minus, nan = seen_specials(problem)
    out = torch.full_like(problem.query, 7.0)
    lse = torch.full(out.shape[:2], 7.0, device=gpu)
    problem.call(shared_prefix_attention, out, lse)
    bad = nan | (plus & minus)
    plus, minus = plus & ~bad, minus & ~bad
    assert int(bad.sum()) and int(plus.sum()) and int(minus.sum())
    assert torch.isnan(out[bad]).all(), "a token that sees NaN, or infinities of both signs"
    assert (out[plus] == INF).all(), "a token that sees infinity"
    assert (out[minus] == -INF).all(), "a token that sees minus infinity"
    finite = ~(bad | plus | minus)
    # The answer without them: what is not finite counts as zero, and its elements are left out.
    values = problem.pool.values
    values.copy_(torch.where(torch.isfinite(values), values, 0.0))
    want = problem.answer()
    for field in ("out", "mass", "spread"):
        setattr(want, field, getattr(want, field)[finite])
    check(out[finite], None, want, dim)
    assert torch.isfinite(lse).all()
    off = (lse.double() - want.lse).abs()
    limit = 4 * math.sqrt(dim) * 2.0 ** -24 * want.size + 2.0 ** -20 * (1 + want.lse.abs())
    assert float((off / limit).max()) <= 1.0


@pytest.mark.parametrize("heads,most", [(1, 1), (1, 20), (1, 48), (4, 30), (4, 48)])   # 16, 32, 64, 128, 256 rows
def test_infinities_of_later_tokens_stay_away(gpu, heads, most):
    """Each token's own V row holds an infinity: token i gets those of its own and of earlier keys, and no later ones."""
    count, length, dim = 48, 64, 64
    problem = make_problem(gpu, heads=heads, kv_heads=1, dim=dim, lengths=[length], counts=[count], prefixes=None,
                           magnitude=1.0, seed=5)
    for i in range(count):
        position = length - count + i
        problem.pool.values[int(problem.tables[0, position // 16]), position % 16, 0, i] = INF
    out = torch.zeros_like(problem.query)
    problem.call(shared_prefix_attention, out, max_query=most)
    want = torch.ones((count, count), dtype=torch.bool, device=gpu).tril()
    for head in range(heads):
        assert torch.equal(out[:, head, :count] == INF, want)
    assert torch.isfinite(out[:, :, count:]).all()
    assert torch.isfinite(out[:, :, :count][(~want).unsqueeze(1).expand(-1, heads, -1)]).all()
