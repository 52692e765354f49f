"""block_attention with the output in the query's place: the bits of a call with an output of its own."""

import pytest
import torch

from adaptive_sparse.attention import block_attention

from attention_cases import check
from block_cases import make_block_problem

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16

CASES = [
    # heads, KV heads, head size, lengths, query tokens, block, chosen, lists
    (16, 2, 128, [700, 90, 333], None, 64, 4, 2),
    (8, 1, 128, [9000], None, 64, 130, 1),                 # one list for many workgroups, joined behind them
    (200, 1, 64, [300, 515], None, 64, 4, 1),              # several tiles of rows
    (70, 1, 256, [300, 515], None, 64, 4, 1),
    (8, 8, 80, [400] * 70, None, 32, 5, 4),                # items of their own workgroups
    (16, 2, 128, [600, 401, 90], [500, 380, 90], 64, 4, 2),
    (16, 16, 64, [300, 201], [200, 64], 32, 3, 1),         # prompts together
    (16, 16, 256, [300, 201], [200, 64], 32, 3, 1),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_the_output_may_be_the_query(gpu, dtype, case):
    heads, kv_heads, dim, lengths, counts, block, chosen, lists = case
    print(f"[blocks] in place {case} {dtype}", flush=True)
    problem = make_block_problem(gpu, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, lengths=lengths, counts=counts,
                                 block=block, chosen=chosen, lists=lists, together=True, tail=2 if counts else 0, seed=dim)
    # A projection's output, of which the queries are a slice.
    both = torch.zeros((problem.query.shape[0], heads + 2, dim), dtype=dtype, device=gpu)
    both[:, :heads] = problem.query
    problem.query = both[:, :heads]
    out, lse = torch.empty_like(problem.query), torch.empty((both.shape[0], heads), device=gpu)
    problem.call(block_attention, out, lse)
    check(out, lse, problem.answer(), dim)
    again = torch.full_like(lse, 7.0)
    problem.call(block_attention, problem.query, again)
    assert torch.equal(problem.query, out) and torch.equal(again, lse)
    assert not bool(both[:, heads:].any())
