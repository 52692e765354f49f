"""block_attention of prompts, whose neighbouring tokens go through their lists together: against a 64-bit answer.

All calls here have as many query rows and heads as the rule for that asks for: 64 rows of a batch row, and 2048 pairs
of a token and a KV head, or more.
"""

import math

import pytest
import torch

from adaptive_sparse.attention import block_attention

from attention_cases import check
from block_cases import make_block_problem

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def pairs_wanted(dim, block):
    """(token, KV head) pairs, more where heads are small or blocks end inside 32 keys."""
    size = 64 if dim <= 64 else 96 if dim <= 96 else 128
    return 2049 * 128 / size * (-(-block // 32) * 32) / block + 1


def run(problem, **extra):
    tokens, heads, dim = problem.query.shape
    kv_heads = problem.pool.keys.shape[2]
    assert max(problem.batch.counts) * heads // kv_heads >= 64
    assert tokens * kv_heads >= pairs_wanted(dim, problem.block)
    out = torch.full_like(problem.query, 7.0)
    lse = torch.full(out.shape[:2], 7.0, device=out.device)
    problem.call(block_attention, out, lse, **extra)
    return out, lse


CASES = [
    # heads, KV heads, head size, page, layout, lengths, query tokens, block, chosen, lists
    (64, 4, 128, 16, "planes", [300, 90, 450], [100, 90, 3], 64, 4, 4),
    (64, 4, 128, 16, "blocks", [1300, 90, 450], [70, 33, 30], 64, 5, 1),
    (64, 2, 64, 1, "planes", [1300, 40], [130, 5], 32, 9, 2),          # 32 heads a KV head: two tokens a tile
    (60, 20, 96, 100, "planes", [150, 330], [110, 40], 96, 3, 10),     # three heads a KV head: tiles end inside tokens
    (63, 9, 80, 64, "blocks", [150, 330], [110, 40], 160, 2, 3),       # seven
    (32, 32, 128, 16, "planes", [300, 200], [201, 70], 32, 8, 32),     # one: 64 tokens a tile
    (72, 24, 8, 16, "planes", [260], [130], 64, 3, 1),
    (64, 4, 128, 16, "planes", [5000, 77], [100, 77], 128, 16, 2),
    (64, 2, 128, 16, "planes", [5000], [130], 2048, 2, 1),             # blocks longer than most of the context
    (64, 4, 128, 16, "planes", [300, 90, 450], [100, 90, 3], 16, 9, 4),    # blocks that 32 keys are too many for
    (64, 4, 128, 16, "planes", [300, 90, 450], [100, 90, 3], 100, 3, 1),
    (63, 9, 80, 64, "blocks", [150, 330], [110, 40], 20, 6, 3),
    (32, 4, 256, 16, "planes", [300, 90], [100, 60], 64, 4, 2),
    (24, 2, 200, 100, "blocks", [300, 90], [100, 60], 33, 5, 1),
]


@pytest.mark.parametrize("dtype,together", [(BF16, True), (F16, False)])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_prompts(gpu, dtype, together, case):
    heads, kv_heads, dim, page, layout, lengths, counts, block, chosen, lists = case
    times = math.ceil(pairs_wanted(dim, block) / (sum(counts) * kv_heads))
    lengths, counts = lengths * times, counts * times
    print(f"[blocks] {case} {dtype} {together}", flush=True)
    problem = make_block_problem(gpu, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, layout=layout,
                                 lengths=lengths, counts=counts, block=block, chosen=chosen, lists=lists,
                                 together=together, index=torch.int32 if together else torch.int64, seed=dim + block)
    out, lse = run(problem)
    check(out, lse, problem.answer(), dim)
    again, _ = run(problem)
    assert torch.equal(again, out), "two calls differ"


def test_empty_lists_tokens_of_no_row_and_requests_that_are_not(gpu):
    problem = make_block_problem(gpu, heads=64, kv_heads=4, lengths=[300] * 5 + [0, 450, 200],
                                 counts=[95] * 5 + [0, 3, 42], tail=3, lists=2, seed=1, together=True)
    problem.blocks[3] = -1
    problem.blocks[5, 1] = 1000                       # behind the position
    problem.batch.rows = problem.batch.rows.clone()
    problem.batch.rows[7] = 9
    for most in (95, 5000):
        out, lse = run(problem, max_query=most)
        check(out, lse, problem.answer(), 128)
        assert not bool(out[-45:].any()) and bool((lse[-45:] == -math.inf).all())
        assert not bool(out[3].any()) and not bool(out[5, 32:].any()) and bool(out[5, :32].any())


def test_bad_pages_and_a_length_past_the_table(gpu):
    problem = make_block_problem(gpu, heads=64, kv_heads=4, lengths=[640] * 4, counts=[140] * 4, chosen=10, block=32,
                                 seed=3, together=True)
    place = int(problem.batch.rows[0])
    tables = problem.batch.tables
    tables[place, 0:2], tables[place, 5], tables[place, 39] = 0, problem.batch.pages, -3
    problem.blocks[7, 0] = torch.arange(10, device=gpu)
    out, lse = run(problem)
    check(out, lse, problem.answer(), 128)
    problem.batch.lengths = [700] * 4                 # more than the table covers
    out, lse = run(problem)
    check(out, lse, problem.answer(), 128)


def test_what_is_not_seen_may_be_anything(gpu):
    problem = make_block_problem(gpu, heads=64, kv_heads=2, lengths=[300] * 8 + [77], counts=[140] * 8 + [2], block=64,
                                 chosen=3, lists=2, seed=4, together=True)
    want = problem.answer()
    keys, values = problem.pool.keys, problem.pool.values
    used = torch.zeros(keys.shape[:2], dtype=torch.bool, device=gpu)
    for b, length in enumerate(problem.batch.lengths):
        for t, page in problem.batch.seen(b, length - 1):
            used[page, t % 16] = True
    for value in (float("nan"), float("inf")):
        keys[~used] = value
        values[~used] = value
        out, lse = run(problem)
        check(out, lse, want, 128)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinities_reach_the_tokens_that_see_them(gpu, dim):
    """Key i of a row's last tokens has an infinity in column i of V: token i sees its own and earlier ones it lists."""
    count, length, heads = 64, 256, 128
    problem = make_block_problem(gpu, heads=heads, kv_heads=heads, dim=dim, lengths=[length], counts=[count], block=32,
                                 chosen=3, seed=5)
    problem.query = problem.query * 0.25
    listed = torch.tensor([[0, 6, 7]] * count, dtype=torch.int32, device=gpu).unsqueeze(1)
    listed[1::2, 0, 2] = 5                            # every other token does not list the newest block
    problem.blocks = listed
    table = problem.batch.table(0)
    seen = torch.zeros((count, count), dtype=torch.bool, device=gpu)
    for i in range(count):
        t = length - count + i
        problem.pool.values[table[t // 16], t % 16, :, i] = math.inf
        for n in range(count):
            seen[n, i] = t <= length - count + n and t // 32 in listed[n, 0].tolist()
    out, lse = run(problem)
    for head in range(heads):
        assert torch.equal(out[:, head, :count] == math.inf, seen)
    assert torch.isfinite(out[:, :, count:]).all() and torch.isfinite(lse).all()
    assert torch.isfinite(out[:, :, :count][(~seen).unsqueeze(1).expand(-1, heads, -1)]).all()


def test_a_block_listed_twice_counts_twice(gpu):
    problem = make_block_problem(gpu, heads=64, kv_heads=4, lengths=[300, 200] * 4, counts=[100, 39] * 4, block=32,
                                 chosen=5, lists=2, seed=6, together=True)
    problem.blocks[:, 0, 1] = problem.blocks[:, 0, 0]
    problem.blocks[::2, 1] = problem.blocks[::2, 1, :1]       # five times
    out, lse = run(problem)
    check(out, lse, problem.answer(), 128)
    again, _ = run(problem)
    assert torch.equal(again, out)


def test_a_replay_of_prompts_on_another_stream(gpu):
    problem = make_block_problem(gpu, heads=64, kv_heads=4, lengths=[300, 200] * 4, counts=[100, 39] * 4, block=32,
                                 chosen=5, lists=2, seed=7, together=True)
    out, lse = torch.empty_like(problem.query), torch.empty(problem.query.shape[:2], device=gpu)
    lengths, starts = problem.batch.ints(problem.batch.lengths), problem.batch.ints(problem.batch.starts())
    from adaptive_sparse.attention import block_workspace
    workspace = torch.empty(block_workspace(556, 5, 32, 64, 4, 128, 100), dtype=torch.uint8, device=gpu)
    call = lambda: block_attention(problem.query, problem.pool.planes, problem.batch.tables,  # noqa: E731
                                   problem.batch.rows, lengths, problem.blocks, out, page_size=16, block_size=32,
                                   kv_heads=4, layer=problem.pool.layer, query_starts=starts, max_query=100, lse=lse,
                                   workspace=workspace)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
    torch.cuda.synchronize()
    for step in range(3):
        problem.batch.counts = [100 - 30 * step, 39 + 30 * step] * 4
        starts.copy_(problem.batch.ints(problem.batch.starts()))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        check(out, lse, problem.answer(), 128)
