"""block_attention against a 64-bit answer, by the bounds of attention_cases.py."""

import math

import pytest
import torch

from adaptive_sparse.attention import block_attention, block_workspace

from attention_cases import check
from block_cases import make_block_problem

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def run(problem, **extra):
    out = torch.full_like(problem.query, 7.0)
    lse = torch.full(out.shape[:2], 7.0, device=out.device)
    problem.call(block_attention, out, lse, **extra)
    return out, lse


CASES = [
    # heads, KV heads, head size, page, layout, lengths, query tokens, block, chosen, lists
    (8, 2, 128, 16, "planes", [1, 500, 40], None, 64, 4, 1),
    (8, 2, 128, 16, "blocks", [1, 500, 40], None, 64, 4, 2),
    (16, 2, 128, 1, "planes", [700, 90], None, 128, 3, 2),
    (4, 4, 64, 64, "planes", [700, 90, 333], None, 16, 9, 4),
    (4, 4, 64, 100, "blocks", [700, 90, 333], None, 100, 2, 2),
    (12, 4, 96, 16, "planes", [300, 77], None, 20, 5, 1),
    (12, 4, 80, 16, "planes", [300, 77], None, 1, 65, 4),
    (6, 2, 8, 16, "planes", [300, 77], None, 7, 11, 2),
    (8, 2, 256, 16, "blocks", [300, 515], None, 64, 4, 2),
    (40, 2, 128, 16, "planes", [300, 515], None, 64, 4, 2),        # 20 rows a KV head
    (128, 2, 64, 16, "planes", [300, 515], None, 64, 4, 1),        # 64
    (200, 1, 64, 16, "planes", [300, 515], None, 64, 4, 1),        # several tiles of rows
    (70, 1, 256, 16, "planes", [300, 515], None, 64, 4, 1),
    (8, 2, 128, 16, "planes", [40, 500, 333], [3, 1, 5], 64, 4, 2),
    (8, 2, 64, 16, "planes", [300, 90, 450], [100, 90, 3], 32, 5, 1),
    (8, 2, 128, 16, "planes", [3000, 90], None, 64, 40, 1),        # most of a list behind its end
    (8, 1, 128, 16, "planes", [9000], None, 64, 130, 1),           # one long list, many workgroups
    (8, 2, 128, 16, "planes", [900] * 3, None, 2048, 1, 2),        # one block that nobody fills
    (16, 2, 128, 16, "planes", [600, 401], [150, 33], 64, 4, 2),
    (2, 2, 128, 16, "planes", [600, 401], [150, 33], 16, 20, 2),
    (16, 1, 256, 16, "blocks", [300, 201], [50, 33], 64, 3, 1),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("together", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_block_attention(gpu, dtype, together, case):
    heads, kv_heads, dim, page, layout, lengths, counts, block, chosen, lists = case
    print(f"[blocks] {case} {dtype} {together}", flush=True)
    problem = make_block_problem(gpu, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, layout=layout,
                                 lengths=lengths, counts=counts, block=block, chosen=chosen, lists=lists,
                                 together=together, index=torch.int64 if together else torch.int32, seed=dim + block)
    out, lse = run(problem)
    check(out, lse, problem.answer(), dim)
    again, _ = run(problem)
    assert torch.equal(again, out), "two calls differ"


def test_empty_lists_tokens_of_no_row_and_requests_that_are_not(gpu):
    problem = make_block_problem(gpu, lengths=[300, 90, 450, 200], counts=[20, 1, 3, 2], tail=3, lists=2, seed=1)
    problem.blocks[3] = -1
    problem.blocks[5, 1] = 1000                       # behind the position
    problem.batch.rows = problem.batch.rows.clone()
    problem.batch.rows[3] = 9
    for most in (20, 1, 500):
        out, lse = run(problem, max_query=most)
        check(out, lse, problem.answer(), 128)
        assert not bool(out[-5:].any()) and bool((lse[-5:] == -math.inf).all())
        assert not bool(out[3].any()) and not bool(out[5, 4:].any()) and bool(out[5, :4].any())


def test_bad_pages_and_lengths(gpu):
    problem = make_block_problem(gpu, lengths=[300, 640], chosen=10, block=32, seed=3)
    place = int(problem.batch.rows[1])
    tables = problem.batch.tables
    tables[place, 0:2], tables[place, 5], tables[place, 9] = 0, problem.batch.pages, -3
    problem.blocks[1, 0] = torch.arange(10, device=gpu)
    out, lse = run(problem)
    check(out, lse, problem.answer(), 128)
    problem.batch.lengths = [-5, 5000]                # nothing, and more than the table covers
    out, lse = run(problem)
    check(out, lse, problem.answer(), 128)


def test_what_is_not_seen_may_be_anything(gpu):
    problem = make_block_problem(gpu, lengths=[300, 77], counts=[40, 2], block=64, chosen=3, lists=2, seed=4,
                                 together=True)
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


@pytest.mark.parametrize("heads", [8, 16])
def test_infinities_reach_the_tokens_that_see_them(gpu, heads):
    """Key i of a row's last tokens has an infinity in column i of V: token i sees its own and earlier ones it lists."""
    count, length, dim = 32, 128, 64
    problem = make_block_problem(gpu, heads=heads, kv_heads=1, dim=dim, lengths=[length], counts=[count], block=16,
                                 chosen=3, seed=5)
    problem.query = problem.query * 0.25
    listed = torch.tensor([[0, 6, 7]] * count, dtype=torch.int32, device=gpu).unsqueeze(1)
    listed[1::2, 0, 2] = 5                            # every other token does not list the newest block
    problem.blocks = listed
    table = problem.batch.table(0)
    seen = torch.zeros((count, count), dtype=torch.bool, device=gpu)
    for i in range(count):
        t = length - count + i
        problem.pool.values[table[t // 16], t % 16, 0, i] = math.inf
        for n in range(count):
            seen[n, i] = t <= length - count + n and t // 16 in listed[n, 0].tolist()
    out, lse = run(problem)
    for head in range(heads):
        assert torch.equal(out[:, head, :count] == math.inf, seen)
    assert torch.isfinite(out[:, :, count:]).all() and torch.isfinite(lse).all()
    assert torch.isfinite(out[:, :, :count][(~seen).unsqueeze(1).expand(-1, heads, -1)]).all()


def test_a_block_listed_twice_counts_twice(gpu):
    problem = make_block_problem(gpu, lengths=[300, 200], counts=[30, 9], block=32, chosen=4, lists=2, seed=6,
                                 together=True)
    problem.blocks[:, 0, 1] = problem.blocks[:, 0, 0]
    problem.blocks[::2, 1] = problem.blocks[::2, 1, :1]
    out, lse = run(problem)
    check(out, lse, problem.answer(), 128)


def test_a_negative_scale_and_strided_tensors(gpu):
    problem = make_block_problem(gpu, lengths=[300, 77], counts=[3, 2], lists=2, seed=7)
    wide = torch.zeros((5, 20, 128), dtype=BF16, device=gpu)
    wide[:, 4:12] = problem.query
    problem.query = wide[:, 4:12]
    problem.blocks = problem.blocks.transpose(0, 2).contiguous().transpose(0, 2)
    problem.scale = -0.05
    out = torch.full((8, 5, 128), 7.0, dtype=BF16, device=gpu).transpose(0, 1)
    lse = torch.empty((8, 5), device=gpu).t()
    problem.call(block_attention, out, lse)
    check(out, lse, problem.answer(), 128)


def test_replays_in_a_graph_with_other_lists(gpu):
    problem = make_block_problem(gpu, lengths=[300, 777], lists=2, seed=8)
    out, lse = torch.empty_like(problem.query), torch.empty(problem.query.shape[:2], device=gpu)
    size = block_workspace(2, 4, 64, 8, 2, 128)
    workspace = torch.empty(size, dtype=torch.uint8, device=gpu)
    lengths = problem.batch.ints(problem.batch.lengths)
    call = lambda: block_attention(problem.query, problem.pool.planes, problem.batch.tables,  # noqa: E731
                                   problem.batch.rows, lengths, problem.blocks, out, page_size=16, block_size=64,
                                   kv_heads=2, layer=problem.pool.layer, lse=lse, workspace=workspace)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
    torch.cuda.synchronize()
    for step in range(3):
        problem.blocks.copy_(problem.blocks.roll(1, 0) if step else problem.blocks)
        problem.batch.lengths = [300 - step, 777 - 100 * step]
        lengths.copy_(problem.batch.ints(problem.batch.lengths))
        workspace.fill_(255)
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        check(out, lse, problem.answer(), 128)


def test_no_blocks_and_no_tokens(gpu):
    problem = make_block_problem(gpu, lengths=[300, 77], seed=9)
    problem.blocks = problem.blocks[:, :, :0]
    out, lse = run(problem)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    none = problem.query[:0]
    block_attention(none, problem.pool.planes, problem.batch.tables, problem.batch.rows[:0],
                    problem.batch.ints([]), problem.blocks[:0], torch.empty_like(none), page_size=16, block_size=64,
                    kv_heads=2)
