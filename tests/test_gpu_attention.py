"""shared_prefix_attention and topk_attention against their definition in 64 bits.

The bounds are derived in attention_cases.py. Sizes: every head size class, head ratios from 1 to 16, pages that end
inside a tile, lengths of zero and one, ragged query counts, groups of every shape; unseen memory holds NaN.
"""

import math

import pytest
import torch

from adaptive_sparse.attention import (shared_prefix_attention, shared_prefix_workspace, topk_attention,
                                       topk_workspace)
from adaptive_sparse.kv_pool import KVPlanes

from attention_cases import Problem, answer_of, attend, check, make_pool, make_problem

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def run(problem, lse=True, **extra):
    out = torch.full_like(problem.query, float("nan"))
    stats = (torch.full(problem.query.shape[:2], float("nan"), dtype=torch.float32, device=out.device)
             if lse else None)
    problem.call(shared_prefix_attention, out, stats, **extra)
    return out, stats


def verify(problem, **extra):
    print(f"[attention] {tuple(problem.query.shape)} lengths {problem.lengths[:8]} counts {problem.counts[:8]} "
          f"prefixes {problem.prefix_lengths[:8]}", flush=True)
    out, lse = run(problem, **extra)
    check(out, lse, problem.answer(), problem.query.shape[2])
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 96, 128, 160, 192, 256])
def test_decode_over_head_sizes(gpu, dtype, dim):
    verify(make_problem(gpu, dtype=dtype, heads=6, kv_heads=2, dim=dim, page=16,
                        lengths=[1, 15, 16, 17, 33, 128, 200, 5], prefixes=[77], seed=dim))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (8, 1), (16, 2), (17, 1), (32, 1), (48, 2), (12, 4),
                                            (64, 1), (100, 1)])
def test_decode_over_head_ratios(gpu, heads, kv_heads):
    verify(make_problem(gpu, heads=heads, kv_heads=kv_heads, dim=64, lengths=[3, 70, 31, 1, 150], prefixes=[213],
                        seed=heads))


@pytest.mark.parametrize("page", [1, 2, 7, 16, 48, 64, 100, 256])
@pytest.mark.parametrize("layout", ["planes", "blocks"])
def test_decode_over_page_sizes_and_layouts(gpu, page, layout):
    verify(make_problem(gpu, page=page, layout=layout, lengths=[1, 63, 64, 65, 300, 129], prefixes=[page + 1],
                        index=torch.int64 if page % 2 else torch.int32, seed=page))


@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 33, 64, 127, 1000])
def test_prefix_lengths(gpu, prefix):
    verify(make_problem(gpu, lengths=[9, 1, 64], prefixes=[prefix], seed=prefix))


@pytest.mark.parametrize("batch", [1, 2, 5, 20, 70])
def test_batches_behind_one_prefix(gpu, batch):
    verify(make_problem(gpu, heads=16, kv_heads=2, lengths=[1 + (37 * i) % 90 for i in range(batch)], prefixes=[515],
                        seed=batch))


def test_no_prefix_and_no_rows(gpu):
    verify(make_problem(gpu, lengths=[100, 3, 0, 77], prefixes=None, permute=False))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_groups_of_every_shape(gpu, dtype):
    # Rows 0 and 11.. lie outside every group, group 1 is empty, group 3's prefix has no tokens.
    verify(make_problem(gpu, dtype=dtype, lengths=[4, 0, 19, 33, 1, 64, 0, 8, 90, 2, 16, 0, 5],
                        prefixes=[65, 10, 130, 0, 7], groups=[1, 4, 4, 7, 9, 11], seed=3))


@pytest.mark.parametrize("counts,lengths", [
    ([1, 2, 3, 4, 5], [1, 2, 3, 40, 500]),
    ([0, 7, 0, 1], [10, 7, 0, 1]),
    ([5, 5], [3, 0]),                            # fewer own tokens than query tokens: the first see the prefix only
    ([33, 64, 65], [33, 200, 65]),
    ([150, 1, 40], [150, 700, 41]),
])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (4, 2, 64), (6, 1, 96)])
def test_several_query_tokens(gpu, counts, lengths, heads, kv_heads, dim):
    verify(make_problem(gpu, heads=heads, kv_heads=kv_heads, dim=dim, lengths=lengths, counts=counts, prefixes=[145],
                        seed=sum(counts)))


def test_several_query_tokens_in_groups(gpu):
    verify(make_problem(gpu, dtype=F16, heads=8, kv_heads=2, dim=64, page=5, lengths=[9, 80, 41, 6, 200, 3],
                        counts=[4, 40, 1, 6, 130, 3], prefixes=[33, 300], groups=[0, 3, 5], layout="blocks", seed=8))


def test_query_tokens_of_no_row_get_zeros(gpu):
    problem = make_problem(gpu, lengths=[9, 20], counts=[2, 3], prefixes=[40], tail=4)
    out, lse = verify(problem)
    assert not out[5:].any() and (lse[5:] == -math.inf).all()


def test_max_query_picks_kernels_not_results(gpu):
    problem = make_problem(gpu, heads=8, kv_heads=1, lengths=[90, 40, 300], counts=[80, 1, 20], prefixes=[200])
    want = problem.answer()
    for most in (1, 3, 20, 80, 5000):
        out, lse = run(problem, max_query=most)
        check(out, lse, want, 128)


def test_a_long_prefix_and_long_rows(gpu):
    verify(make_problem(gpu, heads=16, kv_heads=2, page=64, lengths=[20011, 1, 4097, 300], prefixes=[30001], seed=11))


def test_many_rows_of_query(gpu):
    verify(make_problem(gpu, heads=16, kv_heads=1, page=16, lengths=[900, 300], counts=[300, 290], prefixes=[1500],
                        seed=12))


def poison(pool, problem):
    """NaN in every row that no query may see: the sink, spare pages, tails of last pages."""
    seen = torch.zeros(pool.keys.shape[:2], dtype=torch.bool, device=pool.keys.device)
    place = problem.rows.tolist()
    spans = [(problem.tables[place[b]], n) for b, n in enumerate(problem.lengths)]
    spans += [(problem.prefix_tables[g], n) for g, n in enumerate(problem.prefix_lengths)]
    for table, count in spans:
        for i in range(-(-count // pool.page)):
            page = int(table[i])
            if 1 <= page < pool.keys.shape[0]:
                seen[page, :count - i * pool.page] = True
    keys, values = pool.keys, pool.values
    keys[~seen] = float("nan")
    values[~seen] = float("nan")


@pytest.mark.parametrize("page,layout", [(16, "planes"), (7, "blocks"), (128, "planes")])
@pytest.mark.parametrize("counts", [None, [1, 4, 2, 40]])
def test_memory_that_nobody_sees_may_hold_nan(gpu, page, layout, counts):
    problem = make_problem(gpu, page=page, layout=layout, lengths=[5, 64, 130, 47], counts=counts, prefixes=[97],
                           seed=page)
    poison(problem.pool, problem)
    verify(problem)


def test_page_ids_that_name_no_page_are_not_seen(gpu):
    problem = make_problem(gpu, lengths=[100, 64, 33, 16], prefixes=[90], seed=21)
    place = problem.rows.tolist()
    pages = problem.pool.keys.shape[0]
    problem.tables[place[0], 2] = 0
    problem.tables[place[1], 0] = -5
    problem.tables[place[2], 1] = pages
    problem.tables[place[3], :] = 0x7fffffff           # nothing of its own
    problem.prefix_tables[0, 3] = -1
    poison(problem.pool, problem)
    verify(problem)


def test_bad_rows_lengths_and_starts_read_nothing(gpu):
    problem = make_problem(gpu, lengths=[40, 40, 40, 40], prefixes=[50], seed=22)
    problem.rows = torch.tensor([0, 99, -1, 3], device=gpu)
    problem.lengths = [10 ** 6, 40, 40, -7]             # past the table; no request; no request; negative
    verify(problem)
    problem.prefix_lengths = [10 ** 9]                  # past the prefix table: what the table holds
    verify(problem)


@pytest.mark.parametrize("counts", [[3, 5, 40], [1, 1, 1]])
def test_future_tokens_may_hold_infinities_and_nan(gpu, counts):
    """A token's own future is masked, whatever its K and V hold: earlier tokens' outputs stay finite."""
    problem = make_problem(gpu, heads=8, kv_heads=1, lengths=[20, 70, 90], counts=counts, prefixes=[33], seed=23)
    want = problem.answer()
    place = problem.rows.tolist()
    spoiled = torch.zeros(problem.query.shape[0], dtype=torch.bool, device=gpu)
    starts = problem.starts()
    for b, bad in enumerate((float("nan"), float("inf"), -float("inf"))):
        position = problem.lengths[b] - 1
        page = int(problem.tables[place[b], position // 16])
        problem.pool.keys[page, position % 16] = bad
        problem.pool.values[page, position % 16] = bad
        spoiled[starts[b + 1] - 1] = True               # the newest token sees it
    out, lse = run(problem)
    good = ~spoiled
    for field in ("out", "lse", "mass", "spread"):
        setattr(want, field, getattr(want, field)[good])
    if int(good.sum()):
        check(out[good], lse[good], want, 128)


def test_a_nan_query_spoils_its_own_rows_only(gpu):
    problem = make_problem(gpu, heads=8, kv_heads=2, lengths=[30, 31, 32], counts=[2, 3, 1], prefixes=[64], seed=24)
    want = problem.answer()
    problem.query[3, 5] = float("nan")
    out, lse = run(problem)
    assert torch.isnan(out[3, 5]).all() and torch.isnan(lse[3, 5])
    keep = torch.ones(out.shape[:2], dtype=torch.bool, device=gpu)
    keep[3, 5] = False
    for field in ("out", "lse", "mass", "spread"):
        setattr(want, field, getattr(want, field)[keep])
    check(out[keep], lse[keep], want, 128)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_and_lopsided_scores(gpu, dtype):
    """Scores of several hundred: one key takes all; and a key far below the others counts for nothing."""
    problem = make_problem(gpu, dtype=dtype, lengths=[200, 1, 65], prefixes=[300], magnitude=60.0, seed=25)
    verify(problem)
    problem.pool.keys[problem.prefix_tables[0, 0].long(), 0] = -60.0     # far below for positive queries
    problem.query.copy_(problem.query.abs())
    verify(problem)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_the_type_s_lowest_and_largest_values(gpu, dtype):
    """K rows at the type's bounds: scores of -3e38 and beyond are weights of zero, not NaN."""
    problem = make_problem(gpu, dtype=dtype, heads=2, kv_heads=1, dim=64, lengths=[40, 17], prefixes=[20], seed=26)
    lowest = torch.finfo(dtype).min
    problem.query.fill_(1.0)
    problem.scale = 1.0 if dtype == F16 else 2.0 ** -7
    for page in problem.tables[:, 0].tolist():
        problem.pool.keys[page, 3] = lowest / 64
        problem.pool.keys[page, 4] = -float("inf") if dtype == BF16 else lowest
    problem.pool.keys[int(problem.prefix_tables[0, 0]), 0] = lowest / 64
    out, lse = run(problem)
    want = problem.answer()
    want.size = float((problem.pool.keys[1:].double().abs().clamp(max=8).sum(-1)).max()) * problem.scale
    check(out, lse, want, 64)


def test_scores_of_minus_infinity_everywhere_are_an_empty_row(gpu):
    problem = make_problem(gpu, heads=2, kv_heads=1, dim=64, lengths=[3], prefixes=None, seed=27)
    problem.query.fill_(1.0)
    problem.pool.keys.fill_(-float("inf"))
    out, lse = run(problem)
    assert not out.any() and (lse == -math.inf).all()


def test_strides_of_query_output_lse_and_tables(gpu):
    problem = make_problem(gpu, heads=8, kv_heads=2, dim=64, lengths=[33, 80, 2], counts=[2, 3, 1], prefixes=[70])
    want = problem.answer()
    wide = torch.zeros((6, 3, 8, 72), dtype=BF16, device=gpu)            # rows of 72, every third plane
    wide[:, 1, :, :64] = problem.query
    problem.query = wide[:, 1, :, :64]
    for name in ("tables", "prefix_tables"):
        table = getattr(problem, name)
        spread = torch.full((table.shape[0] * 2, table.shape[1] * 3), 10 ** 9, dtype=table.dtype, device=gpu)
        spread[::2, ::3] = table
        setattr(problem, name, spread[::2, ::3])
    problem.rows = problem.rows.repeat_interleave(2)[::2]
    out = torch.full((8, 6, 64), 7.0, dtype=BF16, device=gpu).transpose(0, 1)
    lse = torch.full((8, 12), 7.0, device=gpu).t()[::2]
    problem.call(shared_prefix_attention, out, lse)
    check(out, lse, want, 64)


def test_padded_strides_leave_the_gaps_alone(gpu):
    problem = make_problem(gpu, heads=4, kv_heads=1, dim=80, lengths=[33, 80], prefixes=[70])
    room = torch.full((2, 4, 96), 7.0, dtype=BF16, device=gpu)
    problem.call(shared_prefix_attention, room[:, :, :80])
    check(room[:, :, :80], None, problem.answer(), 80)
    assert (room[:, :, 80:] == 7.0).all()


def test_offsets_past_32_bits(gpu):
    """A pool of over 6 GiB a plane, with pages at both ends of it."""
    rows, kv_heads, dim, page = 26 << 20, 1, 128, 16
    memory = torch.empty((2, rows, kv_heads, dim), dtype=BF16, device=gpu)
    planes = KVPlanes(base=memory.data_ptr(), device=0, layers=1, kv=2, layer_stride=0,
                      kv_stride=rows * 256, row_stride=256, row_bytes=256, rows=rows, owner=memory)
    problem = make_problem(gpu, heads=8, kv_heads=1, lengths=[90, 33], prefixes=[100], seed=31)
    small = problem.pool
    pages = small.keys.shape[0]
    where = torch.cat([torch.arange(3), rows // page - 1 - torch.arange(pages - 3) * 3]).to(gpu)
    big = memory.view(2, rows // page, page, kv_heads, dim)
    big[0][where], big[1][where] = small.keys, small.values
    want = problem.answer()
    problem.tables = where[problem.tables.long()].to(torch.int32)
    problem.prefix_tables = where[problem.prefix_tables.long()].to(torch.int32)
    small.planes, small.layer = planes, 0
    out, lse = run(problem)
    check(out, lse, want, 128)


def test_repeated_calls_agree_bit_for_bit(gpu):
    problem = make_problem(gpu, heads=16, kv_heads=2, lengths=[777, 30, 2000], counts=[3, 1, 2], prefixes=[3333])
    first = run(problem)
    for _ in range(3):
        again = run(problem)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_another_stream_and_a_dirty_workspace(gpu):
    problem = make_problem(gpu, heads=16, kv_heads=2, lengths=[777, 30, 2000], prefixes=[3333], seed=41)
    size = shared_prefix_workspace(3, 3, 1, 16, 2, 128, 1)
    workspace = torch.full((size,), 255, dtype=torch.uint8, device=gpu)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out, lse = run(problem, workspace=workspace)
    stream.synchronize()
    check(out, lse, problem.answer(), 128)


def test_graph_replays(gpu):
    problem = make_problem(gpu, heads=16, kv_heads=2, lengths=[300, 1, 64], prefixes=[500], seed=42)
    out = torch.zeros_like(problem.query)
    lse = torch.zeros(out.shape[:2], device=gpu)
    lengths = torch.tensor(problem.lengths, dtype=torch.int32, device=gpu)
    prefix_lengths = torch.tensor(problem.prefix_lengths, dtype=torch.int32, device=gpu)
    workspace = torch.empty(shared_prefix_workspace(3, 3, 1, 16, 2, 128), dtype=torch.uint8, device=gpu)

    def call():
        shared_prefix_attention(problem.query, problem.pool.planes, problem.tables, problem.rows, lengths,
                                problem.prefix_tables, prefix_lengths, out, page_size=16, kv_heads=2, layer=1,
                                lse=lse, workspace=workspace)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(4):
        problem.lengths = [300 - 70 * step, 1 + step, 64]
        problem.prefix_lengths = [500 - 100 * step]
        lengths.copy_(torch.tensor(problem.lengths))
        prefix_lengths.copy_(torch.tensor(problem.prefix_lengths))
        problem.query.normal_()
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(out, lse, problem.answer(), 128)


def test_lse_merges_a_split_context(gpu):
    """The prefix alone and the own part alone, merged by their lse, are the whole."""
    problem = make_problem(gpu, heads=8, kv_heads=2, lengths=[100, 40], prefixes=[200], seed=43)
    whole, lse = run(problem)
    own = Problem(problem.pool, problem.query, problem.tables, problem.rows, problem.lengths, None, [], None,
                  problem.counts, problem.scale)
    part, part_lse = run(own)
    front = Problem(problem.pool, problem.query, problem.tables, problem.rows, [0, 0], problem.prefix_tables,
                    problem.prefix_lengths, problem.group_starts, problem.counts, problem.scale)
    other, other_lse = run(front)
    joined = torch.logaddexp(part_lse, other_lse)
    assert torch.allclose(joined, lse, atol=1e-5, rtol=0)
    merged = (part.float() * torch.exp(part_lse - joined).unsqueeze(-1)
              + other.float() * torch.exp(other_lse - joined).unsqueeze(-1))
    # Each side was rounded once more than the whole: three units of an output's size.
    assert float((merged - whole.float()).abs().max()) <= 3 * 2.0 ** -8 * float(whole.float().abs().max())


# ---------------------------------------------------------------- Top-K


def topk_problem(gpu, *, dtype=BF16, tokens=3, lanes=50, heads=8, kv_heads=2, dim=128, seed=0, index=torch.int32,
                 layout_rows=400):
    pool = make_pool(gpu, dtype, layout_rows, 1, kv_heads, dim, seed=seed)
    gen = torch.Generator(device=gpu).manual_seed(seed + 7)
    slots = torch.stack([torch.randperm(layout_rows - 1, generator=gen, device=gpu)[:lanes] + 1
                         for _ in range(tokens)]).to(index) if tokens else torch.zeros((0, lanes), dtype=index,
                                                                                       device=gpu)
    query = (torch.randn((tokens, heads, dim), generator=gen, device=gpu) * 2).to(dtype)
    return pool, query, slots


def topk_answer(pool, query, slots, zero_below=1):
    parts = []
    for t in range(query.shape[0]):
        at = slots[t].long()
        good = (at >= zero_below) & (at < pool.keys.shape[0])
        at = torch.where(good, at, 0)
        parts.append(attend(query[t], pool.keys[at, 0], pool.values[at, 0], query.shape[2] ** -0.5, good))
    return answer_of(parts)


def topk_run(pool, query, slots, **extra):
    out = torch.full_like(query, float("nan"))
    lse = torch.full(query.shape[:2], float("nan"), device=query.device)
    topk_attention(query, pool.planes, slots, out, kv_heads=pool.keys.shape[2], layer=pool.layer, lse=lse, **extra)
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 16, 2), (64, 8, 8), (96, 12, 4), (80, 20, 1), (256, 4, 2),
                                                (8, 3, 3), (128, 40, 1), (64, 130, 1)])
@pytest.mark.parametrize("lanes", [1, 33, 300])
def test_topk_sizes(gpu, dtype, dim, heads, kv_heads, lanes):
    pool, query, slots = topk_problem(gpu, dtype=dtype, lanes=lanes, heads=heads, kv_heads=kv_heads, dim=dim,
                                      seed=lanes + dim, index=torch.int64 if lanes == 33 else torch.int32)
    out, lse = topk_run(pool, query, slots)
    check(out, lse, topk_answer(pool, query, slots), dim)


def test_topk_lanes_that_name_no_row(gpu):
    pool, query, slots = topk_problem(gpu, tokens=5, lanes=100)
    slots[0, ::3] = 0
    slots[1, 20:] = -1
    slots[2, 5:50] = 400
    slots[3] = -1                                       # nothing
    slots[4, :64] = 0x7fffffff
    used = torch.zeros(400, dtype=torch.bool, device=gpu)
    used[slots[(slots >= 1) & (slots < 400)].long()] = True
    pool.keys[~used] = float("nan")
    pool.values[~used] = float("nan")
    out, lse = topk_run(pool, query, slots)
    check(out, lse, topk_answer(pool, query, slots), 128)
    assert not out[3].any()


def test_topk_zero_below_and_repeated_slots(gpu):
    pool, query, slots = topk_problem(gpu, lanes=40)
    slots[:, 10:20] = slots[:, :10]                     # counted twice
    slots[:, 20] = 0
    out, lse = topk_run(pool, query, slots, zero_below=0)
    check(out, lse, topk_answer(pool, query, slots, 0), 128)


def test_topk_strides_and_layers_of_a_lookup(gpu):
    """slots as one layer of [L, B, K], and transposed; an empty batch and no lanes."""
    pool, query, slots = topk_problem(gpu, tokens=6, lanes=70)
    whole = torch.full((3, 6, 70), -1, dtype=torch.int32, device=gpu)
    whole[1] = slots
    want = topk_answer(pool, query, slots)
    for given in (whole[1], slots.t().contiguous().t()):
        out, lse = topk_run(pool, query, given)
        check(out, lse, want, 128)
    out, lse = topk_run(pool, query, slots[:, :0])
    assert not out.any() and (lse == -math.inf).all()
    topk_run(pool, query[:0], slots[:0])


def test_topk_of_a_large_step(gpu):
    pool, query, slots = topk_problem(gpu, tokens=40, lanes=2048, heads=16, layout_rows=30000, seed=5)
    slots.masked_fill_(torch.rand(slots.shape, device=gpu) < 0.05, 0)
    out, lse = topk_run(pool, query, slots, workspace=torch.empty(topk_workspace(40, 2048, 16, 2, 128),
                                                                  dtype=torch.uint8, device=gpu))
    check(out, lse, topk_answer(pool, query, slots), 128)
    again = topk_run(pool, query, slots)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
