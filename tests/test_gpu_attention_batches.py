"""The attention operators over batches of hundreds of rows, and with scales of zero and below, against 64 bits.

A workgroup holds the batch rows of a launch some hundred at a time, and a launch of many query tokens joins its parts
cut by cut instead of token by token: both begin at sizes that the other tests do not reach. The bounds are those of
attention_cases.py.
"""

import math

import pytest
import torch

from adaptive_sparse.attention import shared_prefix_attention, topk_attention

from attention_cases import answer_of, attend, check, make_pool, make_problem

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def run(problem, **extra):
    out = torch.full_like(problem.query, float("nan"))
    lse = torch.full(problem.query.shape[:2], float("nan"), dtype=torch.float32, device=out.device)
    problem.call(shared_prefix_attention, out, lse, **extra)
    return out, lse


def verify(problem, **extra):
    print(f"[attention] {tuple(problem.query.shape)} rows {len(problem.lengths)}", flush=True)
    out, lse = run(problem, **extra)
    check(out, lse, problem.answer(), problem.query.shape[2])


def ragged_lengths(batch, most, seed):
    gen = torch.Generator().manual_seed(seed)
    lengths = (torch.rand(batch, generator=gen) ** 4 * most).long()
    lengths[::17] = 0
    return lengths.tolist()


@pytest.mark.parametrize("batch", [127, 128, 129, 255, 256, 257, 600])
def test_decode_batches_without_a_prefix(gpu, batch):
    verify(make_problem(gpu, heads=4, kv_heads=2, dim=64, lengths=ragged_lengths(batch, 700, batch), prefixes=None,
                        seed=batch))


@pytest.mark.parametrize("batch,groups", [(128, 3), (129, 128), (300, 129), (530, 257)])
def test_decode_batches_in_many_groups(gpu, batch, groups):
    gen = torch.Generator().manual_seed(batch)
    starts = torch.randint(0, batch + 1, (groups + 1,), generator=gen).sort().values.tolist()
    prefixes = ragged_lengths(groups, 400, groups)
    verify(make_problem(gpu, heads=8, kv_heads=2, dim=96, lengths=ragged_lengths(batch, 300, batch), prefixes=prefixes,
                        groups=starts, seed=groups))


@pytest.mark.parametrize("dtype,dim,heads,kv_heads", [(BF16, 128, 16, 8), (F16, 64, 40, 8), (BF16, 256, 16, 8)])
def test_decode_of_more_rows_than_are_joined_by_token(gpu, dtype, dim, heads, kv_heads):
    lengths = ragged_lengths(530, 400, dim)
    lengths[3], lengths[400] = 9000, 2049
    verify(make_problem(gpu, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, lengths=lengths, prefixes=None,
                        seed=dim))


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 80), (BF16, 192)])
@pytest.mark.parametrize("share", [1, 6])
def test_prompt_batches(gpu, dtype, dim, share):
    batch = 270
    counts = [(7 * i) % 17 for i in range(batch)]
    counts[5], counts[200] = 300, 131
    lengths = [n + (31 * i) % 90 for i, n in enumerate(counts)]
    lengths[5] = 5000
    problem = make_problem(gpu, dtype=dtype, heads=4 * share, kv_heads=4, dim=dim, lengths=lengths, counts=counts,
                           prefixes=[70, 0, 333], groups=[2, 90, 91, 260], tail=5, seed=dim + share)
    verify(problem)


@pytest.mark.parametrize("prefixes", [None, [50]])
def test_tokens_in_front_of_the_first_row(gpu, prefixes):
    # 4 + 1300 + 3 tokens of 4 KV heads; the rows' tokens are 4 .. 1303.
    problem = make_problem(gpu, heads=8, kv_heads=4, dim=64, lengths=[700, 640], counts=[660, 640], prefixes=prefixes,
                           tail=7, seed=21)
    want = problem.answer()
    starts = torch.tensor([4 + n for n in problem.starts()], dtype=torch.int32, device=gpu)
    problem.query = problem.query.roll(4, 0)
    out, lse = run(problem, query_starts=starts)
    for t in (*range(4), *range(1304, 1307)):
        assert not out[t].any() and (lse[t] == -math.inf).all()
    check(out.roll(-4, 0), lse.roll(-4, 0), want, 64)


@pytest.mark.parametrize("scale", [-0.11, 0.0, -3.0, 1e-30])
@pytest.mark.parametrize("counts", [None, [30, 2, 90]])
def test_scales(gpu, scale, counts):
    problem = make_problem(gpu, heads=8, kv_heads=2, dim=96, lengths=[200, 9, 90], counts=counts, prefixes=[150],
                           magnitude=1.0, seed=31)
    problem.scale = scale
    verify(problem)


def test_without_statistics(gpu):
    problem = make_problem(gpu, lengths=[40, 3], prefixes=[150], seed=32)
    want, _ = run(problem)
    out = torch.full_like(problem.query, float("nan"))
    problem.call(shared_prefix_attention, out, None)
    assert torch.equal(out, want)


@pytest.mark.parametrize("heads,lanes", [(16, 90), (80, 700)])
def test_topk_of_more_tokens_than_are_joined_by_token(gpu, heads, lanes):
    tokens, kv_heads, dim = 530, 8, 64
    pool = make_pool(gpu, BF16, 3000, 1, kv_heads, dim, seed=lanes)
    gen = torch.Generator(device=gpu).manual_seed(lanes)
    slots = torch.randint(-1, 3000, (tokens, lanes), generator=gen, device=gpu, dtype=torch.int32)
    slots[7] = 0
    query = torch.randn((tokens, heads, dim), generator=gen, device=gpu).to(BF16)
    out, lse = torch.full_like(query, float("nan")), torch.empty((tokens, heads), device=gpu)
    topk_attention(query, pool.planes, slots, out, kv_heads=kv_heads, layer=pool.layer, lse=lse)
    parts = []
    for t in range(tokens):
        at = slots[t].long()
        seen = at >= 1
        at = torch.where(seen, at, 0)
        parts.append(attend(query[t], pool.keys[at, 0], pool.values[at, 0], dim ** -0.5, seen))
    check(out, lse, answer_of(parts), dim)


@pytest.mark.parametrize("tokens", [5, 3000])
@pytest.mark.parametrize("prefixes", [None, [50]])
def test_a_batch_of_no_rows(gpu, tokens, prefixes):
    problem = make_problem(gpu, heads=4, kv_heads=2, dim=64, lengths=[30], prefixes=prefixes, permute=False)
    problem.query = torch.randn((tokens, 4, 64), device=gpu).to(BF16)
    problem.lengths, problem.counts = [], []
    if prefixes is not None:
        problem.group_starts = [0, 0]
    out, lse = run(problem)
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("most", [1, 40])
def test_starts_out_of_order_stay_in_bounds(gpu, most):
    """What such starts give is not defined, but a later call finds its inputs and the memory around as they were."""
    problem = make_problem(gpu, heads=8, kv_heads=2, dim=64, lengths=[40, 40, 40], counts=[4, 4, 4],
                           prefixes=[100, 30], groups=[0, 2, 3], seed=41)
    want = problem.answer()
    memory = torch.full((14, 8, 64), 7.0, dtype=BF16, device=gpu)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    problem.call(shared_prefix_attention, memory[1:13], None, query_starts=ints([0, 9, 3, 12]),
                 group_starts=ints([0, 3, 1]), max_query=most)
    torch.cuda.synchronize()
    assert (memory[0] == 7).all() and (memory[13] == 7).all()
    out, lse = run(problem)
    check(out, lse, want, 64)
