"""append_rotary and append_index against their definitions: rotations in 64 bits, codes on the host.

The angle of a pair is its turns times the position, in whole numbers, so the answer's angles are exact. The kernel's
sine and cosine come from an angle of at most pi / 4 held in 32 bits and a series in 32 bits: 2^-22 off at most. A result
then has that error times both elements, a few roundings of 32 bits, and its own rounding of half a step.
"""

import math

import pytest
import torch

from adaptive_sparse.append import append_index, append_rotary, make_rotary
from adaptive_sparse.kv_pool import KVPlanes

from attention_cases import make_pool
from block_cases import codes_of

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
STEP = {BF16: 2.0 ** -133, F16: 2.0 ** -24}        # the smallest numbers' step


def turned(x, positions, rotary):
    """(result in 64 bits, how far it may be off) of rows [N, H, D]."""
    half = len(rotary.turns)
    turns = [t % 2 ** 64 for t in rotary.turns.tolist()]
    angle = torch.tensor([[2 * math.pi * ((max(p, 0) * t) % 2 ** 64) / 2 ** 64 for t in turns]
                          for p in positions.tolist()], dtype=torch.float64, device=x.device).unsqueeze(1)
    cos, sin = torch.cos(angle) * rotary.magnitude, torch.sin(angle) * rotary.magnitude
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if rotary.interleaved else (i, i + half)
    y, slack = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    m, n = x[..., a].double(), x[..., b].double()
    y[..., a], y[..., b] = m * cos - n * sin, n * cos + m * sin
    slack[..., a] = slack[..., b] = (m.abs() + n.abs()) * 2.0 ** -21 * abs(rotary.magnitude)
    unit = torch.finfo(x.dtype).eps / 2
    bound = unit * y.abs() + 1.01 * slack + STEP[x.dtype]
    return y, torch.where(slack > 0, bound, 0.0)


def near(got, want, bound, what):
    error = (got.double() - want).abs()
    assert bool((error <= bound).all()), f"{what} is {float((error / bound.clamp_min(1e-300)).max()):.3f} of its bound away"


CASES = [
    # tokens, query heads, KV heads, head size, rotated, neighbours, page, layout
    (1, 16, 2, 128, 128, False, 16, "planes"),
    (7, 16, 2, 128, 128, False, 16, "blocks"),
    (1, 1, 1, 8, 8, False, 1, "planes"),
    (5, 3, 1, 8, 2, True, 4, "planes"),
    (9, 6, 2, 64, 64, True, 16, "blocks"),
    (33, 12, 4, 80, 80, False, 100, "planes"),     # 40 pairs: pieces of 8
    (33, 12, 4, 80, 24, True, 100, "blocks"),      # three pieces of 8 rotated
    (33, 12, 4, 80, 24, False, 1, "planes"),       # 12 pairs: pieces of 4
    (18, 4, 2, 96, 20, False, 16, "blocks"),       # 10 pairs: pieces of 2
    (18, 4, 2, 96, 22, False, 16, "planes"),       # 11 pairs: single elements
    (18, 4, 2, 96, 22, True, 16, "planes"),
    (18, 4, 2, 96, 36, True, 16, "planes"),
    (20, 8, 8, 256, 256, False, 64, "planes"),
    (20, 8, 8, 256, 64, True, 64, "blocks"),
    (1100, 8, 2, 128, 64, False, 16, "planes"),    # several tokens a workgroup, the last one's part-filled
    (1027, 2, 2, 64, 64, True, 3, "blocks"),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_append_rotary(gpu, dtype, case):
    tokens, heads, kv_heads, dim, size, neighbours, page, layout = case
    print(f"[append] {case} {dtype}", flush=True)
    gen = torch.Generator(device=gpu).manual_seed(tokens + size)
    pages = 3 + -(-tokens // page)
    pool = make_pool(gpu, dtype, pages, page, kv_heads, dim, layout)
    before = pool.memory.clone()
    both = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=gen, device=gpu).to(dtype)
    query, key, value = both.split([heads, kv_heads, kv_heads], 1)
    slots = (torch.randperm(pages * page - page, generator=gen, device=gpu)[:tokens] + page).to(torch.int32)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen, device=gpu)
    if tokens > 4:
        positions[2] = -1                    # left out
        positions[1] = (1 << 30) + 12345
        slots[3], slots[4] = 0, -1           # rotated, but no row
        slots[0] = pages * page              # past the pool
    rotary = make_rotary(size, device=gpu, interleaved=neighbours, magnitude=1.25 if size % 16 else 1.0)
    output = torch.full((tokens, heads, dim), 7.0, dtype=dtype, device=gpu)
    append_rotary(query, key, value, pool.planes, slots, positions, rotary, output, page_size=page, layer=pool.layer)
    live = positions >= 0
    want, bound = turned(query, positions, rotary)
    near(output[live], want[live], bound[live], "a query")
    assert bool((output[~live] == 7.0).all()), "the output of a token that is left out"
    written = live & (slots >= 1) & (slots < pages * page)
    at = slots[written].long()
    want, bound = turned(key, positions, rotary)
    near(pool.keys[at // page, at % page], want[written], bound[written], "a key")
    assert torch.equal(pool.values[at // page, at % page], value[written])
    # Nothing else was written.
    pool.keys[at // page, at % page] = 0
    pool.values[at // page, at % page] = 0
    other = make_pool(gpu, dtype, pages, page, kv_heads, dim, layout)
    assert torch.equal(other.memory, before)
    other.keys[at // page, at % page] = 0
    other.values[at // page, at % page] = 0
    assert torch.equal(pool.memory, other.memory)


def test_in_place_parts_and_other_index_types(gpu):
    gen = torch.Generator(device=gpu).manual_seed(0)
    rotary = make_rotary(64, device=gpu)
    both = torch.randn((50, 12, 128), generator=gen, device=gpu).to(BF16)
    kept = both.clone()
    query, key, value = both[:, :8], both[:, 8:10], both[:, 10:]
    pool = make_pool(gpu, BF16, 6, 16, 2, 128)
    positions = torch.arange(50, device=gpu, dtype=torch.int32) * 1000
    table = torch.stack([positions.long(), torch.arange(50, device=gpu) + 16], 1)     # columns of one tensor
    append_rotary(query, key, value, pool.planes, table[:, 1], table[:, 0], rotary, query, page_size=16, layer=1)
    want, bound = turned(kept[:, :8], positions, rotary)
    near(query, want, bound, "a query rotated in place")
    assert torch.equal(both[:, 8:], kept[:, 8:])
    keys = pool.keys.reshape(-1, 2, 128)[16:66].clone()
    # Only queries, only keys and values.
    out = torch.empty_like(kept[:, :8])
    append_rotary(kept[:, :8], None, None, None, None, positions, rotary, out)
    assert torch.equal(out, query)
    pool.memory.zero_()
    append_rotary(None, kept[:, 8:10], kept[:, 10:], pool.planes, table[:, 1].int(), positions, rotary, None, page_size=16,
                  layer=1)
    assert torch.equal(pool.keys.reshape(-1, 2, 128)[16:66], keys)
    assert torch.equal(pool.values.reshape(-1, 2, 128)[16:66], kept[:, 10:])


def test_token_rows_behind_the_last_whole_page_are_slots_too(gpu):
    memory = torch.zeros((2, 21, 1, 64), dtype=BF16, device=gpu)
    planes = KVPlanes(base=memory.data_ptr(), device=0, layers=1, kv=2, layer_stride=0, kv_stride=21 * 128,
                      row_stride=128, row_bytes=128, rows=21, owner=memory)
    key = torch.ones((2, 1, 64), dtype=BF16, device=gpu)
    append_rotary(None, key, key, planes, torch.tensor([20, 21], device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu),
                  make_rotary(64, device=gpu), None, page_size=16)
    assert bool((memory[:, 20] == 1).all()) and not bool(memory[:, :20].any())


def test_no_tokens(gpu):
    rotary = make_rotary(64, device=gpu)
    none = torch.empty((0, 4, 64), dtype=BF16, device=gpu)
    ints = torch.empty(0, dtype=torch.int32, device=gpu)
    append_rotary(none, None, None, None, None, ints, rotary, torch.empty_like(none))
    keys = torch.zeros((64, 32), dtype=torch.int8, device=gpu)
    planes = KVPlanes(base=keys.data_ptr(), device=0, layers=1, kv=1, layer_stride=0, kv_stride=0, row_stride=32,
                      row_bytes=32, rows=64, owner=keys)
    append_index(torch.empty((0, 32), dtype=BF16, device=gpu), planes, torch.zeros(64, device=gpu), ints, page_size=16)


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("base", 8.0), ("ramp", 32.0)])
def test_scaled_frequencies_turn_heads(gpu, scaling, factor):
    rotary = make_rotary(128, device=gpu, scaling=scaling, factor=factor, original=4096)
    query = torch.randn((3, 2, 128), device=gpu).to(BF16)
    positions = torch.tensor([1, 4095, 130000], device=gpu)
    out = torch.empty_like(query)
    append_rotary(query, None, None, None, None, positions, rotary, out)
    want, bound = turned(query, positions, rotary)
    near(out, want, bound, scaling)
    # The same by the frequencies themselves: an angle in 64 bits at these positions is 2^-36 off at most.
    angle = positions.double().view(-1, 1, 1) * torch.tensor(rotary.frequencies, dtype=torch.float64, device=gpu)
    first = query[..., :64].double() * angle.cos() - query[..., 64:].double() * angle.sin()
    near(out[..., :64], first * rotary.magnitude, bound[..., :64], scaling)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 128, 176, 256])
def test_append_index(gpu, dtype, dim):
    gen = torch.Generator(device=gpu).manual_seed(dim)
    tokens, page = 301, 16
    key = (torch.randn((tokens, dim + 16), generator=gen, device=gpu)
           * torch.exp(2 * torch.randn((tokens, 1), generator=gen, device=gpu)).clamp_max(1000)).to(dtype)[:, :dim]
    key[5] = 0
    key[6] = 2.0 ** -24                          # equal and small: codes of 127
    key[7, 1:] = 0
    key[8] *= -1
    pages = 22
    memory = torch.full((pages, 2, page, dim), 3, dtype=torch.int8, device=gpu)
    planes = KVPlanes(base=memory.data_ptr(), device=0, layers=2, kv=1, layer_stride=page * dim, kv_stride=page * dim,
                      row_stride=2 * page * dim, row_bytes=page * dim, rows=pages, owner=memory)
    scales = torch.full((2, pages * page), 9.0, device=gpu)
    slots = torch.randperm(pages * page - page, generator=gen, device=gpu)[:tokens] + page
    slots[10], slots[11], slots[12] = 0, -1, pages * page
    append_index(key, planes, scales[1], slots, page_size=page, layer=1)
    codes, scale = codes_of(key)
    good = (slots >= 1) & (slots < pages * page)
    at = slots[good]
    want = torch.full_like(memory[:, 1], 3)
    want[at // page, at % page] = torch.from_numpy(codes).to(gpu).to(torch.int8)[good]
    assert torch.equal(memory[:, 1], want) and bool((memory[:, 0] == 3).all())
    want = torch.full_like(scales, 9.0)
    want[1, at] = torch.from_numpy(scale).to(gpu)[good]
    assert torch.equal(scales, want)


def test_appends_replay_in_a_graph_on_another_stream(gpu):
    gen = torch.Generator(device=gpu).manual_seed(3)
    rotary = make_rotary(128, device=gpu)
    pool = make_pool(gpu, BF16, 5, 16, 2, 128)
    both = torch.randn((20, 8, 128), generator=gen, device=gpu).to(BF16)
    out = torch.empty((20, 4, 128), dtype=BF16, device=gpu)
    positions = torch.arange(20, device=gpu, dtype=torch.int32)
    slots = positions + 16
    args = (both[:, :4], both[:, 4:6], both[:, 6:], pool.planes, slots, positions, rotary, out)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        append_rotary(*args, page_size=16, layer=1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            append_rotary(*args, page_size=16, layer=1)
    torch.cuda.synchronize()
    for step in range(3):
        positions += 1000
        both.normal_(generator=gen)
        out.zero_()
        pool.memory.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, rows = out.clone(), pool.memory.clone()
        out.zero_()
        pool.memory.zero_()
        append_rotary(*args, page_size=16, layer=1)
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(rows, pool.memory)
        want, bound = turned(both[:, :4], positions, rotary)
        near(out, want, bound, f"step {step}")
