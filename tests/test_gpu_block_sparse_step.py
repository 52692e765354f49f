"""The operators of a block-sparse step run together, as a server runs them: tables extended, tokens appended, blocks
selected, attention over them, layer by layer, for prompts' pieces and for single tokens.

Each stage is compared with its definition on what the stages before it left in the pool. While the lists hold the whole
context, the outputs are also compared with attention computed from the projections alone: rotation, cache, lists and
softmax in 64 bits. There a score is off by the two roundings of its query and key, e = scale * sum|q k| * 2^-7 (1.01 for
products of both and the rotation's own error), its weight by a factor within exp(-2 e) .. exp(2 e), so an output by
(exp(2 e) - 1) * sum(w |v|), beside the bound of attention_cases.py.
"""

import math

import pytest
import torch

from adaptive_sparse.append import append_index, append_rotary, make_rotary
from adaptive_sparse.attention import block_attention, block_workspace
from adaptive_sparse.block_selection import select_blocks, selection_workspace
from adaptive_sparse.block_tables import check_table_status, extend_block_tables

from attention_cases import UNIT, check, make_pool
from block_cases import Batch, BlockProblem, codes_of, make_index_pool, selection
from test_gpu_append import near, turned

pytestmark = pytest.mark.gpu

LAYERS, HEADS, KV_HEADS, DIM, INDEX_HEADS, INDEX_DIM = 2, 8, 2, 64, 4, 64
PAGE, BLOCK, CHOSEN, MOST = 16, 32, 5, 640
SCALE = DIM ** -0.5


class Server:
    """A pool of K, V and index keys, and the step's tensors for up to `room` tokens."""

    def __init__(self, gpu, requests, room, dtype=torch.bfloat16):
        self.requests, self.room = requests, room
        pages = 1 + requests * MOST // PAGE
        self.pools = [make_pool(gpu, dtype, pages, PAGE, KV_HEADS, DIM, layers=LAYERS, layer=i) for i in range(LAYERS)]
        # One memory of all layers.
        for p in self.pools[1:]:
            p.memory, p.planes = self.pools[0].memory, self.pools[0].planes
            p.keys, p.values = self.pools[0].memory[p.layer, 0], self.pools[0].memory[p.layer, 1]
        self.index = [make_index_pool(gpu, pages, PAGE, INDEX_DIM, layers=1, layer=0, seed=i) for i in range(LAYERS)]
        self.rotary, self.index_rotary = make_rotary(DIM, device=gpu), make_rotary(32, device=gpu, interleaved=True)
        ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=gpu)  # noqa: E731
        self.tables, self.lengths, self.new_lengths = ints(requests, MOST // PAGE), ints(requests), ints(requests)
        self.rows = torch.arange(requests - 1, -1, -1, device=gpu)
        gen = torch.Generator(device=gpu).manual_seed(3)
        self.free = (torch.randperm(pages - 1, generator=gen, device=gpu) + 1).to(torch.int32)
        self.head, self.new_head, self.status = ints(1), ints(1), ints(1)
        self.slots, self.positions, self.starts = ints(room), ints(room), ints(requests + 1)
        self.blocks = ints(LAYERS, room, 1, CHOSEN)
        self.outputs = torch.zeros((LAYERS, room, HEADS, DIM), dtype=dtype, device=gpu)
        self.queries, self.index_parts = torch.zeros_like(self.outputs), torch.zeros(
            (LAYERS, room, INDEX_HEADS + 1, INDEX_DIM), dtype=dtype, device=gpu)
        size = selection_workspace(room, 1, MOST // PAGE, PAGE, BLOCK)
        self.selecting = torch.empty(size, dtype=torch.uint8, device=gpu)
        size = block_workspace(room, CHOSEN, BLOCK, HEADS, KV_HEADS, DIM, room)
        self.attending = torch.empty(size, dtype=torch.uint8, device=gpu)

    def step(self, added, projections, index_projections, most):
        """`added` tokens of each batch row: projections [L, room, (Hq + 2 Hkv) * D] and [L, room, (Hi + 1) * Di]."""
        extend_block_tables(self.tables, self.rows, self.lengths, added, self.free, self.head, PAGE, slots=self.slots,
                            positions=self.positions, starts=self.starts, new_lengths=self.new_lengths,
                            new_head=self.new_head, status=self.status)
        self.lengths.copy_(self.new_lengths)
        self.head.copy_(self.new_head)
        for i in range(LAYERS):
            parts = projections[i].view(self.room, HEADS + 2 * KV_HEADS, DIM)
            query, key, value = parts.split([HEADS, KV_HEADS, KV_HEADS], 1)
            append_rotary(query, key, value, self.pools[i].planes, self.slots, self.positions, self.rotary,
                          self.queries[i], page_size=PAGE, layer=self.pools[i].layer)
            append_rotary(index_projections[i].view(self.room, INDEX_HEADS + 1, INDEX_DIM), None, None, None, None,
                          self.positions, self.index_rotary, self.index_parts[i])
            append_index(self.index_parts[i][:, INDEX_HEADS], self.index[i].planes, self.index[i].scales, self.slots,
                         page_size=PAGE)
            select_blocks(self.index_parts[i][:, :INDEX_HEADS], self.index[i].planes, self.index[i].scales, self.tables,
                          self.rows, self.lengths, self.blocks[i], page_size=PAGE, block_size=BLOCK,
                          query_starts=self.starts, max_query=most, first=1, last=2, workspace=self.selecting)
            block_attention(self.queries[i], self.pools[i].planes, self.tables, self.rows, self.lengths, self.blocks[i],
                            self.outputs[i], page_size=PAGE, block_size=BLOCK, kv_heads=KV_HEADS,
                            layer=self.pools[i].layer, query_starts=self.starts, max_query=most, scale=SCALE,
                            workspace=self.attending)

    def state(self):
        return [self.pools[0].memory, *[p.memory for p in self.index], *[p.scales for p in self.index], self.tables,
                self.lengths, self.head, self.blocks, self.outputs]


def inputs(gpu, room, seed, dtype=torch.bfloat16):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    shape = (LAYERS, room, (HEADS + 2 * KV_HEADS) * DIM)
    index = (LAYERS, room, (INDEX_HEADS + 1) * INDEX_DIM)
    return [torch.randn(s, generator=gen, device=gpu).to(dtype) for s in (shape, index)]


def from_projections(held, query, positions, rotary):
    """(output, bound) of one query token over a request's keys and values as they were projected."""
    keys, values = held
    turned_q, _ = turned(query.unsqueeze(0), positions[-1:], rotary)
    turned_k, _ = turned(keys, positions, rotary)
    share = HEADS // KV_HEADS
    k, v = (x.double().repeat_interleave(share, 1) for x in (turned_k, values))        # [T, Hq, D]
    products = k * turned_q
    score, size = SCALE * products.sum(-1), SCALE * products.abs().sum(-1)             # [T, Hq]
    weight = torch.softmax(score, 0).unsqueeze(-1)
    out, mass = (weight * v).sum(0), (weight * v.abs()).sum(0)
    off = 1.01 * 2.0 ** -7 * size.amax(0).unsqueeze(-1)
    unit = UNIT[query.dtype]
    far = torch.expm1(2 * off) * mass
    return out, unit * (out.abs() + far) + (unit + 2.0 ** -12) * (mass + far) + far + 2.0 ** -24


def test_prompts_and_single_tokens(gpu):
    server = Server(gpu, 3, 300)
    held = [[[torch.zeros((0, KV_HEADS, DIM), dtype=torch.bfloat16, device=gpu)] * 2 for _ in range(LAYERS)]
            for _ in range(3)]
    lengths = [0, 0, 0]
    whole = 0
    for turn, added in enumerate(([40, 1, 90], [1, 1, 1], [0, 33, 5], [150, 100, 50], [1, 1, 1], [1, 0, 1])):
        print(f"[step] {turn} {added}", flush=True)
        given = inputs(gpu, 300, turn)
        server.outputs.fill_(5.0)
        server.step(torch.tensor(added, dtype=torch.int32, device=gpu), *given, max(added))
        check_table_status(server.status)
        lengths = [n + m for n, m in zip(lengths, added)]
        total = sum(added)
        assert server.lengths.tolist() == lengths
        batch = Batch(lengths, added, server.tables, server.rows, server.pools[0].keys.shape[0], PAGE, torch.int32)
        at = server.slots[:total].long()
        assert bool((server.slots[total:] == -1).all()) and bool((server.positions[total:] == -1).all())
        for i in range(LAYERS):
            parts = given[0][i].view(300, HEADS + 2 * KV_HEADS, DIM)[:total]
            query, key, value = parts.split([HEADS, KV_HEADS, KV_HEADS], 1)
            pool, index, positions = server.pools[i], server.index[i], server.positions[:total]
            want, bound = turned(query, positions, server.rotary)
            near(server.queries[i, :total], want, bound, "a query")
            want, bound = turned(key, positions, server.rotary)
            near(pool.keys[at // PAGE, at % PAGE], want, bound, "a key")
            assert torch.equal(pool.values[at // PAGE, at % PAGE], value)
            codes, scales = codes_of(server.index_parts[i, :total, INDEX_HEADS])
            assert torch.equal(index.keys[at // PAGE, at % PAGE].cpu().long(), torch.from_numpy(codes))
            assert torch.equal(index.scales[at].cpu(), torch.from_numpy(scales))
            want = selection(batch, index, server.index_parts[i, :, :INDEX_HEADS], 1, CHOSEN, BLOCK, 1, 2)
            assert torch.equal(server.blocks[i].cpu(), want)
            problem = BlockProblem(batch, pool, server.queries[i], server.blocks[i], BLOCK, SCALE)
            check(server.outputs[i], None, problem.answer(), DIM)
            # From the projections alone, where all blocks are chosen.
            start = 0
            for b, n in enumerate(added):
                held[b][i] = [torch.cat([old, new[start:start + n]]) for old, new in zip(held[b][i], (key, value))]
                for m in range(n):
                    seen = lengths[b] - n + m + 1
                    if seen <= CHOSEN * BLOCK:
                        keys, values = (x[:seen] for x in held[b][i])
                        out, bound = from_projections((keys, values), query[start + m],
                                                      torch.arange(seen, device=gpu), server.rotary)
                        assert bool(((server.outputs[i, start + m].double() - out).abs() <= bound).all())
                        whole += 1
                start += n
        assert bool((server.outputs[:, total:] == 0).all())          # rows behind the last sequence see nothing
    assert whole > 2 * 300 and math.ceil(max(lengths) / BLOCK) > CHOSEN


def test_a_captured_step_is_replayed(gpu):
    """Steps of single tokens from a graph, against the same steps called one by one on another copy."""
    requests = 3
    servers = [Server(gpu, requests, requests) for _ in range(2)]
    prompt = Server(gpu, requests, 200)
    prompt.step(torch.tensor([100, 30, 70], dtype=torch.int32, device=gpu), *inputs(gpu, 200, 50), 100)
    for server in servers:
        for mine, other in zip(server.state()[:-2], prompt.state()[:-2]):
            mine.copy_(other)
        for mine, other in zip((server.free, server.head), (prompt.free, prompt.head)):
            mine.copy_(other)
    one = torch.ones(requests, dtype=torch.int32, device=gpu)
    given = inputs(gpu, requests, 0)
    kept = [x.clone() for x in servers[0].state()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        servers[0].step(one, *given, 1)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        servers[0].step(one, *given, 1)
    for mine, old in zip(servers[0].state(), kept):
        mine.copy_(old)
    for turn in range(5):
        fresh = inputs(gpu, requests, 100 + turn)
        for mine, new in zip(given, fresh):
            mine.copy_(new)
        graph.replay()
        servers[1].step(one, *fresh, 1)
        torch.cuda.synchronize()
        for mine, other in zip(servers[0].state(), servers[1].state()):
            assert torch.equal(mine, other), f"step {turn}"
        check_table_status(servers[0].status)
        assert servers[0].lengths.tolist() == [101 + turn, 31 + turn, 71 + turn]
