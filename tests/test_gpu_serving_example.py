"""The serving loop of examples/shared_prefix_serving.py: its operators' outputs against the rows that it wrote.

K and V are kept by the test as they are written, so that a wrong page, slot, length or start anywhere in the chain
shows as a wrong output. The bounds are those of attention_cases.py.
"""

import sys

import pytest
import torch

from attention_cases import answer_of, attend, check
from conftest import PACKAGE

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, str(PACKAGE / "examples"))
    try:
        import shared_prefix_serving
    finally:
        sys.path.pop(0)
    return shared_prefix_serving


def test_the_loop_runs(gpu, example):
    outputs = example.run(torch.device("cuda:0"), steps=3)
    assert len(outputs) == 3
    for dense, sparse in outputs:
        assert torch.isfinite(dense).all() and torch.isfinite(sparse).all() and dense.any() and sparse.any()


def test_every_step_attends_to_what_was_written(gpu, example):
    torch.manual_seed(3)
    prompts, prefix = [20, 1, 77], 130
    serving = example.Serving(3, prefix, 90, gpu)
    try:
        pool = serving.pool
        planes = [[pool.plane_rows(layer, kv).view(torch.bfloat16).view(-1, example.KV_HEADS, example.DIM)
                   for kv in range(2)] for layer in range(example.LAYERS)]
        at = torch.arange(prefix, device=gpu)
        shared = serving.prefix_table[0].long()[at // example.PAGE] * example.PAGE + at % example.PAGE
        shared = [[plane[shared].clone() for plane in pair] for pair in planes]
        held = [[[torch.empty(0, example.KV_HEADS, example.DIM, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
                 for _ in range(example.LAYERS)] for _ in prompts]
        for added in (prompts, [1, 1, 1], [0, 5, 3], [1, 1, 1]):
            rows = serving.extend(torch.tensor(added, dtype=torch.int32, device=gpu), sum(added))
            start = 0
            for b, n in enumerate(added):
                for layer in range(example.LAYERS):
                    for kv in range(2):
                        held[b][layer][kv] = torch.cat([held[b][layer][kv], rows[layer, kv, start:start + n]])
                start += n
            everything = torch.arange(90, dtype=torch.int32, device=gpu).expand(example.LAYERS, 3, 90)
            slots = serving.select(everything)
            for layer in range(example.LAYERS):
                query = example.queries(sum(added), gpu)
                want, first, scale = [], 0, example.DIM ** -0.5
                for b, n in enumerate(added):
                    for i in range(n):
                        keys, values = (torch.cat([shared[layer][kv],
                                                   held[b][layer][kv][:held[b][layer][kv].shape[0] - n + i + 1]])
                                        for kv in range(2))
                        seen = torch.ones(keys.shape[0], dtype=torch.bool, device=gpu)
                        want.append(attend(query[first + i], keys, values, scale, seen))
                    first += n
                check(serving.attend(layer, query, max(added)), None, answer_of(want), example.DIM)
                query = example.queries(3, gpu)
                lse = torch.empty(query.shape[:2], device=gpu)
                out = serving.attend_selected(layer, query, slots, lse)
                want = [attend(query[b], *held[b][layer], scale,
                               torch.ones(held[b][layer][0].shape[0], dtype=torch.bool, device=gpu)) for b in range(3)]
                check(out, lse, answer_of(want), example.DIM)
        example.check_table_status(serving.status)
    finally:
        serving.close()
