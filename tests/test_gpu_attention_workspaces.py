"""The attentions write inside the workspace that they ask for, whatever is around it, at sizes with more items than parts.

The bounds are those of attention_cases.py.
"""

import pytest
import torch

from adaptive_sparse.attention import (shared_prefix_attention, shared_prefix_workspace, topk_attention,
                                       topk_workspace)

from attention_cases import answer_of, attend, check, make_pool, make_problem

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
GUARD = 1 << 20


def guarded(size, device):
    """A workspace of exactly `size` bytes between two guards, NaN in all of its words."""
    whole = torch.full((GUARD + size + GUARD,), 255, dtype=torch.uint8, device=device)
    return whole, whole[GUARD:GUARD + size]


def untouched(whole, size):
    return bool((whole[:GUARD] == 255).all()) and bool((whole[GUARD + size:] == 255).all())


@pytest.mark.parametrize("name,dtype,heads,kv_heads,dim,batch,count,prefixes", [
    ("16 rows", BF16, 8, 4, 128, 400, 1, None),
    ("16 rows, by cuts", F16, 16, 8, 64, 400, 1, None),
    ("32 rows", BF16, 60, 2, 64, 400, 1, None),
    ("64 rows", F16, 128, 2, 128, 300, 1, None),
    ("128 rows", BF16, 16, 4, 128, 200, 20, None),
    ("256 rows", BF16, 16, 4, 128, 30, 180, None),
    ("128 rows of 256", F16, 16, 4, 256, 100, 25, None),
    ("256 rows behind their prefixes", BF16, 16, 4, 96, 30, 180, [300]),
    ("prefixes of their own", BF16, 16, 4, 128, 300, 1, [500, 2000]),
])
def test_attention_stays_in_its_workspace(gpu, name, dtype, heads, kv_heads, dim, batch, count, prefixes):
    print(f"[attention] {name}", flush=True)
    counts = [1 + (count * (i % 7)) // 4 if count > 1 else 1 for i in range(batch)]
    lengths = [n + int(700 * ((i * 0.6180339887498949) % 1.0) ** 4) for i, n in enumerate(counts)]
    lengths[batch // 2] = 9000
    groups = None if prefixes is None else [0, batch] if len(prefixes) == 1 else [0, batch // 3, batch]
    problem = make_problem(gpu, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, lengths=lengths, counts=counts,
                           prefixes=prefixes, groups=groups, seed=dim)
    size = shared_prefix_workspace(sum(counts), batch, len(prefixes or []), heads, kv_heads, dim, max(counts))
    whole, workspace = guarded(size, gpu)
    out = torch.full_like(problem.query, float("nan"))
    lse = torch.full(out.shape[:2], float("nan"), device=gpu)
    problem.call(shared_prefix_attention, out, lse, workspace=workspace)
    assert untouched(whole, size)
    check(out, lse, problem.answer(), dim)


@pytest.mark.parametrize("heads,kv_heads,dim,tokens,lanes", [(16, 2, 128, 300, 900), (16, 8, 64, 300, 777),
                                                             (64, 1, 64, 600, 300), (256, 1, 96, 270, 300)])
def test_topk_stays_in_its_workspace(gpu, heads, kv_heads, dim, tokens, lanes):
    print(f"[attention] Top-K {heads} heads {kv_heads} KV heads {tokens} tokens", flush=True)
    pool = make_pool(gpu, BF16, 3000, 1, kv_heads, dim, seed=lanes)
    gen = torch.Generator(device=gpu).manual_seed(lanes)
    slots = torch.randint(-1, 3000, (tokens, lanes), generator=gen, device=gpu, dtype=torch.int32)
    query = torch.randn((tokens, heads, dim), generator=gen, device=gpu).to(BF16)
    size = topk_workspace(tokens, lanes, heads, kv_heads, dim)
    whole, workspace = guarded(size, gpu)
    out, lse = torch.full_like(query, float("nan")), torch.empty((tokens, heads), device=gpu)
    topk_attention(query, pool.planes, slots, out, kv_heads=kv_heads, layer=pool.layer, lse=lse, workspace=workspace)
    assert untouched(whole, size)
    parts = []
    for t in range(tokens):
        at = slots[t].long()
        at = torch.where(at >= 1, at, 0)
        parts.append(attend(query[t], pool.keys[at, 0], pool.values[at, 0], dim ** -0.5, at >= 1))
    check(out, lse, answer_of(parts), dim)
