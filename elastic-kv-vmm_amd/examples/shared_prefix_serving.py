"""A serving loop over the paged pool: requests behind a shared prefix, dense and Top-K attention of each step.

    python elastic-kv-vmm_amd/examples/shared_prefix_serving.py

Every step is four calls on the device, with no host round trip between them:

    extend_block_tables      pages and slots of the step's new tokens, from the request lengths
    scatter_kv               their K and V rows into the pool
    shared_prefix_attention  each layer; a decode step reads the prefix once per 128 query rows of all requests
    topk_attention           each layer, over the slots that resolve_resident finds for selected positions

K, V, queries and selections are random numbers in place of a model's. The reference's counterpart is its serving
coordinator's step (adaptive_sparse/request_residency.py:739-839), which leaves the attention to its engine.
"""

import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from adaptive_sparse.attention import (shared_prefix_attention, shared_prefix_workspace, topk_attention,
                                       topk_workspace)
from adaptive_sparse.block_tables import check_table_status, extend_block_tables
from adaptive_sparse.migration_engine import PlanePagedPool
from adaptive_sparse.resident_lookup import resolve_resident
from adaptive_sparse.sparse_read import scatter_kv

LAYERS, HEADS, KV_HEADS, DIM, PAGE = 2, 16, 2, 128, 16


class Serving:
    """Requests with one shared prefix: their pages, lengths and the buffers of a step."""

    def __init__(self, requests, prefix, most, device):
        self.device, self.requests, self.prefix, self.most = device, requests, prefix, most
        columns = -(-most // PAGE)
        pages = -(-prefix // PAGE) + requests * columns
        self.pool = PlanePagedPool(LAYERS, 2, pages, PAGE, KV_HEADS * DIM * 2, device=device.index or 0)
        ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
        self.free = torch.tensor(list(self.pool.take(pages)), dtype=torch.int32, device=device)
        self.head, self.next_head = ints(1), ints(1)
        self.tables, self.prefix_table = ints(requests, columns), ints(1, -(-prefix // PAGE))
        self.lengths, self.next_lengths = ints(requests), ints(requests)
        self.prefix_length = ints(1) + prefix
        self.starts, self.status = ints(requests + 1), ints(1)
        # Position -> slot of every request's own tokens, what the resident lookup reads.
        self.resident = ints(requests, most)
        self.rows = torch.arange(requests, device=device)
        self.workspaces = {}
        self.write(self.prefix_table, ints(1), ints(1) + prefix, prefix, ints(2), ints(1))

    def write(self, tables, lengths, added, tokens, starts, new_lengths):
        """Pages for `added` tokens of each row of `tables`, and random K and V in them: (slots, positions, K and V)."""
        slots = torch.empty(tokens, dtype=torch.int32, device=self.device)
        positions = torch.empty_like(slots)
        extend_block_tables(tables, None, lengths, added, self.free, self.head, PAGE, slots=slots,
                            positions=positions, starts=starts, new_lengths=new_lengths, new_head=self.next_head,
                            status=self.status)
        self.head, self.next_head = self.next_head, self.head
        rows = torch.randn((1, LAYERS, 2, tokens, KV_HEADS, DIM), device=self.device).to(torch.bfloat16)
        scatter_kv(self.pool.planes, slots.expand(LAYERS, 1, tokens), rows)
        return slots, positions, rows[0]

    def workspace(self, name, size):
        if name not in self.workspaces or self.workspaces[name].numel() < size:
            self.workspaces[name] = torch.empty(size, dtype=torch.uint8, device=self.device)
        return self.workspaces[name]

    def extend(self, added, tokens):
        """The step's new tokens, written; `tokens` is the sum of `added`."""
        slots, positions, rows = self.write(self.tables, self.lengths, added, tokens, self.starts, self.next_lengths)
        self.lengths, self.next_lengths = self.next_lengths, self.lengths
        request = torch.repeat_interleave(self.rows, added, output_size=tokens)
        self.resident[request, positions.long()] = slots
        return rows

    def attend(self, layer, query, max_query):
        """Attention of the step's query tokens to the prefix and to their requests' tokens."""
        output = torch.empty_like(query)
        size = shared_prefix_workspace(query.shape[0], self.requests, 1, HEADS, KV_HEADS, DIM, max_query)
        shared_prefix_attention(query, self.pool.planes, self.tables, None, self.lengths, self.prefix_table,
                                self.prefix_length, output, page_size=PAGE, kv_heads=KV_HEADS, layer=layer,
                                query_starts=self.starts, max_query=max_query,
                                workspace=self.workspace("prefix", size))
        return output

    def select(self, positions):
        """Slots [L, B, K] of selected positions [L, B, K]: 0 not resident, -1 past the length."""
        slots = torch.full(positions.shape, -1, dtype=torch.int32, device=self.device)
        resolve_resident(positions, self.resident, None, self.rows, self.lengths, self.rows, slots, 1)
        return slots

    def attend_selected(self, layer, query, slots, lse=None):
        output = torch.empty_like(query)
        size = topk_workspace(query.shape[0], slots.shape[2], HEADS, KV_HEADS, DIM)
        topk_attention(query, self.pool.planes, slots[layer], output, kv_heads=KV_HEADS, layer=layer, lse=lse,
                       workspace=self.workspace("topk", size))
        return output

    def close(self):
        self.pool.close()


def queries(tokens, device):
    return torch.randn((tokens, HEADS, DIM), device=device).to(torch.bfloat16)


def run(device, prompts=(40, 7, 100, 33), prefix=1000, steps=4, lanes=64):
    """Prompts, then decode steps. Returns each step's dense and Top-K outputs of the last layer."""
    torch.manual_seed(0)
    serving = Serving(len(prompts), prefix, max(prompts) + steps, device)
    try:
        added = torch.tensor(prompts, dtype=torch.int32, device=device)
        serving.extend(added, sum(prompts))
        for layer in range(LAYERS):
            serving.attend(layer, queries(sum(prompts), device), max(prompts))
        one = torch.ones_like(added)
        outputs = []
        for _ in range(steps):
            serving.extend(one, len(prompts))
            selected = torch.rand((LAYERS, len(prompts), lanes), device=device) * serving.lengths.view(1, -1, 1)
            slots = serving.select(selected.int())
            for layer in range(LAYERS):
                query = queries(len(prompts), device)
                dense = serving.attend(layer, query, 1)
                sparse = serving.attend_selected(layer, query, slots)
            outputs.append((dense, sparse))
        check_table_status(serving.status)
        torch.cuda.synchronize(device)
        return outputs
    finally:
        serving.close()


if __name__ == "__main__":
    for step, (dense, sparse) in enumerate(run(torch.device("cuda:0"))):
        print(f"step {step}: dense {tuple(dense.shape)} rms {float(dense.float().square().mean().sqrt()):.4f}, "
              f"Top-K rms {float(sparse.float().square().mean().sqrt()):.4f}")
