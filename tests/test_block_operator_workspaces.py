"""What the block-sparse operators ask of their workspaces, on the host and before any launch (CPU only)."""

import pytest

from test_block_operator_refusals import PROMPTS, blocks_call, lib, place, select_call  # noqa: F401
from test_operator_refusals import ADDRESS, BF16, F32, INT32, tensor

PLANE = ADDRESS + (1 << 20)          # of the layer; V of block_attention's 2^19 behind it


@pytest.mark.parametrize("batch", [0, 5])
def test_no_selections_need_no_workspace(lib, batch):  # noqa: F811
    none = dict(index_query=tensor((0, 8, 128), BF16, data=None), blocks=tensor((0, 2, 4), INT32, data=None), rows=None,
                lengths=tensor((batch,), INT32, data=place(4)),
                query_starts=tensor((batch + 1,), INT32, data=place(6)))
    assert lib.ekv_select_workspace_bytes(0, 2, 9, 16, 64) == 0
    status, error = select_call(lib, None, 0, **none)
    assert status == 0, error


@pytest.mark.parametrize("at,other", [
    (place(0), "index_query"), (PLANE, "the layer's plane"), (PLANE + (1 << 17) - 256, "the layer's plane"),
    (place(1), "scales"), (place(2), "block_tables"), (place(3), "rows"), (place(4), "lengths"), (place(5), "blocks"),
    (place(6), "query_starts"),
])
def test_a_selection_s_workspace_shares_no_memory(lib, at, other):  # noqa: F811
    given = dict(query_starts=tensor((6,), INT32, data=place(6)))
    size = lib.ekv_select_workspace_bytes(5, 2, 9, 16, 64)
    # It ends in the tensor, and begins in it.
    for begin in (at - size // 256 * 256 + 256, at):
        status, error = select_call(lib, begin, size, **given)
        assert status == -1 and f"the workspace must not share memory with {other}" in error, error


@pytest.mark.parametrize("given", [{}, PROMPTS], ids=["tokens", "prompts"])
@pytest.mark.parametrize("at,other", [
    (place(0), "query"), (PLANE, "the layer's planes"), (PLANE + (1 << 19), "the layer's planes"),
    (place(2), "block_tables"), (place(3), "rows"), (place(4), "lengths"), (place(5), "blocks"), (place(6), "output"),
    (place(7), "lse"), (place(8), "query_starts"),
])
def test_an_attention_s_workspace_shares_no_memory(lib, at, other, given):  # noqa: F811
    changes = dict(given)
    if other == "rows":
        changes["rows"] = tensor((5,), INT32, data=place(3))
    tokens, heads = (4096, 16) if given else (5, 6)
    if other == "lse":
        changes["lse"] = tensor((tokens, heads), F32, data=place(7))
    changes["query_starts"] = tensor((6,), INT32, data=place(8))
    size = lib.ekv_block_workspace_bytes(tokens, 4, 64, heads, 2, 64, changes.get("max_query", 1))
    status, error = blocks_call(lib, at, size, **changes)
    assert status == -1 and f"the workspace must not share memory with {other}" in error, error
