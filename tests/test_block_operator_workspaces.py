"""What the block-sparse operators ask of their workspaces, on the host and before any launch (CPU only)."""

import pytest

from test_block_operator_refusals import lib, place, select_call  # noqa: F401
from test_operator_refusals import BF16, INT32, tensor


@pytest.mark.parametrize("batch", [0, 5])
def test_no_selections_need_no_workspace(lib, batch):  # noqa: F811
    none = dict(index_query=tensor((0, 8, 128), BF16, data=None), blocks=tensor((0, 2, 4), INT32, data=None), rows=None,
                lengths=tensor((batch,), INT32, data=place(4)),
                query_starts=tensor((batch + 1,), INT32, data=place(6)))
    assert lib.ekv_select_workspace_bytes(0, 2, 9, 16, 64) == 0
    status, error = select_call(lib, None, 0, **none)
    assert status == 0, error
