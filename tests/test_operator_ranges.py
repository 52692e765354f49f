"""What extend_block_tables refuses because a count could not be written (CPU only)."""

import pytest

from test_operator_refusals import ADDRESS, INT32, INT64, lib, tables_call, tensor  # noqa: F401

FAR = 1 << 50      # where nothing else lies; never read: each call ends before a launch


@pytest.mark.parametrize("kind", [INT32, INT64])
def test_counts_that_int32_cannot_hold(lib, kind):  # noqa: F811
    for changes in (dict(slots=tensor((1 << 31,), kind, data=FAR), positions=None),
                    dict(free_pages=tensor((1 << 31,), kind, data=FAR))):
        status, error = tables_call(lib, **changes)
        assert status == -1 and "count at most 2^31 - 1 slots and free pages" in error, error
