"""extend_block_tables refuses outputs that share memory with an input or with one another (CPU only).

Workgroups read the inputs while others write the outputs, so such a call would be a race. Each call below is refused on
the host, before any launch.
"""

import pytest

from test_operator_refusals import ADDRESS, INT32, INT64, lib, tables_call, tensor  # noqa: F401

# The arrays of a call apart from each other; "status" is one more.
SIZES = dict(rows=(5, INT64), lengths=(5, INT32), added=(5, INT32), free_pages=(50, INT32), free_head=(1, INT32),
             slots=(40, INT32), positions=(40, INT32), starts=(6, INT32), new_lengths=(5, INT32), new_head=(1, INT32),
             status=(1, INT32))
PLACES = {name: ADDRESS + 4096 * (i + 1) for i, name in enumerate(SIZES)}
INPUTS = ("lengths", "added", "rows", "free_pages", "free_head")
OUTPUTS = ("new_lengths", "new_head", "starts", "slots", "positions", "status")


def refused(lib, **moved):  # noqa: F811
    given = {name: tensor((n,), kind, data=PLACES[name]) for name, (n, kind) in SIZES.items()}
    given.update(moved)
    status, error = tables_call(lib, block_tables=tensor((7, 9), INT32, data=ADDRESS + (1 << 18)), **given)
    assert status == -1
    return error


@pytest.mark.parametrize("out", OUTPUTS)
@pytest.mark.parametrize("other", INPUTS)
def test_an_output_in_an_input(lib, out, other):  # noqa: F811
    count, kind = SIZES[out]
    item = 8 if SIZES[other][1] == INT64 else 4
    # On its last element's last word.
    at = PLACES[other] + SIZES[other][0] * item - 4
    assert f"{out} must not share memory with {other}" in refused(lib, **{out: tensor((count,), kind, data=at)})


@pytest.mark.parametrize("out,other", [(a, b) for i, a in enumerate(OUTPUTS) for b in OUTPUTS[:i]])
def test_an_output_in_another(lib, out, other):  # noqa: F811
    count, kind = SIZES[out]
    assert f"{out} must not share memory with {other}" in refused(
        lib, **{out: tensor((count,), kind, data=PLACES[other])})


def test_columns_that_share_elements(lib):  # noqa: F811
    # Every second word, and every third from the second on: both have the fifth.
    lengths = tensor((5,), INT32, (2,), PLACES["lengths"])
    grown = tensor((5,), INT32, (3,), PLACES["lengths"] + 4)
    assert "new_lengths must not share memory with lengths" in refused(lib, lengths=lengths, new_lengths=grown)
    # int64 columns whose halves meet.
    lengths = tensor((5,), INT64, (2,), PLACES["lengths"])
    grown = tensor((5,), INT64, (2,), PLACES["lengths"] + 4)
    assert "new_lengths must not share memory with lengths" in refused(lib, lengths=lengths, new_lengths=grown)
