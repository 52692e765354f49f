"""What the append, selection and block attention entry points refuse, on the host and before any launch (CPU only).

Every call is right but for one argument. Calls that are right in all of them have no tokens, or no workspace, which is
the last check of all.
"""

import ctypes as ct
import math
from fractions import Fraction

import pytest
import torch

from test_operator_refusals import ADDRESS, BF16, F16, F32, I8, INT32, INT64, lib, planes, tensor  # noqa: F401

FAR = 1 << 30              # apart from the planes and the other tensors


def structure(names):
    class Args(ct.Structure):
        _fields_ = [(name, {"scale": ct.c_double, "magnitude": ct.c_double}.get(
            name, ct.c_int64 if name in ("layer", "page_size", "block_size", "kv_heads", "max_query", "first", "last",
                                         "zero_below", "interleaved") else ct.c_void_p)) for name in names]
    return Args


APPEND = structure(["query", "key", "value", "planes", "layer", "page_size", "slots", "zero_below", "positions", "turns",
                    "magnitude", "interleaved", "output"])
SELECT = structure(["index_query", "planes", "layer", "page_size", "block_size", "scales", "block_tables", "rows",
                    "lengths", "query_starts", "max_query", "first", "last", "blocks"])
BLOCKS = structure(["query", "planes", "layer", "kv_heads", "page_size", "block_size", "block_tables", "rows", "lengths",
                    "blocks", "query_starts", "max_query", "scale", "output", "lse"])


def place(i):
    return FAR + (i << 24)


def call(lib, kind, entry, given, *rest):  # noqa: F811
    args = kind()
    for name, value in given.items():
        setattr(args, name, ct.addressof(value) if isinstance(value, ct.Structure) else value)
    status = getattr(lib, entry)(ct.byref(args), *rest)
    return status, lib.ev_error().decode()


def append_call(lib, tokens=5, **changes):  # noqa: F811
    given = dict(query=tensor((tokens, 6, 64), BF16, data=place(0)), key=tensor((tokens, 2, 64), BF16, data=place(1)),
                 value=tensor((tokens, 2, 64), BF16, data=place(2)), planes=planes(), layer=1, page_size=16,
                 slots=tensor((tokens,), INT32, data=place(3)), zero_below=1,
                 positions=tensor((tokens,), INT64, data=place(4)), turns=tensor((32,), INT64, data=place(5)),
                 magnitude=1.0, interleaved=0, output=tensor((tokens, 6, 64), BF16, data=place(6)))
    given.update(changes)
    return call(lib, APPEND, "ekv_append_rotary", given, None)


Q, K = place(0), place(1)
REFUSED_APPENDS = [
    (dict(query=None), "query and output are given together"),
    (dict(output=None), "query and output are given together"),
    (dict(value=None), "key, value, planes and slots are given together"),
    (dict(planes=None), "key, value, planes and slots are given together"),
    (dict(slots=None), "key, value, planes and slots are given together"),
    (dict(query=None, output=None, key=None, value=None, planes=None, slots=None), "query or key is required"),
    (dict(positions=None), "positions is required"),
    (dict(turns=None), "turns is required"),
    (dict(query=tensor((5, 6, 64), F32, data=Q)), "query must be bfloat16 or float16"),
    (dict(key=tensor((5, 2, 64), F16, data=K)), "key must have the type of query"),
    (dict(output=tensor((5, 6, 64), F16, data=place(6))), "output must have the type of query"),
    (dict(query=tensor((5, 6, 64), BF16, (768, 128, 2), Q)), "query must be dense in its last dimension"),
    (dict(query=tensor((5, 6, 64), BF16, data=Q + 8)), "query address must be a multiple of 16 bytes"),
    (dict(key=tensor((5, 2, 64), BF16, (132, 64, 1), K)), "key token stride must be a multiple of 16 bytes"),
    (dict(output=tensor((5, 6, 64), BF16, (480, 68, 1), place(6))), "output head stride must be a multiple of 16"),
    (dict(output=tensor((5, 6, 64), BF16, (0, 64, 1), place(6))), "output must not repeat its elements"),
    (dict(output=tensor((5, 6, 64), BF16, (384, 32, 1), place(6))), "output must not repeat its elements"),
    (dict(output=tensor((5, 6, 64), BF16, (64, 64, 1), place(6))), "output must not repeat its elements"),
    (dict(output=tensor((4, 6, 64), BF16, data=place(6))), "output dimension 0 is 4, expected 5"),
    (dict(output=tensor((5, 5, 64), BF16, data=place(6))), "output dimension 1 is 5, expected 6"),
    (dict(value=tensor((5, 3, 64), BF16, data=place(2))), "value dimension 1 is 3, expected 2"),
    (dict(key=tensor((5, 2, 72), BF16, data=K)), "key dimension 2 is 72, expected 64"),
    (dict(query=tensor((5, 6, 60), BF16, (384, 64, 1), Q)), "multiple of 8 from 8 to 256"),
    (dict(query=tensor((5, 6, 264), BF16, data=Q)), "multiple of 8 from 8 to 256"),
    (dict(query=tensor((5, 6, 0), BF16, data=Q)), "multiple of 8 from 8 to 256"),
    (dict(query=tensor((5, 1 << 16, 64), BF16, data=Q)), "from 1 to 65535 heads"),
    (dict(key=tensor((5, 0, 64), BF16, data=K)), "from 1 to 65535 heads"),
    (dict(tokens=(1 << 24) + 1), "more than 2^24 tokens"),
    (dict(slots=tensor((4,), INT32)), "slots dimension 0 is 4, expected 5"),
    (dict(slots=tensor((5,), F32)), "slots"),
    (dict(positions=tensor((6,), INT32)), "positions dimension 0 is 6, expected 5"),
    (dict(turns=tensor((32,), INT32)), "turns must be dense int64"),
    (dict(turns=tensor((32,), INT64, (2,))), "turns must be dense int64"),
    (dict(turns=tensor((32,), INT64, data=place(5) + 4)), "turns must be dense int64"),
    (dict(turns=tensor((33,), INT64, data=place(5))), "from 1 to half the head size's pairs"),
    (dict(turns=tensor((0,), INT64)), "from 1 to half the head size's pairs"),
    (dict(magnitude=float("nan")), "magnitude must be finite"),
    (dict(magnitude=1e39), "magnitude must be finite"),
    (dict(zero_below=-1), "zero_below must not be negative"),
    (dict(page_size=0), "page_size must be from 1"),
    (dict(layer=2), "layer 2 outside the pool's 2"),
    (dict(planes=planes(kv=1)), "planes must hold K and V"),
    (dict(planes=planes(row_bytes=512)), "neither a token's 256 nor a page's 4096"),
    (dict(planes=planes(row_stride=128)), "plane rows must not overlap"),
    (dict(planes=planes(row_stride=0)), "plane rows must not overlap"),
    (dict(planes=planes(kv_stride=128)), "the layer's K plane must not share memory with its V plane"),
    (dict(planes=planes(row_stride=264)), "plane row stride must be a multiple of 16 bytes"),
    # K of layer 1 begins at ADDRESS + 2^20, V 2^19 behind it.
    (dict(key=tensor((5, 2, 64), BF16, data=ADDRESS + (1 << 20) + 256)), "key must not share memory with the layer's"),
    (dict(value=tensor((5, 2, 64), BF16, data=ADDRESS + (3 << 19))), "value must not share memory with the layer's"),
    (dict(query=tensor((5, 6, 64), BF16, data=ADDRESS + (1 << 20))), "query must not share memory with the layer's"),
    (dict(output=tensor((5, 6, 64), BF16, data=ADDRESS + (1 << 20))), "output must not share memory with the layer's"),
    (dict(positions=tensor((5,), INT32, data=ADDRESS + (1 << 20))), "positions must not share memory with the layer's"),
    (dict(slots=tensor((5,), INT64, data=ADDRESS + (1 << 20))), "slots must not share memory with the layer's"),
    (dict(turns=tensor((32,), INT64, data=ADDRESS + (1 << 20))), "turns must not share memory with the layer's"),
    (dict(output=tensor((5, 6, 64), BF16, data=Q + 768)), "output must not share memory with query, unless"),
    (dict(output=tensor((5, 6, 64), BF16, data=K - 768)), "output must not share memory with key"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(2))), "output must not share memory with value"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(3))), "output must not share memory with slots"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(4))), "output must not share memory with positions"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(5))), "output must not share memory with turns"),
]


def ids(cases):
    return [f"{i}-{'-'.join(c)}" for i, (c, _) in enumerate(cases)]


@pytest.mark.parametrize("changes,message", REFUSED_APPENDS, ids=ids(REFUSED_APPENDS))
def test_append_rotary_refuses(lib, changes, message):  # noqa: F811
    status, error = append_call(lib, **changes)
    assert status == -1 and message in error, error


def slices(tokens, at=place(0)):
    """q, k and v as slices of one projection of 10 heads of 64."""
    return dict(query=tensor((tokens, 6, 64), BF16, (640, 64, 1), at),
                key=tensor((tokens, 2, 64), BF16, (640, 64, 1), at + 6 * 128),
                value=tensor((tokens, 2, 64), BF16, (640, 64, 1), at + 8 * 128))


@pytest.mark.parametrize("changes", [
    {}, dict(query=None, output=None), dict(key=None, value=None, planes=None, slots=None), dict(interleaved=1),
    dict(planes=planes(row_bytes=4096, row_stride=8192, rows=64)), dict(slices(0), output=slices(0)["query"]),
    dict(positions=tensor((0,), INT32, data=None)),
])
def test_appending_no_tokens_is_no_launch(lib, changes):  # noqa: F811
    assert append_call(lib, tokens=0, **changes)[0] == 0


def test_slices_of_one_projection_are_apart(lib):  # noqa: F811
    # The output in the query's place passes the checks of overlaps, which come before that of the planes' rows.
    bad = planes(kv_stride=128)
    given = slices(5)
    status, error = append_call(lib, **given, output=given["query"], planes=bad)
    assert status == -1 and "its V plane" in error, error
    # One head further it meets the key.
    moved = tensor((5, 6, 64), BF16, (640, 64, 1), place(0) + 128)
    status, error = append_call(lib, **given, output=moved, planes=bad)
    assert status == -1 and "output must not share memory with query" in error, error


def index_planes(**changes):
    at = dict(kv=1, row_stride=128, row_bytes=128)
    at.update(changes)
    return planes(**at)


def index_call(lib, **changes):  # noqa: F811
    given = dict(index_key=tensor((5, 128), BF16, data=place(0)), planes=index_planes(), layer=1, page_size=16,
                 scales=tensor((1024,), F32, data=place(1)), slots=tensor((5,), INT32, data=place(2)), zero_below=1)
    given.update(changes)
    at = [ct.byref(v) if isinstance(v, ct.Structure) else v for v in given.values()]
    return lib.ekv_append_index(*at, None), lib.ev_error().decode()


REFUSED_INDEXES = [
    (dict(index_key=None), "index_key is required"),
    (dict(index_key=tensor((5, 1, 128), BF16)), "index_key"),
    (dict(index_key=tensor((5, 128), F32)), "index_key must be bfloat16 or float16"),
    (dict(index_key=tensor((5, 120), BF16)), "multiple of 16 from 16 to 256"),
    (dict(index_key=tensor((5, 272), BF16)), "multiple of 16 from 16 to 256"),
    (dict(index_key=tensor((5, 0), BF16)), "multiple of 16 from 16 to 256"),
    (dict(index_key=tensor((5, 128), BF16, (256, 2), place(0))), "index_key must be dense in its last dimension"),
    (dict(index_key=tensor((5, 128), BF16, data=place(0) + 2)), "index_key address must be a multiple of 16 bytes"),
    (dict(index_key=tensor((5, 128), BF16, (130, 1), place(0))), "index_key token stride must be a multiple of 16"),
    (dict(index_key=tensor(((1 << 24) + 1, 128), BF16, data=place(0))), "more than 2^24 tokens"),
    (dict(slots=None), "slots is required"),
    (dict(slots=tensor((6,), INT32)), "slots dimension 0 is 6, expected 5"),
    (dict(planes=None), "planes are required"),
    (dict(planes=planes(row_bytes=128)), "planes must hold one plane a layer"),
    (dict(planes=index_planes(row_bytes=64)), "neither a token's 128 nor a page's 2048"),
    (dict(planes=index_planes(row_stride=64)), "plane rows must not overlap"),
    (dict(planes=index_planes(row_stride=136)), "plane row stride must be a multiple of 16 bytes"),
    (dict(layer=-1), "layer -1 outside"),
    (dict(zero_below=-1), "zero_below must not be negative"),
    (dict(scales=None), "scales is required"),
    (dict(scales=tensor((1023,), F32)), "scales must have an element for each of the pool's 1024 slots, got 1023"),
    (dict(scales=tensor((1024,), BF16)), "scales must be float32"),
    (dict(scales=tensor((1024,), F32, (0,), place(1))), "scales must not repeat its elements"),
    (dict(scales=tensor((1024,), F32, data=ADDRESS + (1 << 20))), "scales must not share memory with the layer's"),
    (dict(scales=tensor((1024,), F32, data=place(0))), "scales must not share memory with index_key"),
    (dict(scales=tensor((1024,), F32, data=place(2) - 4092)), "scales must not share memory with slots"),
    (dict(index_key=tensor((5, 128), BF16, data=ADDRESS + (1 << 20))), "index_key must not share memory with the layer"),
    (dict(slots=tensor((5,), INT32, data=ADDRESS + (1 << 20) + 4)), "slots must not share memory with the layer's"),
]


@pytest.mark.parametrize("changes,message", REFUSED_INDEXES, ids=ids(REFUSED_INDEXES))
def test_append_index_refuses(lib, changes, message):  # noqa: F811
    status, error = index_call(lib, **changes)
    assert status == -1 and message in error, error


def test_no_index_keys_is_no_launch(lib):  # noqa: F811
    none = dict(index_key=tensor((0, 128), BF16, data=None), slots=tensor((0,), INT32, data=None))
    assert index_call(lib, **none)[0] == 0


def select_call(lib, workspace=0, size=0, **changes):  # noqa: F811
    given = dict(index_query=tensor((5, 8, 128), BF16, data=place(0)), planes=index_planes(), layer=1, page_size=16,
                 block_size=64, scales=tensor((1024,), F32, data=place(1)),
                 block_tables=tensor((7, 9), INT32, data=place(2)), rows=tensor((5,), INT64, data=place(3)),
                 lengths=tensor((5,), INT32, data=place(4)), query_starts=None, max_query=1, first=1, last=1,
                 blocks=tensor((5, 2, 4), INT32, data=place(5)))
    given.update(changes)
    return call(lib, SELECT, "ekv_select_blocks", given, workspace, size, None)


REFUSED_SELECTIONS = [
    (dict(index_query=None), "index_query is required"),
    (dict(index_query=tensor((5, 8, 128), F32, data=place(0))), "index_query must be bfloat16 or float16"),
    (dict(index_query=tensor((5, 8, 120), BF16, data=place(0))), "multiple of 16 from 16 to 256"),
    (dict(index_query=tensor((5, 8, 272), BF16, data=place(0))), "multiple of 16 from 16 to 256"),
    (dict(index_query=tensor((5, 8, 128), BF16, data=place(0) + 8)), "index_query address must be a multiple of 16"),
    (dict(index_query=tensor((5, 8, 128), BF16, (1028, 128, 1), place(0))), "index_query token stride"),
    (dict(blocks=None), "blocks is required"),
    (dict(blocks=tensor((5, 8), INT32)), "blocks"),
    (dict(blocks=tensor((4, 2, 4), INT32)), "blocks dimension 0 is 4, expected 5"),
    (dict(blocks=tensor((5, 2, 4), INT64, data=place(5))), "blocks must be int32"),
    (dict(blocks=tensor((5, 2, 4), INT32, (8, 0, 1), place(5))), "blocks must not repeat its elements"),
    (dict(blocks=tensor((5, 2, 4), INT32, (8, 3, 1), place(5))), "blocks must not repeat its elements"),
    (dict(blocks=tensor((5, 3, 4), INT32, data=place(5))), "a divisor of the index heads"),
    (dict(blocks=tensor((5, 0, 4), INT32, data=place(5))), "a divisor of the index heads"),
    (dict(index_query=tensor((5, 129, 128), BF16, data=place(0)), blocks=tensor((5, 1, 4), INT32, data=place(5))),
     "at most 128 heads"),
    (dict(blocks=tensor((5, 2, 0), INT32, data=place(5))), "from 1 to 2^30 blocks a list"),
    (dict(first=-1), "first and last must not be negative"),
    (dict(last=-1), "first and last must not be negative"),
    (dict(first=3, last=2), "not more together than a list holds"),
    (dict(first=1 << 62, last=1 << 62), "not more together than a list holds"),
    (dict(page_size=0), "at most 2^30 - 1 tokens"),
    (dict(block_size=0), "block_size must be from 1 to 2^30"),
    (dict(block_size=(1 << 30) + 1), "block_size must be from 1 to 2^30"),
    (dict(block_tables=None), "block_tables is required"),
    (dict(block_tables=tensor((63,), INT32)), "block_tables"),
    (dict(block_tables=tensor((7, 1 << 27), INT32)), "at most 2^30 - 1 tokens"),
    (dict(planes=None), "planes are required"),
    (dict(planes=planes(row_bytes=128)), "planes must hold one plane a layer"),
    (dict(layer=2), "layer 2 outside"),
    (dict(scales=None), "scales is required"),
    (dict(scales=tensor((1000,), F32)), "scales must have an element for each of the pool's 1024 tokens, got 1000"),
    (dict(scales=tensor((1024,), F16)), "scales must be float32"),
    (dict(lengths=None), "lengths is required"),
    (dict(lengths=tensor((5,), F32)), "lengths"),
    (dict(lengths=tensor((4,), INT32), rows=None), "without query_starts every batch row has one query token"),
    (dict(lengths=tensor((1 << 21,), INT32), rows=None), "more than 2^20 batch rows"),
    (dict(rows=tensor((4,), INT32)), "rows dimension 0 is 4, expected 5"),
    (dict(query_starts=tensor((5,), INT32)), "query_starts dimension 0 is 5, expected 6"),
    (dict(max_query=0), "max_query must be positive"),
    (dict(blocks=tensor((5, 2, 4), INT32, data=place(0) + 64)), "blocks must not share memory with index_query"),
    (dict(blocks=tensor((5, 2, 4), INT32, data=ADDRESS + (1 << 20))), "blocks must not share memory with the layer's"),
    (dict(blocks=tensor((5, 2, 4), INT32, data=place(1))), "blocks must not share memory with scales"),
    (dict(blocks=tensor((5, 2, 4), INT32, data=place(2) + 248)), "blocks must not share memory with block_tables"),
    (dict(blocks=tensor((5, 2, 4), INT32, data=place(4))), "blocks must not share memory with lengths"),
    (dict(blocks=tensor((5, 2, 4), INT32, data=place(3))), "blocks must not share memory with rows"),
    (dict(query_starts=tensor((6,), INT32, data=place(5) + 156)), "blocks must not share memory with query_starts"),
]


@pytest.mark.parametrize("changes,message", REFUSED_SELECTIONS, ids=ids(REFUSED_SELECTIONS))
def test_select_blocks_refuses(lib, changes, message):  # noqa: F811
    status, error = select_call(lib, **changes)
    assert status == -1 and message in error, error


@pytest.mark.parametrize("changes", [
    {}, dict(rows=None), dict(first=0, last=0), dict(block_size=1), dict(page_size=64), dict(max_query=1 << 40),
    dict(planes=index_planes(row_bytes=2048, row_stride=4096, rows=64)),
    dict(query_starts=tensor((6,), INT64, data=place(6))),
    # Lists in another order of dimensions.
    dict(blocks=tensor((5, 2, 4), INT32, (1, 5, 10), place(5))),
])
def test_select_blocks_s_last_check_is_the_workspace(lib, changes):  # noqa: F811
    status, error = select_call(lib, **changes)
    assert status == -1 and "workspace bytes, got 0" in error, error
    status, error = select_call(lib, workspace=ADDRESS + 16, size=1 << 40, **changes)
    assert status == -1 and "256-byte aligned device buffer" in error, error


def test_no_selections_are_no_launch(lib):  # noqa: F811
    none = dict(index_query=tensor((0, 8, 128), BF16, data=None), blocks=tensor((0, 2, 4), INT32, data=None),
                query_starts=tensor((6,), INT32, data=place(6)))
    size = lib.ekv_select_workspace_bytes(0, 2, 9, 16, 64)
    assert select_call(lib, ADDRESS, size, **none)[0] == 0


@pytest.mark.parametrize("sizes", [(-1, 2, 9, 16, 64), (5, 0, 9, 16, 64), (5, 1025, 9, 16, 64), (5, 2, -1, 16, 64),
                                   (5, 2, 9, 0, 64), (5, 2, 9, 16, 0), (5, 2, 1 << 26, 16, 64), (5, 2, 1, 1 << 31, 64),
                                   (1 << 22, 1, 9, 16, 64), (1 << 20, 8, 9, 16, 64), (1 << 62, 2, 9, 16, 64)])
def test_selection_workspaces_that_cannot_be(lib, sizes):  # noqa: F811
    from adaptive_sparse.block_selection import selection_workspace

    assert lib.ekv_select_workspace_bytes(*sizes) == (1 << 64) - 1
    with pytest.raises(ValueError):
        selection_workspace(*sizes)


def test_selection_workspaces_hold_a_score_for_each_block(lib):  # noqa: F811
    from adaptive_sparse.block_selection import selection_workspace

    for tokens, groups, columns, page, block in ((1, 1, 1, 16, 64), (128, 1, 2048, 16, 1), (4096, 4, 64, 64, 64)):
        lists = tokens * groups
        assert selection_workspace(tokens, groups, columns, page, block) >= lists * -(-columns * page // block) * 4
    # The largest that the sizes allow is held in 64 bits.
    assert selection_workspace((1 << 22) - 1, 1, (1 << 30) - 1, 1, 1) > 1 << 53


def blocks_call(lib, workspace=0, size=0, **changes):  # noqa: F811
    given = dict(query=tensor((5, 6, 64), BF16, data=place(0)), planes=planes(), layer=1, kv_heads=2, page_size=16,
                 block_size=64, block_tables=tensor((7, 9), INT32, data=place(2)),
                 rows=tensor((5,), INT64, data=place(3)), lengths=tensor((5,), INT32, data=place(4)),
                 blocks=tensor((5, 2, 4), INT32, data=place(5)), query_starts=None, max_query=1, scale=0.125,
                 output=tensor((5, 6, 64), BF16, data=place(6)), lse=tensor((5, 6), F32, data=place(7)))
    given.update(changes)
    return call(lib, BLOCKS, "ekv_block_attention", given, workspace, size, None)


REFUSED_BLOCKS = [
    (dict(query=None), "query is required"),
    (dict(query=tensor((5, 6, 64), F16, data=place(0))), "output must have the query's type"),
    (dict(query=tensor((5, 6, 60), BF16, (384, 64, 1)), output=tensor((5, 6, 60), BF16, (384, 64, 1))),
     "multiple of 8 from 8 to 256"),
    (dict(kv_heads=4), "kv_heads must divide"),
    (dict(scale=float("inf")), "scale must be finite"),
    (dict(planes=None), "planes are required"),
    (dict(planes=planes(kv=1)), "planes must hold K and V"),
    (dict(layer=2), "layer 2 outside"),
    (dict(page_size=0), "page_size must be from 1"),
    (dict(block_size=0), "a list of blocks may name at most 2^30 - 1 tokens"),
    (dict(block_size=1 << 30), "a list of blocks may name at most 2^30 - 1 tokens"),
    (dict(blocks=None), "blocks is required"),
    (dict(blocks=tensor((5, 8), INT32)), "blocks"),
    (dict(blocks=tensor((5, 2, 4), F32)), "blocks"),
    (dict(blocks=tensor((4, 2, 4), INT32)), "blocks dimension 0 is 4, expected 5"),
    (dict(blocks=tensor((5, 3, 4), INT32)), "blocks must have a divisor of kv_heads as lists"),
    (dict(blocks=tensor((5, 0, 4), INT32)), "blocks must have a divisor of kv_heads as lists"),
    (dict(blocks=tensor((5, 2, 4), INT32, (8, 4, 1 << 30), place(5))), "columns more than 2 GiB apart"),
    (dict(blocks=tensor((5, 2, 1 << 24), INT32, (0, 0, 0), place(5))), "at most 2^30 - 1 tokens"),
    (dict(block_tables=None), "block_tables is required"),
    (dict(block_tables=tensor((7, 1 << 27), INT32)), "at most 2^30 - 1 tokens"),
    (dict(lengths=tensor((4,), INT32), rows=None), "without query_starts every batch row has one query token"),
    (dict(rows=tensor((4,), INT64)), "rows dimension 0 is 4, expected 5"),
    (dict(query_starts=tensor((5,), INT32)), "query_starts dimension 0 is 5, expected 6"),
    (dict(max_query=0), "max_query must be positive"),
    (dict(lse=tensor((5, 6), BF16)), "lse must be float32"),
    (dict(output=tensor((5, 6, 64), BF16, (64, 64, 1), place(6))), "output must not repeat its elements"),
    (dict(lse=tensor((5, 6), F32, (6, 0), place(7))), "lse must not repeat its elements"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(0) + 128)), "output must not share memory with query, unless"),
    (dict(output=tensor((5, 6, 64), BF16, data=ADDRESS + (1 << 20))), "output must not share memory with the layer's"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(2))), "output must not share memory with block_tables"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(3))), "output must not share memory with rows"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(4))), "output must not share memory with lengths"),
    (dict(output=tensor((5, 6, 64), BF16, data=place(5))), "output must not share memory with blocks"),
    (dict(lse=tensor((5, 6), F32, data=place(0))), "lse must not share memory with query"),
    (dict(lse=tensor((5, 6), F32, data=place(6))), "lse must not share memory with output"),
    (dict(lse=tensor((5, 6), F32, data=place(5))), "lse must not share memory with blocks"),
]


@pytest.mark.parametrize("changes,message", REFUSED_BLOCKS, ids=ids(REFUSED_BLOCKS))
def test_block_attention_refuses(lib, changes, message):  # noqa: F811
    status, error = blocks_call(lib, **changes)
    assert status == -1 and message in error, error


PROMPTS = dict(query=tensor((4096, 16, 64), BF16, data=place(0)), output=tensor((4096, 16, 64), BF16, data=place(6)),
               lse=None, blocks=tensor((4096, 1, 4), INT32, data=place(5)), rows=None,
               query_starts=tensor((6,), INT32, data=place(8)), max_query=1024)


@pytest.mark.parametrize("changes", [
    {}, dict(lse=None), dict(rows=None), dict(scale=0.0), dict(blocks=tensor((5, 1, 4), INT64, data=place(5))),
    dict(blocks=tensor((5, 2, 0), INT32, data=None)), dict(output=tensor((5, 6, 64), BF16, data=place(0))),
    dict(blocks=tensor((5, 2, 4), INT32, (0, 0, 1), place(5))), PROMPTS,
])
def test_block_attention_s_last_check_is_the_workspace(lib, changes):  # noqa: F811
    status, error = blocks_call(lib, **changes)
    assert status == -1 and "workspace bytes, got 0" in error, error
    status, error = blocks_call(lib, workspace=ADDRESS + 16, size=1 << 40, **changes)
    assert status == -1 and "256-byte aligned device buffer" in error, error


@pytest.mark.parametrize("sizes", [(-1, 4, 64, 6, 2, 64, 1), (5, -1, 64, 6, 2, 64, 1), (5, 4, 0, 6, 2, 64, 1),
                                   (5, 4, 64, 6, 4, 64, 1), (5, 4, 64, 6, 2, 300, 1), (5, 4, 64, 6, 2, 64, 0),
                                   (5, 1 << 24, 64, 6, 2, 64, 1), (1 << 24, 4, 64, 6, 2, 64, 1)])
def test_block_workspaces_that_cannot_be(lib, sizes):  # noqa: F811
    from adaptive_sparse.attention import block_workspace

    assert lib.ekv_block_workspace_bytes(*sizes) == (1 << 64) - 1
    with pytest.raises(ValueError):
        block_workspace(*sizes)


@pytest.mark.parametrize("entry", ["ekv_append_rotary", "ekv_select_blocks", "ekv_block_attention"])
def test_calls_without_arguments(lib, entry):  # noqa: F811
    rest = (None,) if entry == "ekv_append_rotary" else (0, 0, None)
    assert getattr(lib, entry)(None, *rest) == -1 and "args is required" in lib.ev_error().decode()


def test_the_python_calls_refuse():
    from adaptive_sparse.append import append_index, append_rotary, make_rotary
    from adaptive_sparse.attention import block_attention
    from adaptive_sparse.block_selection import select_blocks
    from adaptive_sparse.kv_pool import KVPlanes

    memory = torch.zeros((2, 64, 2, 64), dtype=torch.bfloat16)
    pool = KVPlanes(base=memory.data_ptr(), device=0, layers=1, kv=2, layer_stride=0, kv_stride=64 * 256,
                    row_stride=256, row_bytes=256, rows=64, owner=memory)
    query = torch.zeros((3, 6, 64), dtype=torch.bfloat16)
    ints, tables = torch.zeros(3, dtype=torch.int32), torch.zeros((3, 4), dtype=torch.int32)
    lists = torch.zeros((3, 1, 2), dtype=torch.int32)
    rotary = make_rotary(64, device="cpu")
    with pytest.raises(TypeError, match="rotary must be a Rotary"):
        append_rotary(query, None, None, None, None, ints, rotary.turns, query)
    with pytest.raises(TypeError, match="planes must be a KVPlanes"):
        append_rotary(None, query, query, memory, ints, ints, rotary, None)
    with pytest.raises(TypeError, match="planes must be a KVPlanes"):
        append_index(query[:, 0], memory, torch.zeros(64), ints)
    with pytest.raises(TypeError, match="planes must be a KVPlanes"):
        select_blocks(query, memory, torch.zeros(64), tables, None, ints, lists, page_size=16, block_size=64)
    with pytest.raises(ValueError, match=r"blocks must be shaped \[tokens, groups, K\]"):
        select_blocks(query, pool, torch.zeros(64), tables, None, ints, lists[0], page_size=16, block_size=64)
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        select_blocks(query, pool, torch.zeros(64), tables, None, ints, lists, page_size=16, block_size=64,
                      workspace=torch.zeros((4, 4), dtype=torch.uint8)[:, :2])
    with pytest.raises(TypeError, match="planes must be a KVPlanes"):
        block_attention(query, memory, tables, None, ints, lists, query, page_size=16, block_size=64, kv_heads=2)
    with pytest.raises(ValueError, match=r"blocks must be shaped \[tokens, lists, K\]"):
        block_attention(query, pool, tables, None, ints, lists[0], query, page_size=16, block_size=64, kv_heads=2)
    with pytest.raises(ValueError, match=r"query must be shaped \[tokens, heads, head_dim\]"):
        block_attention(query[0], pool, tables, None, ints, lists, query, page_size=16, block_size=64, kv_heads=2)


@pytest.mark.parametrize("given", [
    dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=64.0), dict(scaling="other"),
    dict(base=0.0), dict(base=float("inf")), dict(factor=-1.0), dict(factor=float("nan")),
    dict(rotary_dim=2, scaling="base"), dict(scaling="ramp"), dict(scaling="ramp", original=0),
    dict(scaling="ramp", original=4096, fast=1.0, slow=1.0), dict(scaling="ramp", original=4096, slow=0.0),
    dict(scaling="ramp", original=4096, base=1.0),
])
def test_rotations_that_cannot_be(given):
    from adaptive_sparse.append import make_rotary

    with pytest.raises(ValueError):
        make_rotary(**{"rotary_dim": 64, "device": "cpu", **given})


def test_frequencies():
    from adaptive_sparse.append import make_rotary, rotary_frequencies

    plain, one = rotary_frequencies(64, base=500000.0)
    assert one == 1.0 and len(plain) == 32 and plain[0] == 1.0
    assert all(math.isclose(f, 500000.0 ** (-i / 32), rel_tol=1e-14) for i, f in enumerate(plain))
    linear, _ = rotary_frequencies(64, base=500000.0, scaling="linear", factor=8.0)
    assert linear == [f / 8 for f in plain]
    # The first pair keeps its frequency, the last one's is divided by the factor.
    raised, _ = rotary_frequencies(64, base=500000.0, scaling="base", factor=8.0)
    assert raised[0] == 1.0 and math.isclose(raised[-1], plain[-1] / 8, rel_tol=1e-12)
    ramp, magnitude = rotary_frequencies(64, scaling="ramp", factor=16.0, original=4096)
    plain, _ = rotary_frequencies(64)
    assert math.isclose(magnitude, 0.1 * math.log(16.0) + 1.0, rel_tol=1e-15)
    for f, p in zip(ramp, plain):
        turns = 4096 * p / (2 * math.pi)
        # The pairs' places are whole numbers, so a pair next to a limit may be a step inside the ramp.
        if turns > 2 * 32:
            assert f == p
        if turns < 0.5:
            assert f == p / 16
        assert p / 16 * (1 - 1e-15) <= f <= p
    assert rotary_frequencies(64, scaling="ramp", factor=0.5, original=4096)[1] == 1.0
    assert make_rotary(64, device="cpu", scaling="ramp", factor=16.0, original=4096).magnitude == magnitude
    assert make_rotary(64, device="cpu", scaling="ramp", factor=16.0, original=4096, magnitude=1).magnitude == 1.0


@pytest.mark.parametrize("given", [dict(rotary_dim=128), dict(rotary_dim=64, base=500000.0),
                                   dict(rotary_dim=128, scaling="linear", factor=4.0), dict(rotary_dim=2),
                                   dict(rotary_dim=256, base=0.5)])        # frequencies above a turn a position
def test_turns_are_the_nearest_64_bit_fractions(given):
    from adaptive_sparse.append import make_rotary

    rotary = make_rotary(device="cpu", **given)
    assert rotary.turns.dtype == torch.int64 and len(rotary.turns) == given["rotary_dim"] // 2
    for turn, frequency in zip(rotary.turns.tolist(), rotary.frequencies):
        exact = Fraction(frequency / (2 * math.pi)) * 2 ** 64
        off = (turn - exact) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2)
