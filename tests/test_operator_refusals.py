"""What the block-table and attention entry points refuse, on the host and before any launch (CPU only).

Every call below is right but for one argument. The attention calls that are right in all of them are given no
workspace, which is the last check of all, so its message shows that nothing else was refused.
"""

import ctypes as ct

import pytest
import torch

from elastic_kv import _native

INT32, INT64, BF16, F16, F32, I8 = 1, 2, 6, 7, 8, 4
ADDRESS = 1 << 20          # never read: every call ends before a launch


def tensor(shape, dtype, stride=None, data=ADDRESS):
    t = _native.EkvTensor()
    t.data, t.dtype, t.ndim = data, dtype, len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        t.shape[i] = shape[i]
        t.stride[i] = step if stride is None else stride[i]
        step *= shape[i]
    return t


@pytest.fixture(scope="module")
def lib():
    assert _native._DTYPE_CODES[torch.bfloat16] == BF16 and _native._DTYPE_CODES[torch.float16] == F16
    assert _native._DTYPE_CODES[torch.float32] == F32 and _native._DTYPE_CODES[torch.int8] == I8
    return _native.kernel_library()


def planes(**changes):
    # 2 layers of K and V, 1024 tokens of 2 heads of 64.
    at = dict(base=ADDRESS, layers=2, kv=2, layer_stride=1 << 20, kv_stride=1 << 19, row_stride=256, row_bytes=256,
              rows=1024)
    at.update(changes)
    return _native.EkvPlanes(*at.values())


class Args(ct.Structure):
    _fields_ = [("query", ct.c_void_p), ("planes", ct.c_void_p), ("layer", ct.c_int64), ("kv_heads", ct.c_int64),
                ("page_size", ct.c_int64), ("block_tables", ct.c_void_p), ("rows", ct.c_void_p),
                ("lengths", ct.c_void_p), ("prefix_tables", ct.c_void_p), ("prefix_lengths", ct.c_void_p),
                ("group_starts", ct.c_void_p), ("query_starts", ct.c_void_p), ("max_query", ct.c_int64),
                ("scale", ct.c_double), ("output", ct.c_void_p), ("lse", ct.c_void_p)]


def prefix_call(lib, workspace=0, size=0, **changes):
    """(status, message) of a decode of 5 rows in 2 groups, 6 query heads, with `changes`."""
    given = dict(query=tensor((5, 6, 64), BF16), planes=planes(), layer=1, kv_heads=2, page_size=16,
                 block_tables=tensor((7, 9), INT32), rows=tensor((5,), INT64), lengths=tensor((5,), INT32),
                 prefix_tables=tensor((2, 4), INT32), prefix_lengths=tensor((2,), INT32),
                 group_starts=tensor((3,), INT32), query_starts=None, max_query=1, scale=0.125,
                 output=tensor((5, 6, 64), BF16), lse=tensor((5, 6), F32))
    given.update(changes)
    args = Args()
    for name, value in given.items():
        setattr(args, name, ct.addressof(value) if isinstance(value, ct.Structure) else value)
    status = lib.ekv_shared_prefix_attention(ct.byref(args), workspace, size, None)
    return status, lib.ev_error().decode()


PREFIX = [
    (dict(query=None), "query is required"),
    (dict(query=tensor((5, 384), BF16)), "query"),
    (dict(query=tensor((5, 6, 64), F32)), "query must be bfloat16 or float16"),
    (dict(query=tensor((5, 6, 64), F16)), "output must have the query's type"),
    (dict(query=tensor((5, 6, 64), BF16, data=None)), "query"),
    (dict(query=tensor((5, 6, 64), BF16, (768, 128, 2))), "query must be dense in its last dimension"),
    (dict(query=tensor((5, 6, 64), BF16, data=ADDRESS + 8)), "query address must be a multiple of 16 bytes"),
    (dict(query=tensor((5, 6, 64), BF16, (388, 64, 1))), "query token stride must be a multiple of 16 bytes"),
    (dict(output=tensor((5, 6, 64), BF16, (480, 68, 1))), "output head stride must be a multiple of 16 bytes"),
    (dict(output=tensor((4, 6, 64), BF16)), "output dimension 0 is 4, expected 5"),
    (dict(kv_heads=4), "kv_heads must divide"),
    (dict(kv_heads=0), "kv_heads must divide"),
    (dict(query=tensor((5, 6, 60), BF16, (384, 64, 1)), output=tensor((5, 6, 60), BF16, (384, 64, 1))),
     "multiple of 8 from 8 to 256"),
    (dict(query=tensor((5, 6, 264), BF16), output=tensor((5, 6, 264), BF16)), "multiple of 8 from 8 to 256"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(scale=1e39), "scale must be finite"),
    (dict(planes=None), "planes are required"),
    (dict(planes=planes(kv=1)), "planes must hold K and V"),
    (dict(planes=planes(base=None)), "null plane base"),
    (dict(planes=planes(base=ADDRESS + 2)), "plane address must be a multiple of 16 bytes"),
    (dict(planes=planes(kv_stride=8)), "kv stride must be a multiple of 16 bytes"),
    (dict(planes=planes(row_stride=264)), "plane row stride must be a multiple of 16 bytes"),
    (dict(planes=planes(row_bytes=512)), "neither a token's 256 nor a page's 4096"),
    (dict(planes=planes(row_stride=1 << 33)), "row stride must be below 4 GiB"),
    (dict(planes=planes(row_stride=1 << 30)), "a page must lie within 4 GiB"),
    (dict(layer=2), "layer 2 outside the pool's 2"),
    (dict(layer=-1), "layer -1 outside"),
    (dict(page_size=0), "page_size must be from 1"),
    (dict(block_tables=None), "block_tables is required"),
    (dict(block_tables=tensor((7, 9), I8)), "block_tables"),
    (dict(block_tables=tensor((7, 1 << 27), INT32)), "at most 2^30 - 1 tokens"),
    (dict(block_tables=tensor((7, 9), INT32, (9, 1 << 30))), "columns more than 2 GiB apart"),
    (dict(lengths=tensor((4,), INT32), rows=None), "without query_starts every batch row has one query token"),
    (dict(lengths=tensor((1 << 21,), INT32), rows=None), "more than 2^20 batch rows"),
    (dict(rows=tensor((4,), INT64)), "rows dimension 0 is 4, expected 5"),
    (dict(query_starts=tensor((5,), INT32)), "query_starts dimension 0 is 5, expected 6"),
    (dict(max_query=0), "max_query must be positive"),
    (dict(prefix_lengths=None), "prefix_tables and prefix_lengths are given together"),
    (dict(prefix_tables=None), "prefix_tables and prefix_lengths are given together"),
    (dict(prefix_tables=None, prefix_lengths=None), "group_starts without prefix_tables"),
    (dict(prefix_lengths=tensor((3,), INT32)), "prefix_lengths dimension 0 is 3, expected 2"),
    (dict(group_starts=tensor((2,), INT32)), "group_starts dimension 0 is 2, expected 3"),
    (dict(group_starts=None), "more than one prefix needs group_starts"),
    (dict(lse=tensor((5, 6), BF16)), "lse must be float32"),
    (dict(lse=tensor((5, 5), F32)), "lse dimension 1 is 5, expected 6"),
]


@pytest.mark.parametrize("changes,message", PREFIX, ids=[f"{i}-{'-'.join(c)}" for i, (c, _) in enumerate(PREFIX)])
def test_shared_prefix_attention_refuses(lib, changes, message):
    status, error = prefix_call(lib, **changes)
    assert status == -1 and message in error, error


@pytest.mark.parametrize("changes", [
    {}, dict(lse=None), dict(rows=None), dict(prefix_tables=None, prefix_lengths=None, group_starts=None),
    dict(planes=planes(row_bytes=4096, row_stride=8192, rows=64)), dict(scale=0.0), dict(scale=-2.0),
    dict(query=tensor((9, 6, 64), BF16), output=tensor((9, 6, 64), BF16), lse=None, query_starts=tensor((6,), INT64)),
])
def test_shared_prefix_attention_s_last_check_is_the_workspace(lib, changes):
    status, error = prefix_call(lib, **changes)
    assert status == -1 and "workspace bytes, got 0" in error, error
    status, error = prefix_call(lib, workspace=ADDRESS + 16, size=1 << 40, **changes)
    assert status == -1 and "256-byte aligned device buffer" in error, error


def topk_call(lib, workspace=0, size=0, **changes):
    given = dict(query=tensor((5, 6, 64), BF16), planes=planes(), layer=0, kv_heads=2, slots=tensor((5, 40), INT32),
                 zero_below=1, scale=0.125, output=tensor((5, 6, 64), BF16), lse=None)
    given.update(changes)
    at = {k: ct.byref(v) if isinstance(v, ct.Structure) else v for k, v in given.items()}
    status = lib.ekv_topk_attention(at["query"], at["planes"], at["layer"], at["kv_heads"], at["slots"],
                                    at["zero_below"], at["scale"], at["output"], at["lse"], workspace, size, None)
    return status, lib.ev_error().decode()


@pytest.mark.parametrize("changes,message", [
    (dict(slots=None), "slots is required"),
    (dict(slots=tensor((5, 8, 5), INT32)), "slots"),
    (dict(slots=tensor((4, 40), INT32)), "slots dimension 0 is 4, expected 5"),
    (dict(slots=tensor((5, 40), F32)), "slots"),
    (dict(slots=tensor((5, 1 << 30), INT32)), "more than 2^30 - 1 lanes"),
    (dict(zero_below=-1), "zero_below must be from 0"),
    (dict(zero_below=1 << 31), "zero_below must be from 0"),
    (dict(planes=planes(row_bytes=4096, row_stride=4096)), "neither a token's 256 nor a page's 256"),
    (dict(layer=5), "layer 5 outside"),
    (dict(scale=float("inf")), "scale must be finite"),
])
def test_topk_attention_refuses(lib, changes, message):
    status, error = topk_call(lib, **changes)
    assert status == -1 and message in error, error


def test_topk_attention_s_last_check_is_the_workspace(lib):
    for changes in ({}, dict(slots=tensor((5, 40), INT64)), dict(slots=tensor((5, 0), INT32))):
        status, error = topk_call(lib, **changes)
        assert status == -1 and "workspace bytes, got 0" in error, error


def test_no_query_tokens_is_no_launch(lib):
    none = dict(query=tensor((0, 6, 64), BF16, data=None), output=tensor((0, 6, 64), BF16, data=None))
    size = lib.ekv_topk_workspace_bytes(0, 40, 6, 2, 64)
    assert topk_call(lib, ADDRESS, size, slots=tensor((0, 40), INT32, data=None), **none)[0] == 0


@pytest.mark.parametrize("sizes", [(-1, 5, 1, 6, 2, 64, 1), (5, 5, 1, 6, 4, 64, 1), (5, 5, 1, 0, 0, 64, 1),
                                   (5, 5, 1, 6, 2, 300, 1), (5, 5, -1, 6, 2, 64, 1), (5, 5, 1, 6, 2, 64, 0),
                                   (1 << 24, 5, 1, 6, 2, 64, 1), (5, 1 << 21, 1, 6, 2, 64, 1),
                                   (5, 5, 1, 1 << 17, 1, 64, 1)])
def test_workspace_sizes_that_cannot_be(lib, sizes):
    from adaptive_sparse.attention import shared_prefix_workspace

    assert lib.ekv_shared_prefix_workspace_bytes(*sizes) == (1 << 64) - 1
    with pytest.raises(ValueError):
        shared_prefix_workspace(*sizes)


def tables_call(lib, **changes):
    given = dict(block_tables=tensor((7, 9), INT32), rows=tensor((5,), INT64), lengths=tensor((5,), INT32),
                 added=tensor((5,), INT32), free_pages=tensor((50,), INT32),
                 free_head=tensor((1,), INT32, data=ADDRESS + 512), page_size=16, slots=tensor((40,), INT32),
                 positions=tensor((40,), INT32), starts=tensor((6,), INT32),
                 new_lengths=tensor((5,), INT32, data=ADDRESS + 256), new_head=tensor((1,), INT32, data=ADDRESS + 768),
                 status=None)
    given.update(changes)
    at = [ct.byref(v) if isinstance(v, ct.Structure) else v for v in given.values()]
    status = lib.ekv_extend_block_tables(*at, None)
    return status, lib.ev_error().decode()


@pytest.mark.parametrize("changes,message", [
    (dict(block_tables=None), "block_tables is required"),
    (dict(block_tables=tensor((63,), INT32)), "block_tables"),
    (dict(block_tables=tensor((7, 9), F32)), "block_tables"),
    (dict(page_size=0), "page_size must be positive"),
    (dict(page_size=1 << 40), "at most 2^30 - 1 tokens"),
    (dict(block_tables=tensor((7, 1 << 27), INT32)), "at most 2^30 - 1 tokens"),
    (dict(added=tensor((4,), INT32)), "added dimension 0 is 4, expected 5"),
    (dict(rows=tensor((6,), INT32)), "rows dimension 0 is 6, expected 5"),
    (dict(starts=tensor((5,), INT32)), "starts dimension 0 is 5, expected 6"),
    (dict(positions=tensor((39,), INT32)), "positions dimension 0 is 39, expected 40"),
    (dict(new_head=tensor((2,), INT32)), "new_head dimension 0 is 2, expected 1"),
    (dict(free_head=None), "free_head is required"),
    (dict(free_pages=tensor((50,), INT32, data=None)), "free_pages"),
    (dict(new_lengths=tensor((5,), INT32, data=ADDRESS + 16)), "new_lengths must not share memory with lengths"),
    (dict(new_head=tensor((1,), INT32, data=ADDRESS + 512)), "new_head must not share memory with free_head"),
    (dict(status=tensor((1,), INT64)), "status must be int32"),
])
def test_extend_block_tables_refuses(lib, changes, message):
    status, error = tables_call(lib, **changes)
    assert status == -1 and message in error, error


def test_the_python_calls_refuse():
    from adaptive_sparse.attention import shared_prefix_attention, topk_attention, topk_workspace
    from adaptive_sparse.kv_pool import KVPlanes

    memory = torch.zeros((2, 64, 2, 64), dtype=torch.bfloat16)
    pool = KVPlanes(base=memory.data_ptr(), device=0, layers=1, kv=2, layer_stride=0, kv_stride=64 * 256,
                    row_stride=256, row_bytes=256, rows=64, owner=memory)
    query = torch.zeros((3, 6, 64), dtype=torch.bfloat16)
    slots = torch.zeros((3, 10), dtype=torch.int32)
    ints = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError, match="planes must be a KVPlanes"):
        topk_attention(query, memory, slots, query, kv_heads=2)
    with pytest.raises(ValueError, match=r"query must be shaped \[tokens, heads, head_dim\]"):
        topk_attention(query[0], pool, slots, query, kv_heads=2)
    with pytest.raises(ValueError, match=r"slots must be shaped \[tokens, K\]"):
        topk_attention(query, pool, slots[None], query, kv_heads=2)
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        shared_prefix_attention(query, pool, slots, None, ints, None, None, query, page_size=16, kv_heads=2,
                                workspace=torch.zeros((4, 4), dtype=torch.uint8)[:, :2])
    with pytest.raises(ValueError):
        topk_workspace(3, -1, 6, 2, 64)


def test_a_head_size_of_zero_is_refused_as_any_other():
    from adaptive_sparse.attention import shared_prefix_attention, topk_attention
    from adaptive_sparse.kv_pool import KVPlanes

    memory = torch.zeros((2, 64, 2, 64), dtype=torch.bfloat16)
    pool = KVPlanes(base=memory.data_ptr(), device=0, layers=1, kv=2, layer_stride=0, kv_stride=64 * 256,
                    row_stride=256, row_bytes=256, rows=64, owner=memory)
    query = torch.zeros((3, 6, 0), dtype=torch.bfloat16)
    ints, workspace = torch.zeros((3, 10), dtype=torch.int32), torch.zeros(4096, dtype=torch.uint8)
    with pytest.raises((ValueError, RuntimeError)):
        topk_attention(query, pool, ints, query, kv_heads=2, workspace=workspace)
    with pytest.raises((ValueError, RuntimeError)):
        shared_prefix_attention(query, pool, ints, None, ints[:, 0], None, None, query, page_size=16, kv_heads=2,
                                workspace=workspace)
