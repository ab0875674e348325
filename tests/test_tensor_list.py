"""The chunk plan of a gradient list and the refusals of its entry points: host
code, no device needed."""
import ctypes

import numpy as np
import pytest

from nntrain_b200.native import GradientTensorList

INVALID = 1   # cudaErrorInvalidValue
TENSOR = GradientTensorList._TENSOR


def table_of(lengths, kind=0, block=0):
    """Tensors of these lengths, one behind the other in an address space of their own."""
    table = np.zeros(len(lengths), dtype=TENSOR)
    table["length"], table["kind"], table["block_size"] = lengths, kind, block
    table["values"] = 4096 + np.concatenate([[0], np.cumsum(lengths)[:-1]]).astype(np.uint64) * 4
    if kind == 2:
        table["scales"] = table["values"] + np.uint64(1 << 60)
    return table


def plan(lib, table, chunk_map=None, capacity=None):
    chunks, values = ctypes.c_longlong(), ctypes.c_int()
    status = lib.nntrain_gradient_list_plan(
        table.ctypes.data, len(table), None if chunk_map is None else chunk_map.ctypes.data,
        (0 if chunk_map is None else len(chunk_map)) if capacity is None else capacity,
        ctypes.addressof(chunks), ctypes.addressof(values))
    return status, chunks.value, values.value


@pytest.mark.parametrize("lengths", (
    [1], [0, 5, 0], [4096, 4097, 1, 0, 8191, 8192], [233_373_696] + [1536, 256, 2_359_296] * 28, [1] * 400, [3_000_000_000]))
def test_plan_covers_every_value_once(lib, lengths):
    table = table_of(lengths)
    status, chunks, size = plan(lib, table)
    assert status == 0 and 4096 <= size <= 65536 and size % 4096 == 0
    chunk_map = np.full((max(chunks, 1), 2), -1, dtype=np.int32)
    status, again, size_again = plan(lib, table, chunk_map, chunks)
    assert status == 0 and (again, size_again) == (chunks, size)
    assert chunks == sum(-(-n // size) for n in lengths)
    first = np.concatenate([[0], np.cumsum([-(-n // size) for n in lengths])])
    assert (table["first_chunk"] == first[:-1]).all()
    for t, n in enumerate(lengths):
        mine = chunk_map[first[t]:first[t + 1]]
        assert (mine[:, 0] == t).all() and (mine[:, 1] == np.arange(len(mine))).all()
        assert (len(mine) - 1) * size < n <= len(mine) * size if n else len(mine) == 0


@pytest.mark.parametrize("kind", (0, 1, 2))
def test_a_chunk_is_as_many_bytes_for_every_kind(lib, kind):
    n = 100_000
    status, chunks, size = plan(lib, table_of([n], kind=kind, block=32))
    assert status == 0 and size == 4096 and chunks == -(-n // (size << kind))


def test_plan_bounds_the_partials_of_one_finish_block(lib):
    status, chunks, _ = plan(lib, table_of([1_543_714_304]))
    assert status == 0 and chunks <= 65536


def test_plan_refusals(lib):
    chunks, values = ctypes.c_longlong(), ctypes.c_int()
    a, b = ctypes.addressof(chunks), ctypes.addressof(values)
    good = table_of([10])
    assert lib.nntrain_gradient_list_plan(None, 1, None, 0, a, b) == INVALID
    assert lib.nntrain_gradient_list_plan(good.ctypes.data, 0, None, 0, a, b) == INVALID
    assert lib.nntrain_gradient_list_plan(good.ctypes.data, 1, None, 0, None, b) == INVALID
    assert lib.nntrain_gradient_list_plan(good.ctypes.data, 1, None, -1, a, b) == INVALID
    for field, value in (("length", -1), ("kind", 3), ("kind", -1), ("block_size", -1), ("values", 0),
                         ("values", 4098), ("destination", 4097)):
        bad = table_of([10])
        bad[field] = value
        assert plan(lib, bad)[0] == INVALID, (field, value)
    unscaled = table_of([10], kind=2, block=32)
    unscaled["scales"] = 0
    assert plan(lib, unscaled)[0] == INVALID
    huge = table_of([4, 4])
    huge["length"] = 1 << 62                                                    # the sum would overflow
    assert plan(lib, huge)[0] == INVALID
    small = np.zeros((1, 2), dtype=np.int32)
    assert plan(lib, table_of([10_000]), small, 1)[0] == INVALID                # room for one chunk of three


def test_plan_refuses_tensors_that_share_what_is_written(lib):
    def status(**changed):
        """Three fp32 tensors of 10 values at 0x1000, 0x2000, 0x3000; changed: field -> (tensor, value)."""
        table = table_of([10, 10, 10])
        table["values"] = [0x1000, 0x2000, 0x3000]
        for field, (tensor, value) in changed.items():
            table[field][tensor] = value
        return plan(lib, table)[0]
    assert status() == 0
    assert status(destination=(0, 0x1000)) == 0                     # in place, said twice
    assert status(destination=(0, 0x4000)) == 0
    assert status(destination=(0, 0x2000 - 40)) == 0                # up to its neighbour
    assert status(values=(1, 0x1000)) == INVALID                    # the same tensor twice
    assert status(values=(1, 0x1000 + 36)) == INVALID               # one value shared
    assert status(destination=(0, 0x1004)) == INVALID               # over itself, moved
    assert status(destination=(0, 0x2000)) == INVALID               # over a neighbour
    assert status(destination=(0, 0x2000 - 36)) == INVALID
    twice = table_of([10, 10])
    twice["values"], twice["destination"] = 0x1000, [0x3000, 0x4000]
    assert plan(lib, twice)[0] == 0                                 # read twice, written apart
    twice["destination"] = 0x3000
    assert plan(lib, twice)[0] == INVALID
    encoded = table_of([64, 64], kind=2, block=32)
    encoded["values"], encoded["scales"] = 0x1000, [0x2000, 0x2008]
    assert plan(lib, encoded)[0] == 0                               # a payload is only read
    encoded["scales"] = [0x2000, 0x2004]
    assert plan(lib, encoded)[0] == INVALID
    empty = table_of([10, 0])
    empty["values"] = 0x1000
    assert plan(lib, empty)[0] == 0


@pytest.mark.parametrize("length,block", ((64, 4), (4, 0), (4, 8), (8, 4), (64, 32)))
def test_plan_refuses_scales_written_over_their_own_payload(lib, length, block):
    """Blocks of four values have as many bytes of scales as of codes: the two ranges are then the same one."""
    table = table_of([length], kind=2, block=block)
    table["values"], table["scales"] = 0x1000, 0x2000
    assert plan(lib, table)[0] == 0
    for destination, status in ((0x2000, 0), (0x1000 + length, 0), (0x1000, INVALID)):
        table["destination"] = destination
        assert plan(lib, table)[0] == status, hex(destination)
    table["scales"], table["destination"] = 0x1000, 0
    assert plan(lib, table)[0] == INVALID                           # in place, scales where the payload is
    table["destination"] = 0x3000
    assert plan(lib, table)[0] == 0                                 # both are only read


def test_clip_refusals_come_before_the_device(lib):
    def call(tensors=4096, count=1, chunk_map=4096, chunks=1, values=4096, workspace=4096, max_norm=1.0, out=4096):
        return lib.nntrain_gradient_list_clip(0, tensors, count, chunk_map, chunks, values, workspace, max_norm, 1, out,
                                              None, None, None)
    assert call(tensors=None) == INVALID
    assert call(count=0) == INVALID
    assert call(chunk_map=None) == INVALID
    assert call(chunk_map=4100) == INVALID
    assert call(chunks=-1) == INVALID
    assert call(chunks=1 << 31) == INVALID
    assert call(values=4095) == INVALID
    assert call(values=1 << 20) == INVALID
    assert call(workspace=None) == INVALID
    assert call(workspace=4100) == INVALID
    assert call(out=None) == INVALID
    for max_norm in (0.0, -1.0, float("nan")):
        assert call(max_norm=max_norm) == INVALID


def test_refused_calls_land_in_the_error_ring(lib):
    from nntrain_b200.library import last_error
    chunks, values = ctypes.c_longlong(), ctypes.c_int()
    for operation, call in (
            (219, lambda: lib.nntrain_gradient_list_plan(None, 1, None, 0, ctypes.addressof(chunks), ctypes.addressof(values))),
            (219, lambda: lib.nntrain_gradient_list_clip(0, None, 1, None, 0, 4096, None, 1.0, 1, None, None, None, None)),
            (220, lambda: lib.nntrain_rms_norm_backward_workspace(-1, 1, None)),
            (221, lambda: lib.nntrain_embedding_gradient_workspace(-1, 1, 1, None))):
        before = last_error().sequence
        assert call() == INVALID
        info = last_error()
        assert info.sequence == before + 1 and info.operation == operation and info.status == INVALID


def test_a_list_refuses_tensors_that_are_not_on_a_device():
    import torch
    with pytest.raises(ValueError, match="CUDA"):
        GradientTensorList(0, [torch.zeros(4)])
    with pytest.raises(ValueError, match="needs tensors"):
        GradientTensorList(0, [])
    with pytest.raises(ValueError, match="float32, bfloat16 or an int8"):
        GradientTensorList(0, [torch.zeros(4, dtype=torch.float16)])
