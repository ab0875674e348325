"""Refusals and scratch sizes of the token table's entry points: host code only."""
import ctypes

import pytest

INVALID = 1   # cudaErrorInvalidValue


def lookup(lib, **changed):
    a = dict(device=0, table_kind=0, table=4096, scales=None, block_size=0, first_value=0, vocab=10, width=64, tokens=4096,
             token_bytes=8, count=3, padding=-1, scale=1.0, out_kind=0, out=4096, out_stride=64, status=None, stream=None)
    a.update(changed)
    return lib.nntrain_embedding_lookup(*a.values())


def gradient(lib, **changed):
    a = dict(device=0, gradient_kind=0, out_gradient=4096, stride=64, tokens=4096, token_bytes=8, count=3, padding=-1,
             scale=1.0, table_kind=0, table=4096, vocab=10, width=64, accumulate=0, status=None, workspace=4096,
             workspace_bytes=1 << 20, stream=None)
    a.update(changed)
    return lib.nntrain_embedding_gradient(*a.values())


@pytest.mark.parametrize("changed", (
    dict(table_kind=3), dict(table_kind=-1), dict(table=None), dict(table_kind=2), dict(table_kind=2, scales=4098),
    dict(block_size=-1), dict(first_value=-1), dict(vocab=0), dict(vocab=(1 << 31) + 1), dict(width=0),
    dict(width=(1 << 24) + 1, out_stride=1 << 25), dict(tokens=None), dict(token_bytes=2), dict(tokens=4100), dict(count=-1),
    dict(count=1 << 31), dict(out_kind=2), dict(out=None), dict(out=4098), dict(out_stride=63), dict(table=4098),
    dict(status=4097)))
def test_lookup_refuses(lib, changed):
    assert lookup(lib, **changed) == INVALID


@pytest.mark.parametrize("changed", (
    dict(gradient_kind=2), dict(table_kind=2), dict(table=None), dict(out_gradient=None), dict(stride=63), dict(tokens=None),
    dict(token_bytes=1), dict(count=-1), dict(count=1 << 31), dict(vocab=0), dict(width=0), dict(workspace=None),
    dict(workspace=4104), dict(workspace_bytes=100), dict(out_gradient=4097), dict(table=4098), dict(tokens=4100),
    dict(status=4098)))
def test_gradient_refuses(lib, changed):
    assert gradient(lib, **changed) == INVALID


def test_no_tokens_are_no_work(lib):
    assert lookup(lib, count=0, tokens=None, out=None) == 0
    assert gradient(lib, count=0, tokens=None, out_gradient=None, accumulate=1) == 0


def test_scratch_size(lib):
    out = ctypes.c_longlong()

    def size(count, vocab, width):
        assert lib.nntrain_embedding_gradient_workspace(count, vocab, width, ctypes.addressof(out)) == 0
        return out.value

    # two arrays of a pair per token, a bit per row, two counters, lists of the tokens that cross chunks of 16 or 32,
    # two rows of fp32 a chunk
    for count, vocab, width, chunk in ((0, 1, 1, 16), (1, 10, 64, 16), (32, 10, 64, 16), (33, 10, 64, 16),
                                       (8192, 151936, 1536, 16), (65536, 32000, 512, 16), (131072, 50000, 768, 32)):
        chunks = -(-count // chunk)
        parts = [count * 8] * 2 + [-(-vocab // 32) * 4, 8, chunks * 4, (chunks // 16 + 1) * 4] + [chunks * width * 4] * 2
        assert size(count, vocab, width) == sum(-(-p // 256) * 256 for p in parts)
    for bad in ((-1, 10, 10), (10, 0, 10), (10, 10, 0), (1 << 31, 10, 10)):
        assert lib.nntrain_embedding_gradient_workspace(*bad, ctypes.addressof(out)) == INVALID
    assert lib.nntrain_embedding_gradient_workspace(1, 1, 1, None) == INVALID
