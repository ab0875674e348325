"""Refusals of the RMS norm's entry points that come before any device work."""
import ctypes

import pytest

INVALID = 1   # cudaErrorInvalidValue


def forward(lib, **changed):
    a = dict(device=0, kind=0, x=4096, x_stride=64, residual=None, residual_stride=0, weight=4096, weight_kind=0, rows=2,
             width=64, epsilon=1e-6, residual_out=None, y=4096, y_kind=0, payload=None, scales=None, block_size=0,
             inverse_rms=None, finite_status=None, stream=None)
    a.update(changed)
    return lib.nntrain_rms_norm_forward(*a.values())


def backward(lib, **changed):
    a = dict(device=0, kind=0, y_gradient=4096, y_stride=64, residual_gradient=None, residual_stride=0, h=4096, h_stride=64,
             weight=4096, weight_kind=0, inverse_rms=4096, rows=2, width=64, x_gradient=4096, weight_gradient=4096,
             weight_gradient_kind=0, accumulate=0, workspace=4096, workspace_bytes=1 << 20, stream=None)
    a.update(changed)
    return lib.nntrain_rms_norm_backward(*a.values())


@pytest.mark.parametrize("changed", (
    dict(kind=2), dict(kind=-1), dict(weight_kind=2), dict(y_kind=3), dict(rows=-1), dict(rows=1 << 41), dict(width=0),
    dict(width=-4), dict(width=(1 << 24) + 1, x_stride=1 << 25), dict(epsilon=-1e-6), dict(epsilon=float("nan")),
    dict(epsilon=float("inf")), dict(x_stride=63), dict(residual=4096, residual_stride=63), dict(weight=None), dict(x=None),
    dict(y=None), dict(payload=4096), dict(payload=4096, scales=4096, block_size=-1),
    dict(payload=4096, scales=4096, block_size=48), dict(residual_out=4096), dict(x=4098), dict(y=4097),
    dict(scales=4097), dict(weight=4098), dict(inverse_rms=4098), dict(finite_status=4098)))
def test_forward_refuses(lib, changed):
    assert forward(lib, **changed) == INVALID


@pytest.mark.parametrize("changed", (
    dict(kind=2), dict(weight_kind=-1), dict(weight_gradient_kind=2), dict(rows=-1), dict(width=0), dict(y_stride=63),
    dict(h_stride=63), dict(residual_gradient=4096, residual_stride=0), dict(weight=None), dict(weight_gradient=None),
    dict(y_gradient=None), dict(h=None), dict(inverse_rms=None), dict(x_gradient=None), dict(workspace=None),
    dict(workspace_bytes=2 * 64 * 4 - 1), dict(workspace=4097), dict(x_gradient=4098)))
def test_backward_refuses(lib, changed):
    assert backward(lib, **changed) == INVALID


def test_workspace_is_one_row_for_each_block_that_leaves_a_partial(lib):
    out = ctypes.c_longlong(-1)
    for rows, width, want in ((0, 8, 0), (1, 8, 32), (1000, 10, 40_000), (10 ** 6, 10, 1184 * 40)):
        assert lib.nntrain_rms_norm_backward_workspace(rows, width, ctypes.addressof(out)) == 0
        assert out.value == want
    assert lib.nntrain_rms_norm_backward_workspace(-1, 8, ctypes.addressof(out)) == INVALID
    assert lib.nntrain_rms_norm_backward_workspace(1, 0, ctypes.addressof(out)) == INVALID
    assert lib.nntrain_rms_norm_backward_workspace(1, 8, None) == INVALID


def test_no_rows_are_no_work(lib):
    assert forward(lib, rows=0, x=None) == 0
