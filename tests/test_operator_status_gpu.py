"""The status of a training operator's call is its own: neither a refused call
before it nor an error that another library left behind shows in it, and a
refused call leaves no error behind for the next library to find."""
import ctypes

import pytest
import torch

from nntrain_b200.library import load
from nntrain_b200.native import GradientTensorList

pytestmark = pytest.mark.gpu

NO_SUCH_DEVICE, INVALID_DEVICE = 99, 101     # cudaErrorInvalidDevice
ROWS, WIDTH, VOCAB = 3000, 64, 700


@pytest.fixture(scope="module")
def calls():
    """name -> call(device) of every entry point that launches, on every path of its launches."""
    lib = load()

    def zeros(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    x, y, w, dw, inverse = zeros(ROWS, WIDTH), zeros(ROWS, WIDTH), zeros(WIDTH), zeros(WIDTH), zeros(ROWS)
    table, tokens = zeros(VOCAB, WIDTH), zeros(ROWS, dtype=torch.int64)
    scratch, norm = zeros(1 << 24, dtype=torch.uint8), zeros(2)
    short, long = GradientTensorList(0, [zeros(5000)]), GradientTensorList(0, [zeros(8_000_000)])

    def forward(width):
        return lambda device: lib.nntrain_rms_norm_forward(
            device, 0, x.data_ptr(), width, 0, 0, w.data_ptr(), 0, ROWS, width, 1e-6, 0, y.data_ptr(), 0, 0, 0, 0, 0, 0, 0)

    def backward(width):
        return lambda device: lib.nntrain_rms_norm_backward(
            device, 0, x.data_ptr(), width, 0, 0, x.data_ptr(), width, w.data_ptr(), 0, inverse.data_ptr(), ROWS, width,
            y.data_ptr(), dw.data_ptr(), 0, 0, scratch.data_ptr(), scratch.numel(), 0)

    def lookup(device):
        return lib.nntrain_embedding_lookup(device, 0, table.data_ptr(), 0, 0, 0, VOCAB, WIDTH, tokens.data_ptr(), 8, ROWS, -1,
                                            1.0, 0, y.data_ptr(), WIDTH, 0, 0)

    def gradient(count):
        return lambda device: lib.nntrain_embedding_gradient(
            device, 0, x.data_ptr(), WIDTH, tokens.data_ptr(), 8, count, -1, 1.0, 0, table.data_ptr(), VOCAB, WIDTH, 0, 0,
            scratch.data_ptr(), scratch.numel(), 0)

    def clip(plan):
        return lambda device: lib.nntrain_gradient_list_clip(
            device, plan.table_address, plan.count, plan.map_address, plan.chunks, plan.chunk_values, scratch.data_ptr(), 1.0,
            1, norm.data_ptr(), 0, 0, 0)

    yield {"forward": forward(WIDTH), "forward, single values": forward(WIDTH - 1), "backward": backward(WIDTH),
           "backward, single values": backward(WIDTH - 1), "lookup": lookup, "gradient, one CTA": gradient(500),
           "gradient, a cluster": gradient(ROWS), "clip, short": clip(short), "clip, long": clip(long)}
    torch.cuda.synchronize()


def test_a_refused_device_shows_in_its_own_call_only(cuda, calls):
    for name, call in calls.items():
        assert [call(0), call(NO_SUCH_DEVICE), call(0)] == [0, INVALID_DEVICE, 0], name
        assert float((torch.ones(4, device="cuda") + 1.0).sum()) == 8.0          # and torch finds no error either


def test_an_error_that_another_library_left_behind_is_not_the_call_s(cuda, calls):
    runtime = ctypes.CDLL("libcudart.so.12")
    for name, call in calls.items():
        assert runtime.cudaSetDevice(NO_SUCH_DEVICE) == INVALID_DEVICE
        try:
            status = call(0)
        finally:
            runtime.cudaGetLastError()
        assert status == 0, name
