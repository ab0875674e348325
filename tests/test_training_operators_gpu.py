"""One training step's operators in a row, as a trainer on the encoded gradient
path calls them: rows of the published (BFP8) table, the norm with its output
encoded, back through both into the fp32 gradient arena, the global norm and
clip over the list of its tensors, and the publication of the arena.

Every stage is checked against numpy in 64 bits on the inputs that the stage
before it left on the device, with that stage's own bounds; the recorded step
has to leave the same bits as the eager one."""
import numpy as np
import pytest
import torch

import test_rms_norm_gpu as norm_tests
import test_tensor_list_gpu as list_tests
import test_token_embedding_gpu as embedding_tests
from gpu_helpers import assert_bits_equal, dev, host
from nntrain_b200.native import (CudaBfp8GradientNative, CudaBfp8Native, GradientNorm, GradientTensorList, RmsNorm,
                                 TokenEmbedding, scale_count)

pytestmark = pytest.mark.gpu

VOCAB, WIDTH, BATCH, LENGTH, BLOCK, MAX_NORM = 515, 96, 3, 70, 32, 0.5
EPS = 1e-6


class Step:
    """Buffers of one step.  The arena holds the table's gradient, the norm
    weight's and a leaf of another layer, one behind the other."""

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.rows = BATCH * LENGTH
        table = (rng.standard_normal(VOCAB * WIDTH) * 0.05).astype(np.float32)
        self.payload = torch.zeros(VOCAB * WIDTH, dtype=torch.int8, device="cuda")
        self.scales = torch.zeros(scale_count(VOCAB * WIDTH, BLOCK), device="cuda")
        CudaBfp8Native.block_encode(0, dev(table), self.payload, self.scales, BLOCK)
        tokens = embedding_tests.some_tokens(rng, self.rows, VOCAB, 0.0)
        tokens.reshape(BATCH, LENGTH)[1, 40:] = -1                       # a padded sequence
        self.tokens = dev(tokens.reshape(BATCH, LENGTH))
        self.weight = dev((1.0 + 0.2 * rng.standard_normal(WIDTH)).astype(np.float32))
        self.residual = dev(rng.standard_normal((self.rows, WIDTH)).astype(np.float32)).to(torch.bfloat16)
        self.y_gradient = dev((rng.standard_normal((self.rows, WIDTH)) * 1e-2).astype(np.float32)).to(torch.bfloat16)
        self.other = dev((rng.standard_normal(1001) * 1e-2).astype(np.float32))

        def empty(*shape, dtype=torch.float32):
            return torch.zeros(*shape, dtype=dtype, device="cuda")

        self.x, self.h, self.y, self.x_gradient = (empty(self.rows, WIDTH, dtype=torch.bfloat16) for _ in range(4))
        self.codes, self.code_scales = empty(self.rows, WIDTH, dtype=torch.int8), empty(self.rows * (WIDTH // BLOCK))
        self.inverse = empty(self.rows)
        self.lengths = [VOCAB * WIDTH, WIDTH, 1001]
        offsets = np.concatenate([[0], np.cumsum(self.lengths)]).astype(np.int64)
        self.total = int(offsets[-1])
        self.offsets = dev(offsets)
        self.arena = empty(self.total)
        self.table_gradient = self.arena[:VOCAB * WIDTH].view(VOCAB, WIDTH)
        self.weight_gradient = self.arena[offsets[1]:offsets[2]]
        self.leaf = self.arena[offsets[2]:offsets[3]]
        self.published, self.published_scales = empty(self.total, dtype=torch.int8), empty(3)
        self.maxima, self.flag, self.token_status = (empty(n, dtype=torch.int32) for n in (3, 1, 1))
        self.norm_and_coefficient, self.tensor_norms = empty(2), empty(3)
        # the leaf of the other layer lies elsewhere and is gathered into the arena by the clip
        self.list = GradientTensorList(0, [self.table_gradient, self.weight_gradient, self.other],
                                       destinations=[None, None, self.leaf])

    def forward(self):
        TokenEmbedding.lookup(0, self.tokens, self.payload.view(VOCAB, WIDTH), self.x, scale=WIDTH ** 0.5,
                              table_scales=self.scales, block_size=BLOCK, token_status=self.token_status)
        RmsNorm.forward(0, self.x, self.weight, EPS, residual=self.residual, residual_out=self.h, y=self.y, payload=self.codes,
                        scales=self.code_scales, block_size=BLOCK, inverse_rms=self.inverse, finite_status=self.flag)

    def backward(self):
        RmsNorm.backward(0, self.y_gradient, self.h, self.weight, self.inverse, self.x_gradient, self.weight_gradient)
        TokenEmbedding.gradient(0, self.tokens, self.x_gradient, self.table_gradient, scale=WIDTH ** 0.5)

    def finish(self):
        GradientNorm.clip_tensors(0, self.list, MAX_NORM, self.norm_and_coefficient, self.tensor_norms, self.flag)
        CudaBfp8GradientNative.publish_tensors(0, self.arena, self.published, self.published_scales, self.offsets, self.maxima,
                                               self.flag)

    def run(self):
        self.flag.zero_()
        self.forward()
        self.backward()
        self.finish()

    def results(self):
        return (self.y, self.codes, self.code_scales, self.x_gradient, self.arena, self.published, self.published_scales,
                self.norm_and_coefficient, self.tensor_norms)


def test_a_step_stage_by_stage(cuda, oracle):
    s = Step(1)
    s.forward()
    torch.cuda.synchronize()
    table = torch.zeros(VOCAB * WIDTH, device="cuda")
    CudaBfp8Native.block_decode(0, s.payload, s.scales, table, BLOCK)
    tokens = host(s.tokens).ravel()
    rows = host(table).reshape(VOCAB, WIDTH)[tokens.clip(0)] * np.float32(WIDTH ** 0.5)
    want = torch.from_numpy(np.where((tokens >= 0)[:, None], rows, 0).astype(np.float32)).to(torch.bfloat16)
    assert torch.equal(s.x.cpu(), want)
    assert torch.equal(s.h.cpu(), (s.x.float() + s.residual.float()).to(torch.bfloat16).cpu())
    _, inverse, y = norm_tests.reference(s.x, s.residual, s.weight)
    ti = norm_tests.tolerance_i(WIDTH)
    assert (np.abs(norm_tests.f64(s.inverse) - inverse) <= inverse * ti).all()
    q = y.reshape(-1, BLOCK) / (np.abs(y.reshape(-1, BLOCK)).max(axis=1) / 127.0)[:, None]
    assert (np.abs(norm_tests.f64(s.codes).reshape(-1, BLOCK) - q) <= 0.5 + 127.0 * (2 * (ti + 3 * norm_tests.E) + 2 * norm_tests.E)).all()

    s.backward()
    torch.cuda.synchronize()
    norm_tests.check_gradient(s.x_gradient, s.weight_gradient, s.y_gradient, s.h, s.weight, s.inverse, None)
    embedding_tests.check_gradient(tokens, s.x_gradient, s.table_gradient, np.float64(np.float32(WIDTH ** 0.5)), VOCAB)

    before = [t.clone() for t in (s.table_gradient, s.weight_gradient, s.other)]
    s.finish()
    torch.cuda.synchronize()
    squares = [float((t.double() ** 2).sum()) for t in before]
    norm, c = host(s.norm_and_coefficient)
    assert abs(norm - np.sqrt(sum(squares))) <= np.sqrt(sum(squares)) * list_tests.HALF * 1.001
    assert norm > MAX_NORM and abs(c - MAX_NORM / (norm + 1e-6)) <= c * 3 * list_tests.HALF
    assert (np.abs(host(s.tensor_norms) - np.sqrt(squares)) <= np.sqrt(squares) * list_tests.HALF * 1.001).all()
    assert torch.equal(s.other, before[2])                                # gathered, not clipped where it lies
    assert int(s.flag.item()) == 0 and int(s.token_status.item()) == 0
    for t, (clipped, length) in enumerate(zip(before, s.lengths)):
        start = int(host(s.offsets)[t])
        decoded, payload, scale, flag, _ = oracle.gradient_publish((host(clipped).ravel() * c).astype(np.float32), 0)
        assert flag == 0
        assert np.array_equal(host(s.published)[start:start + length], payload)
        assert_bits_equal(host(s.published_scales)[t:t + 1], scale, f"scale of tensor {t}")
        assert_bits_equal(host(s.arena)[start:start + length], decoded, f"arena, tensor {t}")


def test_recorded_step_leaves_the_same_bits(cuda):
    s = Step(2)
    s.run()
    torch.cuda.synchronize()
    eager = [t.clone() for t in s.results()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    for t in s.results():
        t.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager, s.results()):
        assert torch.equal(a, b)


def test_a_gradient_that_is_not_finite_ends_the_step_closed(cuda):
    s = Step(3)
    s.y_gradient[5, 7] = float("nan")
    s.published_scales.fill_(9.0)
    s.flag.zero_()
    s.forward()
    s.backward()
    before = s.arena[:VOCAB * WIDTH + WIDTH].clone()
    s.finish()
    torch.cuda.synchronize()
    assert int(s.flag.item()) == 1 and host(s.norm_and_coefficient)[1] == 1.0
    assert (s.published_scales == 1.0).all() and not s.published.any()    # nothing is published
    assert torch.equal(s.arena[:VOCAB * WIDTH + WIDTH].view(torch.int32), before.view(torch.int32))
