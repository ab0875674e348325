"""The norm and the list's clip on tensors of more than 2^31 values, whose offsets
pass 32 bits (the token table's are in test_token_embedding_gpu.py)."""
import math

import pytest
import torch

from nntrain_b200.native import GradientNorm, GradientTensorList, RmsNorm

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.mark.parametrize("width,block", ((2048, 32), (16416, 32), (771, 0)))
def test_norm_of_more_than_31_bits_of_values(cuda, width, block):
    rows = (1 << 31) // width + 1000
    pattern = torch.randn(7, width, generator=torch.Generator(device="cuda").manual_seed(width), device="cuda").to(torch.bfloat16)
    x = pattern.repeat(-(-rows // 7), 1)[:rows]
    w = torch.rand(width, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    y, payload = torch.empty_like(x), torch.empty(rows, width, dtype=torch.int8, device="cuda")
    scales, inverse = torch.empty(rows, width // (block or width), device="cuda"), torch.empty(rows, device="cuda")
    RmsNorm.forward(0, x, w, EPS, y=y, payload=payload, scales=scales, block_size=block, inverse_rms=inverse)
    dx, dw = torch.empty_like(x), torch.empty(width, device="cuda")
    RmsNorm.backward(0, y, x, w, inverse, dx, dw)
    torch.cuda.synchronize()
    for out in (y, payload, scales, inverse, dx):          # every row is the one seven rows before it
        for begin in range(0, rows - 7, 1 << 17):
            end = min(begin + (1 << 17), rows - 7)
            assert torch.equal(out[begin:end], out[begin + 7:end + 7]), begin
    few = 7 * 22                                           # rows enough for the same kernel
    first = [torch.empty_like(t[:few]) for t in (y, payload, scales, inverse, dx)]
    RmsNorm.forward(0, x[:few], w, EPS, y=first[0], payload=first[1], scales=first[2], block_size=block, inverse_rms=first[3])
    RmsNorm.backward(0, first[0], x[:few], w, first[3], first[4], torch.empty(width, device="cuda"))
    for whole, part in zip((y, payload, scales, inverse, dx), first):
        assert torch.equal(whole[:few], part)


@pytest.mark.parametrize("offset", (0, 3))
def test_clip_of_tensors_of_more_than_31_bits_of_values(cuda, offset):
    n = (1 << 31) + 12345
    x = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    x[-1] = 4096.0
    to = torch.zeros(n + offset + 9, dtype=torch.bfloat16, device="cuda")
    payload = torch.ones(n, dtype=torch.int8, device="cuda")
    payload[-1] = 127
    scales = torch.full((-(-n // 32),), 0.25, device="cuda")
    scales[-1] = 64.0
    last = n - (len(scales) - 1) * 32                      # values of the last block
    plan = GradientTensorList(0, [x, payload], [None, scales], [0, 32], [to[offset:offset + n], None])
    out, norms = torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")
    GradientNorm.clip_tensors(0, plan, 1.0, out, norms)
    torch.cuda.synchronize()
    squares = [(n - 1) * 0.25 + 4096.0 ** 2, (n - last) * 0.0625 + (last - 1 + 127 ** 2) * 4096.0]
    for got, want in zip(norms.tolist(), squares):         # binary64 sums, the root rounded once: 2^-24
        assert abs(got - math.sqrt(want)) <= math.sqrt(want) * 2.0 ** -24 * 1.001
    c = out[1]
    assert 0.0 < float(c) < 1.0
    assert torch.equal(to[offset:offset + n - 1].amin(), (0.5 * c).to(torch.bfloat16))
    assert torch.equal(to[offset:offset + n - 1].amax(), (0.5 * c).to(torch.bfloat16))
    assert torch.equal(to[offset + n - 1], (4096.0 * c).to(torch.bfloat16))
    assert not to[:offset].any() and not to[offset + n:].any()
    assert (scales[:-1] == 0.25 * c).all() and scales[-1] == 64.0 * c
    assert int(payload.sum(dtype=torch.int64)) == n - 1 + 127
