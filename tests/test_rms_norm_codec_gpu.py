"""The norm's encoded output is the codec's encode of y = (h * i) * w, bit for bit,
for the i that the call itself gives: two products in fp32, then the codec's
launch.  (Not of the y of another call: forms that take different kernels add a
row's squares in different orders, and i may differ in its last bit.)"""
import pytest
import torch

from nntrain_b200.native import CudaBfp8Native, RmsNorm

pytestmark = pytest.mark.gpu

EPS = 1e-6


def inputs(rows, width, dtype):
    """Rows of ordinary size, of zeros, very small and very large ones, ties of the rounding, and some that are not
    finite; weights from 2^-80 to 2^80 in one stretch, so that blocks differ as much."""
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    x = torch.randn(rows, width, generator=g, device="cuda")
    x[1] = 0.0
    x[2] *= 1e-25
    x[3] *= 1e15
    x[4] = torch.arange(width, device="cuda").remainder(255).sub(127).float()
    x[5, width // 2] = float("nan")
    x[6, width // 3] = float("inf")
    x[7, ::2] = 0.0
    w = 1.0 + 0.3 * torch.randn(width, generator=g, device="cuda")
    part = slice(width // 4, width // 4 + 16)
    w[part] *= torch.exp2(torch.linspace(-80, 80, len(w[part]), device="cuda"))
    return x.to(dtype), w


SHAPES = ((9, 64), (9, 33), (200, 96), (200, 771), (200, 1536), (1501, 2048), (200, 4096), (9, 16384), (9, 16416), (9, 8193))


@pytest.mark.parametrize("rows,width,block", [(rows, width, block) for rows, width in SHAPES for block in (0, 32, 64, 128, 96, 3)
                                              if not block or width % block == 0])
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("aligned", (True, False))
def test_the_encode_is_the_codec_s(cuda, rows, width, block, dtype, aligned):
    b = block or width
    x, w = inputs(rows, width, dtype)
    if not aligned:
        base = torch.zeros(rows * width + 8, dtype=dtype, device="cuda")
        base[1:1 + rows * width] = x.view(-1)
        x = base[1:1 + rows * width].view(rows, width)
    payload, scales = torch.zeros(rows, width, dtype=torch.int8, device="cuda"), torch.zeros(rows * (width // b), device="cuda")
    inverse = torch.zeros(rows, device="cuda")
    RmsNorm.forward(0, x, w, EPS, payload=payload, scales=scales, block_size=block, inverse_rms=inverse)
    y = (x.float() * inverse[:, None]) * w
    codes, code_scales = torch.zeros_like(payload), torch.zeros_like(scales)
    CudaBfp8Native.block_encode(0, y.view(-1), codes.view(-1), code_scales, b)
    torch.cuda.synchronize()
    assert torch.equal(scales.view(torch.int32), code_scales.view(torch.int32))
    assert torch.equal(payload, codes)
