"""Decoding blocks whose size is not a multiple of four: a 32-bit payload word
then holds values of two blocks, each with its own scale."""
import numpy as np
import pytest
import torch

from gpu_helpers import assert_bits_equal, dev, host
from nntrain_b200.native import CudaBfp8Native, scale_count

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,block", ((99, 33), (515, 5), (4097, 1), (70001, 771), (1000, 7), (1000, 998), (70000, 6)))
def test_odd_blocks_decode_with_their_own_scale(cuda, oracle, n, block):
    source = oracle.generate_gradient(n, 0xB2000031, 0)
    payload, scales = oracle.encode(source, block, strict=False)
    d_payload, d_scales = torch.zeros(n, dtype=torch.int8, device="cuda"), torch.zeros(scale_count(n, block), device="cuda")
    CudaBfp8Native.block_encode(0, dev(source), d_payload, d_scales, block)
    decoded, again = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    CudaBfp8Native.block_decode(0, d_payload, d_scales, decoded, block)
    CudaBfp8Native.dequantize_float32(0, d_payload, d_scales, again, block)
    torch.cuda.synchronize()
    want = oracle.decode(payload, scales, block, strict=False)
    assert np.array_equal(host(d_payload), payload)
    assert_bits_equal(host(decoded), want, "block_decode")
    assert_bits_equal(host(again), want, "dequantize_float32")
