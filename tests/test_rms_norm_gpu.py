"""The RMS norm with an encoded output and its gradient against numpy in 64 bits.

Tolerances, with e = 2^-24 (half a step of binary32, relative) and o = half a
step of the output's type (0 where it is fp32 and counted already):
  squares  a sum of `width` non-negative products; no value passes more than
           d = terms of a thread + 5 butterfly steps + 16 warps additions:
           (d + 2) e, the 2 for h = fl(x + r) squared
  i        the mean, a product with fl(1/width), adds 2 e, + epsilon e; the root
           halves; its Newton step is 3/2 e off
  y        i's, and h, two products: 3 e more
  code     |code - y/scale| <= 1/2 + 127 (2 y's + 2 e), for y and scale both
  dx       i (g - n c) + r with c = mean(g n): (d + 5) e of mean|g n| in c, a
           step for each of g, n, their product, the sums and the result
  dw       rows / 148 terms a block, 37 + 5 in the join, 2 e for the product"""
import numpy as np
import pytest
import torch

from gpu_helpers import assert_bits_equal, dev, host
from nntrain_b200.native import CudaBfp8Native, RmsNorm

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
EPS = 1e-6
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def depth(width):
    """Most additions a term of a row's sum passes: 32 terms a thread in registers (widths to 16384), more beyond."""
    return max(32, -(-width // 256)) + 5 + 16


def tolerance_i(width):
    return ((depth(width) + 5) / 2 + 1.5) * E


def f64(t):
    return t.detach().double().cpu().numpy()


def values(rng, rows, width, dtype, sigma=1.0):
    return dev((rng.standard_normal((rows, width)) * sigma).astype(np.float32)).to(dtype)


def placed(t, shift, stride):
    """The same matrix `shift` values off the allocation's start with rows `stride` apart."""
    rows, width = t.shape
    base = torch.full((shift + rows * stride + 64,), 7.0, dtype=t.dtype, device="cuda")
    view = base[shift:shift + rows * stride].view(rows, stride)[:, :width]
    view.copy_(t)
    return view


def reference(x, r, w):
    h = f64(x) + (f64(r) if r is not None else 0.0)
    i = 1.0 / np.sqrt((h * h).mean(axis=1) + EPS)
    return h, i, h * i[:, None] * f64(w)


def round_to(a64, dtype):
    return torch.from_numpy(a64).float().to(dtype)


SHAPES = ((1, 1), (1, 8), (2, 32), (3, 33), (5, 771), (7, 1536), (149, 96), (1, 4096), (200, 4096), (3, 8192), (2, 16384),
          (2, 16416), (3, 2049), (2, 8193), (1500, 64))


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("rows,width,block", [(rows, width, block) for rows, width in SHAPES
                                              for block in (None, 0, 32, 64, 128, 96) if not block or width % block == 0])
def test_forward(cuda, rows, width, dtype, block):
    rng = np.random.default_rng(rows * 1000 + width)
    x, r = values(rng, rows, width, dtype), values(rng, rows, width, dtype, 3.0)
    w = dev((1.0 + 0.3 * rng.standard_normal(width)).astype(np.float32))
    h, i, y = reference(x, r, w)
    out_h, inverse = torch.zeros_like(x), torch.zeros(rows, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out_y = torch.zeros(rows, width, dtype=dtype, device="cuda")
    if block is None:
        RmsNorm.forward(0, x, w, EPS, residual=r, residual_out=out_h, y=out_y, inverse_rms=inverse, finite_status=flag)
    else:
        b = width if block == 0 else block
        payload = torch.zeros(rows, width, dtype=torch.int8, device="cuda")
        scales = torch.zeros(rows * (width // b), device="cuda")
        RmsNorm.forward(0, x, w, EPS, residual=r, residual_out=out_h, y=out_y, payload=payload, scales=scales,
                        block_size=block, inverse_rms=inverse, finite_status=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    assert torch.equal(out_h.cpu(), (x.float() + r.float()).to(dtype).cpu())
    ti = tolerance_i(width)
    assert (np.abs(f64(inverse) - i) <= i * ti).all()
    ty = ti + 3 * E
    if block is None:
        assert (np.abs(f64(out_y) - y) <= np.abs(y) * (ty + 1.01 * HALF_STEP[dtype])).all()
        return
    largest = np.abs(y.reshape(-1, b)).max(axis=1)
    assert (np.abs(f64(scales) - largest / 127.0) <= largest / 127.0 * (ty + 2 * E)).all()
    codes = f64(payload).reshape(-1, b)
    q = y.reshape(-1, b) / (largest / 127.0)[:, None]
    assert (np.abs(codes - q) <= 0.5 + 127.0 * (2 * ty + 2 * E)).all() and np.abs(codes).max() <= 127
    # y is what the codes stand for, and what the codec decodes
    per_value = np.repeat(host(scales), b).reshape(rows, width)
    want = (host(payload).astype(np.float32) * per_value).astype(np.float32)
    assert_bits_equal(out_y.float().cpu().numpy().ravel(), torch.from_numpy(want).to(dtype).float().numpy().ravel(), "decoded y")
    decoded = torch.zeros(rows * width, device="cuda")
    CudaBfp8Native.block_decode(0, payload.view(-1), scales, decoded, b)
    assert_bits_equal(host(decoded), want.ravel(), "the codec's decode")


@pytest.mark.parametrize("width", (64, 771, 1536, 16416))
@pytest.mark.parametrize("shift,extra", ((0, 8), (1, 0), (3, 5), (8, 16)))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_any_place_and_stride_gives_the_same_bits(cuda, width, shift, extra, dtype):
    """Rows off the 16-byte grid take another kernel; within a kernel the place does not matter."""
    rows = 5
    rng = np.random.default_rng(width)
    x, r = values(rng, rows, width, dtype), values(rng, rows, width, dtype)
    w = dev((1.0 + 0.3 * rng.standard_normal(width)).astype(np.float32)).to(dtype)
    block = 0 if width == 771 else 32

    def run(x, r):
        y = torch.zeros(rows, width, device="cuda")
        payload, scales = torch.zeros(rows, width, dtype=torch.int8, device="cuda"), torch.zeros(rows * max(1, width // 32 if block else 1), device="cuda")
        h = torch.zeros(rows, width, dtype=dtype, device="cuda")
        RmsNorm.forward(0, x, w, EPS, residual=r, residual_out=h, y=y, payload=payload, scales=scales, block_size=block)
        torch.cuda.synchronize()
        return y, h, scales

    y, h, scales = run(placed(x, shift, width + extra), placed(r, shift, width + extra))
    _, i, want = reference(x, r, w)
    ty = tolerance_i(width) + 3 * E
    b = width if block == 0 else block
    largest = np.abs(want.reshape(-1, b)).max(axis=1)
    assert (np.abs(f64(scales) - largest / 127) <= largest / 127 * (ty + 2 * E)).all()
    step = np.repeat(largest / 127, b).reshape(rows, width)
    assert (np.abs(f64(y) - want) <= step * (0.5 + 127 * (3 * ty + 4 * E))).all()
    assert torch.equal(h.cpu(), (x.float() + r.float()).to(dtype).cpu())
    again = run(placed(x, shift, width + extra), placed(r, shift, width + extra))
    assert all(torch.equal(a, b) for a, b in zip((y, h, scales), again))


@pytest.mark.parametrize("width", (1536, 771, 16416, 8193))
@pytest.mark.parametrize("block", (0, 32))
def test_the_sum_may_take_the_place_of_an_input(cuda, width, block):
    if block and width % block:
        block = 0
    rows = 4
    rng = np.random.default_rng(3)
    x, r = values(rng, rows, width, torch.bfloat16), values(rng, rows, width, torch.bfloat16)
    w = dev(rng.standard_normal(width).astype(np.float32))
    results = []
    for place in ("apart", "x", "residual"):
        a, b = x.clone(), r.clone()
        h = {"apart": torch.zeros_like(x), "x": a, "residual": b}[place]
        payload = torch.zeros(rows, width, dtype=torch.int8, device="cuda")
        scales = torch.zeros(rows * (width // 32 if block else 1), device="cuda")
        RmsNorm.forward(0, a, w, EPS, residual=b, residual_out=h, payload=payload, scales=scales, block_size=block)
        torch.cuda.synchronize()
        results.append((h.clone(), payload, scales))
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], other))


@pytest.mark.parametrize("width", (1536, 771, 16416, 8193))
@pytest.mark.parametrize("block", (None, 0, 32))
def test_y_may_take_the_place_of_x(cuda, width, block):
    if block and width % block:
        block = 0
    rows = 700                                        # some CTAs have several rows on their way
    rng = np.random.default_rng(4)
    x = values(rng, rows, width, torch.bfloat16)
    w = dev(rng.standard_normal(width).astype(np.float32))
    results = []
    for place in (torch.zeros_like(x), x.clone()):
        source = x if not results else place
        kwargs = {}
        if block is not None:
            kwargs = dict(payload=torch.zeros(rows, width, dtype=torch.int8, device="cuda"), block_size=block,
                          scales=torch.zeros(rows * (width // 32 if block else 1), device="cuda"))
        RmsNorm.forward(0, source, w, EPS, y=place, **kwargs)
        torch.cuda.synchronize()
        results.append(place)
    assert torch.equal(results[0], results[1])


def test_without_a_residual_and_bits_for_bf16(cuda):
    rng = np.random.default_rng(4)
    x = values(rng, 6, 256, torch.bfloat16)
    w = dev(rng.standard_normal(256).astype(np.float32)).to(torch.bfloat16)
    y, bits = torch.zeros(6, 256, dtype=torch.bfloat16, device="cuda"), torch.zeros(6, 256, dtype=torch.int16, device="cuda")
    RmsNorm.forward(0, x, w, EPS, y=y)
    RmsNorm.forward(0, x.view(torch.int16), w.view(torch.int16), EPS, y=bits)
    torch.cuda.synchronize()
    _, _, want = reference(x, None, w)
    assert (np.abs(f64(y) - want) <= np.abs(want) * (tolerance_i(256) + 3 * E + 1.01 * 2.0 ** -8)).all()
    assert torch.equal(y.view(torch.int16), bits)


@pytest.mark.parametrize("width,block", ((64, 32), (64, 0), (771, 0), (16416, 32), (16416, 0)))
def test_zero_rows_and_values_that_are_not_finite(cuda, width, block):
    rows = 5
    rng = np.random.default_rng(5)
    x = values(rng, rows, width, torch.float32)
    x[0] = 0.0
    x[2, 3], x[3, 5] = float("nan"), float("inf")
    w = dev(np.ones(width, np.float32))
    b = width if block == 0 else block
    payload = torch.zeros(rows, width, dtype=torch.int8, device="cuda")
    scales, flag = torch.zeros(rows * (width // b), device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    RmsNorm.forward(0, x, w, EPS, payload=payload, scales=scales, block_size=block, finite_status=flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 1
    s, p = host(scales).reshape(rows, -1), host(payload)
    assert (s[0] == 1.0).all() and not p[0].any()              # a block of zeros has scale 1
    assert not p[2].any() and (s[2] == 1.0).all()              # every y of the row is NaN: no maximum, codes 0
    assert not p[3].any()                                      # 1 / inf: zeros, and NaN in the place of the inf
    flag.zero_()
    RmsNorm.forward(0, x[[0, 1, 4]], w, EPS, payload=payload[:3], scales=scales[:3 * (width // b)], block_size=block, finite_status=flag)
    assert int(flag.item()) == 0                               # the rows without them raise nothing


def test_an_overflowing_mean_square_raises_the_flag(cuda):
    x = torch.full((1, 64), 1e20, device="cuda")
    y, flag = torch.zeros_like(x), torch.zeros(1, dtype=torch.int32, device="cuda")
    RmsNorm.forward(0, x, torch.ones(64, device="cuda"), EPS, y=y, finite_status=flag)
    assert int(flag.item()) == 1


# ---- gradient -----------------------------------------------------------------

def gradient_reference(dy, h, w, i, r):
    dy, h, w, i = f64(dy), f64(h), f64(w), f64(i)[:, None]
    n, g = h * i, dy * w
    c = (g * n).mean(axis=1, keepdims=True)
    dx = i * (g - n * c) + (0.0 if r is None else f64(r))
    return dx, (dy * n).sum(axis=0), n, g, c, i


def check_gradient(dx, dw, dy, h, w, i, r, before=None, dtype=None):
    rows, width = h.shape
    want, want_w, n, g, c, i = gradient_reference(dy, h, w, i, r)
    size = np.abs(g * n).mean(axis=1, keepdims=True)
    bound = E * (i * (3 * np.abs(g) + np.abs(n) * (size * (depth(width) + 6) + 3 * np.abs(c))) + 2 * np.abs(want))
    bound = bound + np.abs(want) * (HALF_STEP[dx.dtype] * 1.01 if dx.dtype == torch.bfloat16 else 0.0)
    assert (np.abs(f64(dx) - want) <= bound).all()
    terms = np.abs(f64(dy) * n).sum(axis=0)
    bound = (-(-rows // 148) + 45 + 2) * E * terms
    if before is not None:
        want_w = want_w + f64(before)
        bound = bound + E * (np.abs(want_w) + terms)
    if dw.dtype == torch.bfloat16:
        bound = bound + np.abs(want_w) * 2.0 ** -8 * 1.01
    assert (np.abs(f64(dw) - want_w) <= bound).all()


@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("residual", (False, True))
def test_backward(cuda, rows, width, dtype, residual):
    rng = np.random.default_rng(rows + width)
    h, dy = values(rng, rows, width, dtype, 3.0), values(rng, rows, width, dtype, 1e-3)
    r = values(rng, rows, width, dtype, 1e-3) if residual else None
    w = dev((1.0 + 0.3 * rng.standard_normal(width)).astype(np.float32))
    i = torch.rsqrt(h.float().square().mean(dim=1) + EPS)
    dx, dw = torch.zeros_like(h), torch.full((width,), 9.0, device="cuda")
    RmsNorm.backward(0, dy, h, w, i, dx, dw, residual_gradient=r)
    torch.cuda.synchronize()
    check_gradient(dx, dw, dy, h, w, i, r)
    again, weight_again = torch.zeros_like(h), torch.zeros(width, device="cuda")
    RmsNorm.backward(0, dy, h, w, i, again, weight_again, residual_gradient=r)
    assert torch.equal(again, dx) and torch.equal(weight_again, dw)


@pytest.mark.parametrize("kind", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("width", (96, 771, 16416))
def test_weight_gradient_is_added_at_an_arena_offset(cuda, kind, width):
    rows = 300
    rng = np.random.default_rng(7)
    h, dy = values(rng, rows, width, torch.bfloat16), values(rng, rows, width, torch.bfloat16, 1e-2)
    arena = dev(rng.standard_normal(width + 9).astype(np.float32)).to(kind)
    weight_arena = dev(rng.standard_normal(width + 9).astype(np.float32)).to(kind)
    before = arena.clone()
    i = torch.rsqrt(h.float().square().mean(dim=1) + EPS)
    dx = torch.zeros_like(h)
    RmsNorm.backward(0, dy, h, weight_arena[3:3 + width], i, dx, arena[5:5 + width], accumulate=True)
    torch.cuda.synchronize()
    check_gradient(dx, arena[5:5 + width], dy, h, weight_arena[3:3 + width], i, None, before=before[5:5 + width])
    assert torch.equal(arena[:5], before[:5]) and torch.equal(arena[5 + width:], before[5 + width:])


@pytest.mark.parametrize("width", (1536, 771, 16416))
def test_the_gradient_may_take_the_place_of_an_input_and_rows_may_be_apart(cuda, width):
    rows = 6
    rng = np.random.default_rng(8)
    h, dy, r = (values(rng, rows, width, torch.float32) for _ in range(3))
    w, i = dev(rng.standard_normal(width).astype(np.float32)), torch.rsqrt(h.square().mean(dim=1) + EPS)
    results = []
    for place in ("apart", "dy", "residual"):
        a, b = dy.clone(), r.clone()
        dx = {"apart": torch.zeros_like(h), "dy": a, "residual": b}[place]
        dw = torch.zeros(width, device="cuda")
        RmsNorm.backward(0, a, h, w, i, dx, dw, residual_gradient=b)
        torch.cuda.synchronize()
        results.append((dx.clone(), dw))
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], other))
    dx, dw = torch.zeros_like(h), torch.zeros(width, device="cuda")
    RmsNorm.backward(0, placed(dy, 1, width + 3), placed(h, 2, width + 1), w, i, dx, dw, residual_gradient=placed(r, 0, width + 8))
    torch.cuda.synchronize()
    check_gradient(dx, dw, dy, h, w, i, r)


def test_no_rows_leave_a_zero_weight_gradient(cuda):
    w, dw = torch.ones(40, device="cuda"), torch.full((40,), 3.0, device="cuda")
    empty, i = torch.zeros(0, 40, device="cuda"), torch.zeros(0, device="cuda")
    RmsNorm.backward(0, empty, empty, w, i, empty, dw, accumulate=True)
    assert (dw == 3.0).all()
    RmsNorm.backward(0, empty, empty, w, i, empty, dw)
    assert not dw.any()
    RmsNorm.forward(0, empty, w, EPS, y=empty)


def test_gradient_against_differences(cuda):
    """f = sum(y * dy) in 64 bits, central differences of 1e-5: they are off by
    third derivatives times 1e-10 and by 1e-16 / 1e-5 times f, both below 1e-8."""
    rows, width = 2, 40
    rng = np.random.default_rng(9)
    h, dy = values(rng, rows, width, torch.float32), values(rng, rows, width, torch.float32)
    w = dev(rng.standard_normal(width).astype(np.float32))

    def f(h64, w64):
        i = 1.0 / np.sqrt((h64 * h64).mean(axis=1, keepdims=True) + EPS)
        return (h64 * i * w64 * f64(dy)).sum()

    y, i = torch.zeros_like(h), torch.zeros(rows, device="cuda")
    RmsNorm.forward(0, h, w, EPS, y=y, inverse_rms=i)
    dx, dw = torch.zeros_like(h), torch.zeros(width, device="cuda")
    RmsNorm.backward(0, dy, h, w, i, dx, dw)
    torch.cuda.synchronize()
    step, h64, w64 = 1e-5, f64(h), f64(w)
    for a in range(rows):
        for b in range(width):
            up, down = h64.copy(), h64.copy()
            up[a, b] += step
            down[a, b] -= step
            difference = (f(up, w64) - f(down, w64)) / (2 * step)
            # every term of dx is at most a few units: 100 steps of binary32 cover its roundings and i's
            assert abs(f64(dx)[a, b] - difference) <= 100 * E * 10 + 1e-8
    for b in range(width):
        up, down = w64.copy(), w64.copy()
        up[b] += step
        down[b] -= step
        assert abs(f64(dw)[b] - (f(h64, up) - f(h64, down)) / (2 * step)) <= 100 * E * 10 + 1e-8


def test_on_a_stream_of_its_own_and_replayed(cuda):
    rng = np.random.default_rng(10)
    rows, width = 300, 512
    h, dy = values(rng, rows, width, torch.bfloat16), values(rng, rows, width, torch.bfloat16)
    w, i = torch.ones(width, device="cuda"), torch.rsqrt(h.float().square().mean(dim=1) + EPS)

    def outputs():
        return torch.zeros_like(h), torch.zeros(width, device="cuda")

    eager, side, recorded = outputs(), outputs(), [outputs(), outputs()]
    RmsNorm.backward(0, dy, h, w, i, *eager)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    RmsNorm.backward(0, dy, h, w, i, *side, stream=stream)
    stream.synchronize()
    graphs = []
    for out in recorded:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            RmsNorm.backward(0, dy, h, w, i, *out)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for out in [side, *recorded]:
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_refusals(cuda):
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    y, i = torch.zeros_like(x), torch.zeros(4, device="cuda")
    payload, scales = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(8, device="cuda")
    with pytest.raises(ValueError, match="needs an output"):
        RmsNorm.forward(0, x, w, EPS)
    with pytest.raises(ValueError, match="divides the width"):
        RmsNorm.forward(0, x, w, EPS, payload=payload, scales=scales, block_size=48)
    with pytest.raises(ValueError, match="scales"):
        RmsNorm.forward(0, x, w, EPS, payload=payload, block_size=32)
    with pytest.raises(ValueError, match="scales has 8 values, expected 4"):
        RmsNorm.forward(0, x, w, EPS, payload=payload, scales=scales)
    with pytest.raises(ValueError, match="shape"):
        RmsNorm.forward(0, x.view(-1), w, EPS, y=y)
    with pytest.raises(ValueError, match="residual has type"):
        RmsNorm.forward(0, x, w, EPS, residual=x.to(torch.bfloat16), y=y)
    with pytest.raises(ValueError, match="residual has shape"):
        RmsNorm.forward(0, x, w, EPS, residual=x[:2], y=y)
    with pytest.raises(ValueError, match="without a residual"):
        RmsNorm.forward(0, x, w, EPS, residual_out=torch.zeros_like(x), y=y)
    with pytest.raises(ValueError, match="contiguous"):
        RmsNorm.forward(0, torch.zeros(64, 4, device="cuda").t(), w, EPS, y=y)
    with pytest.raises(ValueError, match="overlap"):
        RmsNorm.forward(0, torch.zeros(64, device="cuda").expand(4, 64), w, EPS, y=y)
    with pytest.raises(ValueError, match="device"):
        RmsNorm.forward(0, x.cpu(), w, EPS, y=y)
    with pytest.raises(ValueError, match="weight has 63"):
        RmsNorm.forward(0, x, w[:63], EPS, y=y)
    with pytest.raises(ValueError, match="type"):
        RmsNorm.forward(0, x.half(), w, EPS, y=y)
    with pytest.raises(ValueError, match="x_gradient has type"):
        RmsNorm.backward(0, x, x, w, i, y.to(torch.bfloat16), w.clone())
    with pytest.raises(ValueError, match="inverse_rms"):
        RmsNorm.backward(0, x, x, w, i[:2], y, w.clone())
    with pytest.raises(ValueError, match="workspace"):
        RmsNorm.backward(0, x, x, w, i, y, w.clone(), workspace=torch.zeros(8, dtype=torch.uint8, device="cuda"))
