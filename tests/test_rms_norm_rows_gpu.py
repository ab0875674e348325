"""The RMS norm over many more rows than the device holds at once, so that every
CTA walks rows: its ring of staged rows turns, the slots of its reductions take
turns, and what it writes may lie where rows ahead of it are still read.

A row's result does not depend on the other rows or on the CTA that makes it.
So the rows of a long call have the bits of the same rows called in slices that
are short enough for a CTA for each row, and long enough (148 rows and more) for
the same kernel.  The slices are the shapes of test_rms_norm_gpu.py; one of them
is checked against the 64-bit definition here again.  The weight's gradient is
a sum over all rows and has that module's bound."""
import numpy as np
import pytest
import torch

import test_rms_norm_gpu as small
from nntrain_b200.native import RmsNorm

pytestmark = pytest.mark.gpu

EPS, SLICE = small.EPS, 150
# 148 SMs hold at most 4736 CTAs of 32 threads, 1480 of 192, 1184 of 256: 5 rows a CTA and more, 2 of the longest rows
SHAPES = ((23701, 64), (23701, 33), (7501, 1536), (7501, 771), (6001, 2048), (6001, 4096), (6001, 4001), (2501, 16384),
          (2501, 16416))


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, sigma=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * sigma).to(dtype)


def slices(rows):
    """(begin, end) of slices of SLICE rows that cover all rows; the last one overlaps its neighbour."""
    return [(min(i, rows - SLICE), min(i, rows - SLICE) + SLICE) for i in range(0, rows, SLICE)]


def forward(x, residual, w, block, in_place=None):
    """The outputs of one call; in_place: None, 'y' over x, or 'sum' over the residual."""
    rows, width = x.shape
    out = {"inverse": torch.zeros(rows, device="cuda")}
    out["y"] = x if in_place == "y" else torch.zeros_like(x)
    if residual is not None:
        out["sum"] = residual if in_place == "sum" else torch.zeros_like(x)
    if block is not None:
        out["payload"] = torch.zeros(rows, width, dtype=torch.int8, device="cuda")
        out["scales"] = torch.zeros(rows * (width // (block or width)), device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    RmsNorm.forward(0, x, w, EPS, residual=residual, residual_out=out.get("sum"), y=out["y"], payload=out.get("payload"),
                    scales=out.get("scales"), block_size=block or 0, inverse_rms=out["inverse"], finite_status=flag)
    out["flag"] = int(flag.item())
    return out


@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("block", (None, 0, 32))
@pytest.mark.parametrize("with_residual", (False, True))
def test_forward_over_many_rows(cuda, rows, width, dtype, block, with_residual):
    if block and width % block:
        block = 0
    g = generator(rows + width)
    x = normal(g, rows, width, dtype=dtype)
    residual = normal(g, rows, width, dtype=dtype, sigma=3.0) if with_residual else None
    w = 1.0 + normal(g, width, sigma=0.3)
    whole = forward(x, residual, w, block)
    assert whole["flag"] == 0
    per_row = 1 if block is None else width // (block or width)
    for begin, end in slices(rows):
        part = forward(x[begin:end], None if residual is None else residual[begin:end], w, block)
        for name in part:
            if name == "scales":
                assert torch.equal(part[name], whole[name][begin * per_row:end * per_row]), (name, begin)
            elif name != "flag":
                assert torch.equal(part[name], whole[name][begin:end]), (name, begin)
    for place in ("y", "sum") if with_residual else ("y",):
        again = forward(x.clone(), None if residual is None else residual.clone(), w, block, in_place=place)
        for name in again:
            assert name == "flag" or torch.equal(again[name], whole[name]), (place, name)
    end = rows - 7                                   # and a few of the last rows by the definition
    part = slice(end - 40, end)
    h, i, y = small.reference(x[part], None if residual is None else residual[part], w)
    ty = small.tolerance_i(width) + 3 * small.E
    assert (np.abs(small.f64(whole["inverse"][part]) - i) <= i * small.tolerance_i(width)).all()
    if block is None:
        assert (np.abs(small.f64(whole["y"][part]) - y) <= np.abs(y) * (ty + 1.01 * small.HALF_STEP[dtype])).all()
    else:
        b = block or width
        step = np.abs(y.reshape(-1, b)).max(axis=1) / 127.0
        codes = small.f64(whole["payload"][part]).reshape(-1, b)
        assert (np.abs(codes - y.reshape(-1, b) / step[:, None]) <= 0.5 + 127.0 * (2 * ty + 2 * small.E)).all()


@pytest.mark.parametrize("rows,width", ((23701, 64), (7501, 1536), (7501, 771), (2501, 16416)))
@pytest.mark.parametrize("block", (None, 0, 32))
def test_a_row_that_is_not_finite_stays_alone(cuda, rows, width, block):
    if block and width % block:
        block = 0
    g = generator(width)
    x, w = normal(g, rows, width), 1.0 + normal(g, width, sigma=0.3)
    clean = forward(x, None, w, block)
    bad = rows - 900
    x[bad, width // 2] = float("nan")
    got = forward(x, None, w, block)
    assert clean["flag"] == 0 and got["flag"] == 1
    others = torch.arange(rows, device="cuda") != bad
    for name in got:
        if name == "scales":
            assert torch.equal(got[name].view(rows, -1)[others], clean[name].view(rows, -1)[others])
        elif name != "flag":
            assert torch.equal(got[name][others], clean[name][others]), name
    assert got["inverse"][bad].isnan()


def backward(dy, h, w, i, residual, in_place=None):
    dx = {None: None, "dy": dy, "residual": residual}[in_place]
    dx = torch.zeros_like(h) if dx is None else dx
    dw = torch.full((h.shape[1],), 9.0, device="cuda")
    RmsNorm.backward(0, dy, h, w, i, dx, dw, residual_gradient=residual)
    return dx, dw


@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("with_residual", (False, True))
def test_gradient_over_many_rows(cuda, rows, width, dtype, with_residual):
    g = generator(rows * 3 + width)
    h, dy = normal(g, rows, width, dtype=dtype, sigma=3.0), normal(g, rows, width, dtype=dtype, sigma=1e-3)
    residual = normal(g, rows, width, dtype=dtype, sigma=1e-3) if with_residual else None
    w = 1.0 + normal(g, width, sigma=0.3)
    i = torch.rsqrt(h.float().square().mean(dim=1) + EPS)
    dx, dw = backward(dy, h, w, i, residual)
    for begin, end in slices(rows):
        part, _ = backward(dy[begin:end], h[begin:end], w, i[begin:end], None if residual is None else residual[begin:end])
        assert torch.equal(part, dx[begin:end]), begin
    for place in ("dy", "residual") if with_residual else ("dy",):
        again, weight_again = backward(dy.clone(), h, w, i, None if residual is None else residual.clone(), in_place=place)
        assert torch.equal(again, dx) and torch.equal(weight_again, dw), place
    # the weight's gradient of all rows (a lost row of them shows: its share is some 1e-4, the bound some 1e-6)
    n = h.double() * i.double()[:, None]
    terms = dy.double() * n
    bound = (-(-rows // 148) + 45 + 2) * small.E * terms.abs().sum(dim=0)
    assert ((dw.double() - terms.sum(dim=0)).abs() <= bound).all()
    part = slice(rows - 47, rows - 7)
    small.check_gradient(dx[part], backward(dy[part], h[part], w, i[part], None)[1], dy[part], h[part], w, i[part],
                         None if residual is None else residual[part])


PLACES = {"on the grid": ((0, 0), (0, 8), (8, 16), (16, 24)), "off the grid": ((1, 0), (3, 5), (5, 3), (2, 1))}


@pytest.mark.parametrize("width,places", [(w, p) for w in (64, 1536, 16416) for p in PLACES] + [(771, "off the grid")])
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("block", (None, 0, 32))
def test_places_that_take_one_kernel_give_the_same_bits(cuda, width, places, dtype, block):
    if block and width % block:
        block = 0
    rows = 200
    g = generator(width)
    x, residual, dy = (normal(g, rows, width, dtype=dtype) for _ in range(3))
    w, i = 1.0 + normal(g, width, sigma=0.3), None
    results = []
    for shift, extra in PLACES[places]:
        at = lambda t: small.placed(t, shift, width + extra)
        got = forward(at(x), at(residual), w, block)
        i = got["inverse"] if i is None else i
        dx, dw = backward(at(dy), at(x), w, i, at(residual))
        results.append({**got, "dx": dx, "dw": dw})
    for other in results[1:]:
        for name in other:
            assert name == "flag" or torch.equal(results[0][name], other[name]), name
